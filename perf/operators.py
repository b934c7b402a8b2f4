"""Cases of the serving and training operators around masked attention.

rope   norms of queries and keys for each head with the position rotation in the same pass, forward
       (grad false) or forward and gradients (grad true)
cache  keys and values quantised as they are written into a paged cache, and the sequence read back
tree   attention of a tree of drafted tokens (or of a chain: plain decoding) over such a cache

Where `own` is false, run() computes a case in elementary torch operations; where it is true it makes
the calls a user makes of this repository's modules.
"""
import functools
import math
import os
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6


@functools.lru_cache(maxsize=None)  # (a user's program imports a module once, not with each call)
def _mod(name):
    import importlib
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(here, "graph-processing-attention-ipdps-2025_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    return importlib.import_module(name)


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _rope(name, batch, tokens, hq, hk, d, rot, interleaved, dtype, grad, heads_first):
    return {"name": name, "op": "rope", "batch": batch, "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": rot,
            "interleaved": interleaved, "dtype": dtype, "grad": grad, "heads_first": heads_first}


def _cache(name, seqs, new, length, hk, d, page, dtype, code, head_pages):
    return {"name": name, "op": "cache", "seqs": seqs, "new": new, "length": length, "hk": hk, "d": d, "page": page,
            "dtype": dtype, "code": code, "head_pages": head_pages}


def _tree(name, seqs, ctx, nodes, chain, hk, group, d, page, dtype, code, head_pages):
    return {"name": name, "op": "tree", "seqs": seqs, "ctx": ctx, "nodes": nodes, "chain": chain, "hk": hk,
            "group": group, "d": d, "page": page, "dtype": dtype, "code": code, "head_pages": head_pages}


def listed():
    return [
        # the queries and keys of one token: a decoding step of a single stream
        _rope("rope_one_token", 1, 1, 32, 8, 128, 128, False, "bf16", False, False),
        # an odd-length prompt, half of each head rotated in adjacent pairs, written head by head
        _rope("rope_prompt_f16", 1, 4099, 16, 2, 64, 32, True, "f16", False, True),
        # a training step over two long sequences, grouped heads
        _rope("rope_train_bf16", 2, 8192, 32, 8, 128, 128, False, "bf16", True, True),
        # fp32 training, odd lengths, heads that are not a power of two
        _rope("rope_train_f32", 3, 1021, 12, 12, 96, 64, False, "f32", True, False),
        # a decoding step appends one token to each of four short sequences, which are read back
        _cache("cache_step_int8", 4, 1, 333, 8, 128, 16, "bf16", "int8", True),
        # a chunk of a long prompt is appended and the whole prefix read back for the next layer call
        _cache("cache_chunk_e4m3", 1, 2048, 32768, 8, 128, 64, "bf16", "e4m3", True),
        # whole prompts of fp32 keys written at once, odd head size and page size, token-major pages
        _cache("cache_prompts_f32", 3, 5001, 5001, 5, 80, 48, "f32", "int8", False),
        # one stream, one token at a time, unquantised cache
        _tree("tree_one_token", 1, 700, 1, True, 8, 4, 128, 16, "bf16", "none", True),
        # plain decoding of a full batch of ragged sequences over an 8-bit floating-point cache
        _tree("tree_batch_e4m3", 64, 8191, 1, True, 8, 4, 128, 64, "bf16", "e4m3", True),
        # small draft trees for a ragged batch over an int8 cache with small token-major pages
        _tree("tree_drafts_int8", 16, 12345, 13, False, 4, 7, 128, 16, "f16", "int8", False),
        # a small batch over very long contexts, unquantised: the largest cache
        _tree("tree_long_bf16", 2, 200001, 8, False, 8, 4, 128, 64, "bf16", "none", True),
        # wide trees over medium contexts: many rows for every key
        _tree("tree_wide_f16", 6, 5000, 61, False, 8, 8, 64, 32, "f16", "none", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "cache", "tree"])
    if op == "rope":
        d = rng.choice([64, 80, 96, 128, 256])
        hk = rng.choice([1, 2, 4, 8])
        hq = hk * rng.randint(1, 6)
        tokens = max(1, min(_log(rng, 1, 16000), int(6.0e7 / (d * (hq + hk)))))
        batch = rng.randint(1, 3) if tokens > 8 else 1
        return _rope(None, batch, tokens, hq, hk, d, rng.choice([d, d, d // 2, d // 4 * 2]), rng.random() < 0.4,
                     rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5, rng.random() < 0.5)
    if op == "cache":
        d = rng.choice([64, 80, 128, 256])
        seqs, hk = rng.randint(1, 6), rng.choice([1, 2, 5, 8])
        length = max(2, min(_log(rng, 2, 32000), int(3.0e7 / (d * hk * seqs))))
        return _cache(None, seqs, min(length, _log(rng, 1, 4000)), length, hk, d, rng.choice([16, 32, 48, 64, 128]),
                      rng.choice(["bf16", "f16", "f32"]), rng.choice(["int8", "e4m3", "none"]), rng.random() < 0.5)
    d = rng.choice([64, 80, 128, 256])
    hk, group, seqs = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]), rng.randint(1, 32)
    nodes = _log(rng, 1, 64)
    ctx = min(_log(rng, 1, 60000), int(2.0e8 / (seqs * hk * d)), int(1.5e8 / (seqs * hk * group * nodes)))
    return _tree(None, seqs, max(1, ctx), nodes, rng.random() < 0.4, hk, group, d, rng.choice([16, 24, 32, 64, 128]),
                 rng.choice(["bf16", "f16"]), rng.choice(["int8", "e4m3", "none"]), rng.random() < 0.6)


def _spread(n, top, least):
    """n lengths between `least` and `top`, ragged, the first one `top`: the same for every seed."""
    return [top - ((i * 2654435761) % (1 << 32)) * (top - least) // (1 << 32) for i in range(n)]


def _lengths(case):
    """Tokens before the tree, and nodes of the tree, of each sequence."""
    ctx = _spread(case["seqs"], case["ctx"], case["ctx"] // 4)
    nodes = _spread(case["seqs"], case["nodes"], (case["nodes"] + 1) // 2)
    return ctx, nodes


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _pages(n_pages, case):
    """The shape of a cache's pages in memory: by head, then token (head_pages), or by token."""
    if case["head_pages"]:
        return (n_pages, case["hk"], case["page"]), (0, 2, 1)
    return (n_pages, case["page"], case["hk"]), (0, 1, 2)


def _filled_cache(n_pages, case, g):
    """(codes, scales) [pages, page, heads, d] / [pages, page, heads] of normal values as they stand
    in the cache, quantised row by row; scales is None for a cache of the inputs' own type."""
    shape, order = _pages(n_pages, case)
    x = torch.randn(*shape, case["d"], generator=g, device=DEV)
    x *= torch.rand(*shape, 1, generator=g, device=DEV) + 0.5
    code = case["code"]
    if code == "none":
        return x.to(TYPES[case["dtype"]]).permute(*order, 3), None
    c, s = _quantise(x, code)
    return c.permute(*order, 3), s.permute(*order)


def _quantise(x, code):
    """Codes and scales of rows: code = round(x * top / amax), ties to even, scale = amax / top.
    The quotient of 16-bit values stays on its side of a border in 32 bits; that of 32-bit values
    needs 64."""
    amax = x.abs().amax(-1, keepdim=True).float()
    y = x.double() if x.dtype == torch.float32 else x.float()
    y = y * TOP[code] / torch.where(amax == 0, torch.ones_like(amax), amax)
    if code == "int8":
        y = y.round()
    elif y.dtype == torch.float64:  # (rounded here: the cast goes by way of 32 bits)
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)
        y = (y / step).round() * step
    return y.to(CODES[code]), (amax / TOP[code]).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case)
    dt = TYPES[case["dtype"]]
    if case["op"] == "rope":
        b, t, hq, hk, d = (case[x] for x in ("batch", "tokens", "hq", "hk", "d"))
        # the projection of a layer gives queries, keys and values of a token side by side
        qkv = torch.randn(b, t, (hq + 2 * hk) * d, generator=g, device=DEV).to(dt)
        s["q"] = qkv[..., :hq * d].view(b, t, hq, d)
        s["k"] = qkv[..., hq * d:(hq + hk) * d].view(b, t, hk, d)
        s["w_q"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
        s["w_k"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
        start = torch.randint(0, 100000, (b, 1), generator=g, device=DEV, dtype=torch.int64)
        s["positions"] = start + torch.arange(t, device=DEV)
        n = case["rot"] // 2
        s["inv_freq"] = 500000.0 ** (-torch.arange(n, device=DEV, dtype=torch.float32) / max(n, 1))
        if case["grad"]:
            s["d_q_out"] = _heads(s, hq).normal_(generator=g)
            s["d_k_out"] = _heads(s, hk).normal_(generator=g)
        return s
    if case["op"] == "cache":
        n, new, length, page = case["seqs"], case["new"], case["length"], case["page"]
        per = -(-length // page)
        n_pages = n * per + 3
        s["k_cache"], s["k_scale"] = _filled_cache(n_pages, case, g)
        s["v_cache"], s["v_scale"] = _filled_cache(n_pages, case, g)
        table = torch.randperm(n_pages, generator=g, device=DEV)[:n * per].view(n, per)
        at = torch.arange(length, device=DEV)
        slots = table[:, at // page] * page + at % page
        s["write_slots"] = slots[:, length - new:].reshape(-1).contiguous()
        s["read_slots"] = slots.reshape(-1).contiguous()
        s["k"] = torch.randn(n * new, case["hk"], case["d"], generator=g, device=DEV).to(dt)
        s["v"] = torch.randn(n * new, case["hk"], case["d"], generator=g, device=DEV).to(dt)
        return s
    ctx, nodes = _lengths(case)
    n, page, total = case["seqs"], case["page"], sum(nodes)
    need = [-(-(c + m) // page) for c, m in zip(ctx, nodes)]
    n_pages = sum(need) + 2
    s["k_cache"], s["k_scale"] = _filled_cache(n_pages, case, g)
    s["v_cache"], s["v_scale"] = _filled_cache(n_pages, case, g)
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    s["page_table"] = table
    s["ctx_lens"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    off = [0]
    for m in nodes:
        off.append(off[-1] + m)
    s["q_offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
    s["q"] = (1.5 * torch.randn(total, case["hk"] * case["group"], case["d"], generator=g, device=DEV)).to(dt)
    s["tree_mask"] = None
    if not case["chain"]:
        # node i hangs on one of the nodes before it (or on the last cached token); its row of bits
        # is its ancestors' and its own
        pick = torch.rand(n, max(nodes), generator=g, device=DEV).cpu().tolist()
        rows = []
        for i, m in enumerate(nodes):
            mine = []
            for j in range(m):
                parent = int(pick[i][j] * (j + 1)) - 1
                mine.append((mine[parent] if parent >= 0 else 0) | (1 << j))
            rows += mine
        words = -(-max(nodes) // 64)
        split = [[(r >> (64 * w)) & ((1 << 64) - 1) for w in range(words)] for r in rows]
        split = [[x - (1 << 64) if x >> 63 else x for x in r] for r in split]
        s["tree_mask"] = torch.tensor(split, dtype=torch.int64, device=DEV)
    return s


def _heads(s, heads):
    """An output of the rope: [batch, tokens, heads, d], in memory head by head where asked."""
    b, t, d, dt = s["batch"], s["tokens"], s["d"], TYPES[s["dtype"]]
    if s["heads_first"]:
        return torch.empty(b, heads, t, d, dtype=dt, device=DEV).transpose(1, 2)
    return torch.empty(b, t, heads, d, dtype=dt, device=DEV)


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _pairs(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _rotate(x, cos, sin, rot, interleaved):
    a, b = _pairs(x, rot, interleaved)
    y = x.clone()
    ya, yb = _pairs(y, rot, interleaved)
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    return y


def _plain_rope(s):
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"].double()
    cos, sin = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    rot, inter, dt = s["rot"], s["interleaved"], TYPES[s["dtype"]]

    def one(x, w, heads, d_out):
        x, w = x.float(), w.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        n = x * r
        out = _heads(s, heads)
        out.copy_(_rotate(n * w, cos, sin, rot, inter))
        if d_out is None:
            return (out,)
        gr = _rotate(d_out.float(), cos, -sin, rot, inter)
        gn = gr * w
        dx = r * (gn - n * (gn * n).mean(-1, keepdim=True))
        return out, dx.to(dt), (gr * n).sum((0, 1, 2))

    return (one(s["q"], s["w_q"], s["hq"], s.get("d_q_out")), one(s["k"], s["w_k"], s["hk"], s.get("d_k_out")))


def _plain_write(x, slots, cache, scale, code):
    page = cache.shape[1]
    at = (slots // page, slots % page)
    if code == "none":
        cache[at] = x
        return
    c, sc = _quantise(x, code)
    if code == "e4m3":  # (copied as bytes: torch indexes no 8-bit floating-point tensors in place)
        c, cache = c.view(torch.uint8), cache.view(torch.uint8)
    cache[at] = c
    scale[at] = sc


def _values(cache, scale, code, at):
    """fp32 values of the cache's rows at `at` (an index)."""
    if code == "e4m3":
        x = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    else:
        x = cache[at].float()
    return x if scale is None else x * scale[at].unsqueeze(-1)


def _plain_cache(s):
    out = []
    page, rs, dt = s["page"], s["read_slots"], TYPES[s["dtype"]]
    for x in ("k", "v"):
        _plain_write(s[x], s["write_slots"], s[x + "_cache"], s[x + "_scale"], s["code"])
        y = _values(s[x + "_cache"], s[x + "_scale"], s["code"], (rs // page, rs % page))
        out.append(y.to(dt).transpose(0, 1).contiguous().transpose(0, 1))
    return out


def _plain_tree(s):
    hk, group, d, n = s["hk"], s["group"], s["d"], s["seqs"]
    total, most = s["q"].shape[0], s["nodes"]
    pages = s["page_table"].clamp(min=0).long()
    k = _values(s["k_cache"], s["k_scale"], s["code"], (pages,)).flatten(1, 2).permute(0, 2, 3, 1).contiguous()
    v = _values(s["v_cache"], s["v_scale"], s["code"], (pages,)).flatten(1, 2).transpose(1, 2).contiguous()
    length = v.shape[2]
    off = s["q_offsets"].long()
    node = torch.arange(most, device=DEV)
    row = (off[:-1, None] + node).clamp(max=total - 1)                       # [n, most]
    there = node < (off[1:] - off[:-1])[:, None]
    q = s["q"].float()[row].view(n, most, hk, group, d).transpose(1, 2).reshape(n, hk, most * group, d)
    ctx = s["ctx_lens"].long()[:, None, None]
    j = torch.arange(length, device=DEV)[None, None, :] - ctx                # draft index of a key
    if s["tree_mask"] is None:
        mine = j <= node[None, :, None]
    else:
        bits = s["tree_mask"][row]                                           # [n, most, words]
        jj = j.clamp(0, 64 * bits.shape[2] - 1).expand(n, most, length)
        mine = ((bits.gather(2, jj // 64) >> (jj % 64)) & 1) == 1
        mine = mine & (j < 64 * bits.shape[2])
    live = ((j < 0) | mine) & (j < (off[1:] - off[:-1])[:, None, None]) & there[..., None]
    score = torch.matmul(q, k).view(n, hk, most, group, length) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~live[:, None, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp()
    total_p = p.sum(-1, keepdim=True)
    p = p / torch.where(total_p == 0, torch.ones_like(total_p), total_p)
    out = torch.matmul(p.view(n, hk, most * group, length), v)
    out = out.view(n, hk, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, hk * group, d)
    t = torch.arange(total, device=DEV)
    seq = torch.searchsorted(off, t, right=True) - 1
    return out[seq, t - off[seq]].to(TYPES[s["dtype"]])


# ------------------------------------------------------------------------------------------------
# the repository's operators
# ------------------------------------------------------------------------------------------------
def _own_rope(s):
    m = _mod("spfa_rope")
    args = (s["q"], s["k"], s["w_q"], s["w_k"], s["positions"], s["inv_freq"])
    q_out, k_out = _heads(s, s["hq"]), _heads(s, s["hk"])
    m.forward(*args, q_out, k_out, EPS, s["interleaved"])
    if not s["grad"]:
        return (q_out,), (k_out,)
    d_q, d_k = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV), torch.empty(s["k"].shape, dtype=s["q"].dtype, device=DEV)
    d_wq, d_wk = torch.empty(s["d"], device=DEV), torch.empty(s["d"], device=DEV)
    m.backward(*args, s["d_q_out"], s["d_k_out"], d_q, d_k, d_wq, d_wk, EPS, s["interleaved"])
    return (q_out, d_q, d_wq), (k_out, d_k, d_wk)


def _own_cache(s):
    m = _mod("spfa_cache")
    cache = (s["k_cache"], s["v_cache"])
    m.write(s["k"], s["v"], s["write_slots"], *cache, s["k_scale"], s["v_scale"])
    n, dt = s["read_slots"].shape[0], TYPES[s["dtype"]]
    k = torch.empty(s["hk"], n, s["d"], dtype=dt, device=DEV).transpose(0, 1)
    v = torch.empty(s["hk"], n, s["d"], dtype=dt, device=DEV).transpose(0, 1)
    m.read(*cache, s["read_slots"], k, v, s["k_scale"], s["v_scale"])
    return k, v


def _own_tree(s):
    out = torch.empty_like(s["q"])
    return _mod("spfa_tree").forward(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["ctx_lens"], s["q_offsets"],
                                     out, s["tree_mask"], s["k_scale"], s["v_scale"])


def run(state):
    if own:
        return {"rope": _own_rope, "cache": _own_cache, "tree": _own_tree}[state["op"]](state)
    return {"rope": _plain_rope, "cache": _plain_cache, "tree": _plain_tree}[state["op"]](state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["batch"] * case["tokens"]
        x = n * (case["hq"] + case["hk"]) * case["d"]
        # forward: read, write; gradients: inputs (still the same ones) and output gradients read, gradients written
        moved = (4 if case["grad"] else 2) * x * size + n * 8
        return {"bytes": moved + 2 * case["d"] * size, "flops": (24 if case["grad"] else 9) * x}
    bits = size if case["code"] == "none" else 1
    scale = 0 if case["code"] == "none" else 4
    if case["op"] == "cache":
        rows_in, rows = 2 * case["seqs"] * case["new"] * case["hk"], 2 * case["seqs"] * case["length"] * case["hk"]
        d = case["d"]
        moved = rows_in * (d * size + d * bits + scale) + rows * (d * bits + scale + d * size)
        return {"bytes": moved + 8 * case["seqs"] * (case["new"] + case["length"]), "flops": 3 * rows_in * d + rows * d}
    ctx, nodes = _lengths(case)
    keys = sum(ctx) + sum(nodes)
    d, hk, group = case["d"], case["hk"], case["group"]
    moved = 2 * keys * hk * (d * bits + scale) + 2 * sum(nodes) * hk * group * d * size + 4 * keys // case["page"]
    return {"bytes": moved, "flops": 4 * d * hk * group * sum((c + 1) * m for c, m in zip(ctx, nodes))}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"rope": _exact_rope, "cache": _exact_cache, "tree": _exact_tree}[case["op"]](case, prepare(case, seed))


def _exact_rope(case, s):
    """The rotation as a product of complex numbers, the gradients from the norm's Jacobian."""
    rot, d, pos = case["rot"], case["d"], s["positions"].double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos[..., None] * s["inv_freq"].double())[:, :, None]

    def pairs(x):
        if case["interleaved"]:
            return torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous())
        return torch.complex(x[..., :rot // 2], x[..., rot // 2:rot])

    def flat(z, rest):
        if case["interleaved"]:
            return torch.cat((torch.view_as_real(z).flatten(-2), rest), -1)
        return torch.cat((z.real, z.imag, rest), -1)

    res = []
    for x, w, d_out in ((s["q"], s["w_q"], s.get("d_q_out")), (s["k"], s["w_k"], s.get("d_k_out"))):
        x, w = x.double(), w.double()
        root = (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
        y = x / root * w
        mine = [flat(pairs(y) * turn, y[..., rot:])]
        if d_out is not None:
            g = d_out.double()
            g = flat(pairs(g) * turn.conj(), g[..., rot:])
            mine.append(w * g / root - x * (w * g * x).sum(-1, keepdim=True) / (d * root ** 3))
            mine.append((g * x / root).flatten(0, 2).sum(0))
        res.append(tuple(mine))
    return tuple(res)


def _exact_cache(case, s):
    """What the slots hold afterwards: the old rows' values, or the new rows rounded to their grid."""
    out = []
    page, rs, ws = case["page"], s["read_slots"], s["write_slots"]
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        held = (cache.view(torch.uint8)[rs // page, rs % page].view(torch.float8_e4m3fn) if case["code"] == "e4m3"
                else cache[rs // page, rs % page]).double()
        x = s[name].double()
        if scale is not None:
            held *= scale[rs // page, rs % page].double()[..., None]
            top = TOP[case["code"]]
            amax = x.abs().amax(-1, keepdim=True)
            y = x * top / amax
            if case["code"] == "int8":
                y = y.round()
            else:  # 3 bits after the first one, the smallest step 2^-9
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                y = (y / step).round() * step
            x = y * amax / top
        held = held.view(case["seqs"], case["length"], case["hk"], case["d"])
        held[:, case["length"] - case["new"]:] = x.view(case["seqs"], case["new"], case["hk"], case["d"])
        out.append(held.flatten(0, 1))
    return out


def _exact_tree(case, s):
    ctx, nodes = _lengths(case)
    hk, group, d = case["hk"], case["group"], case["d"]
    res, at = [], 0
    for b in range(case["seqs"]):
        c, n = ctx[b], nodes[b]
        pos = torch.arange(c + n, device=DEV)
        page, slot = s["page_table"][b].long()[pos // case["page"]], pos % case["page"]

        def rows(cache, scale):
            x = (cache.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn) if case["code"] == "e4m3" else cache[page, slot]).double()
            return x if scale is None else x * scale[page, slot].double()[..., None]

        if s["tree_mask"] is None:
            mine = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        else:
            word, bit = pos[:n] // 64, pos[:n] % 64
            mine = ((s["tree_mask"][at:at + n][:, word] >> bit) & 1).bool()
        live = torch.cat((torch.ones(n, c, dtype=torch.bool, device=DEV), mine), 1)
        k, v = rows(s["k_cache"], s["k_scale"]), rows(s["v_cache"], s["v_scale"])
        q = s["q"][at:at + n].double().view(n, hk, group, d)
        mine = torch.empty(n, hk, group, d, dtype=torch.float64, device=DEV)
        for h in range(hk):
            sc = (q[:, h].reshape(n * group, d) @ k[:, h].t().contiguous() / math.sqrt(d)).view(n, group, c + n)
            sc = sc.masked_fill(~live[:, None], float("-inf"))
            mine[:, h] = (torch.softmax(sc, -1).view(n * group, c + n) @ v[:, h].contiguous()).view(n, group, d)
        res.append(mine.view(n, hk * group, d))
        at += n
    return torch.cat(res)
