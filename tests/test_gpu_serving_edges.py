"""Inputs at the edges of what the operators around masked attention take, on the GPU against the
float64 oracle: the cases, tolerances' units and helpers are those of test_gpu_serving.py."""
import math

import numpy as np
import pytest
import torch

from helpers import np64
from oracle import serve_oracle as sv
from test_gpu_serving import (BF16, DEV, F16, F32, HALF, ROOM, TINY, U, Run, _close, _gen, _mod, _ones, _pair_size,
                              _rope_inputs)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------
# rope
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", [
    (F32, 5, 3, 1, 96, 64, False, F32, True, False),
    (F16, 5, 3, 1, 64, 32, True, F16, False, False),
    (BF16, 5, 3, 1, 128, 128, False, BF16, True, False),
    (BF16, 1, 1, 1, 128, 128, False, BF16, False, False),
    (F32, 3, 1, 2, 33, 10, False, F32, False, False),      # single elements
    (BF16, 701, 5, 3, 128, 128, False, F32, True, False),  # several rounds of a workgroup, the last one not full
], ids=lambda c: "%s_t%d_h%d_%d_d%d" % (str(c[0])[6:], *c[1:5]))
def test_rope_gradients_without_eps(case):
    """eps = 0: the norms of the vectors are what they are, and lanes without a vector add nothing."""
    dt, tokens, hq, hk, d, rot, inter, wdt, fused, _ = case
    q, k, w, pos, f = _rope_inputs(case, 21)
    m = _mod("spfa_rope")
    qo, ko = [torch.empty(x.shape, dtype=dt, device=DEV) for x in (q, k)]
    m.forward(q, k, *w, pos, f, qo, ko, 0.0, inter)
    g = _gen(22)
    dqo, dko = [torch.randn(x.shape, generator=g, device=DEV).to(dt) for x in (q, k)]
    dq, dk = torch.empty_like(dqo), torch.empty_like(dko)
    dw = [torch.empty(d, device=DEV) for _ in range(2)]
    m.backward(q, k, *w, pos, f, dqo, dko, dq, dk, *dw, 0.0, inter)
    p, fr = pos.cpu().numpy(), np64(f)
    for x, y, dy, dx, ww, dww, heads in ((q, qo, dqo, dq, w[0], dw[0], hq), (k, ko, dko, dk, w[1], dw[1], hk)):
        want = sv.norm_rope(np64(x), _ones(ww, d), p, fr, 0.0, inter)
        _close(y, want, HALF[dt] * np.abs(want) + TINY[dt] + (d / 2 + 28) * U * _pair_size(want, rot, inter) * 1.5, "forward")
        gx, gw, sx, sw = sv.norm_rope_backward(np64(x), _ones(ww, d), p, fr, 0.0, inter, np64(dy))
        _close(dx, gx, HALF[dt] * np.abs(gx) + TINY[dt] + (d + 60) * U * sx, "gradient")
        _close(dww, gw, (d + 60 + tokens * heads) * U * sw + TINY[F32], "weights' gradient")


def test_rope_in_place_of_one_token_by_another_view():
    """The stride of a dimension of one is nobody's: the same place stays the same place."""
    m = _mod("spfa_rope")
    x = torch.randn(3, 6, 64, generator=_gen(24), device=DEV).to(BF16)[1:2]
    q, k = x[:, :4], x[:, 4:]
    pos, f = torch.tensor([5], device=DEV), 100.0 ** (-torch.arange(32, device=DEV, dtype=F32) / 32)
    want = m.forward(q, k, None, None, pos, f, torch.empty_like(q), torch.empty_like(k))
    other = [y[0].unsqueeze(0) for y in (q, k)]
    assert other[0].data_ptr() == q.data_ptr() and other[0].stride() != q.stride()
    m.forward(q, k, None, None, pos, f, *other)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rope_positions_that_are_broadcast():
    """One row of positions for all of a batch, as [1, tokens] or expanded, and rows of a wider table."""
    m = _mod("spfa_rope")
    case = (BF16, 7, 2, 1, 64, 64, False, BF16, True, False)
    q, k, w, pos, f = _rope_inputs(case, 23, batch=4)
    new = lambda: [torch.empty(x.shape, dtype=BF16, device=DEV) for x in (q, k)]
    for dt in (torch.int32, torch.int64):
        row = pos[2].to(dt)
        want = m.forward(q, k, *w, row, f, *new())
        table = torch.full((4, 20), 99, dtype=dt, device=DEV)
        table[:, 3:10] = row
        for p in (row.view(1, 7), row.expand(4, 7), row.repeat(4, 1), table[:, 3:10], table[:1, 3:10]):
            got = m.forward(q, k, *w, p, f, *new())
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = [x[:1] for x in (q, k)]
    got = m.forward(*one, *w, pos[2].view(1, 7), f, *[torch.empty(x.shape, dtype=BF16, device=DEV) for x in one])
    assert torch.equal(got[0][0], want[0][0])
    for p in (pos[:2], pos[:3].contiguous(), pos.t().contiguous().t(), pos[..., None], pos[:, :6]):
        with pytest.raises((RuntimeError, ValueError)):
            m.forward(q, k, *w, p, f, *new())


def test_rope_outputs_over_weights_positions_and_each_other_are_refused():
    m = _mod("spfa_rope")
    q, k = [torch.randn(4, h, 64, generator=_gen(h), device=DEV) for h in (2, 1)]
    w = [torch.ones(64, device=DEV) for _ in range(2)]
    pos, f = torch.arange(64, device=DEV)[:4], torch.ones(32, device=DEV)
    new = lambda: [torch.empty_like(q), torch.empty_like(k)]
    buf = torch.zeros(4 * 2 * 64, device=DEV)
    on_w, on_f, on_pos = buf[64:128], buf[300:332], buf[100:108].view(torch.int64)
    for args in ((q, k, on_w, w[1], pos, f), (q, k, w[0], on_w, pos, f), (q, k, *w, on_pos, f), (q, k, *w, pos, on_f)):
        for i in (0, 1):
            out = new()
            out[i] = buf[:out[i].numel()].view(out[i].shape) if i == 0 else buf[64:320].view(out[i].shape)
            with pytest.raises(RuntimeError, match="overlaps"):
                m.forward(*args, *out)
            with pytest.raises(RuntimeError, match="overlaps"):
                m.backward(*args, *new(), *out, None, None)
    grads = lambda **kw: m.backward(q, k, *w, pos, f, kw.get("dqo", torch.ones_like(q)), kw.get("dko", torch.ones_like(k)),
                                    kw.get("dq", torch.empty_like(q)), kw.get("dk", torch.empty_like(k)),
                                    kw.get("dwq", torch.empty(64, device=DEV)), kw.get("dwk", torch.empty(64, device=DEV)))
    a, b = new()
    for kw in (dict(dq=a, dwq=a[1, 1]), dict(dq=a, dwk=a[3, 0]), dict(dk=b, dwq=b[2, 0]), dict(dqo=a, dwk=a[0, 0]), dict(dko=b, dwk=b[3, 0]),
               dict(dwq=q[1, 0]), dict(dwk=q[0, 0]), dict(dwq=k[3, 0]), dict(dwq=w[1]), dict(dwk=w[0])):
        with pytest.raises(RuntimeError, match="overlaps"):
            grads(**kw)
    # in place of its own weights
    want = [torch.empty(64, device=DEV) for _ in range(2)]
    grads(dwq=want[0], dwk=want[1])
    grads(dwq=w[0], dwk=w[1])
    assert torch.equal(w[0], want[0]) and torch.equal(w[1], want[1])


def test_rope_angles_next_to_quarter_turns():
    """The sine or cosine of an angle next to a quarter of a turn is as small as what the angle lacks of it: only an
    angle of more than 24 bits gives its leading digits."""
    d, eps = 64, 1e-6
    f = 500000.0 ** (-np.arange(32, dtype=np.float64) / 32)
    f = f.astype(np.float32)
    pos = np.arange(1 << 20, dtype=np.int64)
    rows = []  # per frequency the positions whose angle is nearest to a whole number of quarter turns
    for x in f[:8]:
        t = pos[1:] * (float(x) / (math.pi / 2))
        rows += list(pos[1:][np.argsort(np.abs(t - np.rint(t)))[:8]])
    p = np.array(rows)
    x = torch.zeros(len(p), 1, d, device=DEV)
    x[..., :32] = 1  # pairs (1, 0): they become (cos, sin) of the norm
    out = torch.empty_like(x)
    _mod("spfa_rope").forward(x, x[:, :0], None, None, torch.from_numpy(p).to(DEV), torch.from_numpy(f).to(DEV), out, x[:, :0].clone(), eps)
    want = sv.norm_rope(np64(x), np.ones(d), p.tolist(), f.astype(np.float64), eps, False)
    # angles: two roundings of the product in 64 bits, here and in the oracle (half a step of the position's
    # angle each); sine, cosine, norm and product: 20 roundings of fp32
    angle = np.concatenate([np.abs(p[:, None] * f[None].astype(np.float64))] * 2, 1)[:, None]
    _close(out, want, 20 * U * np.abs(want) + 4 * 2.0 ** -52 * angle * math.sqrt(2) + 2.0 ** -48, "next to a quarter")


# ------------------------------------------------------------------------------------------------
# cache
# ------------------------------------------------------------------------------------------------
def test_cache_outputs_over_scales_rows_and_slots_are_refused():
    m = _mod("spfa_cache")
    pages, page, heads, d, n = 3, 4, 2, 64, 6
    codes = lambda: torch.zeros(pages, page, heads, d, dtype=torch.int8, device=DEV)
    scales = lambda: torch.zeros(pages, page, heads, device=DEV)
    buf = torch.zeros(pages * page * heads * d, dtype=torch.int8, device=DEV)
    over = buf.view(pages, page, heads, d)
    on_scale = buf[512:512 + 4 * pages * page * heads].view(F32).view(pages, page, heads)
    on_rows = buf[256:256 + n * heads * d].view(BF16).view(n, heads, d // 2)
    on_slots = buf[128:128 + 8 * n].view(torch.int64)
    k = torch.randn(n, heads, d, generator=_gen(1), device=DEV).to(BF16)
    slots = torch.arange(n, device=DEV)
    for args in ((k, k, slots, over, codes(), on_scale, scales()), (k, k, slots, over, codes(), scales(), on_scale),
                 (k, k, slots, codes(), over, on_scale, scales()), (k, k, slots, codes(), over, scales(), on_scale),
                 (k, k, on_slots, over, codes(), scales(), scales()), (k, k, on_slots, codes(), over, scales(), scales())):
        with pytest.raises(RuntimeError, match="overlaps"):
            m.write(*args)
    half = [torch.zeros(pages, page, heads, d // 2, dtype=torch.int8, device=DEV) for _ in range(2)]
    rows = torch.zeros(n, heads, d // 2, dtype=BF16, device=DEV)
    for i in (0, 1):  # a scale over rows and over slots
        for x, s, y in ((on_rows, slots, on_scale), (rows, on_slots, buf[64:64 + 4 * pages * page * heads].view(F32).view(pages, page, heads))):
            sc = [scales(), scales()]
            sc[i] = y
            with pytest.raises(RuntimeError, match="overlaps"):
                m.write(x, rows, s, *half, *sc)
            with pytest.raises(RuntimeError, match="overlaps"):
                m.write(rows, x if s is slots else rows, s, *half, *sc)
            out = [torch.zeros_like(rows), torch.zeros_like(rows)]
            out[i] = on_rows
            with pytest.raises(RuntimeError, match="overlaps"):
                m.read(*half, slots, *out, on_scale, scales())
    # codes and scales side by side in one buffer lie in each other's gaps
    packed = torch.zeros(2, pages, page, heads, d + 8, dtype=torch.int8, device=DEV)
    kc, vc = packed[0, ..., :d], packed[1, ..., :d]
    ks, vs = [packed[i, ..., d:d + 4].view(F32).squeeze(-1) for i in (0, 1)]
    m.write(k, k, slots, kc, vc, ks, vs)
    out = [torch.empty_like(k), torch.empty_like(k)]
    m.read(kc, vc, slots, *out, ks, vs)
    want, amax = sv.quantise(np64(k), "int8")
    want = want * (amax / 127)[..., None]
    for x in out:
        _close(x, want, (HALF[BF16] + 4 * U) * np.abs(want), "read back")


# ------------------------------------------------------------------------------------------------
# tree attention
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("far", [14.25, 17.46875])
@pytest.mark.parametrize("nodes", [1, 20, 90])
def test_tree_one_key_far_above_many(nodes, far):
    """f16 weights: one key whose score is `far` (20.6 or 25.2 powers of two) above those of all the others,
    which still show in the result.

    What the other weights lose: they are f16 numbers next to a largest one of at least 2^7, each off by at
    most half of f16's smallest step, 2^-25, where that is more than 2^-11 of it: 2^-32 of the sum a key."""
    d, hk, n, seqs = 64, 8, 1500, 64  # (so many that a workgroup has all keys of an item)
    r = Run(41, F16, "none", d, 64, hk, 1, True, [n - nodes] * seqs, [nodes] * seqs, "chain", strided=False)
    kc, vc, _, _ = r.cache
    k = torch.zeros(seqs, n, hk, d, device=DEV)
    k[:, 1:, :, 0] = -far / 2  # exact in f16, and so are the scores: -16 * far / 2 / 8
    v = 64 * (1 + 0.25 * torch.rand(seqs, n, hk, d, generator=_gen(42), device=DEV))
    v[:, 0] = 0
    k, v = k.to(F16), v.to(F16)
    _mod("spfa_cache").write(k.flatten(0, 1), v.flatten(0, 1), torch.cat(r.slots), kc, vc)
    r.q = torch.zeros(seqs * nodes, hk, d, dtype=F16, device=DEV)
    r.q[..., 0] = 16
    out = torch.empty(r.q.shape, dtype=F16, device=DEV)
    r.call(out)
    for s in (0, 33, seqs - 1):
        for h in (0, hk - 1):
            for i in sorted({0, nodes // 2, nodes - 1}):
                live = n - nodes + i + 1
                row = s * nodes + i
                o, _, _, a, s_abs = sv.tree_attention(np64(r.q[row:row + 1, h]), np64(k[s, :live, h]), np64(v[s, :live, h]),
                                                      np.ones((1, live), dtype=bool), 1 / math.sqrt(d))
                rel = HALF[F16] + (2 * n + 40) * U + 4 * (d + 8) * U * s_abs[0]
                _close(out[row, h], o[0], HALF[F16] * np.abs(o[0]) + a[0] * rel + live * 2.0 ** -32 * 80 + TINY[F16],
                       "sequence %d head %d row %d" % (s, h, i))


@pytest.mark.parametrize("dt,code", [(BF16, "none"), (F16, "none"), (BF16, "e4m3"), (F16, "e4m3"), (BF16, "int8"), (F16, "int8")])
@pytest.mark.parametrize("d,nodes", [(64, 1), (64, 20), (128, 1), (128, 40), (256, 9), (64, 250), (128, 250), (256, 250)])
def test_tree_infinities_in_front_of_the_tree(dt, code, d, nodes):
    """Cached tokens that every row attends hold infinities and NaN, some where weights are tiny."""
    r = Run(43, dt, code, d, 16, 1, 2, True, [700, 140, 9], [nodes, 4, 3], "random", **(ROOM if nodes > 100 else {}))
    kc, vc, ks, vs = r.cache
    sick = {0: [7, 200, 699], 1: [40], 2: []}
    for i in sick:
        for j in sick[i]:
            slot = int(r.slots[i][j])
            p, at = slot // 16, slot % 16
            if code == "none":
                vc[p, at, 0, 5] = float("inf")
                vc[p, at, 0, d - 3] = float("-inf")
                vc[p, at, 0, 9] = float("nan") if j == 200 else float("inf") if j == 7 else 0.0
            elif code == "e4m3" and j != 200:
                vc[p, at, 0].view(torch.uint8)[7] = 0x7f
            else:
                vs[p, at, 0] = float("inf")
    if code == "none":  # the keys of one of them: scores far below the others'
        slot = int(r.slots[0][7])
        kc[slot // 16, slot % 16, 0] = (-4 * r.q[r.off[0], 0].float()).to(dt)
    out = torch.empty(r.q.shape, dtype=dt, device=DEV)
    r.call(out)
    o, q = np64(out), np64(r.q)
    for i in range(3):
        kk, vv = r.read(i)
        lv = r.live(i)
        for hq in range(2):
            rows = np.arange(r.off[i], r.off[i + 1])
            with np.errstate(all="ignore"):
                want, _, _, a, s_abs = sv.tree_attention(q[rows, hq], kk[:, 0], vv[:, 0], lv, 1 / math.sqrt(d))
            for n, row in enumerate(rows):
                w, g = want[n], o[row, hq]
                fine = np.isfinite(w)
                assert np.array_equal(g[~fine], w[~fine], equal_nan=True), (i, n, hq)
                eps_p = 2.0 ** -16 if (code != "none" and dt == F16) else HALF[dt]
                rel = eps_p + (2 * lv.shape[1] + 40) * U + 4 * (d + 8) * U * s_abs[n]
                tol = HALF[dt] * np.abs(w[fine]) + a[n][fine] * rel * (1 + HALF[dt]) + TINY[dt]
                assert (np.abs(g[fine] - w[fine]) <= tol).all(), (i, n, hq)


def test_tree_outputs_over_what_the_call_reads_are_refused():
    r = Run(47, BF16, "int8", 64, 16, 2, 2, True, [20], [3], "tree", strided=False)
    kc, vc, ks, vs = r.cache
    rows = 3
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)
    over = lambda like, dt=None: buf[:like.numel() * like.element_size()].view(dt or like.dtype).view(like.shape)
    new = lambda: torch.empty(r.q.shape, dtype=BF16, device=DEV)
    state = lambda: [torch.full((rows, 4), float("-inf"), device=DEV), torch.zeros(rows, 4, device=DEV)]
    m = _mod("spfa_tree")
    names = ["q", "k_cache", "v_cache", "page_table", "ctx_lens", "q_offsets", "out", "tree_mask", "k_scale", "v_scale"]
    args = lambda **kw: {**dict(zip(names, (r.q, kc.contiguous(), vc.contiguous(), r.table, r.ctx_t, r.off_t, new(), r.mask, ks.contiguous(), vs.contiguous()))), **kw}
    m.forward(**args())
    base = args()
    for name in names:
        if name == "out":
            continue
        at = over(base[name])
        at.copy_(base[name])
        with pytest.raises(RuntimeError, match="out overlaps"):
            m.forward(**args(**{name: at, "out": over(new(), BF16)}))
        for i, what in enumerate("ml"):
            ml = state()
            ml[i] = buf[:48].view(F32).view(rows, 4)
            with pytest.raises(RuntimeError, match="%s overlaps" % what):
                m.forward(**args(**{name: at}), m=ml[0], l=ml[1])
    for i in (0, 1):
        ml = state()
        ml[i] = buf[16:64].view(F32).view(rows, 4)
        with pytest.raises(RuntimeError, match="out overlaps"):
            m.forward(**args(out=over(new(), BF16)), m=ml[0], l=ml[1])


@pytest.mark.parametrize("nodes", [5, 130])
@pytest.mark.parametrize("code", ["none", "int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tree_weights_of_bf16_calls_have_two_parts(d, code, nodes):
    """Two keys whose values nearly cancel in some elements of each row: what is left of them shows the
    weights' rounding, which is to 16 bits in the tiles of few rows and of many."""
    r = Run(44, BF16, code, d, 16, 1, 2, True, [2], [nodes], "random", strided=False, **(dict(spare=50000, wide=50000) if nodes > 100 else {}))
    r.mask.zero_()
    kc, vc, ks, vs = r.cache
    gaps = torch.tensor([0.21, 0.37, 0.58, 0.81, 1.17, 1.51, 1.93, 2.6], device=DEV)
    r.q = torch.zeros(nodes, 2, d, dtype=BF16, device=DEV)
    r.q[:, 0, 0] = (gaps * math.sqrt(d)).to(BF16)[torch.arange(nodes, device=DEV) % 8]
    r.q[:, 1, 0] = (gaps * math.sqrt(d)).to(BF16)[(torch.arange(nodes, device=DEV) + 3) % 8]
    k, v = torch.zeros(2, 1, d, device=DEV), torch.zeros(2, 1, d, device=DEV)
    k[1, 0, 0] = -1
    v[1] = 1 + torch.rand(1, d, generator=_gen(45), device=DEV)
    write = lambda: _mod("spfa_cache").write(k.to(BF16), v.to(BF16), r.slots[0][:2], kc, vc, ks, vs)
    write()
    p = torch.exp(-(gaps * math.sqrt(d)).to(BF16).double() / math.sqrt(d))[torch.arange(d, device=DEV) % 8]
    v[0, 0] = -(p * torch.from_numpy(r.read(0)[1][1, 0]).to(DEV)).float()  # takes the second key's back where e % 8 is the row's gap
    write()
    out = torch.empty(r.q.shape, dtype=BF16, device=DEV)
    r.call(out)
    kk, vv = r.read(0)
    for h in (0, 1):
        o, _, _, a, s_abs = sv.tree_attention(np64(r.q)[:, h], kk[:2, 0], vv[:2, 0], np.ones((nodes, 2), dtype=bool), 1 / math.sqrt(d))
        rel = 2.0 ** -16 + (2 * 2 + 40) * U + 4 * (d + 8) * U * s_abs
        _close(out[:, h], o, HALF[BF16] * np.abs(o) + a * rel[:, None] * (1 + HALF[BF16]) + TINY[BF16], "head %d" % h)


@pytest.mark.parametrize("code", ["none", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
def test_tree_tight_and_roomy_tables(d, code):
    """The table's width and the cache's size choose the kernel, and with it the order of the sums: the same
    rows, keys and lengths stay within their bounds of the exact result and of each other."""
    args = (46, BF16, code, d, 16, 1, 4, True, [500, 90], [60, 50], "chain")
    tight = Run(*args)
    roomy = Run(*args, **ROOM)
    assert torch.equal(tight.q, roomy.q)
    outs = []
    for r in (tight, roomy):
        out = torch.empty(r.q.shape, dtype=BF16, device=DEV)
        r.call(out)
        r.check(out)
        outs.append(np64(out))
    # of each: half a step of itself, and of sum p |v| / l, at most the largest |v|, the weights' 2^-16 and
    # what Run.check allows for sums and scores (of 560 keys)
    v = max(np.abs(tight.read(i)[1]).max() for i in range(2))
    q = np.abs(np64(tight.q)).sum(-1).max() * max(np.abs(tight.read(i)[0]).max() for i in range(2)) / math.sqrt(d)
    rel = 2.0 ** -16 + (2 * 560 + 40) * U + 4 * (d + 8) * U * q
    bound = HALF[BF16] * (np.abs(outs[0]) + np.abs(outs[1])) * 1.01 + 2 * v * rel
    assert (np.abs(outs[0] - outs[1]) <= bound).all()
