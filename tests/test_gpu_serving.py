"""Head norms with the position rotation, the paged cache and the tree attention on the GPU against
the float64 oracle.

Tolerances.  One rounding to a type is off by at most eps / 2 of the value (HALF).  fp32 arithmetic in
between is counted in units U = 2^-24 of the size of what is added up:
  rope       a sum of d squares, its mean, root and quotient, weight and rotation: d / 2 + 20 roundings
             of a pair's elements; the angle reduced to fp32 within 2^-26 turns: 8 more
  gradients  two such sums: d + 60; the weights' sum over n vectors: n + 60 more, of the absolute terms
  tree       weights are rounded to the type of the second product (f16 over 8-bit caches: to 16 bits),
             scores err by (d + 8) U of sum |q k| * scale, which the exponential turns into a relative
             error of numerator and denominator; sums over n keys: 2 n + 40; a move of the reference
             by the slack costs nothing more
"""
import gc
import importlib
import math

import numpy as np
import pytest
import torch

import spfa_autograd
import spfa_masks
from helpers import np64
from oracle import serve_oracle as sv

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _leave_nothing():
    """Large tensors that refused calls' tracebacks hold go now, not while a later test counts memory."""
    yield
    gc.collect()


def _mod(name):
    return importlib.import_module(name)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _close(got, want, bound, what):
    got = np64(got)
    assert np.isfinite(got).all(), what
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), "%s: off by %.3e where %.3e is allowed" % (
        what, np.abs(got - want).flat[over.argmax()], np.broadcast_to(bound, over.shape).flat[over.argmax()])


# ------------------------------------------------------------------------------------------------
# rope
# ------------------------------------------------------------------------------------------------
def _pair_size(y, rot, interleaved):
    """|a| + |b| of the pair an element belongs to."""
    s = np.abs(y).copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        s[..., a] = s[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    return s


ROPE = [  # dtype, tokens, heads of q and k, d, rot, interleaved, weights' dtype, fused, heads first
    (BF16, 1, 4, 1, 128, 128, False, BF16, True, False),
    (BF16, 67, 5, 2, 128, 128, False, F32, True, True),
    (F16, 33, 3, 3, 64, 32, True, F16, False, True),
    (F16, 9, 2, 1, 256, 256, False, None, True, False),
    (F32, 21, 3, 2, 96, 64, False, F32, True, False),
    (F32, 5, 1, 1, 1024, 1024, False, F32, False, False),
    (BF16, 5, 2, 1, 1024, 512, True, BF16, False, True),
    (F32, 40, 2, 1, 128, 0, False, F32, False, False),
    (BF16, 17, 3, 1, 80, 40, False, BF16, True, False),   # pieces do not divide the rotated part
    (F16, 17, 3, 1, 33, 10, False, F16, False, False),    # odd heads
    (F32, 6, 2, 2, 7, 6, True, F32, False, True),
    (BF16, 6, 2, 2, 1, 0, False, BF16, False, False),
    (F32, 300, 1, 1, 2, 2, False, F32, False, False),
]


def _rope_inputs(case, seed, batch=None):
    dt, tokens, hq, hk, d, rot, inter, wdt, fused, first = case
    g = _gen(seed)
    lead = (tokens,) if batch is None else (batch, tokens)
    if fused:
        x = torch.randn(*lead, (hq + 2 * hk) * d, generator=g, device=DEV).to(dt)
        q = x[..., :hq * d].unflatten(-1, (hq, d))
        k = x[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    else:
        q = torch.randn(*lead, hq, d, generator=g, device=DEV).to(dt)
        k = torch.randn(*lead, hk, d, generator=g, device=DEV).to(dt)
    w = [None, None] if wdt is None else [(1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(wdt) for _ in range(2)]
    pos = torch.randint(-50, 1 << 20, lead, generator=g, device=DEV, dtype=torch.int64)
    f = 10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=F32) / max(rot // 2, 1))
    return q, k, w, pos, f


def _ones(w, d):
    return np.ones(d) if w is None else np64(w)


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "%s_t%d_h%d_%d_d%d_r%d" % (str(c[0])[6:], *c[1:6]))
def test_rope_forward_and_gradients(case):
    dt, tokens, hq, hk, d, rot, inter, wdt, fused, first = case
    q, k, w, pos, f = _rope_inputs(case, 5)
    mk = lambda x: (torch.empty(x.shape[1], x.shape[0], d, dtype=dt, device=DEV).transpose(0, 1) if first
                    else torch.empty(x.shape, dtype=dt, device=DEV))
    m = _mod("spfa_rope")
    qo, ko = mk(q), mk(k)
    back = m.forward(q, k, *w, pos, f, qo, ko, 1e-5, inter)
    assert back[0].data_ptr() == qo.data_ptr() and back[1].data_ptr() == ko.data_ptr()
    dqo, dko = mk(q).normal_(generator=_gen(6)), mk(k).normal_(generator=_gen(7))
    dq, dk = torch.empty(q.shape, dtype=dt, device=DEV), torch.empty(k.shape, dtype=dt, device=DEV)
    dw = [torch.full((d,), 77.0, device=DEV) for _ in range(2)]  # written, not added to
    m.backward(q, k, *w, pos, f, dqo, dko, dq, dk, *dw, 1e-5, inter)
    p, fr = pos.cpu().numpy(), np64(f)
    for x, y, dy, dx, ww, dww, heads in ((q, qo, dqo, dq, w[0], dw[0], hq), (k, ko, dko, dk, w[1], dw[1], hk)):
        want = sv.norm_rope(np64(x), _ones(ww, d), p, fr, 1e-5, inter)
        _close(y, want, HALF[dt] * np.abs(want) + TINY[dt] + (d / 2 + 28) * U * _pair_size(want, rot, inter) * 1.5, "forward")
        gx, gw, sx, sw = sv.norm_rope_backward(np64(x), _ones(ww, d), p, fr, 1e-5, inter, np64(dy))
        _close(dx, gx, HALF[dt] * np.abs(gx) + TINY[dt] + (d + 60) * U * sx, "gradient")
        _close(dww, gw, (d + 60 + tokens * heads) * U * sw + TINY[F32], "weights' gradient")
    # in place, and again into the same tensors: the same bits
    q2, k2 = q.clone(), k.clone()
    m.forward(q2, k2, *w, pos, f, q2, k2, 1e-5, inter)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    dw2 = [torch.empty(d, device=DEV) for _ in range(2)]
    m.backward(q, k, *w, pos, f, dqo, dko, dqo, dko, *dw2, 1e-5, inter)
    assert torch.equal(dqo, dq) and torch.equal(dko, dk) and torch.equal(dw2[0], dw[0]) and torch.equal(dw2[1], dw[1])


@pytest.mark.parametrize("case,batch", [
    ((BF16, 11, 6, 2, 128, 128, False, BF16, True, False), 901),   # more rows of a batch than tokens in a workgroup's share
    ((F32, 4713, 12, 2, 64, 32, True, F32, True, False), 1),
    ((F16, 2100, 3, 1, 33, 10, False, F16, False, False), 2),
    ((BF16, 1, 5, 1, 256, 64, False, F32, False, False), 6007),    # one token of each
], ids=["bf16", "f32", "odd", "steps"])
def test_rope_of_many_vectors(case, batch):
    """Calls that fill the device: workgroups with several rounds and shares, and weights at odd addresses."""
    dt, tokens, hq, hk, d, rot, inter, wdt, fused, _ = case
    q, k, w, pos, f = _rope_inputs(case, 8, batch)
    m = _mod("spfa_rope")
    qo, ko = torch.empty(q.shape, dtype=dt, device=DEV), torch.empty(k.shape, dtype=dt, device=DEV)
    m.forward(q, k, *w, pos, f, qo, ko, 1e-5, inter)
    g = _gen(9)
    dqo, dko = [torch.randn(x.shape, generator=g, device=DEV).to(dt) for x in (q, k)]
    dq, dk = torch.empty_like(dqo), torch.empty_like(dko)
    dw = [torch.empty(d, device=DEV) for _ in range(2)]
    m.backward(q, k, *w, pos, f, dqo, dko, dq, dk, *dw, 1e-5, inter)
    p, fr = pos.flatten().cpu().numpy(), np64(f)
    flat = lambda x: np64(x).reshape(batch * tokens, -1, d)
    for x, y, dy, dx, ww, dww, heads in ((q, qo, dqo, dq, w[0], dw[0], hq), (k, ko, dko, dk, w[1], dw[1], hk)):
        want = sv.norm_rope(flat(x), _ones(ww, d), p, fr, 1e-5, inter)
        _close(y.reshape(want.shape), want, HALF[dt] * np.abs(want) + TINY[dt] + (d / 2 + 28) * U * _pair_size(want, rot, inter) * 1.5, "forward")
        gx, gw, sx, sw = sv.norm_rope_backward(flat(x), _ones(ww, d), p, fr, 1e-5, inter, flat(dy))
        _close(dx.reshape(gx.shape), gx, HALF[dt] * np.abs(gx) + TINY[dt] + (d + 60) * U * sx, "gradient")
        _close(dww, gw, (d + 60 + batch * tokens * heads) * U * sw + TINY[F32], "weights' gradient")
    # weights that do not start at a multiple of 16 bytes
    odd = [torch.cat((x[:1], x))[1:] for x in w]
    q2, k2 = torch.empty_like(qo), torch.empty_like(ko)
    m.forward(q, k, *odd, pos, f, q2, k2, 1e-5, inter)
    for y, y2 in ((qo, q2), (ko, k2)):
        # (other lanes sum the squares: either is within the bound above of the exact value)
        want = np64(y).reshape(batch * tokens, -1, d)
        _close(y2.reshape(want.shape), want, 2 * HALF[dt] * np.abs(want) * 1.01 + 2 * TINY[dt]
               + (d + 56) * U * _pair_size(want, rot, inter) * 1.6, "weights at an odd address")


def test_rope_batches_positions_and_empty_sides():
    m = _mod("spfa_rope")
    case = (BF16, 3, 2, 1, 64, 64, False, BF16, True, False)
    q, k, w, pos, f = _rope_inputs(case, 8, batch=5)
    whole = [torch.empty(x.shape, dtype=BF16, device=DEV) for x in (q, k)]
    m.forward(q, k, *w, pos, f, *whole)
    for b in range(5):
        one = [torch.empty(x.shape[1:], dtype=BF16, device=DEV) for x in (q, k)]
        m.forward(q[b], k[b], *w, pos[b].to(torch.int32), f, *one)
        assert torch.equal(one[0], whole[0][b]) and torch.equal(one[1], whole[1][b])
    # one row of positions for every batch entry
    shared = [torch.empty(x.shape, dtype=BF16, device=DEV) for x in (q, k)]
    m.forward(q, k, *w, pos[2], f, *shared)
    assert torch.equal(shared[0][2], whole[0][2]) and not torch.equal(shared[0][1], whole[0][1])
    # no keys; no tokens: the weights' gradients are zeros
    none = k[:, :, :0]
    only = torch.empty(q.shape, dtype=BF16, device=DEV)
    m.forward(q, none, *w, pos, f, only, none.clone())
    assert torch.equal(only, whole[0])
    dw = [torch.full((64,), 3.0, device=DEV) for _ in range(2)]
    m.backward(q[:, :0], k[:, :0], *w, pos[:, :0].contiguous(), f, q[:, :0], k[:, :0], q[:, :0].clone(), k[:, :0].clone(), *dw)
    assert not dw[0].any() and not dw[1].any()
    # zeros and a NaN: only the vector that holds it
    q = q.clone()
    q[1, 1] = 0
    q[2, 0, 1, 5] = float("nan")
    m.forward(q, k, *w, pos, f, *shared)
    assert not shared[0][1, 1].any()
    bad = torch.isnan(shared[0]).any(-1)
    assert bad.sum() == 1 and bad[2, 0, 1]


def test_rope_far_positions_are_exact():
    """Angles of positions up to 2^31 keep their fraction of a turn: fp32 products would lose it."""
    m = _mod("spfa_rope")
    d = 64
    pos = torch.tensor([0, 1, (1 << 31) - 1, 12345678901, -(1 << 31)], device=DEV)
    f = 500000.0 ** (-torch.arange(32, device=DEV, dtype=F32) / 32)
    q = torch.randn(5, 2, d, generator=_gen(1), device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(q)
    m.forward(q, q, None, None, pos, f, qo, ko)
    want = sv.norm_rope(np64(q), np.ones(d), pos.tolist(), np64(f), 1e-6, False)
    # (the oracle's own angle, up to 2^34, is good to 2^-19)
    _close(qo, want, HALF[F32] * np.abs(want) + ((d / 2 + 28) * U * 1.5 + 2.0 ** -19) * _pair_size(want, d, False), "far")


def test_rope_autograd_feeds_attention_and_its_gradients():
    """q and k of a fused projection through qk_norm_rope and windowed attention, against the chain's
    gradients in float64 by torch's own differentiation on the CPU."""
    n, h, d, w = 96, 2, 32, 7
    g = _gen(3)
    x = torch.randn(1, n, 3 * h * d, generator=g, device=DEV, requires_grad=True)
    wq, wk = [(1 + 0.2 * torch.randn(d, generator=g, device=DEV)).requires_grad_(True) for _ in range(2)]
    pos = torch.arange(n, device=DEV) + 7
    f = 100.0 ** (-torch.arange(d // 2, device=DEV, dtype=F32) / (d // 2))
    d_out = torch.randn(1, h, n, d, generator=g, device=DEV)

    def parts(x):
        q, k, v = x.split(h * d, -1)
        return q.unflatten(-1, (h, d)), k.unflatten(-1, (h, d)), v.unflatten(-1, (h, d)).transpose(1, 2)

    q, k, v = parts(x)
    q, k = spfa_autograd.qk_norm_rope(q, k, wq, wk, pos, f)
    assert tuple(q.shape) == (1, h, n, d) and q.is_contiguous()
    spfa_autograd.attention(q, k, v, [("local", w)]).backward(d_out)
    got = [t.grad for t in (x, wq, wk)]
    xr, wr = x.detach().double().cpu().requires_grad_(True), [t.detach().double().cpu().requires_grad_(True) for t in (wq, wk)]
    ang = pos.double().cpu()[:, None] * f.double().cpu()
    co, si = ang.cos()[:, None], ang.sin()[:, None]

    def rope(t, wt):
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wt
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat((a * co - b * si, a * si + b * co), -1).transpose(1, 2)

    q, k, v = parts(xr)
    s = rope(q, wr[0]) @ rope(k, wr[1]).transpose(-1, -2) / math.sqrt(d)
    i = torch.arange(n)
    s = s.masked_fill((i[:, None] - i).abs() > w, float("-inf"))
    (s.softmax(-1) @ v).backward(d_out.double().cpu())
    for a, b, what in zip(got, (xr.grad, wr[0].grad, wr[1].grad), ("x", "w_q", "w_k")):
        # the attention's own gradient bar is 2e-4 of the largest value (its fp32 sums); the rope's adds U's
        err = (a.double().cpu() - b).abs().max().item()
        assert err <= 4e-4 * max(1.0, b.abs().max().item()), (what, err)


def test_rope_expanded_gradients_and_missing_weights():
    x = torch.randn(4, 2, 16, generator=_gen(1), device=DEV, requires_grad=True)
    y = torch.randn(4, 1, 16, generator=_gen(2), device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    pos, f = torch.arange(4, device=DEV), torch.ones(8, device=DEV)
    a, b = spfa_autograd.qk_norm_rope(x, y, w, None, pos, f)
    (a.sum() + b.sum()).backward()
    ones = lambda t: np.ones(t.shape)
    for t, ww in ((x, np.ones(16)), (y, np.ones(16))):
        gx, gw, sx, sw = sv.norm_rope_backward(np64(t), ww, range(4), np.ones(8), 1e-6, False, ones(t))
        _close(t.grad, gx, HALF[F32] * np.abs(gx) + 76 * U * sx, "gradient")
        if t is x:
            _close(w.grad, gw, 84 * U * sw, "weights' gradient")


def test_rope_refusals():
    m = _mod("spfa_rope")
    q, k = torch.zeros(4, 2, 16, device=DEV), torch.zeros(4, 1, 16, device=DEV)
    pos, f, w = torch.arange(4, device=DEV), torch.ones(8, device=DEV), torch.ones(16, device=DEV)
    call = lambda q=q, k=k, wq=w, wk=w, p=pos, f=f, qo=None, ko=None, **kw: m.forward(
        q, k, wq, wk, p, f, torch.empty_like(q) if qo is None else qo, torch.empty_like(k) if ko is None else ko, **kw)
    call()
    bad = [dict(q=q.double(), k=k.double()), dict(q=q.half()), dict(k=k[:3]), dict(k=torch.zeros(4, 1, 8, device=DEV)),
           dict(f=torch.ones(9, device=DEV)), dict(f=f.double()), dict(f=f.view(2, 4)), dict(p=pos[:3].contiguous()), dict(p=pos.float()),
           dict(p=pos.view(1, 4)), dict(wq=w[:8].contiguous()), dict(wq=w.half(), wk=w.half()), dict(wq=w.cpu()),
           dict(q=torch.zeros(4, 16, 2, device=DEV).transpose(1, 2)), dict(qo=torch.zeros(4, 1, 16, device=DEV).expand(4, 2, 16)),
           dict(qo=torch.zeros(4, 2, 16, device=DEV, dtype=F16)), dict(eps=-1.0), dict(q=q[0], k=k[0])]
    buf = torch.zeros(4 * 32 + 16, device=DEV)
    bad.append(dict(q=buf[:128].view(4, 2, 16), qo=buf[16:].view(4, 2, 16)))  # half on its input
    for kw in bad:
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)
    wide = torch.zeros(1, 1, 1025, device=DEV)
    with pytest.raises(ValueError):
        m.forward(wide, wide, None, None, pos[:1], f, wide.clone(), wide.clone())
    with pytest.raises(RuntimeError):
        m.backward(q, k, w, w, pos, f, q, k, q.clone(), k.clone(), torch.empty(16, device=DEV, dtype=F16), None)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------
# cache
# ------------------------------------------------------------------------------------------------
CODES = {"none": None, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _new_cache(pages, page, heads, d, dt, code, head_pages, fill=0):
    """(k_cache, v_cache, k_scale, v_scale) with every byte of the codes set to `fill`."""
    shape = (pages, heads, page) if head_pages else (pages, page, heads)
    order = (0, 2, 1) if head_pages else (0, 1, 2)
    cd = CODES[code] or dt
    out = []
    for _ in range(2):
        raw = torch.full((*shape, d * torch.empty(0, dtype=cd).element_size()), fill, dtype=torch.uint8, device=DEV)
        out.append(raw.view(cd).permute(*order, 3))
    if code == "none":
        return out + [None, None]
    return out + [torch.full(shape, -7.0, device=DEV).permute(*order) for _ in range(2)]


def _as_float(codes):
    return codes.float() if codes.dtype != torch.int8 else codes.to(F32)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("code", ["none", "int8", "e4m3"])
@pytest.mark.parametrize("d,heads,page,head_pages", [(64, 3, 16, True), (128, 2, 48, False), (256, 1, 5, True), (80, 5, 1, False),
                                                     (272, 2, 7, True), (1024, 1, 3, False), (40, 2, 16, True), (33, 3, 9, False),
                                                     (1, 1, 4, True), (500, 1, 2, True)])
def test_cache_write_and_read(dt, code, d, heads, page, head_pages):
    m = _mod("spfa_cache")
    g = _gen(d + heads)
    pages, tokens = 70 // page + 2, 61
    kc, vc, ks, vs = _new_cache(pages, page, heads, d, dt, code, head_pages, fill=17)
    before = [x.clone() for x in (kc, vc) ] + [None if x is None else x.clone() for x in (ks, vs)]
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].to(torch.int32 if heads > 2 else torch.int64)
    slots[3], slots[4], slots[7] = -1, pages * page, 2 ** 31 - 1  # skipped
    fused = torch.randn(tokens, 2 * heads * d, generator=g, device=DEV)
    fused *= torch.exp(4 * torch.randn(tokens, 1, generator=g, device=DEV))
    fused[10] = 0
    fused = fused.to(dt)
    k, v = fused[:, :heads * d].unflatten(-1, (heads, d)), fused[:, heads * d:].unflatten(-1, (heads, d))
    k[11, 0] = torch.arange(d, device=DEV).to(dt) * (k[11, 0, 0] if d == 1 else 0.5)  # ties
    m.write(k, v, slots, kc, vc, ks, vs)
    live = [i for i in range(tokens) if i not in (3, 4, 7)]
    sl = slots.long()[live]
    at = (sl // page, sl % page)
    if code == "none":
        assert torch.equal(kc.contiguous()[at], k[live]) and torch.equal(vc.contiguous()[at], v[live])
    else:
        for x, c, s in ((k, kc, ks), (v, vc, vs)):
            # (f16 rows may hold an infinity here: their scale is no finite number, whatever their codes)
            fine = torch.isfinite(x[live]).all(-1).cpu().numpy()
            want, amax = sv.quantise(np.where(fine[..., None], np64(x[live]), 0.0), code)
            codes = _as_float(c.contiguous())[at]
            assert np.array_equal(np64(codes)[fine], want[fine])
            top = np.float32(sv.TOP[code])
            scales = s.contiguous()[at].cpu().numpy()
            assert np.array_equal(scales[fine], amax.astype(np.float32)[fine] / top)
            assert not np.isfinite(scales[~fine]).any()
    # nothing else was touched
    keep = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    keep[sl] = False
    for x, y in zip((kc, vc, ks, vs), before):
        if x is not None:
            b = lambda t: t.contiguous().flatten(0, 1).view(torch.uint8 if t.element_size() == 1 else t.dtype)[keep]
            assert torch.equal(b(x), b(y))
    # read back: into [heads, tokens, d], any order, a slot twice, skipped rows as they were
    want_slots = torch.cat((slots[20:], slots[:8], slots[20:22]))
    n = want_slots.numel()
    ko = torch.full((heads, n, d), 5.0, dtype=dt, device=DEV).transpose(0, 1)
    vo = torch.full((n, heads, d), 5.0, dtype=dt, device=DEV)
    m.read(kc, vc, want_slots, ko, vo, ks, vs)
    src = list(range(20, tokens)) + list(range(8)) + [20, 21]
    for c, s, o, x in ((kc, ks, ko, k), (vc, vs, vo, v)):
        for i, t in enumerate(src):
            if t in (3, 4, 7):
                assert (o[i] == 5.0).all()
            elif code == "none":
                assert torch.equal(o[i], x[t])
            else:
                p, r = int(slots[t]) // page, int(slots[t]) % page
                fine = torch.isfinite(x[t]).all(-1)
                # code * scale is at most U of itself off in fp32 and half a step in the output's type
                # (a multiplication that rounds to f16 at once need not agree with two roundings)
                val = np64(_as_float(c[p, r])) * np64(s[p, r])[:, None]
                _close(o[i][fine], val[fine.cpu().numpy()], ((HALF[dt] + U * (1 + HALF[dt])) * np.abs(val) + TINY[dt])[fine.cpu().numpy()], "read back")
                assert torch.isnan(o[i][~fine]).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=str)
def test_cache_borders_and_extremes(dt, code):
    """Values on and next to the borders between codes, the type's smallest and largest numbers,
    infinities and NaN."""
    m = _mod("spfa_cache")
    d = 64
    top = sv.TOP[code]
    rows = []
    for amax in (top, 1.0, 0.3, 254.0, 2.0 ** -14, float(torch.finfo(dt).max), float(torch.finfo(dt).tiny)):
        a = torch.tensor(amax, dtype=dt).double()
        codes = torch.arange(1, 63, dtype=torch.float64)
        y = torch.cat((a.view(1), (codes + 0.5) * a / top, a.view(1) / 2))
        rows += [y, -y, y * (1 + 2.0 ** -11), y.flip(0) * (1 - 2.0 ** -9)]
    x = torch.stack(rows).to(dt).to(DEV).clamp(min=torch.finfo(dt).min, max=torch.finfo(dt).max).view(len(rows), 1, d)
    kc, vc, ks, vs = _new_cache(len(rows), 1, 1, d, dt, code, True)
    slots = torch.arange(len(rows), device=DEV)
    m.write(x, x, slots, kc, vc, ks, vs)
    want, _ = sv.quantise(np64(x), code)
    assert np.array_equal(np64(_as_float(kc))[:, 0], want) and np.array_equal(np64(_as_float(vc))[:, 0], want)
    for special in (float("inf"), float("-inf"), float("nan")):
        x[0, 0, 5] = special
        m.write(x[:2], x[:2], slots[:2], kc, vc, ks, vs)
        o = torch.zeros(2, 1, d, dtype=dt, device=DEV)
        m.read(kc, vc, slots[:2], o, o.clone(), ks, vs)
        assert torch.isnan(o[0]).all() and torch.isfinite(o[1]).all()


def test_cache_refusals():
    m = _mod("spfa_cache")
    kc, vc, ks, vs = _new_cache(3, 4, 2, 16, BF16, "int8", True)
    k = torch.zeros(5, 2, 16, dtype=BF16, device=DEV)
    s = torch.arange(5, device=DEV)
    m.write(k, k, s, kc, vc, ks, vs)
    bad = [(k, k, s, kc, vc), (k, k, s, kc, vc, ks, vs.double()), (k, k, s[:4].contiguous(), kc, vc, ks, vs), (k, k, s.float(), kc, vc, ks, vs),
           (k, k.half(), s, kc, vc, ks, vs), (k.double(), k.double(), s, kc, vc, ks, vs), (k, k[:, :1], s, kc, vc, ks, vs),
           (k[:, :1], k[:, :1], s, kc, vc, ks, vs), (k, k, s, kc, vc.view(torch.float8_e4m3fn), ks, vs), (k, k, s, kc[:2], vc, ks, vs),
           (k, k, s, kc, vc, ks[:2], vs), (k, k, s, k.view(5, 2, 1, 16), k.view(5, 2, 1, 16), None, None),
           (k, k, s, kc, vc, ks.cpu(), vs), (k, k, s, kc[:1].expand(3, 4, 2, 16), vc, ks, vs), (k, k, s.cpu(), kc, vc, ks, vs)]
    for args in bad:
        with pytest.raises((RuntimeError, ValueError)):
            m.write(*args)
    o = torch.zeros(5, 1, 16, dtype=BF16, device=DEV).expand(5, 2, 16)
    with pytest.raises(RuntimeError):
        m.read(kc, vc, s, o, k, ks, vs)
    plain = torch.zeros(3, 4, 2, 16, dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError):
        m.write(k, k, s, plain, plain.clone(), ks, vs)
    with pytest.raises(RuntimeError):
        m.write(k.half(), k.half(), s, plain, plain.clone())
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------
# tree attention
# ------------------------------------------------------------------------------------------------
class Run:
    """A batch of sequences in a cache, and what each row attends, in numbers."""

    def __init__(self, seed, dt, code, d, page, hk, group, head_pages, ctx, nodes, mask, front=0, behind=0, spare=3, wide=0,
                 strided=True):
        g = _gen(seed)
        rng = np.random.default_rng(seed)
        self.dt, self.code, self.d, self.hk, self.group, self.ctx, self.nodes, self.page = dt, code, d, hk, group, ctx, nodes, page
        n, total = len(ctx), front + sum(nodes) + behind
        need = [-(-(c + m) // page) for c, m in zip(ctx, nodes)]
        pages = sum(need) + spare
        # bytes of ones: NaN in every 16-bit and e4m3 place that is not written
        self.cache = _new_cache(pages, page, hk, d, dt, code, head_pages, fill=0xff)
        kc, vc, ks, vs = self.cache
        if ks is not None:
            ks.fill_(float("nan"))
            vs.fill_(float("nan"))
        order = rng.permutation(pages)[:sum(need)]
        table = np.full((n, max(need + [0]) + wide), -1, dtype=np.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m]
            at += m
        self.table_np = table
        t = torch.from_numpy(table).to(DEV)
        self.table = torch.cat((t, t), 1)[:, :t.shape[1]] if strided else t
        self.slots = [torch.from_numpy((table[i, np.arange(c + m) // page].astype(np.int64) * page + np.arange(c + m) % page)).to(DEV)
                      for i, (c, m) in enumerate(zip(ctx, nodes))]
        allslots = torch.cat(self.slots) if n else torch.zeros(0, dtype=torch.int64, device=DEV)
        k, v = [torch.randn(allslots.numel(), hk, d, generator=g, device=DEV).to(dt) for _ in range(2)]
        if allslots.numel():
            _mod("spfa_cache").write(k, v, allslots, kc, vc, ks, vs)
        self.ctx_t = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32) + front
        self.off = off
        self.off_t = torch.from_numpy(off).to(DEV)
        hq = hk * group
        x = (1.5 * torch.randn(total, hq + 3, d + (8 if strided else 0), generator=g, device=DEV)).to(dt)
        self.q = x[:, 1:hq + 1, :d] if strided else x[:, :hq, :d].contiguous()
        words = max(1, -(-max(nodes + [0]) // 64))
        self.mask = None
        self.tree = [np.tril(np.ones((m, m), dtype=bool)) for m in nodes]
        if mask != "chain":
            bits = torch.zeros(total, words, dtype=torch.int64, device=DEV)
            if mask == "tree":
                parents = [-1] * front
                for m in nodes:
                    parents += [int(rng.integers(-1, j)) if j else -1 for j in range(m)]
                parents += [-1] * behind
                bits = spfa_masks.tree_mask(parents, off.tolist(), device=DEV)
            else:  # any bits, also such as leave a row of an empty context nothing, and bits past the tree
                low, high = torch.randint(0, 1 << 32, (2, total, words), generator=g, device=DEV)
                bits = (high << 32) | low
                bits[::3] = 0
            self.mask = bits.contiguous()
            b = self.mask.cpu().numpy().astype(np.uint64)
            for i, m in enumerate(nodes):
                j = np.arange(m)
                rows = b[off[i]:off[i] + m]
                self.tree[i] = ((rows[:, j // 64] >> (j % 64).astype(np.uint64)) & np.uint64(1)).astype(bool)

    def read(self, i):
        """Keys and values of sequence i as numbers."""
        kc, vc, ks, vs = self.cache
        p = torch.from_numpy(self.table_np[i].astype(np.int64)).to(DEV)
        x = np.arange(self.ctx[i] + self.nodes[i])
        pg, at = p[x // self.page], torch.from_numpy(x % self.page).to(DEV)
        out = []
        for c, s in ((kc, ks), (vc, vs)):
            y = np64(_as_float(c.contiguous())[pg, at]) if c.dtype not in (F16, BF16) else np64(c.contiguous()[pg, at])
            out.append(y if s is None else y * np64(s.contiguous()[pg, at])[..., None])
        return out

    def live(self, i):
        return np.concatenate([np.ones((self.nodes[i], self.ctx[i]), dtype=bool), self.tree[i]], 1)

    def call(self, out, **kw):
        kc, vc, ks, vs = self.cache
        return _mod("spfa_tree").forward(self.q, kc, vc, self.table, self.ctx_t, self.off_t, out, self.mask, ks, vs, **kw)

    def check(self, out, m=None, l=None, scale=None, live=None, base=None, want_nan=()):
        scale = 1 / math.sqrt(self.d) if scale is None else scale
        q = np64(self.q)
        eps_p = 2.0 ** -16 if (self.code != "none" and self.dt == F16) else HALF[self.dt]
        for i in range(len(self.ctx)):
            if not self.nodes[i]:
                continue
            ks, vs = self.read(i)
            lv = self.live(i) if live is None else live(i)
            n = lv.shape[1]
            for hq in range(self.hk * self.group):
                rows = slice(self.off[i], self.off[i + 1])
                o, mm, ll, a, s_abs = sv.tree_attention(q[rows, hq], ks[:, hq // self.group], vs[:, hq // self.group], lv, scale)
                rel = eps_p + (2 * n + 40) * U + 4 * (self.d + 8) * U * s_abs
                tol = HALF[self.dt] * np.abs(o) + (a * rel[:, None]) * (1 + HALF[self.dt]) + TINY[self.dt]
                has = ll > 0
                got = out[rows, hq]
                _close(got[torch.from_numpy(has).to(DEV)], o[has], tol[has], "out of sequence %d head %d" % (i, hq))
                empty = torch.from_numpy(~has).to(DEV)
                if m is None:
                    assert not got[empty].any()
                else:
                    assert torch.equal(got[empty], base[rows, hq][empty])
                    e = np64(m[rows, hq])[has] + np.log(np64(l[rows, hq])[has]) - (mm + np.log(np.where(ll > 0, ll, 1)))[has]
                    assert (np.abs(e) <= rel[has] + 2.0 ** -20).all()


# places for many more tokens than the sequences have: calls over as much are worked on in larger tiles
ROOM = dict(spare=33000, wide=16500)
TREES = [  # dtype, code, d, page, kv heads, group, head_pages, ctx, nodes, mask
    (BF16, "none", 128, 16, 2, 4, True, [700], [1], "chain"),
    (F16, "none", 64, 32, 1, 8, True, [0, 31, 32, 33, 500], [1, 1, 1, 1, 1], "chain"),
    (BF16, "e4m3", 128, 64, 2, 4, True, [127, 128, 129, 0, 1500, 1], [1, 1, 1, 1, 1, 1], "chain"),
    (F16, "int8", 128, 16, 2, 7, False, [300, 0, 1023], [13, 5, 1], "tree"),
    (BF16, "int8", 64, 48, 2, 3, True, [95, 96, 1], [9, 33, 64], "tree"),
    (F16, "e4m3", 256, 16, 1, 2, True, [77, 400], [3, 20], "random"),
    (BF16, "none", 256, 5, 1, 5, False, [64, 3], [7, 30], "random"),
    (F16, "none", 64, 32, 1, 8, True, [256, 129], [61, 70], "tree"),       # many rows, two words of bits
    (BF16, "none", 128, 64, 1, 8, True, [260, 0], [40, 17], "random"),
    (F16, "int8", 64, 24, 1, 4, False, [200, 37], [130, 65], "random"),    # three words
    (BF16, "e4m3", 128, 128, 1, 1, True, [900], [200], "chain"),            # a chunk of a prompt
    (F16, "e4m3", 96, 16, 2, 2, True, [150, 40], [4, 2], "tree"),           # heads shorter than the kernel's
    (BF16, "none", 40, 16, 3, 1, False, [150, 40], [4, 2], "chain"),
    (BF16, "int8", 208, 16, 1, 2, True, [50], [3], "tree"),
    (F16, "none", 33, 7, 2, 2, False, [70, 0], [3, 6], "random"),           # odd heads
    (BF16, "e4m3", 7, 1, 1, 3, True, [40], [2], "chain"),                   # pages of one token
    (F16, "int8", 130, 3, 1, 2, False, [97], [5], "tree"),
    (BF16, "none", 1, 4, 1, 1, True, [9], [2], "chain"),
    (BF16, "none", 128, 4096, 1, 2, True, [2000, 5], [0, 2], "chain"),      # a sequence without rows
    (F16, "none", 128, 16, 8, 1, True, [3] * 70, [1] * 70, "chain"),        # more sequences than lanes
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "%s_%s_d%d_p%d_%s_%d" % (str(c[0])[6:], c[1], c[2], c[3], c[9], max(c[7])))
def test_tree_attention(case):
    r = Run(11, *case, front=2, behind=3)
    out = torch.full(r.q.shape, 9.0, dtype=r.dt, device=DEV)
    back = r.call(out)
    assert back.data_ptr() == out.data_ptr()
    r.check(out)
    assert (out[:2] == 9.0).all() and (out[r.off[-1]:] == 9.0).all()  # rows of no sequence
    # the same bits again, into a strided output
    other = torch.full((r.q.shape[1], r.q.shape[0], r.d + 3), 4.0, dtype=r.dt, device=DEV)
    r.call(other.transpose(0, 1)[..., :r.d])
    assert torch.equal(other.transpose(0, 1)[2:r.off[-1], :, :r.d], out[2:r.off[-1]])
    assert (other[..., r.d:] == 4.0).all()


LARGE_TREES = [  # all with more than 192 rows per head
    (F16, "none", 64, 16, 2, 8, True, [700, 0, 31, 128], [61, 40, 2, 50], "tree"),
    (BF16, "none", 128, 16, 2, 8, False, [513, 90], [70, 33], "random"),
    (BF16, "none", 96, 16, 2, 4, True, [300], [130], "chain"),
    (F16, "none", 256, 16, 1, 4, True, [127, 1], [100, 29], "tree"),
    (BF16, "int8", 64, 16, 1, 4, True, [400, 129], [64, 65], "random"),
    (F16, "int8", 128, 16, 2, 7, False, [640, 5], [31, 33], "tree"),
    (F16, "e4m3", 128, 16, 2, 8, True, [100, 3], [70, 10], "random"),
    (BF16, "e4m3", 208, 16, 2, 3, True, [256], [128], "chain"),
    (F16, "int8", 32, 16, 2, 5, True, [50, 0, 0], [70, 0, 60], "random"),
    (BF16, "e4m3", 256, 16, 2, 1, True, [1000], [260], "tree"),
]


@pytest.mark.parametrize("case", LARGE_TREES, ids=lambda c: "%s_%s_d%d_%s_%d" % (str(c[0])[6:], c[1], c[2], c[9], max(c[7])))
def test_tree_attention_of_many_rows(case):
    r = Run(12, *case, front=1, behind=2, **ROOM)
    out = torch.full(r.q.shape, 9.0, dtype=r.dt, device=DEV)
    r.call(out)
    r.check(out)
    assert (out[:1] == 9.0).all() and (out[r.off[-1]:] == 9.0).all()
    again = torch.full(r.q.shape, 9.0, dtype=r.dt, device=DEV)
    r.call(again)
    assert torch.equal(again, out)


def test_tree_of_no_rows_no_pages_and_no_sequences():
    m = _mod("spfa_tree")
    r = Run(2, BF16, "none", 64, 16, 1, 2, True, [0, 0], [1, 2], "random")
    r.mask.zero_()
    r.tree = [t & False for t in r.tree]
    out = torch.full(r.q.shape, 9.0, dtype=BF16, device=DEV)
    r.call(out)
    assert not out.any()  # nothing to attend
    kc, vc, _, _ = r.cache
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert m.forward(r.q[:0], kc, vc, r.table, r.ctx_t, torch.zeros_like(r.off_t), out[:0]).shape[0] == 0
    out.fill_(9.0)
    m.forward(r.q, kc, vc, r.table[:0], z, z.new_zeros(1), out)
    assert (out == 9.0).all()
    m.forward(r.q, kc[:0], vc[:0], r.table, r.ctx_t + 5, r.off_t, out)  # a cache without pages
    assert not out.any()
    out.fill_(9.0)
    m.forward(r.q, kc, vc, r.table[:, :0], r.ctx_t + 5, r.off_t, out)  # a table without columns
    assert not out.any()


@pytest.mark.parametrize("nodes", [40, 130])
@pytest.mark.parametrize("code,dt", [("none", BF16), ("none", F16), ("int8", BF16), ("e4m3", F16)])
def test_tree_state_chains(code, dt, nodes):
    """Two caches one after the other on one (m, l, out), and scale of either sign."""
    room = ROOM if nodes > 100 else {}
    a = Run(3, dt, code, 64, 16, 2, 2, True, [300, 0, 40], [4, 3, nodes], "random", **room)
    b = Run(4, dt, code, 64, 16, 2, 2, False, [129, 2, 0], [4, 3, nodes], "tree", **room)
    b.q = a.q
    # the second one without its trees: whole contexts only
    b.mask.zero_()
    b.tree = [t & False for t in b.tree]
    for scale in (0.125, -0.2, 0.0):
        m = torch.full(a.q.shape[:2], float("-inf"), device=DEV)
        l = torch.zeros(a.q.shape[:2], device=DEV)
        base = torch.full(a.q.shape, 3.0, dtype=dt, device=DEV)
        out = base.clone()
        a.call(out, m=m, l=l, scale=scale)
        a.check(out, m, l, scale=scale, base=base)
        b.call(out, m=m, l=l, scale=scale)
        q = np64(a.q)
        for i in range(3):
            ka, va = a.read(i)
            kb, vb = b.read(i)
            lv = np.concatenate([a.live(i), b.live(i)], 1)
            for hq in range(4):
                rows = slice(a.off[i], a.off[i + 1])
                o, mm, ll, size, s_abs = sv.tree_attention(q[rows, hq], np.concatenate([ka[:, hq // 2], kb[:, hq // 2]]),
                                                           np.concatenate([va[:, hq // 2], vb[:, hq // 2]]), lv, scale)
                eps_p = 2.0 ** -16 if (code != "none" and dt == F16) else HALF[dt]
                rel = eps_p + (2 * lv.shape[1] + 60) * U + 4 * 72 * U * s_abs
                has = ll > 0
                got = out[rows, hq]
                # (out is rounded twice: between the calls, and that value weighs at most size)
                _close(got[torch.from_numpy(has).to(DEV)], o[has], (2 * HALF[dt] * size + size * rel[:, None] + TINY[dt])[has], "chained")
                assert (got[torch.from_numpy(~has).to(DEV)] == 3.0).all()
                e = np64(m[rows, hq]) + np.log(np.where(has, np64(l[rows, hq]), 1)) - (mm + np.log(np.where(has, ll, 1)))
                assert (np.abs(e[has]) <= rel[has] + 2.0 ** -20).all()
                assert (np64(l[rows, hq])[~has] == 0).all()


@pytest.mark.parametrize("code", ["none", "int8", "e4m3"])
def test_tree_lost_pages_are_masked(code):
    r = Run(5, BF16, code, 64, 16, 1, 4, True, [200, 90], [5, 3], "tree", wide=4)
    lost = {0: [3, 9], 1: [0, 1, 2, 3, 4, 5]}  # of the second sequence everything
    bad = [-1, 10 ** 9, r.cache[0].shape[0], -2 ** 31]
    t = r.table_np.copy()
    for i, cols in lost.items():
        for j, c in enumerate(cols):
            t[i, c] = bad[j % 4]
    keep = {i: np.ones(r.ctx[i] + r.nodes[i], dtype=bool) for i in (0, 1)}
    for i, cols in lost.items():
        for c in cols:
            keep[i][16 * c:16 * (c + 1)] = False
    r.table = torch.from_numpy(t).to(DEV)
    out = torch.empty(r.q.shape, dtype=BF16, device=DEV)
    r.call(out)
    r.check(out, live=lambda i: r.live(i) & keep[i])
    # lengths past the table: cut; a negative one: an empty context
    r.table = torch.from_numpy(r.table_np[:, :4].copy()).to(DEV)
    for i in (0, 1):
        keep[i] = np.arange(r.ctx[i] + r.nodes[i]) < 64
    r.call(out)
    r.check(out, live=lambda i: r.live(i) & keep[i])


def test_tree_bad_offsets_are_cut():
    r = Run(6, F16, "none", 64, 16, 1, 2, True, [40, 30], [3, 2], "chain")
    out = torch.full(r.q.shape, 9.0, dtype=F16, device=DEV)
    r.off_t = torch.tensor([-5, 3, 10 ** 9], dtype=torch.int32, device=DEV)
    r.ctx_t = torch.tensor([40, -7], dtype=torch.int32, device=DEV)
    r.call(out)  # rows 0 .. 2 and 3 .. 4; the second sequence begins with its first page
    assert torch.isfinite(out).all()
    r.ctx[1] = 0
    r.check(out)
    r.off_t = torch.tensor([4, 2, 1], dtype=torch.int32, device=DEV)  # descending: no rows
    out.fill_(9.0)
    r.call(out)
    assert (out == 9.0).all()


@pytest.mark.parametrize("dt,code", [(BF16, "none"), (F16, "none"), (BF16, "e4m3"), (F16, "e4m3"), (BF16, "int8"), (F16, "int8")])
@pytest.mark.parametrize("d,nodes", [(64, 20), (128, 6), (128, 40), (256, 9), (64, 250), (128, 250), (256, 250)])
def test_tree_infinities_reach_only_the_rows_that_attend_them(dt, code, d, nodes):
    """Drafted tokens whose keys or values hold infinities and NaN, attended by some nodes; places past
    the sequence and unused pages hold NaN throughout (Run fills them)."""
    r = Run(7, dt, code, d, 16, 1, 2, True, [100, 3], [nodes, 4], "random", **(ROOM if nodes > 100 else {}))
    kc, vc, ks, vs = r.cache
    rng = np.random.default_rng(9)
    sick_v = {0: [1, 2, nodes - 1], 1: [0, 3]}
    sick_k = {0: [4], 1: []}
    for i in (0, 1):
        for j in sick_v[i]:
            slot = int(r.slots[i][r.ctx[i] + j])
            p, at = slot // 16, slot % 16
            if code == "none":
                vc[p, at, 0, 5] = float("inf")
                vc[p, at, 0, d - 3] = float("-inf") if j % 2 else float("nan")
            elif code == "e4m3" and j % 2:
                vc[p, at, 0].view(torch.uint8)[7] = 0x7f
            else:
                vs[p, at, 0] = float("inf") if j % 2 else float("nan")
        for j in sick_k[i]:
            slot = int(r.slots[i][r.ctx[i] + j])
            p, at = slot // 16, slot % 16
            if code == "none":
                kc[p, at, 0, 3] = float("nan")
            else:
                ks[p, at, 0] = float("nan")
    out = torch.empty(r.q.shape, dtype=dt, device=DEV)
    r.call(out)
    o = np64(out)
    q = np64(r.q)
    for i in (0, 1):
        kk, vv = r.read(i)
        lv = r.live(i)
        for hq in range(2):
            rows = np.arange(r.off[i], r.off[i + 1])
            with np.errstate(all="ignore"):
                want, _, _, a, s_abs = sv.tree_attention(q[rows, hq], kk[:, 0], vv[:, 0], lv, 1 / math.sqrt(d))
            for n, row in enumerate(rows):
                w, g = want[n], o[row, hq]
                if any(lv[n, r.ctx[i] + j] for j in sick_k[i]):
                    assert np.isnan(g).all()
                    continue
                fine = np.isfinite(w)
                assert np.array_equal(np.isfinite(g), fine), (i, n)
                assert np.array_equal(g[~fine], w[~fine], equal_nan=True), (i, n)
                eps_p = 2.0 ** -16 if (code != "none" and dt == F16) else HALF[dt]
                rel = eps_p + (2 * lv.shape[1] + 40) * U + 4 * (d + 8) * U * s_abs[n]
                tol = HALF[dt] * np.abs(w[fine]) + a[n][fine] * rel * (1 + HALF[dt]) + TINY[dt]
                assert (np.abs(g[fine] - w[fine]) <= tol).all(), (i, n)


def test_tree_large_scores_and_scales():
    """Scores far apart (the reference moves many times), V scales over many powers of two."""
    r = Run(8, F16, "int8", 128, 16, 1, 4, True, [1500], [3], "chain")
    kc, vc, ks, vs = r.cache
    ks *= torch.exp(1.5 * torch.randn(ks.shape, generator=_gen(1), device=DEV))
    vs *= torch.exp2(torch.randint(-18, 10, vs.shape, generator=_gen(2), device=DEV).float())
    r.q = r.q * 3
    out = torch.empty(r.q.shape, dtype=F16, device=DEV)
    r.call(out)
    r.check(out)


def test_tree_and_cache_offsets_beyond_32_bits():
    """Pages whose offsets pass 2^32 elements: rows at both ends of a 5 GiB cache."""
    page, d = 16, 128
    pages = 5 * (1 << 30) // (page * d)
    m, t = _mod("spfa_cache"), _mod("spfa_tree")
    kc, vc = [torch.empty(pages, page, 1, d, dtype=torch.int8, device=DEV) for _ in range(2)]
    ks, vs = [torch.empty(pages, page, 1, device=DEV) for _ in range(2)]
    order = torch.tensor([pages - 1, 0, pages // 2, pages - 2], dtype=torch.int64, device=DEV)
    n = 4 * page
    slots = (order[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
    k, v = [torch.randn(n, 1, d, generator=_gen(i), device=DEV).to(BF16) for i in (1, 2)]
    m.write(k, v, slots, kc, vc, ks, vs)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    m.read(kc, vc, slots, ko, vo, ks, vs)
    for x, y in ((k, ko), (v, vo)):
        want, amax = sv.quantise(np64(x), "int8")
        val = want * (amax / 127)[..., None]
        _close(y, val, (HALF[BF16] + 4 * U) * np.abs(val), "read back")
    q = torch.randn(1, 2, d, generator=_gen(3), device=DEV).to(BF16)
    out = torch.empty_like(q)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    t.forward(q, kc, vc, order.to(torch.int32).view(1, 4), i32(n - 1), i32(0, 1), out, None, ks, vs)
    small = [x.view(pages * page, 1, -1)[slots].view(4, page, 1, -1) for x in (kc, vc)]
    smalls = [x.view(pages * page, 1)[slots].view(4, page, 1) for x in (ks, vs)]
    want = torch.empty_like(q)
    t.forward(q, *small, i32(0, 1, 2, 3).view(1, 4), i32(n - 1), i32(0, 1), want, None, *smalls)
    assert torch.equal(out, want)


def test_outputs_that_are_other_tensors_of_the_call_are_refused():
    """An output in place of its own input is one thing, in place of another tensor a race."""
    q, k = [torch.randn(6, 2, 64, generator=_gen(i), device=DEV).to(BF16) for i in (1, 2)]
    w, f, pos = torch.ones(64, dtype=BF16, device=DEV), torch.ones(32, device=DEV), torch.arange(6, device=DEV)
    m = _mod("spfa_rope")
    qo, ko, dw = torch.empty_like(q), torch.empty_like(k), torch.empty(64, device=DEV)
    for a, b in ((k, ko), (qo, q), (k, q), (qo, qo)):
        with pytest.raises(RuntimeError, match="overlaps"):
            m.forward(q, k, w, w, pos, f, a, b)
        with pytest.raises(RuntimeError, match="overlaps"):
            m.backward(q, k, w, w, pos, f, q, k, a, b, None, None)
    with pytest.raises(RuntimeError, match="overlaps"):
        m.backward(q, k, w, w, pos, f, q, k, qo, ko, dw, dw)
    flat = torch.randn(6, 2, 64, generator=_gen(3), device=DEV).to(BF16)
    with pytest.raises(RuntimeError, match="overlaps"):  # the same memory in another order
        m.forward(flat, k, w, w, pos, f, flat.view(2, 6, 64).transpose(0, 1), ko)
    c = _mod("spfa_cache")
    kc = torch.zeros(2, 16, 2, 64, dtype=torch.int8, device=DEV)
    ks = torch.zeros(2, 16, 2, device=DEV)
    slots = torch.arange(6, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        c.write(q, k, slots, kc, kc, ks, ks.clone())
    with pytest.raises(RuntimeError, match="overlaps"):
        c.write(q, k, slots, kc, kc.clone(), ks, ks)
    with pytest.raises(RuntimeError, match="overlaps"):
        c.read(kc, kc.clone(), slots, qo, qo, ks, ks.clone())
    r = Run(1, BF16, "none", 64, 16, 2, 2, True, [20], [3], "tree")
    out, ml = torch.empty(r.q.shape, dtype=BF16, device=DEV), torch.zeros(3, 4, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        r.call(out, m=ml, l=ml)


def test_tree_refusals():
    m = _mod("spfa_tree")
    r = Run(1, BF16, "int8", 64, 16, 2, 2, True, [20], [3], "tree")
    kc, vc, ks, vs = r.cache
    out = torch.empty(r.q.shape, dtype=BF16, device=DEV)
    ok = dict(q=r.q, k_cache=kc, v_cache=vc, page_table=r.table, ctx_lens=r.ctx_t, q_offsets=r.off_t, out=out, tree_mask=r.mask,
              k_scale=ks, v_scale=vs)
    m.forward(**ok)
    ml = torch.zeros(3, 4, device=DEV)
    big = torch.zeros(3, 16, 2, 264, dtype=BF16, device=DEV)
    bad = [dict(q=r.q.float(), out=out.float()), dict(q=r.q[:, :3], out=out[:, :3]), dict(q=r.q[..., :32], out=out[..., :32]),
           dict(out=out.half()), dict(out=out[:2]), dict(k_scale=None), dict(page_table=r.table.long()), dict(ctx_lens=r.ctx_t.long()),
           dict(q_offsets=r.off_t[:1]), dict(page_table=r.table[0]), dict(tree_mask=r.mask.int()), dict(tree_mask=r.mask[:2]), dict(m=ml),
           dict(m=ml, l=ml.half()), dict(m=ml[:2], l=ml[:2]), dict(out=out[:1].expand(3, 4, 64)), dict(q=out), dict(page_table=r.table.cpu()),
           dict(q=r.q.cpu()), dict(v_cache=vc[..., :32]), dict(tree_mask=r.mask.cpu())]
    for kw in bad:
        with pytest.raises((RuntimeError, ValueError)):
            m.forward(**{**ok, **kw})
    with pytest.raises(ValueError):
        q = torch.zeros(3, 2, 264, dtype=BF16, device=DEV)
        m.forward(q, big, big.clone(), r.table, r.ctx_t, r.off_t, torch.empty_like(q))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------
# together, on streams and in graphs
# ------------------------------------------------------------------------------------------------
def test_prompt_drafts_and_acceptance_together():
    """A prompt goes through rope, cache and attention as one chunk, a tree is drafted on top, one of
    its paths is accepted (its tokens written again behind the prompt), and decoding goes on: every
    step's rows against one attention over the tokens of that path."""
    rope, cache, tree = (_mod("spfa_" + x) for x in ("rope", "cache", "tree"))
    hk, group, d, page, n = 2, 3, 64, 16, 75
    g = _gen(12)
    wq, wk = [(1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(BF16) for _ in range(2)]
    f = 10000.0 ** (-torch.arange(d // 2, device=DEV, dtype=F32) / (d // 2))
    kc, vc, ks, vs = _new_cache(8, page, hk, d, BF16, "e4m3", True)
    table = torch.tensor([[6, 1, 4, 0, 7, 2]], dtype=torch.int32, device=DEV)
    slots_of = lambda p: table[0].long()[p // page] * page + p % page
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)

    def tokens(count, positions):
        """Fused projections of new tokens -> rotated q, rotated k, v."""
        x = torch.randn(count, (group + 2) * hk * d, generator=g, device=DEV).to(BF16)
        q, k, v = (y.unflatten(-1, (-1, d)) for y in x.split([group * hk * d, hk * d, hk * d], -1))
        qo, ko = torch.empty(q.shape, dtype=BF16, device=DEV), torch.empty(k.shape, dtype=BF16, device=DEV)
        rope.forward(q, k, wq, wk, positions, f, qo, ko)
        want = sv.norm_rope(np64(k), np64(wk), positions.tolist(), np64(f), 1e-6, False)
        _close(ko, want, HALF[BF16] * np.abs(want) + (d / 2 + 28) * U * 1.5 * _pair_size(want, d, False), "rotated keys")
        return qo, ko, v

    def held(x):
        """What an e4m3 cache makes of rows."""
        y, amax = sv.quantise(np64(x), "e4m3")
        return y * (amax / 448)[..., None]

    def expect(out, q, k, v, live):
        for hq in range(group * hk):
            o, _, _, a, s = sv.tree_attention(np64(q)[:, hq], k[:, hq // group], v[:, hq // group], live, 1 / 8)
            rel = HALF[BF16] + (2 * live.shape[1] + 44) * U + 4 * 72 * U * s
            _close(out[:, hq], o, HALF[BF16] * np.abs(o) + a * rel[:, None] * 1.01, "attention")

    pos = torch.arange(n, device=DEV)
    q, k, v = tokens(n, pos)
    cache.write(k, v, slots_of(pos), kc, vc, ks, vs)
    out = torch.empty_like(q)
    tree.forward(q, kc, vc, table, i32(0), i32(0, n), out, None, ks, vs)
    K, V = held(k), held(v)
    expect(out, q, K, V, np.tril(np.ones((n, n), dtype=bool)))

    parents = [-1, 0, 0, 1, 2, 2, 4]
    depth = torch.tensor([0, 1, 1, 2, 2, 2, 3], device=DEV)
    q, k, v = tokens(7, n + depth)
    cache.write(k, v, slots_of(n + torch.arange(7, device=DEV)), kc, vc, ks, vs)
    out = torch.empty_like(q)
    tree.forward(q, kc, vc, table, i32(n), i32(0, 7), out, spfa_masks.tree_mask(parents, device=DEV), ks, vs)
    mine = np.zeros((7, 7), dtype=bool)
    for i, p in enumerate(parents):
        mine[i, i] = True
        if p >= 0:
            mine[i] |= mine[p]
    expect(out, q, np.concatenate([K, held(k)]), np.concatenate([V, held(v)]), np.concatenate([np.ones((7, n), dtype=bool), mine], 1))

    path = torch.tensor([0, 2, 4, 6], device=DEV)
    cache.write(k[path], v[path], slots_of(n + torch.arange(4, device=DEV)), kc, vc, ks, vs)
    K, V = np.concatenate([K, held(k[path])]), np.concatenate([V, held(v[path])])
    q, k, v = tokens(1, torch.tensor([n + 4], device=DEV))
    cache.write(k, v, slots_of(torch.tensor([n + 4], device=DEV)), kc, vc, ks, vs)
    out = torch.empty_like(q)
    tree.forward(q, kc, vc, table, i32(n + 4), i32(0, 1), out, None, ks, vs)
    expect(out, q, np.concatenate([K, held(k)]), np.concatenate([V, held(v)]), np.ones((1, n + 5), dtype=bool))
    # the sequence read back for a call over contiguous keys
    pos = torch.arange(n + 5, device=DEV)
    ko, vo = [torch.empty(hk, n + 5, d, dtype=BF16, device=DEV).transpose(0, 1) for _ in range(2)]
    cache.read(kc, vc, slots_of(pos), ko, vo, ks, vs)
    for y, want in ((ko, np.concatenate([K, held(k)])), (vo, np.concatenate([V, held(v)]))):
        _close(y, want, (HALF[BF16] + 4 * U) * np.abs(want), "read back")


def test_two_streams_at_once():
    runs = [Run(20 + i, BF16, "e4m3", 128, 16, 2, 4, True, [3000, 900, 10], [5, 1, 9], "tree") for i in range(2)]
    want = []
    for r in runs:
        out = torch.empty(r.q.shape, dtype=BF16, device=DEV)
        r.call(out)
        want.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[torch.empty(r.q.shape, dtype=BF16, device=DEV) for _ in range(6)] for r in runs]
    torch.cuda.synchronize()
    for n in range(6):
        for r, s, g in zip(runs, streams, got):
            with torch.cuda.stream(s):
                r.call(g[n])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x in g:
            assert torch.equal(x, w)


def test_replays_from_a_graph():
    """A step of rope, cache and tree attention and a training pair of rope calls, captured once and
    replayed on new inputs and lengths; every replay against the eager calls."""
    rope, cache, tree = (_mod("spfa_" + x) for x in ("rope", "cache", "tree"))
    hk, group, d, page, n = 2, 4, 128, 16, 3
    g = _gen(4)
    w = [torch.ones(d, device=DEV, dtype=BF16) for _ in range(2)]
    f = 10000.0 ** (-torch.arange(d // 2, device=DEV, dtype=F32) / (d // 2))
    x = torch.randn(n, (group + 2) * hk * d, generator=g, device=DEV).to(BF16)
    q, k, v = (y.unflatten(-1, (-1, d)) for y in x.split([group * hk * d, hk * d, hk * d], -1))
    store = _new_cache(n * 40, page, hk, d, BF16, "int8", True)
    kc, vc, ks, vs = store
    ks.fill_(1.0)
    vs.fill_(1.0)
    kc.random_(-100, 100, generator=g)
    vc.random_(-100, 100, generator=g)
    table = torch.randperm(n * 40, generator=g, device=DEV).to(torch.int32).view(n, 40)
    ctx = torch.tensor([600, 3, 77], dtype=torch.int32, device=DEV)
    off = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    qo, ko, out = torch.empty(q.shape, dtype=BF16, device=DEV), torch.empty(k.shape, dtype=BF16, device=DEV), torch.empty(q.shape, dtype=BF16, device=DEV)
    dq, dk, dw = torch.empty_like(qo), torch.empty_like(ko), [torch.empty(d, device=DEV) for _ in range(2)]

    def step():
        pos = ctx.long()
        rope.forward(q, k, *w, pos, f, qo, ko)
        slots = table.long().gather(1, (pos // page)[:, None])[:, 0] * page + pos % page
        cache.write(ko, v, slots, kc, vc, ks, vs)
        tree.forward(qo, kc, vc, table, ctx, off, out, None, ks, vs)
        rope.backward(q, k, *w, pos, f, out, ko, dq, dk, *dw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(3):
        x.normal_(generator=g)
        ctx.copy_(torch.tensor([[600, 3, 77], [638, 0, 127], [5, 129, 300]][rep], dtype=torch.int32))
        results = (qo, ko, out, dq, dk, *dw)
        for t in results:
            t.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*results, kc, vc, ks, vs)]
        for t in results:
            t.fill_(6.0)
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (*results, kc, vc, ks, vs)):
            assert torch.equal(a, b), rep


@pytest.mark.parametrize("dt,code,d", [(F16, "none", 64), (BF16, "int8", 128)])
def test_many_rows_replay_with_other_lengths(dt, code, d):
    """The kernel of many rows, captured and replayed while the contexts change, beside eager calls on
    another stream."""
    r = Run(31, dt, code, d, 16, 2, 8, True, [700, 90, 0], [60, 40, 9], "tree", **ROOM)
    out = torch.empty(r.q.shape, dtype=dt, device=DEV)
    r.call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.call(out)
    side = torch.cuda.Stream()
    for ctx in ([700, 90, 0], [10, 89, 0], [333, 0, 0]):  # (fewer cached tokens: nodes are read from other places)
        r.ctx_t.copy_(torch.tensor(ctx, dtype=torch.int32))
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        with torch.cuda.stream(side):
            r.call(want)
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        r.ctx = ctx
        r.check(out)


def test_cache_of_more_slots_than_31_bits():
    """Slot numbers past 2^31 (pages that are all the same memory, for reading)."""
    m = _mod("spfa_cache")
    one = [torch.randn(1, 16, 2, 8, generator=_gen(i), device=DEV).to(BF16) for i in (1, 2)]
    kc, vc = [x.expand((1 << 28) + 5, 16, 2, 8) for x in one]
    slots = torch.tensor([0, 5, (1 << 31) - 1, (1 << 31) + 7, (1 << 32) + 79, (1 << 32) + 80, -1, 1 << 40], device=DEV)
    ko, vo = [torch.full((8, 2, 8), 3.0, dtype=BF16, device=DEV) for _ in range(2)]
    m.read(kc, vc, slots, ko, vo)
    for x, y in zip(one, (ko, vo)):
        assert torch.equal(y[:5], x[0, (slots[:5] % 16)])
        assert (y[5:] == 3.0).all()
