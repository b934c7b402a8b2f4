"""Inputs at the edges of what the operators around masked attention take, on the GPU against the
float64 oracle: the cases, tolerances' units and helpers are those of test_gpu_serving.py."""
import numpy as np
import pytest
import torch

from helpers import np64
from oracle import serve_oracle as sv
from test_gpu_serving import BF16, DEV, F16, F32, HALF, TINY, U, _close, _gen, _mod, _ones, _pair_size, _rope_inputs

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
