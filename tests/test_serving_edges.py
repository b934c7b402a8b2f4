"""Calls at the edges of the C entry points around masked attention, without a GPU: refused before
anything touches a device."""
import ctypes

import pytest

from test_serving import Heads, lib, _rope  # noqa: F401  (a fixture)


@pytest.mark.parametrize("sizes", [
    dict(batch=1 << 62, heads_q=3),                       # 2^62 * 4 = 2^64
    dict(batch=1 << 44, heads_q=(1 << 20) - 1),           # 2^44 * 2^20 = 2^64
    dict(batch=(1 << 63) - 1, heads_q=1),
    dict(batch=1 << 40, tokens=1 << 40),
    dict(batch=3, tokens=(1 << 63) - 1),
], ids=str)
def test_rope_sizes_whose_product_overflows_are_refused(lib, sizes):  # noqa: F811
    h = ctypes.byref(Heads(data=4096))
    assert lib.spfa_qk_norm_rope_forward(_rope(**sizes), h, h, None) == 1
    assert lib.spfa_qk_norm_rope_backward(_rope(**sizes), h, h, h, h, None, None, 4096, 1 << 40, None) == 1
