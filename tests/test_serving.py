"""Head norms with the position rotation, the paged cache and the tree attention without a GPU: the
oracle against its own differences and against torch, helper functions, parameter checks of the C
entry points and of the modules (both return before anything touches a device)."""
import ctypes
import importlib
import os

import numpy as np
import pytest
import torch

import spfa_masks
from oracle import serve_oracle as sv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "graph-processing-attention-ipdps-2025_amd", "libspfa_hip.so")
I64, I32, P, F = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_float


class Heads(ctypes.Structure):
    _fields_ = [("data", P), ("stride_batch", I64), ("stride_token", I64), ("stride_head", I64)]


class Rope(ctypes.Structure):
    _fields_ = [("batch", I64), ("tokens", I64), ("heads_q", I64), ("heads_k", I64), ("d", I64), ("rot", I64),
                ("dtype", I32), ("w_dtype", I32), ("position_bytes", I32), ("interleaved", I32), ("eps", F),
                ("q", Heads), ("k", Heads), ("w_q", P), ("w_k", P), ("positions", P), ("position_stride", I64),
                ("inv_freq", P)]


class Cache(ctypes.Structure):
    _fields_ = ([("k", P), ("v", P), ("k_scale", P), ("v_scale", P)]
                + [(x + "_stride_" + y, I64) for x in ("k", "v", "ks", "vs") for y in ("page", "slot", "head")]
                + [("pages", I64), ("page_size", I64), ("heads", I64), ("d", I64), ("code", I32), ("dtype", I32)])


class Tree(ctypes.Structure):
    _fields_ = [("q", P), ("out", P), ("q_stride_row", I64), ("q_stride_head", I64), ("out_stride_row", I64),
                ("out_stride_head", I64), ("m", P), ("l", P), ("rows", I64), ("heads_q", I64), ("n_seqs", I64),
                ("q_offsets", P), ("ctx_lens", P), ("page_table", P), ("table_width", I64), ("table_stride", I64),
                ("tree_mask", P), ("mask_words", I64), ("scale", F)]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    L.spfa_qk_norm_rope_backward_workspace_bytes.restype = ctypes.c_size_t
    L.spfa_qk_norm_rope_backward_workspace_bytes.argtypes = [I64] * 5
    L.spfa_qk_norm_rope_forward.argtypes = [P, P, P, P]
    L.spfa_qk_norm_rope_backward.argtypes = [P] * 8 + [ctypes.c_size_t, P]
    L.spfa_cache_write.argtypes = [P, P, P, I64, P, ctypes.c_int, P]
    L.spfa_cache_read.argtypes = [P, P, ctypes.c_int, I64, P, P, P]
    L.spfa_tree_workspace_bytes.restype = ctypes.c_size_t
    L.spfa_tree_workspace_bytes.argtypes = [P, P]
    L.spfa_tree_forward.argtypes = [P, P, P, ctypes.c_size_t, P]
    return L


@pytest.mark.parametrize("d,rot,interleaved", [(8, 8, False), (10, 6, True), (7, 4, False), (6, 0, False)])
def test_oracle_gradients_agree_with_differences(d, rot, interleaved):
    rng = np.random.default_rng(d + rot)
    x, w = rng.standard_normal((3, 2, d)), 1 + 0.2 * rng.standard_normal(d)
    f, pos = 100.0 ** (-np.arange(rot // 2) / max(rot // 2, 1)), np.array([0, 5, 1000])
    dy = rng.standard_normal(x.shape)
    loss = lambda x, w: (sv.norm_rope(x, w, pos, f, 1e-3, interleaved) * dy).sum()
    dx, dw, _, _ = sv.norm_rope_backward(x, w, pos, f, 1e-3, interleaved, dy)
    h = 1e-5  # central differences: h^2 and 2^-53 / h, both about 1e-10
    for got, arr, at in ((dx, x, 0), (dw, w, 1)):
        for i in np.ndindex(arr.shape):
            up, down = arr.copy(), arr.copy()
            up[i] += h
            down[i] -= h
            args = [(up, w), (down, w)] if at == 0 else [(x, up), (x, down)]
            assert abs((loss(*args[0]) - loss(*args[1])) / (2 * h) - got[i]) < 1e-7


def test_oracle_rounds_to_e4m3_as_torch_does():
    # every midpoint and neighbour that fp32 holds exactly, so that torch's cast rounds once
    base = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    mid = (base[1:] + base[:-1]) / 2
    y = np.concatenate([base, mid, mid * (1 + 2.0 ** -15), mid * (1 - 2.0 ** -15)])
    y = np.concatenate([y, -y])
    want = torch.from_numpy(y).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(sv.e4m3_round(y), want)


def test_tree_mask_lists_ancestors():
    # 0 - 1 - 3, 0 - 2, 4 alone; a second sequence of 70 nodes in a chain; rows behind it have no bits
    parents = [-1, 0, 0, 1, -1] + list(range(-1, 69)) + [7]
    m = spfa_masks.tree_mask(parents, [0, 5, 75])
    assert m.dtype == torch.int64 and tuple(m.shape) == (76, 2)
    assert m[:5, 0].tolist() == [1, 3, 5, 11, 16] and m[:5, 1].tolist() == [0] * 5
    assert m[5 + 63, 0].item() == -1 and m[5 + 69, 1].item() == (1 << 6) - 1
    assert m[75].tolist() == [0, 0]
    same = spfa_masks.tree_mask(torch.tensor(parents), torch.tensor([0, 5, 75]))
    assert torch.equal(m, same)
    assert tuple(spfa_masks.tree_mask([]).shape) == (0, 1)
    for bad in ([0], [-2], [-1, 1]):
        with pytest.raises(ValueError):
            spfa_masks.tree_mask(bad)
    with pytest.raises(ValueError):
        spfa_masks.tree_mask([-1, 0], [0, 3])
    with pytest.raises(ValueError):
        spfa_masks.tree_mask([-1, 0], [2, 0])


def _rope(**kw):
    p = Rope(batch=1, tokens=2, heads_q=2, heads_k=1, d=8, rot=8, position_bytes=8, eps=1e-6)
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def test_rope_checks(lib):
    f = lambda **kw: lib.spfa_qk_norm_rope_forward(_rope(**kw), None, None, None)
    b = lambda **kw: lib.spfa_qk_norm_rope_backward(_rope(**kw), None, None, None, None, None, None, None, 0, None)
    for call in (f, b):
        assert call(d=0) == 5 and call(d=1025) == 5
        assert call(dtype=3) == 2 and call(dtype=1, w_dtype=2) == 2 and call(dtype=7) == 2
        assert call(rot=3) == 1 and call(rot=10) == 1 and call(rot=-2) == 1
        assert call(position_bytes=2) == 1 and call(tokens=-1) == 1 and call(heads_k=-1) == 1
        assert call(tokens=1 << 62) == 1
        assert call() == 1  # tensors missing
    assert f(tokens=0) == 0 and f(batch=0) == 0 and f(heads_q=0, heads_k=0) == 0  # nothing to do
    assert b(tokens=0) == 0
    assert lib.spfa_qk_norm_rope_forward(None, None, None, None) == 1
    fake = Heads(data=4096)  # never touched: the workspace check comes first
    p = Rope(batch=1, tokens=2, heads_q=2, heads_k=1, d=8, rot=0, position_bytes=8, q=fake, k=fake)
    h = ctypes.byref(fake)
    assert lib.spfa_qk_norm_rope_backward(ctypes.byref(p), h, h, h, h, None, None, None, 0, None) == 3
    assert lib.spfa_qk_norm_rope_backward(ctypes.byref(p), h, h, h, h, None, None, 4096, 64, None) == 3
    assert lib.spfa_qk_norm_rope_backward_workspace_bytes(1, 1 << 20, 32, 8, 128) < 1 << 20


def _cache(**kw):
    c = Cache(pages=4, page_size=16, heads=2, d=64, code=1, dtype=2, k=4096, v=4096, k_scale=4096, v_scale=4096)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def test_cache_checks(lib):
    h = ctypes.byref(Heads(data=4096))
    w = lambda tokens=3, bytes_=8, x=h, slots=4096, **kw: lib.spfa_cache_write(_cache(**kw), x, x, tokens, slots, bytes_, None)
    r = lambda tokens=3, bytes_=8, x=h, slots=4096, **kw: lib.spfa_cache_read(_cache(**kw), slots, bytes_, tokens, x, x, None)
    for call in (w, r):
        assert call(d=0) == 5 and call(d=1025) == 5
        assert call(dtype=3) == 2 and call(code=3) == 2
        assert call(page_size=0) == 1 and call(pages=-1) == 1 and call(heads=-1) == 1
        assert call(tokens=-1) == 1 and call(bytes_=2) == 1
        assert call(pages=1 << 40, page_size=1 << 40) == 1
        assert call(k=None) == 1 and call(v_scale=None) == 1 and call(slots=None) == 1 and call(x=None) == 1
        assert call(tokens=0) == 0 and call(pages=0) == 0 and call(heads=0) == 0  # nothing to do
    assert lib.spfa_cache_write(None, h, h, 1, 4096, 8, None) == 1


def _tree(**kw):
    t = Tree(q=4096, out=8192, rows=6, heads_q=4, n_seqs=2, q_offsets=4096, ctx_lens=4096, page_table=4096,
             table_width=8, table_stride=8, scale=0.1)
    for k, v in kw.items():
        setattr(t, k, v)
    return ctypes.byref(t)


def test_tree_checks(lib):
    f = lambda cache={}, **kw: lib.spfa_tree_forward(_cache(**cache), _tree(**kw), None, 0, None)
    assert f() == 3  # no workspace
    assert f({"d": 257}) == 5 and f({"d": 0}) == 5
    assert f({"dtype": 0}) == 2 and f({"dtype": 3}) == 2 and f({"code": 9}) == 2
    assert f(heads_q=3) == 1 and f(heads_q=0) == 1 and f({"heads": 0}) == 1
    assert f({"page_size": 0}) == 1 and f({"pages": 1 << 31}) == 1
    assert f(rows=-1) == 1 and f(rows=1 << 31) == 1 and f(n_seqs=-1) == 1 and f(table_width=-1) == 1
    assert f(m=4096) == 1 and f(mask_words=1) == 1 and f(q=None) == 1 and f(q_offsets=None) == 1 and f(page_table=None) == 1
    assert f({"v_scale": None}) == 1
    assert f(rows=0) == 0 and f(n_seqs=0) == 0
    assert lib.spfa_tree_forward(None, _tree(), None, 0, None) == 1
    small = lib.spfa_tree_workspace_bytes(_cache(), _tree(table_width=1))
    large = lib.spfa_tree_workspace_bytes(_cache(), _tree(table_width=1 << 16, rows=1 << 12))
    assert 256 <= small < large < (256 << 20)


def test_modules_refuse_host_tensors():
    rope, cache, tree = (importlib.import_module(m) for m in ("spfa_rope", "spfa_cache", "spfa_tree"))
    q = torch.zeros(2, 4, 8)
    i = torch.zeros(2, dtype=torch.int32)
    kc = torch.zeros(1, 4, 4, 8)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        rope.forward(q, q, None, None, i, torch.ones(4), q, q)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        rope.backward(q, q, None, None, i, torch.ones(4), q, q, q, q, None, None)
    with pytest.raises(RuntimeError, match="k and v must be CUDA tensors"):
        cache.write(q, q, i, kc, kc)
    with pytest.raises(RuntimeError, match="k_out and v_out must be CUDA tensors"):
        cache.read(kc, kc, i, q, q)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        tree.forward(q, kc, kc, i.view(1, 2), i[:1], i, q)
    with pytest.raises(TypeError):
        tree.forward(q, kc)
