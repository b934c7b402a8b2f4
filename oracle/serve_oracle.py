"""Float64 oracle of the operators around masked attention (numpy): head norms with the position
rotation and their gradients, the rows of an 8-bit cache, attention of a tree of tokens.  Written
from the formulas, token by token; test infrastructure only."""
import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def _pair(i, rot, interleaved):
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def rotation(position, inv_freq, d, interleaved):
    """The d x d matrix that turns a head's vector at a position."""
    rot = 2 * len(inv_freq)
    m = np.eye(d)
    for i, f in enumerate(np.asarray(inv_freq, dtype=np.float64)):
        a, b = _pair(i, rot, interleaved)
        t = float(position) * float(f)
        m[a, a] = m[b, b] = math.cos(t)
        m[a, b] = -math.sin(t)
        m[b, a] = math.sin(t)
    return m


def norm_rope(x, w, positions, inv_freq, eps, interleaved):
    """x [tokens, heads, d] -> the rotated norms."""
    out = np.empty_like(x, dtype=np.float64)
    for t in range(x.shape[0]):
        r = rotation(positions[t], inv_freq, x.shape[2], interleaved)
        n = x[t] / np.sqrt((x[t] ** 2).mean(-1, keepdims=True) + eps)
        out[t] = (n * w) @ r.T
    return out


def norm_rope_backward(x, w, positions, inv_freq, eps, interleaved, dy):
    """(d_x, d_w), and the sizes their rounding errors go by: (of d_x per element, of d_w: the sum of
    absolute terms)."""
    dx, sx = np.empty_like(x, dtype=np.float64), np.empty_like(x, dtype=np.float64)
    dw, sw = np.zeros(x.shape[2]), np.zeros(x.shape[2])
    rot = 2 * len(inv_freq)
    for t in range(x.shape[0]):
        m = rotation(positions[t], inv_freq, x.shape[2], interleaved)
        r = 1.0 / np.sqrt((x[t] ** 2).mean(-1, keepdims=True) + eps)
        n = x[t] * r
        g = dy[t] @ m
        mag = np.abs(dy[t]).copy()  # of a pair: both its elements
        for i in range(rot // 2):
            a, b = _pair(i, rot, interleaved)
            mag[:, a] = mag[:, b] = np.abs(dy[t][:, a]) + np.abs(dy[t][:, b])
        dx[t] = r * (g * w - n * (g * w * n).mean(-1, keepdims=True))
        sx[t] = r * (mag * np.abs(w) + np.abs(n) * (mag * np.abs(w) * np.abs(n)).mean(-1, keepdims=True))
        dw += (g * n).sum(0)
        sw += (mag * np.abs(n)).sum(0)
    return dx, dw, sx, sw


def e4m3_round(y):
    """Nearest values of 4 significant bits (ties to even), smallest step 2^-9."""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(e, -5) - 4)
    return np.rint(y / step) * step


def quantise(x, code):
    """Rows [..., d] -> (the numbers their codes stand for, amax)."""
    x = np.asarray(x, dtype=np.float64)
    amax = np.abs(x).max(-1, keepdims=True)
    y = x * TOP[code] / np.where(amax == 0, 1.0, amax)
    return (np.rint(y) if code == "int8" else e4m3_round(y)), amax[..., 0]


def tree_attention(q, k, v, live, scale):
    """q [rows, d], k, v [keys, d], live [rows, keys] -> (out, m, l, and the size of the rounding errors
    of out: sum p |v| / l and the largest sum |q k| * scale among a row's live keys).  Rows with nothing
    live: zeros, m = -inf, l = 0.  Masked keys and values are not touched by any arithmetic."""
    rows, d = q.shape
    out, a = np.zeros((rows, d)), np.zeros((rows, d))
    m, l, s_abs = np.full(rows, -np.inf), np.zeros(rows), np.zeros(rows)
    for i in range(rows):
        js = np.nonzero(live[i])[0]
        if not len(js):
            continue
        s = k[js] @ q[i] * scale
        m[i] = s.max()
        p = np.exp(s - m[i])
        l[i] = p.sum()
        out[i] = p @ v[js] / l[i]
        with np.errstate(invalid="ignore"):
            a[i] = p @ np.abs(v[js]) / l[i]
        s_abs[i] = (np.abs(k[js]) @ np.abs(q[i])).max() * abs(scale)
    return out, m, l, a, s_abs
