"""Attention, rotary positions and paged caches by their definitions in 64 bits on the host, and how far a
kernel that rounds as documented may be from them."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def attend(q, k, v, scale, shown, cap=0.0, bias=None, rel=None, u=None, w=None):
    """One head of one sequence: q [n, d], k and v [m, d] in float64; shown [n, m]; bias [n, m] or None; rel
    [n, m, d] (the position row of each pair) or None. Returns the outputs and the largest sum of
    magnitudes behind a shown score (what its rounding errors are relative to)."""
    qu, qw = (q if u is None else q + u), (q if w is None else q + w)
    s, size = qu @ k.T, np.abs(qu) @ np.abs(k).T
    if rel is not None:
        s = s + np.einsum("id,ijd->ij", qw, rel)
        size = size + np.einsum("id,ijd->ij", np.abs(qw), np.abs(rel))
    s, size = s * scale, size * scale
    if cap:
        s = cap * np.tanh(s / cap)
        size = size + cap
    if bias is not None:
        s = s + bias
        size = size + np.where(np.abs(bias) < 1e29, np.abs(bias), 0.0)  # a lower one absorbs the score whole
    s = np.where(shown, s, -np.inf)
    out = np.zeros((q.shape[0], v.shape[1]))
    for i in range(q.shape[0]):
        see = np.flatnonzero(s[i] > -np.inf)
        if see.size:
            e = np.exp(s[i, see] - s[i, see].max())
            out[i] = (e / e.sum()) @ v[see]
    seen = size[shown & np.isfinite(size)]
    return out, float(seen.max()) if seen.size else 0.0


def shown_pairs(n, m, left=None, right=None, prefix=0, q_docs=None, k_docs=None, held=None):
    """Which of m keys each of the last n positions is shown; held [m]: keys that have a place."""
    i, j = np.arange(m - n, m)[:, None], np.arange(m)[None, :]
    ok = np.ones((n, m), bool)
    if left is not None:
        ok &= j >= i - left
    if right is not None:
        ok &= j <= i + right
    ok |= j < prefix
    if q_docs is not None:
        ok &= (q_docs[:, None] == k_docs[None, :]) & (q_docs[:, None] >= 0)
    if held is not None:
        ok &= held[None, :]
    return ok


def tolerance(type, d, keys, size, top, rel):
    """How far an output may be: its weights' relative error times the largest value, and its own
    rounding. A score is a sum of d products (twice that with position rows) and a few more operations,
    each off by half an f32 step of `size` at most; f32 operands held as three 8-bit parts drop products
    of less than a step each, once more the same. Weight and normaliser each carry the score's error (e^x
    moves by as much as x, and their errors may have opposite signs), a rounding to the type where it has
    16 bits, a few f32 steps of exp, and the sums over the keys."""
    f32 = HALF_STEP["f32"]
    score = (2 * (2 * d if rel else d) + 16) * f32 * size
    weight = 2 * math.expm1(score) + (2 * keys + 32) * f32
    if type != "f32":
        weight += HALF_STEP[type]
    if type == "f16":
        weight += keys * 2.0**-25  # weights below f16's normal range, relative to the largest weight
    return top * (weight + (HALF_STEP[type] if type != "f32" else 4 * f32))


def rotate(x, positions, f, amplitude, dim, interleaved):
    """x [rows, heads, d] in float64, its first dim values rotated, by complex products."""
    x = x.copy()
    if dim:
        turn = amplitude * np.exp(1j * positions.astype(np.float64)[:, None] * f)[:, None]
        a, b = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
        z = (x[..., a] + 1j * x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
    return x
