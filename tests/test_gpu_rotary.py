"""Rotary positions and writes into paged caches on an MI355X, against the definitions in 64 bits."""
import itertools

import numpy as np
import pytest

from attention_oracle import HALF_STEP, rotate
from test_gpu_attention import dtype, ints, rows_of, say

pytestmark = pytest.mark.gpu


def bound(want, x, type, amplitude):
    """Two products and a sum of values no larger than the pair's, sine and cosine off by at most 2^-22 (the
    quarter turn's rounding times pi/2, the function's own two steps, the amplitude's), one rounding to the type."""
    size = amplitude * np.abs(x).max(-1, keepdims=True)
    return HALF_STEP[type] * np.abs(want) + size * (2 * 2.0**-22 + 4 * HALF_STEP["f32"]) + (2.0**-25 if type == "f16" else 0.0)


PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "f16")]


def run(tk, type="f32", to=None, rows=5, heads=3, d=64, dim=None, interleaved=False, layout="rows", far=5000, base=10000.0,
        positions=True, in_place=False, **scaling):
    import torch

    import telmo_amd

    to, dim = to or type, d if dim is None else dim
    say("rotary", type, to, rows, heads, d, dim, interleaved, layout, far, scaling)
    rng = np.random.default_rng(rows * 100 + d + dim)
    x, x64 = rows_of(rng, type, rows, heads, d, layout=layout)
    out = x if in_place else torch.full((rows, heads + 1, d + 8), 7.0, dtype=dtype(to), device="cuda")[:, :heads, :d]
    at = rng.integers(0, far, rows).astype(np.int32) if positions else np.arange(far, far + rows)
    rotary = telmo_amd.Rotary(tk, dim, base=base, interleaved=interleaved, **scaling)
    rotary.apply(x, out, ints(at) if positions else None, start=0 if positions else far)
    tk.synchronize()
    f, amplitude = telmo_amd.rotary_frequencies(dim, base, **scaling)
    want = rotate(x64, at, f, amplitude, dim, interleaved)
    got = out.double().cpu().numpy()
    off = np.abs(got - want)
    assert np.all(off <= bound(want, x64, to, amplitude)), float((off - bound(want, x64, to, amplitude)).max())
    if dim < d:  # values past the rotated ones are copied (rounded once)
        assert np.array_equal(got[..., dim:], x64[..., dim:]) or type != to
    if not in_place and to == "f32":
        assert bool((out.as_strided((rows, d + 8), ((heads + 1) * (d + 8), 1))[:, d:] == 7.0).all())


@pytest.mark.parametrize("types,interleaved", itertools.product(PAIRS, (False, True)))
def test_types(tk, types, interleaved):
    run(tk, *types, rows=9, d=128, interleaved=interleaved)
    run(tk, *types, rows=9, d=80, dim=20, interleaved=interleaved)


@pytest.mark.parametrize("d,dim,interleaved", [(d, dim, i) for d, dims in
                                               ((8, (2, 4, 6, 8)), (64, (16, 18, 62, 64)), (256, (2, 128, 254, 256)))
                                               for dim in dims for i in (False, True)])
def test_parts_of_the_head(tk, d, dim, interleaved):
    run(tk, "f32", d=d, dim=dim, interleaved=interleaved)
    run(tk, "bf16", d=d, dim=dim, interleaved=interleaved, rows=4)


@pytest.mark.parametrize("rows,heads", [(1, 1), (3, 1), (4, 32), (5, 7), (1000, 2)])
def test_rows_and_heads(tk, rows, heads):
    run(tk, "bf16", rows=rows, heads=heads, d=128)
    run(tk, "f32", rows=rows, heads=heads, d=64, positions=False, far=17)


@pytest.mark.parametrize("layout", ("rows", "heads", "padded"))
def test_layouts(tk, layout):
    run(tk, "f16", layout=layout, d=72, dim=72)


@pytest.mark.parametrize("far", (1, 1 << 20, 2**31 - 1))
def test_far_positions(tk, far):
    """64 bits hold p f to 2^-53 of it: at 2^31 radians 2^-22, which both sides of the comparison may be off
    by, so the farthest are compared at a base whose pairs turn slowly."""
    run(tk, "f32", rows=50, d=128, far=far, base=1e6 if far < 2**31 - 1 else 1e9, dim=128 if far < 2**31 - 1 else 16)


@pytest.mark.parametrize("scaling", [dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                     dict(scaling="parts", factor=16.0, original=4096, slow=1.0, fast=32.0)])
def test_scaled_frequencies(tk, scaling):
    run(tk, "f32", rows=20, d=128, far=100000, **scaling)
    run(tk, "bf16", rows=20, d=128, dim=64, far=100000, interleaved=True, **scaling)


@pytest.mark.parametrize("interleaved", (False, True))
def test_in_place(tk, interleaved):
    run(tk, "f32", rows=33, d=128, in_place=True, interleaved=interleaved)
    run(tk, "f16", rows=33, d=80, dim=36, in_place=True, interleaved=interleaved, layout="padded")


# ------------------------------------------------------------------------------------------ append

def append(tk, type="f32", to="bf16", kv_heads=2, d=64, new=(1, 1), lengths=(1, 30), page=16, dim=None, interleaved=False,
           layout="rows", starts=True, longest=None, bad=(), k_layout="rows", width=None):
    import torch

    import telmo_amd

    say("append", type, to, kv_heads, d, new, lengths, page, dim, layout, bad)
    rng = np.random.default_rng(abs(sum(lengths)) + page)
    batch, width = len(new), width or max(max(-(-n // page) for n in lengths), 1)
    pages = batch * width + 1
    tables = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int64)
    for b, entry, value in bad:
        tables[b, entry] = value
    shape = (pages, page, kv_heads, d) if layout == "rows" else (pages, kv_heads, page, d)
    caches = [torch.full(shape, 7.0, dtype=dtype(to), device="cuda") for _ in "kv"]
    if layout == "heads":
        caches = [c.transpose(1, 2) for c in caches]
    spare = 2 if starts else 0
    k, k64 = rows_of(rng, type, sum(new) + spare, kv_heads, d, layout=k_layout)
    v, v64 = rows_of(rng, type, sum(new) + spare, kv_heads, d)
    rotary = None if dim is None else telmo_amd.Rotary(tk, dim, interleaved=interleaved)
    telmo_amd.PagedCache(tk, *caches).append(k, v, ints(tables), ints(lengths),
                                             q_starts=ints(np.concatenate([[0], np.cumsum(new)])) if starts else None,
                                             longest=longest, rotary=rotary)
    tk.synchronize()
    want_k, want_v = (np.full((pages, page, kv_heads, d), 7.0) for _ in "kv")
    slack = np.zeros_like(want_k)
    r = 0
    for n, total, table in zip(new, lengths, tables):
        for i in range(n if longest is None else min(n, longest)):
            p = total - n + i
            if 0 <= p < width * page and 0 <= table[p // page] < pages:
                at = (table[p // page], p % page)
                row = k64[r + i:r + i + 1]
                if dim is not None:
                    f, a = telmo_amd.rotary_frequencies(dim)
                    row = rotate(row, np.array([p]), f, a, dim, interleaved)
                want_k[at], want_v[at] = row[0], v64[r + i]
                slack[at] = bound(row, k64[r + i:r + i + 1], to, 1.0)[0]
        r += n
    got_k, got_v = (c.double().cpu().numpy() for c in caches)
    assert np.all(np.abs(got_k - want_k) <= slack)
    assert np.array_equal(got_v, torch.from_numpy(want_v).to(dtype(to)).double().numpy())
    if dim is None:
        assert np.array_equal(got_k, torch.from_numpy(want_k).to(dtype(to)).double().numpy())


@pytest.mark.parametrize("types,dim", itertools.product(PAIRS, (None, 64, 20)))
def test_append_types(tk, types, dim):
    append(tk, *types, dim=dim, new=(3, 1, 0, 20), lengths=(3, 40, 9, 50))


@pytest.mark.parametrize("page,layout", itertools.product((1, 7, 16, 64), ("rows", "heads")))
def test_append_pages(tk, page, layout):
    append(tk, page=page, layout=layout, new=(40, 1, 5), lengths=(40, 128, 70), dim=64, interleaved=True)
    append(tk, "bf16", "bf16", page=page, layout=layout, new=(9, 9), lengths=(9, 23), starts=False, d=128, k_layout="padded")


def test_append_leaves_what_has_no_place(tk):
    append(tk, new=(5, 2), lengths=(3, 0), dim=64)  # fewer positions than rows
    append(tk, new=(20, 20), lengths=(40, 40), bad=[(0, 2, -1), (1, 1, 99)])
    append(tk, new=(20, 5), lengths=(40, 40), longest=6)


def test_append_past_the_table_leaves_older_keys(tk):
    """Lengths that the table has no pages for: the rows behind it have no place, and those before keep
    theirs; so do lengths below zero."""
    append(tk, new=(20, 5, 3), lengths=(40, 90, 2**31 - 1), width=2, dim=64)
    append(tk, new=(6, 6), lengths=(-3, 2), width=2)
