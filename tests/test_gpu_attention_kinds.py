"""Kernels of the attention operators that few calls meet, on an MI355X, against the definition in 64 bits: few rows with
wide heads, caps, prefixes and tables; tables and position rows over pages; wide heads in paged chunks."""
import itertools

import numpy as np
import pytest

from attention_oracle import attend, shown_pairs, tolerance
from test_gpu_attention import TYPES, check, distance_bias, dtype, floats, ints, position_rows, rows_of, run_paged, run_rows, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type,d", itertools.product(TYPES, (136, 192, 256)))
def test_few_rows_of_wide_heads(tk, type, d):
    run_rows(tk, type, heads=4, kv_heads=2, d=d, lengths=(3, 1, 8), k_lengths=(700, 5, 33), right=0)
    run_rows(tk, type, heads=2, d=d, lengths=(1,), k_lengths=(3000,), workspace=False)
    run_paged(tk, type, heads=4, kv_heads=1, d=d, new=(1, 3), lengths=(1500, 70), page=16)
    run_paged(tk, type, heads=4, kv_heads=1, d=d, new=(1, 3), lengths=(333, 70), page=7, slopes=True, bad=[(0, 3, -1)])


@pytest.mark.parametrize("type,d", itertools.product(TYPES, (64, 128, 256)))
def test_few_rows_with_caps_prefixes_and_tables(tk, type, d):
    run_rows(tk, type, heads=4, kv_heads=2, d=d, lengths=(5, 2), k_lengths=(300, 90), cap=20.0, scale=1.0, right=0)
    run_rows(tk, type, heads=4, kv_heads=2, d=d, lengths=(5, 2), k_lengths=(300, 90), left=20, right=0, prefix=(70, 90))
    run_rows(tk, type, heads=4, kv_heads=2, d=d, lengths=(8, 1), k_lengths=(300, 90), table=40, cap=30.0, slopes=True, prefix=(3, 0))
    run_paged(tk, type, heads=4, kv_heads=2, d=d, new=(1, 4), lengths=(300, 77), cap=15.0, left=50, prefix=(40, 9), slopes=True)


@pytest.mark.parametrize("type,d", itertools.product(TYPES, (136, 256)))
def test_chunks_of_wide_heads_over_pages(tk, type, d):
    run_paged(tk, type, heads=4, kv_heads=2, d=d, new=(40, 0, 9), lengths=(70, 3, 200), page=16)
    run_paged(tk, type, heads=4, kv_heads=2, d=d, new=(40, 30), lengths=(290, 41), page=7, left=60, cap=20.0, prefix=(30, 4))
    run_paged(tk, type, heads=8, kv_heads=8, d=d, new=(130,) * 9, lengths=(130, 150, 200, 300, 131, 140, 190, 260, 129))


def run_pages(tk, type="f32", heads=4, kv_heads=2, d=64, new=(40, 9), lengths=(90, 200), page=16, cap=0.0, left=None, right=0,
              prefix=None, slopes=False, table=None, rel=None, uw=False, seed=1):
    """Attention over pages with a table by distance, or with position rows, which the C interface takes there."""
    import torch

    import telmo_amd
    from telmo_amd import _lib, attention

    say("pages", type, heads, kv_heads, d, new, lengths, page, cap, left, right, prefix, table, rel)
    rng = np.random.default_rng(seed)
    width, batch = -(-max(lengths) // page), len(new)
    tables = rng.permutation(batch * width + 2)[:batch * width].reshape(batch, width)
    stores, exact = [], []
    for _ in "kv":
        store = torch.full(((batch * width + 2) * page, kv_heads, d), float("nan"), dtype=dtype(type), device="cuda")
        rows = [rows_of(rng, type, n, kv_heads, d) for n in lengths]
        for b, (x, _) in enumerate(rows):
            j = np.arange(lengths[b])
            store[torch.from_numpy(tables[b][j // page] * page + j % page).cuda()] = x
        stores.append(store.view(-1, page, kv_heads, d))
        exact.append([x64 for _, x64 in rows])
    q, q64 = rows_of(rng, type, sum(new), heads, d)
    out = torch.full_like(q, 7.0)
    sl = (0.5 ** np.arange(1, heads + 1)).astype(np.float32) if slopes else None
    tb = rng.standard_normal((heads, 2 * table + 1)).astype(np.float32) if table is not None else None
    rl = u = w = None
    if rel is not None:
        rl = rng.standard_normal((2 * rel[0] + 1, d if rel[1] else heads * d)).astype(np.float32)
    if uw:
        u, w = (rng.standard_normal((heads, d)).astype(np.float32) for _ in "uw")
    held = [None if x is None else floats(x) for x in (sl, tb, rl, u, w)]
    att = telmo_amd.Attention(tk, heads, d, kv_heads=kv_heads, softcap=cap, left=left, right=right, slopes=held[0], table=held[1])
    cache = telmo_amd.PagedCache(tk, *stores)
    space = torch.empty(att.workspace_bytes(sum(new), max(lengths), batch) + 64, dtype=torch.uint8, device="cuda")
    lens, starts, at = ints(lengths), ints(np.concatenate([[0], np.cumsum(new)])), ints(tables)
    a, pre = attention._begun(att._desc), None if prefix is None else ints(prefix)
    rows = att._fill(a, q, out, pre, space)
    a.type = cache.type
    attention._CACHE.pack_into(a, attention._AT_K, *cache._k, *cache._v)
    cache._name_seqs(a, rows, at, lens, starts, None)
    if rel is not None:
        att._fill_rel(a, *held[2:])
    assert _lib.lib().tg_attention_paged_device(tk._ctx, a) == 0
    tk.synchronize()
    got, r = out.double().cpu().numpy(), 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        shown = shown_pairs(n, m, left, right, 0 if prefix is None else prefix[b])
        for h in range(heads):
            g = h // (heads // kv_heads)
            want, size = attend(q64[r:r + n, h], exact[0][b][:, g], exact[1][b][:, g], d**-0.5, shown, cap,
                                distance_bias(n, m, h, sl, tb), position_rows(n, m, h, rl, d), None if u is None else u[h],
                                None if w is None else w[h])
            check(got[r:r + n, h], want, tolerance(type, d, m, size, np.abs(exact[1][b]).max(), rel is not None))
        r += n


@pytest.mark.parametrize("type,d", itertools.product(TYPES, (64, 128, 256)))
def test_tables_over_pages(tk, type, d):
    run_pages(tk, type, d=d, table=30)
    run_pages(tk, type, d=d, table=300, page=7, cap=20.0, slopes=True, left=80, prefix=(20, 9))
    run_pages(tk, type, d=d, new=(1, 3), lengths=(300, 77), table=30)


MANY = dict(heads=8, kv_heads=8, new=(130,) * 9, lengths=(130, 150, 200, 300, 131, 140, 190, 260, 129))


@pytest.mark.parametrize("d,page,rel", [(64, 16, (299, False)), (128, 7, (40, True)), (128, 16, (299, False)), (48, 25, (299, True)),
                                        (136, 16, (299, False))])
def test_position_rows_over_pages(tk, d, page, rel):
    """d 136 takes a wavefront per row; nine sequences take the tiles of 128 rows, two those of 64."""
    run_pages(tk, d=d, page=page, rel=rel, uw=True)
    run_pages(tk, d=d, page=page, rel=rel, uw=True, new=(1, 2), lengths=(90, 5), right=None)
    run_pages(tk, d=d, page=page, rel=rel, left=70, cap=15.0, slopes=True, prefix=(20, 33))
    if d <= 128:
        run_pages(tk, d=d, page=page, rel=rel, uw=True, **MANY)
        run_pages(tk, d=d, page=page, rel=rel, left=70, cap=15.0, prefix=(20,) * 9, **MANY)
