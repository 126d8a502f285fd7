"""The paged cache in eight bits on an MI355X: attention over it and the writes into it, against the definitions
in 64 bits."""
import itertools

import numpy as np
import pytest

from attention_oracle import attend, rotate, shown_pairs, tolerance
from e4m3_oracle import VALUES, encode, exponent, half_step
from test_gpu_attention import check, distance_bias, dtype, floats, ints, rows_of, say

pytestmark = pytest.mark.gpu

TYPES = ("f32", "f16", "bf16")


def allowed(type, d, keys, size, top):
    """The attention's tolerance with what eight-bit keys change: f16 and f32 rows are multiplied in two or three parts,
    up to three times the sums (counted as four by the form for position rows)."""
    return tolerance(type, d, keys, size, top, type != "bf16")


def pages_of(rng, pages, page, blocks, kv_heads, d, low=-6, high=3):
    """Codes of N(0, 100) values and random exponents, on the host, and what they stand for."""
    codes = encode(np.clip(rng.standard_normal((pages, page, kv_heads, d)) * 100, -448, 448))
    exps = rng.integers(low, high + 1, (pages, blocks, kv_heads)).astype(np.int8)
    return codes, exps, VALUES[codes] * 2.0 ** np.repeat(exps.astype(np.float64), page // blocks, 1)[..., None]


def on_gpu(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def run_paged(tk, type="f16", heads=4, kv_heads=2, d=64, new=(1, 1), lengths=(5, 70), page=16, block=16, cap=0.0, left=None,
              right=0, prefix=None, slopes=False, table=None, starts=True, workspace=True, bad=None, seed=1, layout="rows"):
    import torch

    import telmo_amd

    say("paged e4m3", type, heads, kv_heads, d, new, lengths, page, block, cap, left, right, prefix, bad, layout, seed)
    rng = np.random.default_rng(seed)
    width, batch = max(max(-(-n // page) for n in lengths), 1), len(new)
    pages = batch * width + 2
    tables = rng.permutation(pages)[:batch * width].reshape(batch, width)
    (kc, ke, k64), (vc, ve, v64) = (pages_of(rng, pages, page, page // block, kv_heads, d) for _ in "kv")
    held_rows, held_blocks = np.zeros((pages, page), bool), np.zeros((pages, page // block), bool)
    for b, n in enumerate(lengths):  # what holds no key is NaN, under an exponent of any kind
        j = np.arange(n)
        held_rows[tables[b][j // page], j % page] = True
        held_blocks[tables[b][j // page], j % page // block] = True
    stores = []
    for codes, exps in ((kc, ke), (vc, ve)):
        codes[~held_rows] = 0x7F
        exps[~held_blocks] = 127
        shape = {"rows": codes.shape, "heads": (pages, kv_heads, page, d), "padded": (pages, page + 1, kv_heads, d + 32)}[layout]
        t = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda")
        t = {"rows": t, "heads": t.transpose(1, 2), "padded": t[:, :page, :, :d]}[layout] if layout != "rows" else t
        t.copy_(on_gpu(codes))
        stores.append(t.view(torch.float8_e4m3fn))
        wide = torch.full((pages, page // block + (layout == "padded"), kv_heads), 127, dtype=torch.int8, device="cuda")
        stores.append(wide[:, :page // block])
        stores[-1].copy_(on_gpu(exps))
    kt, kx, vt, vx = stores
    held = [np.ones(n, bool) for n in lengths]
    given = tables.copy().astype(np.int64)
    for b, entry, value in bad or ():
        given[b, entry] = value
        held[b][entry * page:(entry + 1) * page] = False
    q, q64 = rows_of(rng, type, sum(new) + (2 if starts else 0), heads, d, layout="padded" if layout == "padded" else "rows")
    out = torch.full_like(q, 7.0)
    sl = (0.5 ** np.arange(1, heads + 1)).astype(np.float32) if slopes else None
    tb = None if table is None else rng.standard_normal((heads, 2 * table + 1)).astype(np.float32)
    att = telmo_amd.Attention(tk, heads, d, kv_heads=kv_heads, softcap=cap, left=left, right=right,
                              slopes=None if sl is None else floats(sl), table=None if tb is None else floats(tb))
    cache = telmo_amd.PagedCache(tk, kt, vt, k_exps=kx, v_exps=vx)
    space = None
    if workspace:
        space = torch.empty(att.workspace_bytes(sum(new), max(lengths), batch) + 64, dtype=torch.uint8, device="cuda")
    options = dict(q_starts=ints(np.concatenate([[0], np.cumsum(new)])) if starts else None,
                   prefix=None if prefix is None else ints(prefix), workspace=space)
    args = (q, cache, ints(given), ints(lengths), out)
    att.paged(*args, **options)
    tk.synchronize()
    got = out.double().cpu().numpy()
    assert np.all(got[sum(new):] == 7.0)
    r = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        j = np.arange(m)
        at = (tables[b][j // page], j % page)
        shown = shown_pairs(n, m, left, right, 0 if prefix is None else prefix[b], held=held[b])
        for h in range(heads):
            g = h // (heads // kv_heads)
            kk, vv = k64[at][:, g].reshape(m, d), v64[at][:, g].reshape(m, d)
            want, size = attend(q64[r:r + n, h], kk, vv, d**-0.5, shown, cap, distance_bias(n, m, h, sl, tb))
            check(got[r:r + n, h], want, allowed(type, d, m, size, np.abs(vv).max() if m else 0.0))
        r += n
    return att, args, options, out


@pytest.mark.parametrize("type,page", itertools.product(TYPES, ((1, 1), (7, 7), (16, 8), (25, 5), (64, 64), (64, 16), (96, 1))))
def test_single_tokens(tk, type, page):
    run_paged(tk, type, new=(1, 1, 1, 1), lengths=(1, 2, 65, 333), page=page[0], block=page[1])


@pytest.mark.parametrize("type,page", itertools.product(TYPES, ((1, 1), (7, 7), (16, 4), (64, 64), (64, 32))))
def test_chunks(tk, type, page):
    run_paged(tk, type, new=(40, 1, 0, 9, 3), lengths=(40, 70, 12, 200, 3), page=page[0], block=page[1])
    run_paged(tk, type, new=(40, 40), lengths=(41, 300), page=page[0], block=page[1], starts=False, workspace=False)


@pytest.mark.parametrize("type,new", itertools.product(TYPES, ((1, 1), (1, 30))))
@pytest.mark.parametrize("d", (16, 48, 64, 80, 128, 192, 256))
def test_head_sizes(tk, type, d, new):
    run_paged(tk, type, d=d, new=new, lengths=(150, 77))


@pytest.mark.parametrize("type", TYPES)
def test_lengths_of_zero_and_fewer_keys_than_rows(tk, type):
    run_paged(tk, type, new=(1, 1), lengths=(0, 0))
    run_paged(tk, type, new=(5, 2, 0), lengths=(2, 0, 9))
    run_paged(tk, type, new=(30, 2, 0), lengths=(2, 0, 9))


@pytest.mark.parametrize("type,heads", itertools.product(TYPES, ((1, 1), (8, 8), (8, 1), (12, 2), (40, 1))))
def test_heads_and_layouts(tk, type, heads):
    run_paged(tk, type, heads=heads[0], kv_heads=heads[1], d=128, new=(1, 3), lengths=(150, 77))
    run_paged(tk, type, heads=heads[0], kv_heads=heads[1], d=96, new=(1, 3), lengths=(150, 77), layout="heads", slopes=True)
    run_paged(tk, type, heads=heads[0], kv_heads=heads[1], d=64, new=(1, 20), lengths=(150, 77), layout="padded", block=8)


@pytest.mark.parametrize("type,new", itertools.product(TYPES, ((1, 2), (1, 30))))
def test_masks_and_biases(tk, type, new):
    run_paged(tk, type, new=new, lengths=(300, 290), left=100, cap=20.0, slopes=True)
    run_paged(tk, type, new=new, lengths=(300, 290), left=10, prefix=(20, 300))
    run_paged(tk, type, new=new, lengths=(300, 290), left=40, prefix=(4, 0))
    run_paged(tk, type, new=new, lengths=(300, 290), right=None, cap=400.0)
    run_paged(tk, type, new=new, lengths=(300, 290), table=30, block=4)


@pytest.mark.parametrize("type", TYPES)
def test_pages_that_the_cache_does_not_have_are_not_shown(tk, type):
    bad = [(0, 1, -1), (1, 0, 2**31 - 1), (1, 3, -2**31), (1, 17, 10**6)]
    run_paged(tk, type, new=(1, 20), lengths=(70, 280), bad=bad)
    run_paged(tk, type, new=(1, 2), lengths=(70, 280), bad=bad)
    run_paged(tk, type, new=(1,), lengths=(16,), bad=[(0, 0, -1)])  # nothing left


@pytest.mark.parametrize("type,new", itertools.product(TYPES, (1, 30)))
def test_keys_behind_the_window_may_hold_anything(tk, type, new):
    import torch

    import telmo_amd

    heads, d, page, total, left = 2, 64, 16, 200, 40
    rng = np.random.default_rng(8)
    (kc, ke, k64), (vc, ve, v64) = (pages_of(rng, 13, page, 4, heads, d) for _ in "kv")
    k64, v64 = k64.reshape(-1, heads, d), v64.reshape(-1, heads, d)
    q, q64 = rows_of(rng, type, new, heads, d)
    first = total - new - left  # the first key that any query is shown, in the middle of a block
    kc.reshape(-1, heads, d)[:first] = 0x7F
    vc.reshape(-1, heads, d)[:first] = 0xFF
    out = torch.zeros_like(q)
    cache = telmo_amd.PagedCache(tk, on_gpu(kc), on_gpu(vc), k_exps=on_gpu(ke), v_exps=on_gpu(ve))
    telmo_amd.Attention(tk, heads, d, left=left, right=0).paged(q, cache, ints([list(range(13))]), ints([total]), out)
    tk.synchronize()
    got, shown = out.double().cpu().numpy(), shown_pairs(new, total, left, 0)
    for h in range(heads):
        want, size = attend(q64[:, h], k64[:total, h], v64[:total, h], d**-0.5, shown)
        check(got[:, h], want, allowed(type, d, total, size, np.abs(v64).max()))


@pytest.mark.parametrize("type,new", itertools.product(TYPES, (1, 30)))
def test_rows_that_see_a_nan_key_are_nan_and_others_are_not(tk, type, new):
    import torch

    import telmo_amd

    heads, d, page, total = 2, 64, 16, 64
    rng = np.random.default_rng(9)
    (kc, ke, k64), (vc, ve, v64) = (pages_of(rng, 8, page, 1, heads, d) for _ in "kv")
    kc[3, 5, 0, 7] = 0x7F  # key 53 of the first sequence, head 0
    q, q64 = rows_of(rng, type, 2 * new, heads, d)
    out = torch.zeros_like(q)
    cache = telmo_amd.PagedCache(tk, on_gpu(kc), on_gpu(vc), k_exps=on_gpu(ke), v_exps=on_gpu(ve))
    telmo_amd.Attention(tk, heads, d, right=0).paged(q, cache, ints([[0, 1, 2, 3], [4, 5, 6, 7]]), ints([total, total]), out)
    tk.synchronize()
    got = out.double().cpu().numpy()
    sees = np.zeros((2 * new, heads), bool)
    sees[:new, 0] = np.arange(total - new, total) >= 53
    assert np.all(np.isnan(got[sees]))
    for b in range(2):
        k, v = (x[4 * b:4 * b + 4].reshape(-1, heads, d) for x in (k64, v64))
        for h in range(heads):
            rows = ~sees[b * new:(b + 1) * new, h]
            want, size = attend(q64[b * new:(b + 1) * new, h], k[:, h], v[:, h], d**-0.5, shown_pairs(new, total, None, 0))
            check(got[b * new:(b + 1) * new, h][rows], want[rows], allowed(type, d, total, size, np.abs(v).max()))


@pytest.mark.parametrize("type", TYPES)
def test_chunks_of_many_sequences(tk, type):
    lengths = (130, 150, 200, 300, 131, 140, 190, 260, 129)
    run_paged(tk, type, heads=8, kv_heads=8, new=(130,) * 9, lengths=lengths, page=16)
    run_paged(tk, type, heads=8, kv_heads=8, d=128, new=(130,) * 9, lengths=lengths, page=25, block=25, bad=[(3, 2, -1)], slopes=True)


@pytest.mark.parametrize("type,new", itertools.product(TYPES, ((1, 2), (33, 20))))
def test_long_caches_split_and_joined(tk, type, new):
    run_paged(tk, type, heads=2, kv_heads=1, d=64, new=new, lengths=(9000, 4097), page=64, block=64)
    run_paged(tk, type, heads=2, kv_heads=1, d=64, new=new, lengths=(9000, 4097), page=64, block=8, workspace=False)


@pytest.mark.parametrize("type", TYPES)
def test_calls_replayed_from_a_graph(tk, gpu_stream, type):
    import torch

    att, args, options, out = run_paged(tk, type, new=(1, 1, 4), lengths=(3000, 40, 900), heads=4, kv_heads=1)
    want = out.clone()
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        att.paged(*args, **options)
    for i in range(4):
        out.fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:6], want[:6]), i
        att.paged(*args, **options)  # the program's own eager call between replays
        torch.cuda.synchronize()
        assert torch.equal(out[:6], want[:6]), i


@pytest.mark.parametrize("new", (1, 30))
def test_strides_whose_offsets_pass_32_bits(tk, new):
    """Pages whose stride puts the last one beyond 2^32 values, read and written."""
    import torch

    import telmo_amd

    page, d, stride = 16, 64, (1 << 31) + 1024
    store = torch.empty(2 * stride + page * d * 2, dtype=torch.uint8, device="cuda")
    k, v = (torch.as_strided(store[x:], (3, page, 1, d), (stride, d, d, 1)) for x in (0, page * d))
    k_near, v_near = (torch.randint(0, 120, (3, page, 1, d), dtype=torch.uint8, device="cuda") for _ in "kv")
    k.copy_(k_near)
    v.copy_(v_near)
    exps = [torch.full((3, 2, 1), -8, dtype=torch.int8, device="cuda") for _ in range(4)]
    q, rows = torch.randn(new, 1, d, device="cuda").half(), torch.randn(20, 1, d, device="cuda")
    att, tables, lens = telmo_amd.Attention(tk, 1, d), ints([[2, 0, 1]]), ints([3 * page - 5])
    outs = []
    for kk, vv, e in ((k, v, exps[:2]), (k_near, v_near, exps[2:])):
        cache, out = telmo_amd.PagedCache(tk, kk, vv, k_exps=e[0], v_exps=e[1]), torch.zeros_like(q)
        cache.append(rows, rows + 1, tables, lens)
        att.paged(q, cache, tables, lens, out)
        outs.append(out)
    tk.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(k, k_near) and torch.equal(v, v_near) and torch.equal(exps[0], exps[2])


# ------------------------------------------------------------------------------------------ appends

def run_append(tk, type="f32", kv_heads=2, d=64, new=(1, 5), lengths=(5, 40), page=16, block=8, dim=0, interleaved=False, longest=None,
               seed=3, layout="rows", spread=0.0, values=None, width=None, bad=()):
    """Appends against the definition: exponents and codes equal where keys are not rotated; rotated ones may fall on the
    other side of a border that they are nearer to than the rotation is exact (2^-20 of the pair's size)."""
    import torch

    import telmo_amd

    say("append e4m3", type, kv_heads, d, new, lengths, page, block, dim, interleaved, layout, seed)
    rng = np.random.default_rng(seed)
    batch = len(new)
    width = width or max(max(-(-n // page) for n in lengths), 1)
    pages = batch * width + 2
    tables = rng.permutation(pages)[:batch * width].reshape(batch, width)
    given = tables.astype(np.int64)
    for b, entry, value in bad:
        given[b, entry] = value
    cache, stores = {}, {}
    for name in "kv":
        codes, exps, _ = pages_of(rng, pages, page, page // block, kv_heads, d, -10, -4)
        shape = {"rows": codes.shape, "heads": (pages, kv_heads, page, d)}[layout]
        t = torch.empty(shape, dtype=torch.uint8, device="cuda")
        t = t.transpose(1, 2) if layout == "heads" else t
        t.copy_(on_gpu(codes))
        cache[name], stores[name] = (codes, exps.astype(np.int64)), (t, on_gpu(exps))
    total = sum(new)
    rows = {}
    for name in "kv":
        x = rng.standard_normal((total + 1, kv_heads, d)) * 2.0 ** (spread * rng.standard_normal((total + 1, kv_heads, 1)))
        if values is not None:
            x.flat[rng.choice(x.size, x.size // 5, False)] = rng.choice(values, x.size // 5)
        t = torch.from_numpy(x.astype(np.float32)).to(dtype(type))
        rows[name] = (t.cuda(), t.double().numpy())
    rotary = telmo_amd.Rotary(tk, dim, interleaved=interleaved) if dim else None
    c = telmo_amd.PagedCache(tk, stores["k"][0], stores["v"][0], k_exps=stores["k"][1], v_exps=stores["v"][1])
    starts = np.concatenate([[0], np.cumsum(new)])
    args = (rows["k"][0], rows["v"][0], ints(given), ints(lengths))
    options = dict(q_starts=ints(starts), rotary=rotary, longest=longest)
    c.append(*args, **options)
    tk.synchronize()
    for name in "kv":
        codes, exps = (x.copy() for x in cache[name])
        got, got_exps = stores[name][0].cpu().numpy(), stores[name][1].cpu().numpy().astype(np.int64)
        loose = np.zeros(codes.shape, bool)
        for b in range(batch):
            first = lengths[b] - new[b]
            x = rows[name][1][starts[b]:starts[b + 1]][:longest]
            position = np.arange(first, first + len(x))
            if name == "k" and dim:
                f, amplitude = telmo_amd.rotary_frequencies(dim)
                x = rotate(x, position, f, amplitude, dim, interleaved)
            keep = (position >= 0) & (position < width * page)
            x, position = x[keep], position[keep]
            for n in np.unique(position // block):
                p = given[b, n * block // page]
                if not 0 <= p < pages:
                    continue
                at = position // block == n
                part, r0, older = x[at], n * block % page, position[at][0] - n * block
                size = np.where(np.isfinite(part), np.abs(part), 0.0)
                e = exponent(size.max((0, 2)))
                if name == "k" and dim:  # next to a border the largest may lie on either side
                    near = exponent(size.max((0, 2)) * (1 + 2.0**-20)) != exponent(size.max((0, 2)) * (1 - 2.0**-20))
                    e = np.where(near, got_exps[p, r0 // block], e)
                had = exps[p, r0 // block].copy()
                now = np.maximum(e, had) if older else e
                if older:
                    old = codes[p, r0:r0 + older]
                    again = encode(VALUES[old] * 2.0 ** (had - now)[:, None])
                    codes[p, r0:r0 + older] = np.where((now > had)[:, None], again, old)
                exps[p, r0 // block] = now
                r = r0 + older
                codes[p, r:r + len(part)] = encode(np.clip(part, -1.875 * 2.0**127, 1.875 * 2.0**127) * 2.0 ** -now[:, None]
                                                   if values is not None else part * 2.0 ** -now[:, None])
                if values is not None:
                    codes[p, r:r + len(part)][~np.isfinite(part)] = 0x7F
                if name == "k" and dim:
                    loose[p, r:r + len(part)] = True
                    stands = VALUES[got[p, r:r + len(part)]] * 2.0 ** now[:, None]
                    slack = 2.0**-20 * np.abs(x).max()
                    assert np.all(np.abs(stands - part) <= half_step(np.abs(part) + slack, now[:, None]) + slack)
        assert np.array_equal(got_exps, exps), name
        same = (got == codes) | loose | (np.isnan(VALUES[got]) & np.isnan(VALUES[codes]))
        assert np.all(same), (name, np.argwhere(~same)[:5])
        assert np.mean(got == codes) > 0.999 or values is not None
    return c, args, options, stores


@pytest.mark.parametrize("type,page", itertools.product(TYPES, ((1, 1), (7, 7), (16, 16), (16, 4), (64, 32), (256, 256))))
def test_appends(tk, type, page):
    run_append(tk, type, new=(1, 5, 0, 30, 600), lengths=(1, 40, 12, 30, 650), page=page[0], block=page[1], spread=2.0)


@pytest.mark.parametrize("d,dim", ((16, 0), (16, 16), (48, 20), (64, 64), (80, 40), (128, 128), (256, 256), (256, 64)))
@pytest.mark.parametrize("interleaved", (False, True))
def test_rotated_appends(tk, d, dim, interleaved):
    run_append(tk, "f32", d=d, dim=dim, interleaved=interleaved, new=(1, 9, 70), lengths=(500, 40, 90), page=32, block=16)
    run_append(tk, "bf16", kv_heads=3, d=d, dim=dim, interleaved=interleaved, new=(150,), lengths=(180,), page=128, block=128)


def test_append_layouts_and_tables(tk):
    run_append(tk, layout="heads", new=(3, 20), lengths=(9, 33), dim=32)
    run_append(tk, new=(20, 4), lengths=(10, 3))  # rows before the sequence begins are not written
    run_append(tk, new=(20, 4), lengths=(40, 100), width=2)  # nor are those past the table
    run_append(tk, new=(20, 14), lengths=(40, 30), bad=[(0, 1, -1), (1, 1, 10**6)])
    run_append(tk, new=(20, 14), lengths=(40, 30), longest=11)
    run_append(tk, new=(1, 1), lengths=(9, 25), spread=8.0, seed=4)  # blocks whose exponent grows, or not


@pytest.mark.parametrize("values", ((float("nan"), float("inf"), -float("inf")), (3.4028234663852886e38, -3.3e38, 1e-45),
                                    (0.0, -0.0), (448.0, 464.0, 480.0, 1.0625, 2.0**-9, 1.5 * 2.0**-9, 2.0**-10)))
def test_append_of_special_values(tk, values):
    run_append(tk, values=values, new=(1, 9), lengths=(10, 29))
    run_append(tk, values=values, new=(8,), lengths=(8,), block=1)


def test_appends_replayed_from_a_graph(tk, gpu_stream):
    import torch

    c, args, options, stores = run_append(tk, new=(1, 5), lengths=(9, 40), dim=64, spread=3.0)
    want = [x.clone() for pair in stores.values() for x in pair]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        c.append(*args, **options)
    for i in range(3):
        args[2].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([x for pair in stores.values() for x in pair], want)), i
        c.append(*args, **options)


def test_appends_and_attention_token_by_token(tk, gpu_stream):
    """Two prompts in chunks, then single tokens from one captured graph: each step's rows against the definition over
    what the cache stands for then, and that within its rounding of the keys and values that went in."""
    import torch

    import telmo_amd

    heads, kv, d, dim, page, block = 4, 2, 64, 32, 32, 16
    totals, chunks = (90, 77), ((50, 41), (30, 30)) + ((1, 1),) * 5
    rng = np.random.default_rng(12)
    x = [rng.standard_normal((2, max(totals), n, d)).astype(np.float32) for n in (heads, kv, kv)]
    width = -(-max(totals) // page)
    tables = rng.permutation(2 * width).reshape(2, width)
    codes = [torch.full((2 * width, page, kv, d), 0x7F, dtype=torch.uint8, device="cuda") for _ in "kv"]
    exps = [torch.full((2 * width, page // block, kv), 127, dtype=torch.int8, device="cuda") for _ in "kv"]
    cache = telmo_amd.PagedCache(tk, *codes, k_exps=exps[0], v_exps=exps[1])
    rotary, att = telmo_amd.Rotary(tk, dim), telmo_amd.Attention(tk, heads, d, kv_heads=kv, right=0, left=60)
    f, amplitude = telmo_amd.rotary_frequencies(dim)
    lens, table = ints([0, 0]), ints(tables)
    space = torch.empty(att.workspace_bytes(200, max(totals), 2) + 16, dtype=torch.uint8, device="cuda")
    done, graph, bufs = [0, 0], None, None

    def step(q, k, v, positions, turned, out, starts):
        rotary.apply(q, turned, positions)
        cache.append(k, v, table, lens, q_starts=starts, rotary=rotary)
        att.paged(turned, cache, table, lens, out, q_starts=starts, prefix=first, workspace=space)

    first = ints([4, 4])
    for new in chunks:
        q, k, v = (torch.cat([torch.from_numpy(y[b, done[b]:done[b] + new[b]]) for b in (0, 1)]).cuda() for y in x)
        at = ints(np.concatenate([np.arange(done[b], done[b] + new[b]) for b in (0, 1)]))
        lens.copy_(ints([done[b] + new[b] for b in (0, 1)]))
        if new == (1, 1):
            if graph is None:
                bufs = [q, k, v, at, torch.zeros_like(q), torch.zeros_like(q), ints([0, 1, 2])]
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=gpu_stream):
                    step(*bufs)
            for to, y in zip(bufs, (q, k, v, at)):
                to.copy_(y)
            graph.replay()
            out = bufs[5]
        else:
            out = torch.zeros_like(q)
            step(q, k, v, at, torch.zeros_like(q), out, ints([0, new[0], sum(new)]))
        torch.cuda.synchronize()
        got, r = out.double().cpu().numpy(), 0
        held = [VALUES[c.cpu().numpy()] * 2.0 ** np.repeat(e.double().cpu().numpy(), block, 1)[..., None] for c, e in zip(codes, exps)]
        for b in (0, 1):
            n, m = new[b], done[b] + new[b]
            j = np.arange(m)
            kk, vv = (y[tables[b][j // page], j % page] for y in held)
            step_of = [2.0 ** np.repeat(e.double().cpu().numpy(), block, 1)[tables[b][j // page], j % page][..., None] for e in exps]
            true = rotate(x[1][b, :m].astype(np.float64), j, f, amplitude, dim, False), x[2][b, :m].astype(np.float64)
            for y, z, s in zip((kk, vv), true, step_of):  # rounded at most twice: a half step, and one of the wider exponent's
                assert np.all(np.abs(y - z) <= 2 * np.maximum(np.abs(z) * 2.0**-4, s * 2.0**-10) * 1.01)
            turned = rotate(x[0][b, done[b]:m].astype(np.float64), np.arange(done[b], m), f, amplitude, dim, False)
            for h in range(heads):
                want, size = attend(turned[:, h], kk[:, h // 2], vv[:, h // 2], d**-0.5, shown_pairs(n, m, 60, 0, 4))
                check(got[r:r + n, h], want, allowed("f32", d + 64, m, size, np.abs(vv).max()))
            r += n
            done[b] = m
