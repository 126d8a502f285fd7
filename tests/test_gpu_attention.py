"""Attention over rows and over paged caches on an MI355X, against the definition in 64 bits."""
import itertools

import numpy as np
import pytest

from attention_oracle import attend, shown_pairs, tolerance

pytestmark = pytest.mark.gpu


def say(*args):
    print("[case]", *args, flush=True)


def dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def rows_of(rng, type, *shape, layout="rows"):
    """N(0, 1) values of the type on the GPU as [rows, heads, d], and the same in float64 on the host.
    layout: "rows" as they come, "heads" with the heads outermost, "padded" with gaps between rows and heads."""
    import torch

    n, heads, d = shape
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype(type))
    if layout == "heads":
        t = torch.empty((heads, n, d), dtype=dtype(type), device="cuda").transpose(0, 1)
    elif layout == "padded":
        t = torch.full((n, heads + 1, d + 16), float("nan"), dtype=dtype(type), device="cuda")[:, :heads, :d]
    else:
        t = torch.empty(shape, dtype=dtype(type), device="cuda")
    t.copy_(x)
    return t, x.double().numpy()


def ints(values):
    import torch

    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def floats(values):
    import torch

    return torch.from_numpy(np.asarray(values, np.float32)).cuda()


def distance_bias(n, m, h, slopes, table):
    """The bias of head h [n, m] in float64, and whether there is one."""
    c = np.arange(m)[None, :] - np.arange(m - n, m)[:, None]
    bias = None
    if slopes is not None:
        bias = -slopes[h].astype(np.float64) * np.abs(c)
    if table is not None:
        span = table.shape[1] // 2
        t = table[h].astype(np.float64)[np.clip(c, -span, span) + span]
        bias = t if bias is None else bias + t
    return bias


def position_rows(n, m, h, rel, d):
    if rel is None:
        return None
    c = np.arange(m)[None, :] - np.arange(m - n, m)[:, None]
    span = rel.shape[0] // 2
    rows = rel[:, h * d:(h + 1) * d] if rel.shape[1] != d else rel
    return rows.astype(np.float64)[np.clip(c, -span, span) + span]


def check(got, want, tol):
    off = np.abs(got - want)
    assert np.all(np.isfinite(got)), "not finite"
    at = np.unravel_index(off.argmax(), off.shape) if off.size else None
    assert not off.size or off.max() <= tol, (off.max(), tol, at)


def run_rows(tk, type="f32", heads=2, kv_heads=None, d=64, lengths=(37,), k_lengths=None, layout="rows", cap=0.0,
             left=None, right=None, prefix=None, docs=None, slopes=False, table=None, rel=None, uw=False, scale=None,
             starts=True, workspace=True, longest=None, seed=1):
    """Attention.forward of random rows, checked against the definition; returns the outputs."""
    import torch

    import telmo_amd

    kv_heads = heads if kv_heads is None else kv_heads
    k_lengths = lengths if k_lengths is None else k_lengths
    say(type, heads, kv_heads, d, lengths, k_lengths, layout, cap, left, right, prefix, slopes, table, rel, seed)
    rng = np.random.default_rng(seed)
    nq, nk = sum(lengths), sum(k_lengths)
    spare = 3 if starts else 0  # rows behind the last sequence
    q, q64 = rows_of(rng, type, nq + spare, heads, d, layout=layout)
    k, k64 = rows_of(rng, type, nk + (spare if k_lengths is lengths else 2), kv_heads, d, layout=layout)
    v, v64 = rows_of(rng, type, k.shape[0], kv_heads, d, layout=layout)
    if not starts:
        k, v = k[:nk], v[:nk]
    out = torch.full((nq + spare, heads, d), 7.0, dtype=dtype(type), device="cuda")
    if layout == "padded":
        out = torch.full((nq + spare, heads + 2, d + 8), 7.0, dtype=dtype(type), device="cuda")[:, 1:heads + 1, :d]
    sl = (0.5 ** np.arange(1, heads + 1)).astype(np.float32) if slopes else None
    tb = rng.standard_normal((heads, 2 * table + 1)).astype(np.float32) if isinstance(table, int) else table
    rl = u = w = None
    if rel is not None:
        span, shared = rel
        rl = rng.standard_normal((2 * span + 1, d if shared else heads * d)).astype(np.float32)
    if uw:
        u, w = (rng.standard_normal((heads, d)).astype(np.float32) for _ in "uw")
    qd = kd = None
    if docs is not None:
        qd = kd = np.concatenate([np.asarray(docs(n)) for n in lengths] + [np.full(spare, -1)]).astype(np.int32)
    att = telmo_amd.Attention(tk, heads, d, kv_heads=kv_heads, scale=scale, softcap=cap, left=left, right=right,
                              slopes=None if sl is None else floats(sl), table=None if tb is None else floats(tb))
    space = None
    if workspace:
        space = torch.empty(att.workspace_bytes(nq, max(k_lengths + (1,)), len(lengths)) + 64, dtype=torch.uint8, device="cuda")
    options = dict(longest=longest, prefix=None if prefix is None else ints(prefix), q_docs=None if qd is None else ints(qd),
                   rel=None if rl is None else floats(rl), rel_u=None if u is None else floats(u),
                   rel_v=None if w is None else floats(w), workspace=space)
    if starts:
        options["q_starts"] = ints(np.concatenate([[0], np.cumsum(lengths)]))
        if k_lengths is not lengths:
            options["k_starts"] = ints(np.concatenate([[0], np.cumsum(k_lengths)]))
    else:
        options["batch"] = len(lengths)
    att.forward(q, k, v, out, **options)
    tk.synchronize()
    got = out.double().cpu().numpy()
    assert np.all(got[nq:] == 7.0), "rows behind the last sequence were written"
    scale = d**-0.5 if scale is None else float(np.float32(scale))
    q0 = k0 = 0
    for b, (n, m) in enumerate(zip(lengths, k_lengths)):
        shown = shown_pairs(n, m, left, right, 0 if prefix is None else prefix[b], None if qd is None else qd[q0:q0 + n],
                            None if kd is None else kd[k0:k0 + m])
        for h in range(heads):
            g = h // (heads // kv_heads)
            want, size = attend(q64[q0:q0 + n, h], k64[k0:k0 + m, g], v64[k0:k0 + m, g], scale, shown, cap,
                                distance_bias(n, m, h, sl, tb), position_rows(n, m, h, rl, d), None if u is None else u[h],
                                None if w is None else w[h])
            top = np.abs(v64[k0:k0 + m, g][np.isfinite(v64[k0:k0 + m, g])]).max() if m else 0.0
            tol = tolerance(type, d, m, size, top, rl is not None)
            check(got[q0:q0 + n, h], want, tol)
            if (~shown.any(1)).any():
                assert np.all(got[q0:q0 + n, h][~shown.any(1)] == 0.0)
        q0, k0 = q0 + n, k0 + m
    return out, att, (q, k, v), options


TYPES = ("f32", "f16", "bf16")


@pytest.mark.parametrize("type,n", itertools.product(TYPES, (1, 2, 31, 64, 65, 127, 300)))
def test_lengths(tk, type, n):
    run_rows(tk, type, lengths=(n,), seed=n)


@pytest.mark.parametrize("type,d", itertools.product(TYPES, (8, 16, 40, 64, 80, 96, 128, 136, 192, 256)))
def test_head_sizes(tk, type, d):
    run_rows(tk, type, d=d, lengths=(70,), seed=d)


@pytest.mark.parametrize("type,heads", itertools.product(TYPES, ((1, 1), (3, 1), (4, 2), (7, 1), (35, 5), (40, 1))))
def test_shared_heads(tk, type, heads):
    run_rows(tk, type, heads=heads[0], kv_heads=heads[1], lengths=(45,), right=0, slopes=True, table=9, seed=heads[0])


@pytest.mark.parametrize("type,layout", itertools.product(TYPES, ("rows", "heads", "padded")))
def test_layouts(tk, type, layout):
    run_rows(tk, type, heads=4, kv_heads=2, d=72, lengths=(50, 21), layout=layout)


@pytest.mark.parametrize("type", TYPES)
def test_ragged_sequences_with_empty_and_single_ones(tk, type):
    run_rows(tk, type, lengths=(0, 1, 130, 0, 64, 3, 0), right=0)
    run_rows(tk, type, lengths=(0, 0))
    run_rows(tk, type, lengths=(5, 0, 70), k_lengths=(9, 4, 0))  # the last one's queries have no keys
    run_rows(tk, type, lengths=(40, 7), k_lengths=(130, 3), right=0)  # more queries than keys: some see none


@pytest.mark.parametrize("type", TYPES)
def test_equal_sequences_without_starts(tk, type):
    run_rows(tk, type, lengths=(33, 33, 33), starts=False)
    run_rows(tk, type, lengths=(33, 33), k_lengths=(70, 70), starts=False, right=0)
    run_rows(tk, type, lengths=(0, 0), k_lengths=(7, 7), starts=False)


@pytest.mark.parametrize("type,window", itertools.product(TYPES, ((None, 0), (0, 0), (5, None), (None, 70), (17, 3), (64, 64),
                                                                  (200, 0), (2**40, 2**33))))
def test_windows(tk, type, window):
    run_rows(tk, type, heads=4, kv_heads=2, lengths=(150, 33), left=window[0], right=window[1])


@pytest.mark.parametrize("type,prefix", itertools.product(TYPES, ((0, 0), (1, 9), (100, 33), (400, -5))))
def test_prefixes(tk, type, prefix):
    run_rows(tk, type, lengths=(150, 33), right=0, left=20, prefix=prefix)
    run_rows(tk, type, lengths=(190, 10), k_lengths=(190, 150), right=0, left=2, prefix=prefix)


DOCS = {"packed": lambda n: np.arange(n) // 29, "one": lambda n: np.zeros(n), "none": lambda n: np.full(n, -1),
        "padded": lambda n: np.where(np.arange(n) < n * 2 // 3, 4, -1), "mixed": lambda n: np.arange(n) * 7 % 3,
        "far": lambda n: np.where(np.arange(n) < n // 2, 2**31 - 1, 0)}


@pytest.mark.parametrize("type,docs", itertools.product(TYPES, sorted(DOCS)))
def test_documents(tk, type, docs):
    run_rows(tk, type, heads=3, lengths=(150, 41), docs=DOCS[docs])
    run_rows(tk, type, heads=4, kv_heads=1, lengths=(130,), docs=DOCS[docs], left=9, right=30, prefix=(3,))


@pytest.mark.parametrize("type,cap", itertools.product(TYPES, (1.0, 30.0, 50.0)))
def test_caps(tk, type, cap):
    run_rows(tk, type, lengths=(90,), cap=cap, scale=2.0, right=0)


@pytest.mark.parametrize("type,span", itertools.product(TYPES, (0, 1, 40, 500)))
def test_bias_by_distance(tk, type, span):
    run_rows(tk, type, heads=4, kv_heads=2, lengths=(150,), table=span)
    run_rows(tk, type, heads=4, kv_heads=2, lengths=(150,), table=span, slopes=True, cap=20.0, right=0, d=128)


@pytest.mark.parametrize("type,low", itertools.product(TYPES, (-np.inf, np.finfo(np.float32).min, -1e30)))
def test_a_table_of_lowest_values(tk, type, low):
    """Distances past 3 get the lowest value: -infinity hides them, a finite one hides them where there is
    another key and shares the weight where there is none."""
    table = np.full((2, 9), low, np.float32)
    table[:, 1:8] = 0.25
    run_rows(tk, type, lengths=(100,), table=table)
    run_rows(tk, type, lengths=(100,), table=np.full((2, 1), low, np.float32))  # all alike


@pytest.mark.parametrize("n,heads,d,rel,uw", [
    (1, 2, 64, (0, False), True), (2, 1, 128, (1, False), True), (50, 2, 128, (49, False), True),
    (50, 2, 128, (49, False), False), (129, 3, 64, (128, True), False), (200, 2, 32, (199, False), True),
    (200, 2, 128, (20, True), True), (77, 2, 256, (76, False), True), (150, 1, 40, (300, True), False)])
def test_position_rows(tk, n, heads, d, rel, uw):
    run_rows(tk, "f32", heads=heads, d=d, lengths=(n,), rel=rel, uw=uw, seed=n)
    run_rows(tk, "f32", heads=heads, d=d, lengths=(n, 0, n // 2), rel=rel, uw=uw, right=3, prefix=(2, 2, 2), seed=n)


def test_position_rows_with_shared_heads_and_a_cap(tk):
    run_rows(tk, "f32", heads=6, kv_heads=2, d=64, lengths=(90,), rel=(89, False), uw=True, cap=15.0, slopes=True)


@pytest.mark.parametrize("type", TYPES)
def test_longer_rows(tk, type):
    run_rows(tk, type, heads=2, kv_heads=1, d=128, lengths=(700,), right=0)
    run_rows(tk, type, heads=2, kv_heads=1, d=128, lengths=(700,), right=0, workspace=False)
    run_rows(tk, type, heads=1, d=64, lengths=(3,), k_lengths=(5000,), right=0)
    run_rows(tk, type, heads=1, d=64, lengths=(3,), k_lengths=(5000,), right=0, workspace=False)


MANY = (130, 200, 0, 129, 257, 1, 140, 131, 180, 133, 128, 160)


@pytest.mark.parametrize("type", TYPES)
def test_many_sequences(tk, type):
    """Enough rows of enough heads for the f32 tiles of 128 rows, which few tiles do without."""
    run_rows(tk, type, heads=8, lengths=MANY, right=0)
    run_rows(tk, type, heads=8, d=128, lengths=MANY, left=50, right=20, docs=DOCS["packed"], prefix=(7,) * len(MANY))
    run_rows(tk, type, heads=16, kv_heads=8, d=72, lengths=MANY, cap=20.0, slopes=True, table=30)
    run_rows(tk, type, heads=8, d=256, lengths=MANY[:9], right=0)


@pytest.mark.parametrize("d,rel", [(128, (256, False)), (64, (100, True)), (128, (40, True)), (48, (256, False))])
def test_many_sequences_with_position_rows(tk, d, rel):
    run_rows(tk, "f32", heads=8, d=d, lengths=MANY, rel=rel, uw=True)
    run_rows(tk, "f32", heads=8, d=d, lengths=MANY, rel=rel, uw=True, left=60, right=10, prefix=(33,) * len(MANY), docs=DOCS["mixed"])


@pytest.mark.parametrize("type", TYPES)
def test_workspaces_of_any_size(tk, type):
    """Fewer parts than wanted fit a smaller workspace; none fits 16 bytes. Two results may each be off by a weight's
    and an output's rounding and by the sums over the keys."""
    import torch

    out, att, (q, k, v), options = run_rows(tk, type, heads=2, d=128, lengths=(900,), right=0)
    full = options.pop("workspace")
    need = att.workspace_bytes(900, 900)
    assert need > 0 and full.numel() >= need
    for size in (need // 2, need // 3, 16):
        some = torch.full_like(out, 7.0)
        att.forward(q, k, v, some, workspace=full[:size // 16 * 16], **options)
        tk.synchronize()
        half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[type]
        off = float((some.float() - out.float()).abs().max())
        assert off <= 2 * float(v.float().abs().max()) * (2 * half + (2 * 900 + 32) * 2.0**-24)


@pytest.mark.parametrize("type", TYPES)
def test_row_strides_past_the_tiles(tk, type):
    """Keys 2^23 values and more apart, which a tile's 32-bit offsets do not reach."""
    import torch

    import telmo_amd

    n, d, ld = 5, 64, (1 << 23) + 64
    store = torch.empty(n * ld, dtype=dtype(type), device="cuda")
    far = torch.as_strided(store, (n, 1, d), (ld, d, 1))
    near = torch.randn(n, 1, d, device="cuda").to(dtype(type))
    far.copy_(near)
    q = torch.randn(40, 1, d, device="cuda").to(dtype(type))
    outs = [torch.zeros_like(q) for _ in range(2)]
    att = telmo_amd.Attention(tk, 1, d)
    for k, out in zip((near, far), outs):
        att.forward(q, k, k, out)
    tk.synchronize()
    off = float((outs[0].float() - outs[1].float()).abs().max())
    assert off <= 4 * {"f32": 2.0**-20, "f16": 2.0**-11, "bf16": 2.0**-8}[type] * float(near.abs().max())


def test_forward_with_position_rows_replayed_from_a_graph(tk, gpu_stream):
    import torch

    out, att, (q, k, v), options = run_rows(tk, "f32", heads=2, d=128, lengths=(500,), rel=(499, False), uw=True)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        att.forward(q, k, v, out, **options)
    for i in range(4):
        out.fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:500], want[:500]), i
        att.forward(q, k, v, out, **options)
        torch.cuda.synchronize()
        assert torch.equal(out[:500], want[:500]), i


def test_two_contexts_at_once(tk):
    """Two streams' calls overlap, each stream with a context, an Attention and a workspace of its own."""
    import torch

    import telmo_amd

    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    q = torch.randn(700, 4, 128, generator=g, device="cuda").half()
    k, v = (torch.randn(700, 2, 128, generator=g, device="cuda").half() for _ in "kv")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    kerns = [telmo_amd.Kernels(0, stream=s.cuda_stream) for s in streams]
    atts = [telmo_amd.Attention(x, 4, 128, kv_heads=2, right=0) for x in kerns]
    spaces = [torch.empty(a.workspace_bytes(700, 700) + 16, dtype=torch.uint8, device="cuda") for a in atts]
    outs = [[torch.zeros_like(q) for _ in range(6)] for _ in atts]
    torch.cuda.synchronize()
    for i in range(6):
        for a, o, w in zip(atts, outs, spaces):
            a.forward(q, k, v, o[i], workspace=w)
    for x in kerns:
        x.synchronize()
    for o in outs:
        for y in o:
            assert torch.equal(y, outs[0][0])
    for x in kerns:
        x.close()


@pytest.mark.parametrize("type", TYPES)
def test_longest_bounds_the_rows_that_are_written(tk, type):
    import torch

    import telmo_amd

    q = torch.randn(150, 2, 64, device="cuda").to(dtype(type))
    full, part = torch.zeros_like(q), torch.full_like(q, 7.0)
    att = telmo_amd.Attention(tk, 2, 64)
    starts = ints([0, 90, 150])
    att.forward(q, q.clone(), q.clone(), full, q_starts=starts)
    att.forward(q, q.clone(), q.clone(), part, q_starts=starts, longest=40)
    tk.synchronize()
    done = np.r_[0:40, 90:130]
    left = np.setdiff1d(np.arange(150), done)
    assert torch.equal(part[done], full[done]) and bool((part[left] == 7.0).all())


@pytest.mark.parametrize("type,what", itertools.product(TYPES, (np.nan, np.inf, -np.inf)))
def test_keys_that_a_query_is_not_shown_may_hold_anything(tk, type, what):
    """Rows 60 to 69 hold NaN or infinities; causal queries before them and windowed ones past them must not
    notice, and only those that are shown them may be anything."""
    import torch

    import telmo_amd

    n, heads, d = 150, 2, 64
    rng = np.random.default_rng(3)
    q, q64 = rows_of(rng, type, n, heads, d)
    k, k64 = rows_of(rng, type, n, heads, d)
    v, v64 = rows_of(rng, type, n, heads, d)
    for bad_k, bad_v in ((True, False), (False, True), (True, True)):
        kb, vb, out = k.clone(), v.clone(), torch.zeros_like(q)
        if bad_k:
            kb[60:70] = what
        if bad_v:
            vb[60:70] = what
        telmo_amd.Attention(tk, heads, d, left=20, right=0).forward(q, kb, vb, out)
        tk.synchronize()
        got, shown = out.double().cpu().numpy(), shown_pairs(n, n, 20, 0)
        clean = np.r_[0:60, 90:n]  # 89 - 20 = 69 is the last row that a dirty one is in reach of
        for h in range(heads):
            want, size = attend(q64[:, h], k64[:, h], v64[:, h], d**-0.5, shown)
            check(got[clean, h], want[clean], tolerance(type, d, n, size, np.abs(v64).max(), False))
        if bad_v and not bad_k:  # a value of NaN or infinity that is shown reaches the output
            assert not np.isfinite(got[60:90]).any()


@pytest.mark.parametrize("type,d,what", itertools.product(TYPES, (64, 136), (np.nan, np.inf)))
def test_rows_that_see_a_nan_score_are_nan_and_others_are_not(tk, type, d, what):
    """Queries of NaN or infinity, whose scores are NaN (an infinity's have both signs among their products):
    whole rows of NaN, beside rows as they are. Over enough keys for a row to end at the first of them."""
    import torch

    import telmo_amd

    n, heads = 700, 2
    rng = np.random.default_rng(5)
    q, q64 = rows_of(rng, type, n, heads, d)
    k, k64 = rows_of(rng, type, n, heads, d)
    v, v64 = rows_of(rng, type, n, heads, d)
    bad = np.r_[3, 100:140, n - 1]
    q[bad] = what
    out = torch.zeros_like(q)
    telmo_amd.Attention(tk, heads, d).forward(q, k, v, out)
    tk.synchronize()
    got, clean = out.double().cpu().numpy(), np.setdiff1d(np.arange(n), bad)
    assert np.isnan(got[bad]).all()
    shown = np.ones((len(clean), n), bool)
    for h in range(heads):
        want, size = attend(q64[clean, h], k64[:, h], v64[:, h], d**-0.5, shown)
        check(got[clean, h], want, tolerance(type, d, n, size, np.abs(v64).max(), False))


@pytest.mark.parametrize("rel", (False, True))
def test_more_tiles_than_a_launch_holds_are_refused(tk, rel):
    """Ragged sequences of which any might hold all rows: refused before any launch; their longest makes it fit."""
    import torch

    import telmo_amd

    # With position rows heads of 136 take a wavefront per row: 2^26 rows are one workgroup too many for it. All rows but
    # the output's are one (stride 0).
    batch, rows, heads, d = (1, 1 << 26, 1, 136) if rel else (65535, 1 << 17, 16, 8)
    q = torch.ones((1, heads, d), dtype=torch.float32 if rel else torch.float16, device="cuda").expand(rows, heads, d)
    out = torch.zeros((rows, heads, d), dtype=q.dtype, device="cuda")
    starts = torch.full((batch + 1,), 5, dtype=torch.int32, device="cuda")
    starts[0] = 0
    options = dict(rel=torch.zeros((3, d), device="cuda")) if rel else {}
    att = telmo_amd.Attention(tk, heads, d, left=1, right=1)
    with pytest.raises(telmo_amd.TelmoError, match="longest"):
        att.forward(q, q, q, out, q_starts=starts, **options)
    att.forward(q, q, q, out, q_starts=starts, longest=5, **options)
    tk.synchronize()
    assert bool((out[:5] == 1.0).all()) and not bool(out[5:].any())


@pytest.mark.parametrize("type", TYPES)
def test_outputs_do_not_depend_on_the_run(tk, type):
    import torch

    out, att, (q, k, v), options = run_rows(tk, type, heads=2, lengths=(300, 40), right=0)
    for _ in range(3):
        again = torch.full_like(out, 7.0)
        att.forward(q, k, v, again, **options)
        tk.synchronize()
        assert torch.equal(again, out)


# ------------------------------------------------------------------------------------------- paged

def run_paged(tk, type="f16", heads=4, kv_heads=2, d=64, new=(1, 1), lengths=(5, 70), page=16, cap=0.0, left=None, right=0,
              prefix=None, slopes=False, rel=None, starts=True, workspace=True, bad=None, seed=1, layout="rows", poison=True):
    import torch

    import telmo_amd

    say("paged", type, heads, kv_heads, d, new, lengths, page, cap, left, right, prefix, bad, layout, seed)
    rng = np.random.default_rng(seed)
    width = max(max(-(-n // page) for n in lengths), 1)
    batch = len(new)
    pages = batch * width + 2
    shape = {"rows": (pages, page, kv_heads, d), "heads": (pages, kv_heads, page, d)}[layout]
    order = rng.permutation(pages)
    tables = order[:batch * width].reshape(batch, width)
    k64, v64 = rng.standard_normal((2, pages, page, kv_heads, d))
    k, v = (torch.from_numpy(x.astype(np.float32)).to(dtype(type)) for x in (k64, v64))
    k64, v64 = k.double().numpy(), v.double().numpy()
    kt, vt = (torch.full(shape, float("nan"), dtype=dtype(type), device="cuda") for _ in "kv")
    if layout == "heads":
        kt, vt = kt.transpose(1, 2), vt.transpose(1, 2)
    for b, n in enumerate(lengths):  # only rows that hold keys; the rest stays NaN where poisoned
        for j in range(n if poison else width * page):
            at = (tables[b, j // page], j % page)
            kt[at], vt[at] = k[at].cuda(), v[at].cuda()
    held = [np.ones(n, bool) for n in lengths]
    given = tables.copy().astype(np.int64)
    for b, entry, value in bad or ():
        given[b, entry] = value
        held[b][entry * page:(entry + 1) * page] = False
    spare = 2 if starts else 0
    q, q64 = rows_of(rng, type, sum(new) + spare, heads, d)
    out = torch.full_like(q, 7.0)
    sl = (0.5 ** np.arange(1, heads + 1)).astype(np.float32) if slopes else None
    att = telmo_amd.Attention(tk, heads, d, kv_heads=kv_heads, softcap=cap, left=left, right=right,
                              slopes=None if sl is None else floats(sl))
    cache = telmo_amd.PagedCache(tk, kt, vt)
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
            want, size = attend(q64[r:r + n, h], kk, vv, d**-0.5, shown, cap, distance_bias(n, m, h, sl, None))
            check(got[r:r + n, h], want, tolerance(type, d, m, size, np.abs(vv).max() if m else 0.0, False))
        r += n
    return att, args, options, out


@pytest.mark.parametrize("type,page", itertools.product(TYPES, (1, 7, 16, 25, 64, 100)))
def test_single_tokens_over_pages(tk, type, page):
    run_paged(tk, type, new=(1, 1, 1, 1), lengths=(1, 2, 65, 333), page=page)


@pytest.mark.parametrize("type,page", itertools.product(TYPES, (1, 7, 16, 64)))
def test_chunks_over_pages(tk, type, page):
    run_paged(tk, type, new=(40, 1, 0, 9, 3), lengths=(40, 70, 12, 200, 3), page=page)
    run_paged(tk, type, new=(40, 40), lengths=(41, 300), page=page, starts=False, workspace=False)


@pytest.mark.parametrize("type", TYPES)
def test_paged_lengths_of_zero_and_fewer_keys_than_rows(tk, type):
    run_paged(tk, type, new=(1, 1), lengths=(0, 0))
    run_paged(tk, type, new=(5, 2, 0), lengths=(2, 0, 9))


@pytest.mark.parametrize("type,heads", itertools.product(TYPES, ((1, 1), (8, 8), (8, 1), (12, 2), (40, 1))))
def test_paged_heads(tk, type, heads):
    run_paged(tk, type, heads=heads[0], kv_heads=heads[1], d=128, new=(1, 3), lengths=(150, 77))
    run_paged(tk, type, heads=heads[0], kv_heads=heads[1], d=96, new=(1, 3), lengths=(150, 77), layout="heads", slopes=True)


@pytest.mark.parametrize("type", TYPES)
def test_paged_masks(tk, type):
    run_paged(tk, type, new=(1, 30), lengths=(300, 290), left=100, cap=20.0, slopes=True)
    run_paged(tk, type, new=(1, 30), lengths=(300, 290), left=10, prefix=(20, 300))
    run_paged(tk, type, new=(2, 30), lengths=(300, 290), right=None)


@pytest.mark.parametrize("type", TYPES)
def test_pages_that_the_cache_does_not_have_are_not_shown(tk, type):
    bad = [(0, 1, -1), (1, 0, 2**31 - 1), (1, 3, -2**31), (1, 17, 10**6)]
    run_paged(tk, type, new=(1, 20), lengths=(70, 280), bad=bad)
    run_paged(tk, type, new=(1,), lengths=(16,), bad=[(0, 0, -1)])  # nothing left


@pytest.mark.parametrize("type,new", itertools.product(TYPES, (1, 30)))
def test_cached_keys_behind_the_window_may_hold_anything(tk, type, new):
    import torch

    import telmo_amd

    heads, d, page, total, left = 2, 64, 16, 200, 40
    rng = np.random.default_rng(8)
    k, k64 = rows_of(rng, type, 208, heads, d)
    v, v64 = rows_of(rng, type, 208, heads, d)
    q, q64 = rows_of(rng, type, new, heads, d)
    first = total - new - left  # the first key that any query is shown, in the middle of a page
    k[:first], v[:first] = float("nan"), float("inf")
    out = torch.zeros_like(q)
    cache = telmo_amd.PagedCache(tk, k.view(13, page, heads, d), v.view(13, page, heads, d))
    telmo_amd.Attention(tk, heads, d, left=left, right=0).paged(q, cache, ints([list(range(13))]), ints([total]), out)
    tk.synchronize()
    got, shown = out.double().cpu().numpy(), shown_pairs(new, total, left, 0)
    for h in range(heads):
        want, size = attend(q64[:, h], k64[:total, h], v64[:total, h], d**-0.5, shown)
        check(got[:, h], want, tolerance(type, d, total, size, np.abs(v64).max(), False))


@pytest.mark.parametrize("type", TYPES)
def test_chunks_of_many_sequences(tk, type):
    run_paged(tk, type, heads=8, kv_heads=8, new=(130,) * 9, lengths=(130, 150, 200, 300, 131, 140, 190, 260, 129), page=16)
    run_paged(tk, type, heads=8, kv_heads=8, d=128, new=(130,) * 9, lengths=(130, 150, 200, 300, 131, 140, 190, 260, 129), page=25,
              bad=[(3, 2, -1)], slopes=True)


@pytest.mark.parametrize("type", TYPES)
def test_long_caches_split_and_joined(tk, type):
    run_paged(tk, type, heads=2, kv_heads=1, d=64, new=(1, 2), lengths=(9000, 4097), page=64)
    run_paged(tk, type, heads=2, kv_heads=1, d=64, new=(1, 2), lengths=(9000, 4097), page=64, workspace=False)


@pytest.mark.parametrize("type", ("f16", "f32"))
def test_paged_calls_replayed_from_a_graph(tk, gpu_stream, type):
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
    args[3].sub_(1)  # the lengths are read at each replay
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(out[:6], want[:6])


@pytest.mark.parametrize("new", (1, 30))
def test_strides_whose_offsets_pass_32_bits(tk, new):
    """Pages of one head whose stride puts the last one beyond 2^32 elements (8.6 GB of f16 address space)."""
    import torch

    import telmo_amd

    page, d, stride = 16, 64, (1 << 31) + 1024
    store = torch.empty(2 * stride + page * d, dtype=torch.float16, device="cuda")
    k = torch.as_strided(store, (3, page, 1, d), (stride, d, d, 1))
    small = torch.randn(3, page, 1, d, device="cuda").half()
    k.copy_(small)
    q = torch.randn(new, 1, d, device="cuda").half()
    att, tables, lens = telmo_amd.Attention(tk, 1, d), ints([[2, 0, 1]]), ints([3 * page - 5])
    far, near = torch.zeros_like(q), torch.ones_like(q)
    att.paged(q, telmo_amd.PagedCache(tk, k, k), tables, lens, far)
    att.paged(q, telmo_amd.PagedCache(tk, small, small), tables, lens, near)
    tk.synchronize()
    assert torch.equal(far, near)
