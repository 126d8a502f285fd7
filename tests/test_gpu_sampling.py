"""Drawing tokens on an MI355X, against the definition in 64 bits."""
import itertools

import numpy as np
import pytest

from test_gpu_attention import dtype, say

pytestmark = pytest.mark.gpu


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token and its probability, and how near a border the draw came: the least relative distance of a running
    sum to where it was cut or drawn."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not order.size:
        return -1, 0.0, 1.0
    if not temperature > 0:
        return order[0], 1.0, 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temperature)))
    n, near = w.size, [1.0]
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        sums = np.cumsum(w[:n])
        before = np.concatenate([[0.0], sums[:-1]])
        share = np.float64(np.float32(top_p)) * sums[-1]
        near.append(np.abs(before[1:] - share).min() / sums[-1] if n > 1 else 1.0)
        n = max(1, int((before < share).sum()))
    if min_p > 0:
        near.append(np.abs(w[:n] - np.float64(np.float32(min_p))).min() if n > 1 and min_p < 1 else 1.0)
        n = max(1, int((w[:n] >= np.float64(np.float32(min_p))).sum()))
    sums = np.cumsum(w[:n])
    target = np.float64(u) * sums[-1]
    near.append(np.abs(sums[:-1] - target).min() / sums[-1] if n > 1 else 1.0)
    at = min(int(np.searchsorted(sums, target, "right")), n - 1)
    return order[at], w[at] / sums[-1], min(near)


def run(tk, x, type="f32", seed=1, uniforms=None, pad=0, **options):
    """Draws from x [rows, n] and checks each row. Running sums are off by 2^-41 of themselves (half a step of 2^-40 of
    its bin's lower edge for each weight; where a crowded bin is divided, 2^-43 of the largest weight for each token), so a
    draw nearer than n 2^-42 to a border (there is none for n = 1) may fall on its other side."""
    import torch

    import telmo_amd

    say("sample", x.shape, type, options if all(np.ndim(v) == 0 for v in options.values()) else "mixed", seed)
    rows, n = x.shape
    rng = np.random.default_rng(seed)
    u = rng.random(rows).astype(np.float32) if uniforms is None else np.asarray(uniforms, np.float32)
    store = torch.full((rows, n + pad), 6e4, dtype=dtype(type), device="cuda")
    logits = store[:, :n]
    logits.copy_(torch.from_numpy(x.astype(np.float32)).to(dtype(type)))
    kinds = {k: np.int32 if k == "top_k" else np.float32 for k in options}
    given = {k: torch.from_numpy(np.asarray(v, kinds[k])).cuda() if np.ndim(v) else v for k, v in options.items()}
    sampler = telmo_amd.Sampler(tk, **given)
    tokens = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((rows + 1,), -7.0, device="cuda")
    space = torch.full((sampler.workspace_bytes(rows, n),), 0xA5, dtype=torch.uint8, device="cuda")
    args = (logits, torch.from_numpy(u).cuda(), tokens[:rows], probs[:rows])
    sampler.sample(*args, workspace=space)
    tk.synchronize()
    got, p = tokens.cpu().numpy(), probs.double().cpu().numpy()
    assert got[rows] == -7 and p[rows] == -7.0
    held = logits.float().cpu().numpy()
    for r in range(rows):
        each = {k: (np.asarray(v, kinds[k])[r] if np.ndim(v) else v) for k, v in options.items()}
        token, prob, near = draw(held[r], u[r], **each)
        if near > n * 2.0**-42:
            assert got[r] == token, (r, got[r], token, near, each)
        assert abs(p[r] - prob) <= 2.0**-23 * prob, (r, p[r], prob)
    return sampler, args, space, tokens, probs


def normal(rows, n, spread=2.0, seed=0):
    return spread * np.random.default_rng([seed, rows, n]).standard_normal((rows, n))


OPTIONS = [{}, dict(temperature=0.0), dict(temperature=0.1), dict(temperature=1.7), dict(top_k=1), dict(top_k=5), dict(top_k=700), dict(top_p=0.3),
           dict(top_p=0.95), dict(min_p=0.01), dict(min_p=1.0), dict(top_p=0.0), dict(top_k=40, top_p=0.9, min_p=0.05, temperature=0.8),
           dict(top_k=9000, top_p=0.99)]


@pytest.mark.parametrize("options", OPTIONS, ids=str)
@pytest.mark.parametrize("n", (1, 2, 63, 1000, 8198, 16384, 16385, 32767, 32768, 32769, 50001, 131072))
def test_sizes_and_options(tk, n, options):
    run(tk, normal(4, n), **options)


@pytest.mark.parametrize("type,n", itertools.product(("f16", "bf16"), (100, 8198, 32761, 40000)))
def test_types_whose_logits_are_often_equal(tk, type, n):
    for options in ({}, dict(top_k=50), dict(top_p=0.8), dict(min_p=0.1, temperature=0.5)):
        run(tk, normal(5, n), type, pad=3, **options)


@pytest.mark.parametrize("n", (5, 5000, 20000, 70000))
@pytest.mark.parametrize("options", ({}, dict(top_k=4321), dict(top_p=0.37), dict(top_k=60, top_p=0.5), dict(min_p=0.5)), ids=str)
def test_rows_of_equal_logits(tk, n, options):
    """More tokens of one logit than are sorted: they are told apart by their numbers."""
    x = np.zeros((3, n))
    x[1, ::2] = -1.0
    x[2] = -50.0
    x[2, n // 2] = 3.0
    run(tk, x, uniforms=(0.0, 0.61, 0.9999999), **options)


@pytest.mark.parametrize("spread", (1e-7, 1e-3, 30.0, 1e4, 1e30))
@pytest.mark.parametrize("n", (3000, 30000))
def test_narrow_and_wide_rows(tk, n, spread):
    """Spreads at which all tokens fall into a few bins, or nearly none does."""
    for options in ({}, dict(top_p=0.5), dict(top_k=2500), dict(top_k=2500, top_p=0.9, temperature=3.0), dict(min_p=0.999)):
        run(tk, 1000.0 * (spread < 1) + normal(3, n, spread), **options)


def test_uniforms_at_the_ends(tk):
    for n in (10, 9000, 40000):
        run(tk, normal(4, n), uniforms=(0.0, 2.0**-30, 1 - 2.0**-24, 0.5))
        run(tk, normal(4, n), uniforms=(0.0, 2.0**-30, 1 - 2.0**-24, 0.5), top_p=0.7, top_k=n - 1)


@pytest.mark.parametrize("n", (7, 9000, 40000))
def test_masked_and_special_logits(tk, n):
    x = normal(8, n)
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2, ::2] = -np.inf
    x[3] = np.nan
    x[4, 3] = np.nan
    x[5, [2, 5]] = np.inf
    x[6] = -3e38
    x[7, ::3], x[7, 1::3] = 0.0, -0.0
    for options in ({}, dict(top_p=0.6), dict(top_k=3), dict(min_p=0.3), dict(temperature=0.0), dict(temperature=1e30), dict(temperature=1e-30)):
        run(tk, x, **options)
    low = np.full((2, n), np.finfo(np.float32).min)  # a mask of the type's lowest value
    low[1, -1] = 0.0
    run(tk, low)


def test_options_of_each_row(tk):
    rng = np.random.default_rng(4)
    rows = 60
    for n in (900, 30000):
        run(tk, normal(rows, n), temperature=rng.choice([0.0, 0.3, 1.0, 2.0, -1.0, np.nan], rows), top_k=rng.choice([0, 1, 30, 500, -4], rows),
            top_p=rng.choice([0.2, 0.9, 1.0, 1.5], rows), min_p=rng.choice([0.0, 0.1, 2.0, -1.0], rows))


@pytest.mark.parametrize("n", (50, 9000, 40000))
def test_options_of_rows_past_their_ranges(tk, n):
    """A smallest share past 1 leaves the first token (and its equals), whatever it is; NaN stands for none."""
    x = np.round(normal(8, n))
    run(tk, x, min_p=np.array([np.inf, 3e38, 1.0001, 1.0, 1e-45, 1e-30, 0.0, -np.inf]))
    import torch

    import telmo_amd

    logits, u = torch.from_numpy(x.astype(np.float32)).cuda(), torch.linspace(0, 0.99, 8, device="cuda")
    drawn = []
    for options in ({}, dict(top_p=torch.full((8,), np.nan, device="cuda"), min_p=torch.full((8,), np.nan, device="cuda"))):
        sampler = telmo_amd.Sampler(tk, **options)
        drawn.append(torch.zeros(8, dtype=torch.int32, device="cuda"))
        sampler.sample(logits, u, drawn[-1], workspace=torch.zeros(sampler.workspace_bytes(8, n), dtype=torch.uint8, device="cuda"))
    tk.synchronize()
    assert torch.equal(*drawn)


def test_many_rows_and_empty_calls(tk):
    run(tk, normal(1500, 300), top_p=0.9)
    run(tk, normal(0, 300))
    run(tk, np.zeros((3, 0)))


def test_shares_follow_the_probabilities(tk):
    """20000 draws of one row: each token's count within five standard deviations of its share."""
    x = np.tile(normal(1, 40, 1.5, seed=9), (20000, 1))
    sampler, args, space, tokens, probs = run(tk, x[:2])
    import torch

    import telmo_amd

    u = torch.rand(20000, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    out = torch.empty(20000, dtype=torch.int32, device="cuda")
    telmo_amd.Sampler(tk).sample(torch.from_numpy(x.astype(np.float32)).cuda(), u, out)
    tk.synchronize()
    share = np.exp(x[0]) / np.exp(x[0]).sum()
    count = np.bincount(out.cpu().numpy(), minlength=40)
    assert np.all(np.abs(count - 20000 * share) <= 5 * np.sqrt(20000 * share * (1 - share)) + 1)


@pytest.mark.parametrize("n", (8198, 50000))
def test_calls_replayed_from_a_graph(tk, gpu_stream, n):
    import torch

    sampler, args, space, tokens, probs = run(tk, normal(6, n), top_p=0.9, top_k=300)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        sampler.sample(*args, workspace=space)
    for i in range(4):
        args[1].uniform_(generator=torch.Generator("cuda").manual_seed(i))
        tokens.fill_(-7)
        space.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        got = tokens.clone(), probs.clone()
        sampler.sample(*args, workspace=space)
        torch.cuda.synchronize()
        assert torch.equal(got[0], tokens) and torch.equal(got[1], probs)
        held, u = args[0].cpu().numpy(), args[1].cpu().numpy()
        for r in range(6):
            token, prob, near = draw(held[r], u[r], top_p=0.9, top_k=300)
            assert near < n * 2.0**-42 or tokens[r] == token


def test_rows_past_32_bits_of_values(tk):
    import torch

    import telmo_amd

    rows, n, ld = 5, 20000, (1 << 30) + 8
    big = torch.zeros((rows - 1) * ld + n, dtype=torch.float16, device="cuda")
    far, near = torch.as_strided(big, (rows, n), (ld, 1)), torch.randn(rows, n, device="cuda").half()
    far.copy_(near)
    sampler = telmo_amd.Sampler(tk, top_p=0.9)
    u, outs = torch.rand(rows, device="cuda"), []
    space = torch.empty(sampler.workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    for x in (far, near):
        outs.append(torch.zeros(rows, dtype=torch.int32, device="cuda"))
        sampler.sample(x, u, outs[-1], workspace=space)
    tk.synchronize()
    assert torch.equal(*outs)


def test_python_arguments(tk):
    import torch

    import telmo_amd

    logits, u, out = torch.zeros((4, 50), device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    sampler = telmo_amd.Sampler(tk)
    for args in ((logits.double(), u, out), (logits[0], u, out), (logits.cpu(), u, out), (logits, u.double(), out), (logits, u, out.long()),
                 (logits, u.cpu(), out), (logits, u, out, out)):
        with pytest.raises(TypeError):
            sampler.sample(*args)
    for args in ((logits.t(), u, out), (logits, u[:3], out), (logits, u, torch.zeros(8, dtype=torch.int32, device="cuda")[::2])):
        with pytest.raises(ValueError):
            sampler.sample(*args)
    for bad in (dict(top_k=-1), dict(top_k=1 << 31)):
        with pytest.raises(ValueError):
            telmo_amd.Sampler(tk, **bad)
    for bad in (dict(temperature=out), dict(top_k=u), dict(min_p=u.cpu())):
        with pytest.raises(TypeError):
            telmo_amd.Sampler(tk, **bad)
    with pytest.raises(telmo_amd.TelmoError):
        telmo_amd.Sampler(tk, temperature=-1.0).sample(logits, u, out)
    with pytest.raises(telmo_amd.TelmoError):
        telmo_amd.Sampler(tk, top_p=torch.ones(3, device="cuda")).sample(logits, u, out)
    with pytest.raises(telmo_amd.TelmoError):
        sampler.sample(torch.zeros((1, 50000), device="cuda"), u, out)
