"""The product in eight bits by each of its kernels on an MI355X, against the definition in 64 bits: many rows, outputs of 16
bits, values at f32's ends."""
import numpy as np
import pytest

from attention_oracle import HALF_STEP
from test_gpu_attention import dtype, say
from test_gpu_e4m3_product import rounded_rows, run, stood_for

pytestmark = pytest.mark.gpu

# Rows by which 1100 outputs take each kernel. Into f32: a few rows (as they lie, or not aligned), rounded rows by wavefronts
# that spread the inputs, tiles of two groups of wavefronts and of one. Into 16 bits: the tiles' e4m3 products, and 256 x 256.
N = 1100
KERNELS = [(6, "f32"), (40, "f32"), (2100, "f32"), (4200, "f32"), (6, "bf16"), (40, "bf16"), (2100, "bf16"), (4200, "bf16"), (13100, "bf16")]


def test_wide_tiles_past_the_last_scales(tk):
    """Tiles of 256 x 256 whose second half has no outputs and no scales: 1100 outputs are nine blocks of 128."""
    run(tk, 13100, 272, N, "bf16", "bf16")


def multiplied(tk, a, codes, scales, to, bias=None, act=0):
    """c for f32 rows; where no call of it is finite in 64 bits it is not looked at."""
    import torch

    import telmo_amd

    say("product e4m3", a.shape, codes.shape, to, act)
    m, n = len(a), len(codes)
    w = telmo_amd.E4m3Weights.from_parts(tk, codes, scales)
    c = torch.full((m, n), 3.0, dtype=dtype(to), device="cuda")
    space = torch.zeros(w.workspace_bytes(m), dtype=torch.uint8, device="cuda")
    epi = telmo_amd.Epilogue(bias=None if bias is None else torch.from_numpy(bias).cuda(), act=telmo_amd.Act(act))
    tk.linear_e4m3_device(torch.from_numpy(a).cuda(), w, c, epi, workspace=space)
    tk.synchronize()
    return c.double().cpu().numpy()


def off_by(ar, wr, to):
    """How far sums may be off: test_gpu_e4m3_product.run's bound."""
    m, k = ar.shape
    tol = (2 * k + 64) * HALF_STEP["f32"] * (np.abs(ar) @ np.abs(wr).T)
    if to != "f32" and m > 16:
        for x in range(0, k, 128):
            tol += 2.0**-10 * np.abs(ar[:, x:x + 128]).max(1)[:, None] * np.abs(wr[:, x:x + 128]).max(1)
    return tol


@pytest.mark.parametrize("k", (256, 300))
@pytest.mark.parametrize("m,to", KERNELS)
def test_sums_are_finite_where_the_outputs_are(tk, m, to, k):
    """Rows next to f32's largest values by weights of code 448 and small scales, and rows next to the least exponent by scales
    that are as large: what is multiplied is far from f32's ends only with the scale."""
    rng = np.random.default_rng(m + k)
    codes = rng.integers(0, 256, (N, k)).astype(np.uint8)
    codes[codes & 0x7F == 0x7F] = 0x7E
    blocks = (-(-N // 128), -(-k // 128))
    for low, high, lowest, highest in ((2.0**110, 3e38, -14, -11), (2.0**100, 3e38, -126, -100), (2.0**-98, 2.0**-90, 90, 118),
                                       (2.0**-20, 2.0**20, -120, 100)):
        a = (rng.choice([-1, 1], (m, k)) * 2.0 ** rng.uniform(np.log2(low), np.log2(high), (m, k))).astype(np.float32)
        a[rng.random((m, k)) < 0.98] = 0.0
        scales = (2.0 ** rng.uniform(lowest, highest, blocks)).astype(np.float32)
        ar, wr = rounded_rows(a.astype(np.float64)), stood_for(codes, scales)
        want, most = ar @ wr.T, np.abs(ar) @ np.abs(wr).T
        got = multiplied(tk, a, codes, scales, to)
        good = most < 2.0**126  # past that f32's own sums may be infinite
        assert good.mean() > 0.9
        tol = off_by(ar, wr, to) + 2.0**-120
        tol = tol + (0 if to == "f32" else HALF_STEP[to]) * (np.abs(want) + tol)
        off = np.abs(got - want)[good]
        assert np.all(np.isfinite(got[good])) and np.all(off <= tol[good]), (low, lowest, (off - tol[good]).max())


@pytest.mark.parametrize("m,to", KERNELS)
def test_zeros_by_the_largest_scales_are_zeros(tk, m, to):
    scales = np.full((9, 1), 2.0**119, np.float32)
    got = multiplied(tk, np.full((m, 128), 3e38, np.float32), np.zeros((N, 128), np.uint8), scales, to)
    assert np.all(got == 0.0)


@pytest.mark.parametrize("m,to", KERNELS + [(6, "f16"), (2100, "f16"), (13100, "f16")])
def test_silu_of_any_sum(tk, m, to):
    """SiLU of sums of zeros and a bias, over all of f32. It is off by a step of the exponential and of the reciprocal and
    five roundings, 2^-21 in all, or as much as it is below -87, 87 e^-87."""
    rng = np.random.default_rng(9)
    ends = [0.0, -0.0, 2.0**-140, 87.0, 87.5, 88.5, 100.0, 104.0, 127.9, 128.1, 1e10, 1e30, 1e37, 1e38, 2.3586e38, 2.36e38, 3e38, 3.4e38, np.inf]
    v = np.concatenate([ends, np.negative(ends), [np.nan], rng.uniform(-110, 110, 500), rng.standard_normal(300) * 3,
                        rng.choice([-1, 1], N) * 2.0 ** rng.uniform(-126, 127.9, N)])[:N].astype(np.float32)
    got = multiplied(tk, np.zeros((m, 130), np.float32), np.full((N, 130), 0x38, np.uint8), np.ones((9, 2), np.float32), to, bias=v, act=2)
    v = v.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        want = np.where(v == -np.inf, 0.0, v / (1 + np.exp(-v)))
    tol = np.abs(want) * 2.0**-21 + 2.0**-119
    tol += np.abs(want) * (1 + 2.0**-21) * HALF_STEP[to] + (2.0**-25 if to == "f16" else 0.0)
    largest = 65504.0 if to == "f16" else float(np.finfo(np.float32).max) if to == "f32" else 2.0**128 * (1 - 2.0**-8)
    for r in (0, m // 2, m - 1):
        assert np.array_equal(np.isnan(got[r]), np.isnan(v))
        assert np.all(got[r][v > largest * 1.01] == np.inf)
        near = np.abs(want) <= largest
        off = np.abs(got[r][near] - want[near])
        assert np.all(off <= tol[near]), v[near][off > tol[near]]


@pytest.mark.parametrize("type,n", [("f32", 8200), ("f16", 8201), ("bf16", 8200), ("f32", 16400), ("bf16", 32800), ("f16", 32783)])
@pytest.mark.parametrize("m,k", ((1, 256), (16, 300), (5, 1000), (16, 1024)))
def test_few_rows_by_very_many_outputs(tk, m, k, type, n):
    """Two panels of outputs to a workgroup, and four; rows in whole blocks, and not."""
    run(tk, m, k, n, type, "f32" if m == 5 else type, bias=False)


# Tiles of two groups of wavefronts, of one, and of 256 x 256, for about 1100 outputs in 16 bits.
TILES = (1300, 4200, 13100)


@pytest.mark.parametrize("type,to", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("m", TILES)
def test_tiles_into_16_bits(tk, m, type, to):
    run(tk, m, 384, 1100, type, to, act=2, scale=-1.5)
    run(tk, m - 19, 200, 1099, type, to, bias=False)  # outputs that end inside a lane's four
    run(tk, m, 130, 1100, type, to, act=1, accumulate=True, scale=0.5, pad=4, offset=0)
    run(tk, m + 1, 128, 1101, type, to, accumulate=True, pad=3, offset=1)


@pytest.mark.parametrize("m", TILES)
def test_special_rows_into_16_bits(tk, m):
    """Outliers, subnormals, zeros, f32's largest values; NaN and infinities make their rows' outputs NaN alone, NaN weights their
    outputs."""
    rng = np.random.default_rng(5)
    a = rng.standard_normal((m, 300)).astype(np.float32)
    a[0, 7], a[1], a[2, 130:260], a[3] = 1e30, 0.0, 1e-38, 2.0**-140
    a[4, ::2] *= 1e-3
    run(tk, m, 300, N, to="bf16", rows=a, bias=False)
    a[0, 5], a[2, 290], a[5, 0], a[m - 1, 299] = np.nan, np.inf, -np.inf, np.nan
    run(tk, m, 300, N, to="bf16", rows=a, bias=False)
    b = np.full((m, 128), 448.0, np.float32)  # at the border of an exponent, and one step past it
    b[1::2, 3] = np.nextafter(np.float32(448.0), np.float32(500.0))
    b[2, :] = 3.3e38
    run(tk, m, 128, N, to="bf16", rows=b, bias=False, codes=np.full((N, 128), 1, np.uint8))
    codes = rng.integers(0, 127, (N, 200)).astype(np.uint8)
    codes[37, 150], codes[N - 1, 0] = 0x7F, 0xFF
    for to in ("f16", "bf16"):
        run(tk, m, 200, N, to=to, codes=codes, bias=False)


@pytest.mark.parametrize("to", ("f16", "bf16"))
@pytest.mark.parametrize("m", TILES)
def test_products_that_cancel(tk, m, to):
    """Pairs of inputs whose products cancel exactly, and small ones beside them: off by 2^-10 of the largest products at most."""
    rng = np.random.default_rng(m)
    k = 272
    a = rng.standard_normal((m, k)).astype(np.float32)
    a[:, 1::2] = -a[:, ::2]
    codes = rng.integers(0, 0x7F, (N, k)).astype(np.uint8)
    codes[:, 1::2] = codes[:, ::2]
    a[:, 100:104] = rng.standard_normal((m, 4)) * 2.0**-6
    codes[:, 103] = rng.integers(0, 0x40, N)
    run(tk, m, k, N, to=to, rows=a, codes=codes, bias=False)


@pytest.mark.parametrize("m", TILES)
def test_tiles_replayed_from_a_graph(tk, gpu_stream, m):
    import torch

    args, space, c = run(tk, m, 300, N, "bf16", "bf16", act=2)
    want = c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        tk.linear_e4m3_device(*args, workspace=space)
    for i in range(3):
        args[2].fill_(float(i))
        space.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        same = torch.equal(c, want)
        tk.linear_e4m3_device(*args, workspace=space)
        torch.cuda.synchronize()
        assert same and torch.equal(c, want), i
