"""The product in eight bits with a scale for each block of 128 x 128 on an MI355X, against the definition in 64 bits."""
import itertools

import numpy as np
import pytest

from attention_oracle import HALF_STEP
from e4m3_oracle import VALUES, encode, exponent
from test_gpu_attention import dtype, say

pytestmark = pytest.mark.gpu

NONE, RELU, SILU = 0, 1, 2


def rounded_rows(a):
    """a [m, k] in float64 with its groups of 128 inputs rounded to e4m3 times a power of two."""
    out = np.empty_like(a)
    for b in range(0, a.shape[1], 128):
        x = np.clip(a[:, b:b + 128], -1.875 * 2.0**127, 1.875 * 2.0**127) if np.isfinite(a[:, b:b + 128]).all() else a[:, b:b + 128]
        e = exponent(np.where(np.isfinite(x), np.abs(x), 0.0).max(1))[:, None].astype(np.float64)
        out[:, b:b + 128] = VALUES[encode(np.where(np.isfinite(x), np.clip(x * 2.0**-e, -448, 448), np.nan))] * 2.0**e
    return out


def stood_for(codes, scales):
    n, k = codes.shape
    return VALUES[codes] * np.repeat(np.repeat(scales.astype(np.float64), 128, 0)[:n], 128, 1)[:, :k]


def run(tk, m, k, n, type="f32", to="f32", act=NONE, scale=1.0, bias=True, accumulate=False, pad=0, offset=0, host=False, seed=1,
        rows=None, codes=None):
    """Returns the call's arguments. An output is off by its sum's error and roundings: a sum of k products in f32, each
    a step of the magnitudes' sum at most (blocks of 128 in the matrix instruction, one after another outside, and one
    rounding of each block's scaled sum); the epilogue's few operations and the SIMD exp's 2^-21; the output's half step.
    Many rows with 16-bit outputs add products in e4m3 that are aligned first: 2^-10 of a block's largest product more."""
    import torch

    import telmo_amd

    say("product e4m3", m, k, n, type, to, act, scale, bias, accumulate, pad, offset, seed)
    rng = np.random.default_rng(seed)
    a = (rng.standard_normal((m, k)) * 2.0 ** rng.integers(-6, 7, (m, 1)) if rows is None else rows).astype(np.float32)
    codes = rng.integers(0, 127, (n, k)).astype(np.uint8) + 128 * rng.integers(0, 2, (n, k)).astype(np.uint8) if codes is None else codes
    scales = (rng.uniform(0.5, 2.0, (-(-n // 128), -(-k // 128))) * 1e-3).astype(np.float32)
    store = torch.full((m, k + pad + offset), float("nan"), dtype=dtype(type), device="cuda")
    at = store[:, offset:offset + k]
    at.copy_(torch.from_numpy(a).to(dtype(type)))
    a64 = at.double().cpu().numpy()
    c = torch.full((m + 1, n + pad), 3.0, dtype=dtype(to), device="cuda")
    old = rng.standard_normal((m, n)).astype(np.float32)
    if accumulate:
        c[:m, :n] = torch.from_numpy(old).to(dtype(to))
        old = c[:m, :n].double().cpu().numpy()
    b = rng.standard_normal(n).astype(np.float32)
    epi = telmo_amd.Epilogue(bias=torch.from_numpy(b).cuda() if bias else None, act=telmo_amd.Act(act), scale=scale, accumulate=accumulate)
    if host:
        w = telmo_amd.E4m3Weights.from_parts(tk, codes, scales)
    else:
        wide = torch.full((n, k + pad), 0x7F, dtype=torch.uint8, device="cuda")
        wide[:, :k] = torch.from_numpy(codes).cuda()
        w = telmo_amd.E4m3Weights.from_device(tk, wide[:, :k], torch.from_numpy(scales).cuda())
    space = torch.full((w.workspace_bytes(m),), 0xFF, dtype=torch.uint8, device="cuda")
    args = (at, w, c[:m, :n], epi)
    tk.linear_e4m3_device(*args, workspace=space)
    tk.synchronize()
    ar, wr = rounded_rows(a64), stood_for(codes, scales)
    want = ar @ wr.T
    tol = (2 * k + 64) * HALF_STEP["f32"] * (np.abs(ar) @ np.abs(wr).T)
    if to != "f32" and m > 16:
        for x in range(0, k, 128):
            tol = tol + 2.0**-10 * np.abs(ar[:, x:x + 128]).max(1)[:, None] * np.abs(wr[:, x:x + 128]).max(1)
    if bias:
        want = want + b
        tol = tol + 2 * HALF_STEP["f32"] * np.abs(b)
    if act == RELU:
        want = np.maximum(want, 0)
    elif act == SILU:
        want = want / (1 + np.exp(-want))  # its slope is at most 1.1
        tol = 1.1 * tol + np.abs(want) * 2.0**-20 + 2.0**-120
    want, tol = want * scale, tol * abs(scale)
    if accumulate:
        want = want + old
    tol = tol + 8 * HALF_STEP["f32"] * np.abs(want) + 2.0**-120
    if to != "f32":
        tol = tol + HALF_STEP[to] * (np.abs(want) + tol) + (2.0**-25 if to == "f16" else 0.0)
    got = c.double().cpu().numpy()
    assert np.all(got[m] == 3.0) and np.all(got[:, n:] == 3.0)
    good = np.isfinite(want)
    assert np.all(np.isnan(got[:m, :n][~good]))
    off = np.abs(got[:m, :n] - want)[good]
    assert np.all(np.isfinite(got[:m, :n][good])) and np.all(off <= tol[good]), (off - tol[good]).max()
    return args, space, c


@pytest.mark.parametrize("m", (1, 2, 7, 15, 16, 17, 33, 64, 65, 100, 129, 300))
@pytest.mark.parametrize("k,n", ((128, 16), (640, 2560), (1000, 333), (127, 1), (1, 130), (129, 4097)))
def test_sizes(tk, m, k, n):
    run(tk, m, k, n)


@pytest.mark.parametrize("m,k,n", ((4100, 300, 4100), (2000, 1000, 2000), (8200, 130, 2100), (16, 4096, 16400), (1, 8192, 40)))
def test_larger_sizes(tk, m, k, n):
    run(tk, m, k, n, bias=False)


@pytest.mark.parametrize("type,to", itertools.product(("f32", "f16", "bf16"), repeat=2))
@pytest.mark.parametrize("m", (3, 40, 260))
def test_types(tk, type, to, m):
    run(tk, m, 384, 272, type, to, act=SILU)
    run(tk, m, 200, 272, type, to, accumulate=True, scale=0.5)


@pytest.mark.parametrize("act,bias,accumulate", itertools.product((NONE, RELU, SILU), (False, True), (False, True)))
def test_epilogues(tk, act, bias, accumulate):
    for m in (5, 50, 1100):
        run(tk, m, 256, 2100, act=act, bias=bias, accumulate=accumulate, scale=-1.5)


@pytest.mark.parametrize("pad,offset", ((1, 0), (3, 1), (8, 0), (8, 4), (0, 5)))
@pytest.mark.parametrize("type", ("f32", "bf16"))
def test_strides_and_alignments(tk, type, pad, offset):
    for m in (4, 70, 1200):
        run(tk, m, 272, 1200, type, type, pad=pad, offset=offset)


def test_empty_calls_and_sums(tk):
    run(tk, 0, 128, 64)
    run(tk, 5, 0, 64)
    run(tk, 500, 0, 3000, accumulate=True)
    run(tk, 5, 128, 0)


def test_host_weights_and_encoding(tk):
    import telmo_amd

    run(tk, 40, 300, 200, host=True)
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((200, 300)) * np.repeat([1e-3, 50.0], 100)[:, None]).astype(np.float32)
    w[128:, 256:] = 0.0
    codes, scales = telmo_amd.encode_e4m3(w, 200, 300)
    top = np.array([[np.abs(w[i:i + 128, j:j + 128]).max() for j in (0, 128, 256)] for i in (0, 128)])
    assert np.all(np.abs(scales - np.where(top > 0, top / 448, 1.0)) <= 2.0**-23 * scales)
    each = np.repeat(np.repeat(scales.astype(np.float64), 128, 0)[:200], 128, 1)[:, :300]
    assert np.array_equal(codes, encode(np.clip(w / each, -448, 448)))
    weights = telmo_amd.E4m3Weights.encode(tk, w, 200, 300)
    assert (weights.n(), weights.k(), weights.bytes()) == (200, 300, 200 * 300 + 4 * 6)


@pytest.mark.parametrize("m", (6, 40, 1100))
def test_special_rows(tk, m):
    """Outliers, subnormals, zeros, f32's largest values; NaN and infinities make their rows' outputs NaN alone."""
    rng = np.random.default_rng(5)
    a = rng.standard_normal((m, 300)).astype(np.float32)
    a[0, 7], a[1], a[2, 130:260], a[3] = 1e30, 0.0, 1e-38, 2.0**-140
    a[4, ::2] *= 1e-3
    run(tk, m, 300, 1100, rows=a, bias=False)
    a[0, 5], a[2, 290], a[5, 0] = np.nan, np.inf, -np.inf
    run(tk, m, 300, 1100, rows=a, bias=False)
    b = np.full((m, 128), 448.0, np.float32)  # at the border of an exponent, and one step past it
    b[1::2, 3] = np.nextafter(np.float32(448.0), np.float32(500.0))
    b[2, :] = 3.3e38
    run(tk, m, 128, 1100, rows=b, bias=False, codes=np.full((1100, 128), 1, np.uint8))


@pytest.mark.parametrize("m", (4, 40, 1100))
def test_nan_weights_make_their_outputs_nan(tk, m):
    rng = np.random.default_rng(6)
    codes = rng.integers(0, 127, (1100, 200)).astype(np.uint8)
    codes[37, 150], codes[1099, 0] = 0x7F, 0xFF
    run(tk, m, 200, 1100, codes=codes, bias=False)


@pytest.mark.parametrize("m", (1, 16, 60, 1200))
def test_calls_replayed_from_a_graph(tk, gpu_stream, m):
    import torch

    args, space, c = run(tk, m, 500, 1200, act=SILU)
    want = c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu_stream):
        tk.linear_e4m3_device(*args, workspace=space)
    for i in range(3):
        args[2].fill_(float(i))
        space.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want), i
        tk.linear_e4m3_device(*args, workspace=space)
        torch.cuda.synchronize()
        assert torch.equal(c, want), i
    args[0].mul_(2.0)  # the rows are read at each replay
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(c, want)


def test_two_contexts_at_once(tk):
    import torch

    import telmo_amd

    calls = []
    for i in range(2):
        stream = torch.cuda.Stream()
        kern = telmo_amd.Kernels(0, stream=stream.cuda_stream)
        with torch.cuda.stream(stream):
            calls.append((kern, stream) + run(kern, 700, 640, 900, seed=10 + i))
    wants = [call[4].clone() for call in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for kern, stream, args, space, c in calls:
            kern.linear_e4m3_device(*args, workspace=space)
    torch.cuda.synchronize()
    for (kern, stream, args, space, c), want in zip(calls, wants):
        assert torch.equal(c, want)
        args[1].close()
        kern.close()


def test_outputs_past_32_bits_of_values(tk):
    """Rows of outputs whose stride puts the last past 2^32 values."""
    import torch

    import telmo_amd

    m, k, n, ld = 40, 256, 300, (1 << 32) // 39 + 8
    big = torch.zeros((m - 1) * ld + n, dtype=torch.bfloat16, device="cuda")
    c, near = torch.as_strided(big, (m, n), (ld, 1)), torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(7)
    w = telmo_amd.E4m3Weights.encode(tk, rng.standard_normal((n, k)).astype(np.float32), n, k)
    a = torch.randn(m, k, device="cuda")
    space = torch.empty(w.workspace_bytes(m), dtype=torch.uint8, device="cuda")
    for out in (c, near):
        tk.linear_e4m3_device(a, w, out, workspace=space)
    tk.synchronize()
    assert torch.equal(c, near) and bool((near != 0).any())
