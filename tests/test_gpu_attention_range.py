"""Attention far from rows of N(0, 1), on an MI355X, against the definition in 64 bits."""
import itertools

import numpy as np
import pytest

from attention_oracle import attend, shown_pairs, tolerance
from test_gpu_attention import TYPES, check, dtype, floats, position_rows, say

pytestmark = pytest.mark.gpu


def given(type, x):
    """x as a GPU tensor of the type, and what it holds in float64 on the host."""
    import torch

    t = torch.from_numpy(np.asarray(x, np.float32)).to(dtype(type))
    return t.cuda(), t.double().numpy()


def run(tk, q, k, v, split=True, rel=None, rel_u=None, rel_v=None, **options):
    """Attention.forward of one sequence [rows, heads, d], in parts where split; the outputs in float64."""
    import torch

    import telmo_amd

    att = telmo_amd.Attention(tk, q.shape[1], q.shape[2], kv_heads=k.shape[1], **options)
    out = torch.full_like(q, 7.0)
    space = torch.empty(att.workspace_bytes(q.shape[0], k.shape[0]) + 16, dtype=torch.uint8, device="cuda") if split else None
    starts = [torch.tensor([0, x.shape[0]], dtype=torch.int32, device="cuda") for x in (q, k)]
    att.forward(q, k, v, out, q_starts=starts[0], k_starts=starts[1], rel=rel, rel_u=rel_u, rel_v=rel_v, workspace=space)
    tk.synchronize()
    return out.double().cpu().numpy()


def own_size(q, k, scale, shown):
    """The largest sum of magnitudes behind a shown score, without a cap's."""
    return float(((np.abs(q) @ np.abs(k).T) * scale)[shown].max())


# ------------------------------------------------------------------------------------- large scores

@pytest.mark.parametrize("type,n,d", itertools.product(TYPES, (5, 150), (64, 128, 256)))
def test_large_rows_that_see_one_key_get_its_value(tk, type, n, d):
    """Scores of up to 10^9: the one shown key weighs 1 and the output is its value."""
    say("one key", type, n, d)
    rng = np.random.default_rng(n + d)
    (q, _), (k, _), (v, v64) = (given(type, x * rng.standard_normal((n, 2, d))) for x in (1e4, 1e4, 1.0))
    got = run(tk, q, k, v, left=0, right=0)
    # f32: the weight's and the value's parts are sums of three 8-bit ones, each exact, added in f32.
    assert np.all(np.abs(got - v64) <= (2.0**-22 * np.abs(v64) if type == "f32" else 0.0))


@pytest.mark.parametrize("type,n,d,scale", itertools.product(TYPES, (4, 300), (64, 128, 256), (2.0**-7, 2.0)))
def test_scores_that_differ_little_far_from_zero(tk, type, n, d, scale):
    """Every score is a large power of two plus a small multiple of 2^7 scale, exact in f32 (2^30 + 2^7 x in all
    partial sums), so the weights are those of small differences, at 2^23 and their ties at 2^31."""
    say("far scores", type, n, d, scale)
    rng = np.random.default_rng(n + d)
    q, k = np.zeros((n, 2, d)), np.zeros((500, 2, d))
    q[..., 0], k[..., 0] = 2.0**15, 2.0**15
    q[..., 1:5], k[..., 1:5] = 8.0 * rng.integers(-2, 3, (n, 2, 4)), 16.0 * rng.integers(-2, 3, (500, 2, 4))
    (q, q64), (k, k64), (v, v64) = given(type, q), given(type, k), given(type, rng.standard_normal((500, 2, d)))
    for split in (True, False):
        got = run(tk, q, k, v, split, scale=scale)
        for h in range(2):
            want, _ = attend(q64[:, h], k64[:, h], v64[:, h], scale, np.ones((n, 500), bool))
            # The scores are exact; the exponent, at most 32 log2(e) where a weight is more than 2^-46, is off by three
            # half steps of itself (the factor's, its product's, the base's).
            tol = tolerance(type, d, 500, 0.0, np.abs(v64).max(), False)
            check(got[:, h], want, tol + np.abs(v64).max() * 2 * 3 * 47 * 2.0**-24)


# ------------------------------------------------------------------------------------------ caps

@pytest.mark.parametrize("type,n,cap", itertools.product(TYPES, (3, 90), (1e-39, 1e-3, 200.0, 300.0, 1e4, 1e5, 1e7, 1e30)))
def test_caps_of_any_size(tk, type, n, cap):
    """A large cap leaves scores as they are, to the score's own size; a small one leaves next to nothing."""
    say("cap", type, n, cap)
    rng = np.random.default_rng(n)
    d, m, scale = 64, 400, 0.5
    q, k, v = (rng.standard_normal((x, 2, d)) for x in (n, m, m))
    q[1] = 0.0
    (q, q64), (k, k64), (v, v64) = (given(type, x) for x in (q, k, v))
    shown = shown_pairs(n, m, None, 0)
    got = run(tk, q, k, v, softcap=cap, scale=scale, right=0)
    for h in range(2):
        want, _ = attend(q64[:, h], k64[:, h], v64[:, h], scale, shown, float(np.float32(cap)))
        top = np.abs(v64[:, h]).max()
        tol = tolerance(type, d, m, own_size(q64[:, h], k64[:, h], scale, shown), top, False)
        if type != "f32" and cap <= 256:  # such caps of 16-bit rows: scores to 2^-21 of the cap, in weight and sum
            tol += top * 2 * np.expm1(cap * 2.0**-21)
        check(got[:, h], want, tol)


# --------------------------------------------------------------------------- outliers in f32 rows

@pytest.mark.parametrize("n,d,outlier", itertools.product((5, 40, 300), (64, 128, 256), (2.0**18, 2.0**24, 1e9, 1e12, 1e30)))
def test_rows_with_an_outlier_that_meets_zeros(tk, n, d, outlier):
    """One column of q (of k) holds values far past the others and zeros in k (in q): the score is what the small
    values make it."""
    say("outlier", n, d, outlier)
    rng = np.random.default_rng(n + d)
    q, k, v = (rng.standard_normal((x, 2, d)) for x in (n, 700, 700))
    q[..., 0], k[..., 0] = outlier * rng.choice([-1, 1], (n, 2)), 0.0
    k[..., 5], q[..., 5] = outlier, 0.0
    (q, q64), (k, k64), (v, v64) = (given("f32", x) for x in (q, k, v))
    for split in (True, False):
        got = run(tk, q, k, v, split)
        for h in range(2):
            want, size = attend(q64[:, h], k64[:, h], v64[:, h], d**-0.5, np.ones((n, 700), bool))
            check(got[:, h], want, tolerance("f32", d, 700, size, np.abs(v64[:, h]).max(), False))


@pytest.mark.parametrize("n,d,outlier", itertools.product((40, 300), (64, 128), (2.0**24, 1e12)))
def test_position_rows_with_an_outlier_that_meets_zeros(tk, n, d, outlier):
    """A column of the position rows that is zero in the queries, and one of u and w that is zero in the keys and the
    position rows."""
    say("position rows, outlier", n, d, outlier)
    rng = np.random.default_rng(n + d)
    q, k, v = (rng.standard_normal((n, 2, d)) for _ in "qkv")
    rel, u, w = rng.standard_normal((2 * n - 1, 2 * d)), rng.standard_normal((2, d)), rng.standard_normal((2, d))
    rel[:, [3, d + 3]] = outlier
    q[..., 3], u[:, 3], w[:, 3] = 0.0, 0.0, 0.0
    u[:, 7], w[:, 7] = outlier, -outlier
    k[..., 7], rel[:, [7, d + 7]] = 0.0, 0.0
    (q, q64), (k, k64), (v, v64) = (given("f32", x) for x in (q, k, v))
    rel, u, w = (x.astype(np.float32) for x in (rel, u, w))
    got = run(tk, q, k, v, rel=floats(rel), rel_u=floats(u), rel_v=floats(w))
    for h in range(2):
        want, size = attend(q64[:, h], k64[:, h], v64[:, h], d**-0.5, np.ones((n, n), bool),
                            rel=position_rows(n, n, h, rel, d), u=u[h].astype(np.float64), w=w[h].astype(np.float64))
        check(got[:, h], want, tolerance("f32", d, n, size, np.abs(v64[:, h]).max(), True))


@pytest.mark.parametrize("d,huge", itertools.product((64, 256), (1e18, 1e30)))
def test_hidden_keys_far_past_the_others(tk, d, huge):
    """Keys 60 to 69 dwarf the rest: queries that are not shown them get what the others make."""
    say("hidden", d, huge)
    n, rng = 200, np.random.default_rng(d)
    q, k, v = (rng.standard_normal((n, 2, d)) for _ in "qkv")
    k[60:70] = huge
    (q, q64), (k, k64), (v, v64) = (given("f32", x) for x in (q, k, v))
    got, shown = run(tk, q, k, v, left=20, right=0), shown_pairs(n, n, 20, 0)
    clean = ~shown[:, 60:70].any(1)
    for h in range(2):
        want, _ = attend(q64[:, h], k64[:, h], v64[:, h], d**-0.5, shown)
        size = own_size(q64[clean, h], k64[:, h], d**-0.5, shown[clean])
        check(got[clean, h], want[clean], tolerance("f32", d, n, size, np.abs(v64[:, h]).max(), False))


# ------------------------------------------------------------------- values at the end of their type

@pytest.mark.parametrize("n,split", itertools.product((5, 150), (True, False)))
def test_f16_values_at_the_end_of_the_type(tk, n, split):
    """Weights that all round up make the weighted mean of f16's largest value a little more than that, which has no
    f16: it stays the largest."""
    say("f16 values", n, split)
    d, m, high = 64, 900, 65504.0
    part = np.log(0.5 * (1 + 0.6 * 2.0**-10))  # a weight 0.6 of a step past 1/2 of the largest
    q, k = np.zeros((n, 1, d)), np.zeros((m, 1, d))
    q[..., 0], q[..., 1] = 1.0, 2.0**-9
    k[:, 0, 0] = np.float16(part)
    k[:, 0, 1] = np.float16((part - k[1, 0, 0]) * 512)
    k[::100] = 0.0  # the largest weights, some in every part
    signs = np.where(np.arange(d) % 2, 1.0, -1.0)
    (q, q64), (k, k64), (v, v64) = given("f16", q), given("f16", k), given("f16", high * signs * np.ones((m, 1, d)))
    weight = np.exp(k64[1, 0] @ q64[0, 0])
    assert 2.0**-11 < weight / 0.5 - 1 < 0.7 * 2.0**-10
    got = run(tk, q, k, v, split, scale=1.0)
    assert np.all(np.abs(got[:, 0] - high * signs) <= tolerance("f16", d, m, 1.0, high, False))


@pytest.mark.parametrize("n", (5, 40))
def test_f16_values_of_infinity_stay_infinite(tk, n):
    """A shown value of infinity, or NaN, reaches the output; a finite mean beside it does not change."""
    d, m = 64, 90
    q, k, v = (np.random.default_rng(x).standard_normal((x, 1, d)) for x in (n, m, m + 1))
    v = v[:m]
    v[3, 0, 0], v[4, 0, 1], v[5, 0, 2] = np.inf, -np.inf, np.nan
    (q, q64), (k, k64), (v, v64) = (given("f16", x) for x in (q, k, v))
    got = run(tk, q, k, v)
    assert np.all(got[:, 0, 0] == np.inf) and np.all(got[:, 0, 1] == -np.inf) and np.all(np.isnan(got[:, 0, 2]))
    want, size = attend(q64[:, 0], k64[:, 0], v64[:, 0, 3:], d**-0.5, np.ones((n, m), bool))
    check(got[:, 0, 3:], want, tolerance("f16", d, m, size, np.abs(v64[:, 0, 3:]).max(), False))
