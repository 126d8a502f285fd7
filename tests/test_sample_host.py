"""The drawing kernels run on the host, workgroup by workgroup, with each wavefront in turn as far ahead of the others as
barriers let it: a value that is read after another wavefront has put the next one in its place shows as a wrong token, or
as threads that wait for one another for good."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from test_gpu_sampling import draw

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = os.environ.get("HOST_CLANG", "/opt/rocm/llvm/bin/clang++")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("sample") / "sample_host.so")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O2", "-ffp-contract=off", "-mfma", "-fPIC", "-shared", "-I",
                    os.path.join(HERE, "host_gpu"), os.path.join(HERE, "sample_host.cpp"), "-o", out], check=True, capture_output=True)
    return ctypes.CDLL(out).draw_on_host


def drawn(host, x, u, first_wave, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The rows' tokens and probabilities, as test_gpu_sampling.run checks them."""
    x, u = np.ascontiguousarray(x, np.float32), np.asarray(u, np.float32)
    rows, n = x.shape
    tokens, probs = np.full(rows, -7, np.int32), np.zeros(rows, np.float32)
    f = ctypes.c_float
    at = [a.ctypes.data_as(ctypes.c_void_p) for a in (x, u, tokens, probs)]
    rc = host(0, at[0], ctypes.c_long(n), rows, n, f(temperature), top_k, f(top_p), f(min_p), *at[1:], first_wave)
    assert rc == 0, "threads wait for ones that are gone"
    for r in range(rows):
        token, prob, near = draw(x[r], u[r], np.float32(temperature), top_k, top_p, min_p)
        if near > n * 2.0**-42:
            assert tokens[r] == token, (r, tokens[r], token, near)
        assert abs(probs[r] - prob) <= 2.0**-23 * prob, (r, probs[r], prob)


def crowded(rows, n, seed=0):
    """Rows most of whose tokens fall into a few bins, some of them equal: the borders are looked for one by one."""
    rng = np.random.default_rng([seed, rows, n])
    x = rng.choice([0.0, 1e-3, 2e-3, 0.5], (rows, n)) + 1e-5 * rng.standard_normal((rows, n)) * (rng.random((rows, n)) < 0.3)
    return x


# A wavefront that finds the range's ends writes them (0, 1), one that does not (5), and the last.
@pytest.mark.parametrize("first_wave", (0, 1, 5, 15))
@pytest.mark.parametrize("options", (dict(min_p=0.9993), dict(top_k=9000, top_p=0.6, min_p=0.99), dict(top_k=14000, min_p=0.6), dict(top_k=7001), dict(top_p=0.4),
                                     dict(top_k=6000, top_p=0.9, min_p=0.6, temperature=0.8), {}), ids=str)
def test_borders_one_by_one(host, options, first_wave):
    drawn(host, crowded(1, 16000), [0.37], first_wave, **options)


@pytest.mark.parametrize("first_wave", (0, 1, 5))
def test_equal_logits_one_by_one(host, first_wave):
    x = np.zeros((1, 12000))
    x[0, ::3] = -0.25
    for options in (dict(top_k=6001, min_p=0.9), dict(top_k=9001, top_p=0.7, min_p=0.5), dict(min_p=0.9), dict(top_p=0.5)):
        drawn(host, x, [0.61], first_wave, **options)


@pytest.mark.parametrize("first_wave", (0, 1, 5))
def test_bins_of_a_single_logit(host, first_wave):
    """Logits so large that neighbours lie in different bins: a range is one logit from the start, and nothing but its ends
    is worked out between it and the next one."""
    x = 1e7 - np.random.default_rng(8).integers(0, 2, (1, 15000))
    for options in (dict(top_k=9001), dict(top_k=13001, top_p=0.9), dict(top_p=0.3), dict(top_k=13000, min_p=0.2), {}):
        drawn(host, x, [0.9], first_wave, **options)


@pytest.mark.parametrize("first_wave", (0, 7))
def test_rows_in_parts(host, first_wave):
    drawn(host, crowded(1, 40000), [0.8], first_wave, top_k=30000, top_p=0.8, min_p=0.9985)
    drawn(host, crowded(1, 40000), [0.8], first_wave, min_p=0.9985)
    drawn(host, np.random.default_rng(3).standard_normal((1, 40000)), [0.8], first_wave, top_k=50, top_p=0.8)


@pytest.mark.parametrize("n", (1, 63, 3000))
def test_short_rows(host, n):
    for options in ({}, dict(top_k=5, top_p=0.8), dict(min_p=0.2, temperature=0.7), dict(temperature=0.0)):
        drawn(host, np.random.default_rng(n).standard_normal((2, n)), [0.1, 0.9], 0, **options)
