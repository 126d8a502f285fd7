"""Attention over the paged cache in eight bits where values and exponents lie far apart, on an MI355X, against the
definition in 64 bits."""
import numpy as np
import pytest

from attention_oracle import attend, shown_pairs
from test_gpu_attention import check, dtype, ints, say
from test_gpu_cache_e4m3 import allowed, on_gpu, pages_of

pytestmark = pytest.mark.gpu


def attended(tk, type, new, total, low, high, hidden_nan, q_size=1.0, v_low=-6, v_high=3, left=40, heads=2, d=64, page=16, seed=8):
    """Rows of N(0, q_size^2) over keys whose exponents lie from low to high, scaled so that scores are of the order of 1.
    hidden_nan: the keys before all windows are NaN, so that rows are computed again from the definition."""
    import torch

    import telmo_amd

    say("paged e4m3 ends", type, new, total, low, high, hidden_nan, q_size, v_low, v_high)
    rng = np.random.default_rng(seed)
    pages = -(-total // page)
    (kc, ke, k64), (vc, ve, v64) = (pages_of(rng, pages, page, 4, heads, d, *x) for x in ((low, high), (v_low, v_high)))
    k64, v64 = k64.reshape(-1, heads, d), v64.reshape(-1, heads, d)
    q = torch.from_numpy(rng.standard_normal((new, heads, d)).astype(np.float32) * np.float32(q_size)).to(dtype(type))
    q64 = q.double().numpy()
    scale = float(np.float32(1 / (q_size * 100 * 2.0**high * np.sqrt(d))))
    first = total - new - left
    if hidden_nan:
        kc.reshape(-1, heads, d)[:first] = 0x7F
        vc.reshape(-1, heads, d)[:first] = 0xFF
    q = q.cuda()
    out = torch.zeros_like(q)
    cache = telmo_amd.PagedCache(tk, on_gpu(kc), on_gpu(vc), k_exps=on_gpu(ke), v_exps=on_gpu(ve))
    att = telmo_amd.Attention(tk, heads, d, left=left, right=0, scale=scale)
    att.paged(q, cache, ints([list(range(pages))]), ints([total]), out)
    tk.synchronize()
    got, shown = out.double().cpu().numpy(), shown_pairs(new, total, left, 0)
    for h in range(heads):
        want, size = attend(q64[:, h], k64[:total, h], v64[:total, h], scale, shown)
        check(got[:, h], want, allowed(type, d, total, size, np.abs(v64[:total, h]).max()))


@pytest.mark.parametrize("hidden_nan", (False, True))
@pytest.mark.parametrize("type,new", [(t, n) for t in ("f32", "bf16") for n in (1, 30)])
def test_large_rows_by_small_keys(tk, type, new, hidden_nan):
    """q of 2^118 by keys under 2^-100: their products are moderate, q's by the keys' codes are not."""
    attended(tk, type, new, 200, -100, -98, hidden_nan, q_size=2.0**118)


@pytest.mark.parametrize("type,new", [(t, n) for t in ("f32", "bf16") for n in (1, 30)])
@pytest.mark.parametrize("low,high", ((-100, -100), (-100, -92), (-100, 100), (100, 112)))
def test_values_of_the_least_and_largest_exponents(tk, type, new, low, high):
    """The least exponent leaves an f32 weight's three parts normal numbers of bf16; under the largest ones 40
    values of 448 stay below f32's end together."""
    attended(tk, type, new, 200, -6, 3, False, v_low=low, v_high=high)
