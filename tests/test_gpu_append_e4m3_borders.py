"""Rotated keys next to the borders of e4m3, written into the paged cache on an MI355X: the nearest value is chosen as exactly
as f32 holds the rotated key."""
import numpy as np
import pytest

from attention_oracle import rotate
from e4m3_oracle import VALUES, encode, exponent
from test_gpu_attention import ints, say

pytestmark = pytest.mark.gpu


# Blocks of 16 rows, whose sines and cosines fit LDS, and of 128, whose do not; a rotated part of whole pieces, and not.
@pytest.mark.parametrize("block,dim,interleaved", ((16, 64, False), (16, 64, True), (128, 64, False), (128, 64, True), (16, 40, False)))
def test_keys_that_nearly_cancel(tk, block, dim, interleaved):
    """The first value of each pair is 2^-6 of its terms. A rotated key is off by half an f32 step of itself and 2^-40 of its
    terms (a position of 3000 times a frequency in 64 bits is a turn's 2^-44): the value taken may lie twice that further off
    than the nearest one."""
    import torch

    import telmo_amd

    say("append e4m3 borders", block, dim, interleaved)
    rng = np.random.default_rng(block + dim)
    n, heads, d = 4096, 4, 64
    f, amplitude = telmo_amd.rotary_frequencies(dim)
    angle = np.arange(n, dtype=np.float64)[:, None, None] * f
    cos, sin = np.cos(angle), np.sin(angle)
    rows = rng.standard_normal((n, heads, d)).astype(np.float32)
    first, second = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    a = rows[..., first].astype(np.float64)
    small = a * 2.0**-6 * rng.uniform(0.5, 1, a.shape)
    rows[..., second] = np.where(np.abs(sin) > 0.3, (a * cos - small) / np.where(np.abs(sin) > 0.3, sin, 1.0), rows[..., second])
    codes = [torch.zeros((n // 128, 128, heads, d), dtype=torch.uint8, device="cuda") for _ in "kv"]
    exps = [torch.zeros((n // 128, 128 // block, heads), dtype=torch.int8, device="cuda") for _ in "kv"]
    cache = telmo_amd.PagedCache(tk, *codes, k_exps=exps[0], v_exps=exps[1])
    t = torch.from_numpy(rows).cuda()
    cache.append(t, t, ints([list(range(n // 128))]), ints([n]), rotary=telmo_amd.Rotary(tk, dim, interleaved=interleaved))
    tk.synchronize()
    x = rotate(rows.astype(np.float64), np.arange(n), f, amplitude, dim, interleaved)
    e = exps[0].cpu().numpy().astype(np.int64).reshape(-1, heads)
    top = np.abs(x).reshape(-1, block, heads, d).max((1, 3))
    border = exponent(top * (1 + 2.0**-23)) != exponent(top * (1 - 2.0**-23))
    assert np.array_equal(e[~border], exponent(top)[~border])
    up = np.repeat(2.0**e, block, 0)[..., None]
    got, nearest = VALUES[codes[0].cpu().numpy()].reshape(x.shape) * up, VALUES[encode(np.clip(x / up, -448, 448))] * up
    size = np.abs(rows).astype(np.float64)
    terms = np.zeros_like(x)
    terms[..., first] = terms[..., second] = size[..., first] + size[..., second]
    may = 2 * (2.0**-24 * np.abs(x) * (1 + 2.0**-20) + 2.0**-40 * terms)
    further = np.abs(got - x) - np.abs(nearest - x) - may
    assert np.all(further <= 0), ((further > 0).sum(), further.max())
