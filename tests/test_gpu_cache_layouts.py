"""Paged caches of any layout on an MI355X: what is appended to one and read from it is what a contiguous one gives."""
import itertools

import pytest

from test_gpu_attention import dtype, ints, say

pytestmark = pytest.mark.gpu

PAGES, PAGE, HEADS, D = 9, 7, 3, 64


def caches(type, layout):
    """Keys and values [pages, page, heads, d] in their layout, full of sevens, and the storage they lie in."""
    import torch

    axes = {"rows": (0, 1, 2, 3), "heads outermost": (2, 0, 1, 3), "rows outermost": (1, 0, 2, 3), "heads in pages": (0, 2, 1, 3)}
    if layout in axes:
        order = axes[layout]
        sizes = [(PAGES, PAGE, HEADS, D)[i] for i in order]
        stores = [torch.full(sizes, 7.0, dtype=dtype(type), device="cuda") for _ in "kv"]
        return [t.permute([order.index(i) for i in range(4)]) for t in stores], stores
    store = {"pages of both": (PAGES, 2, PAGE, HEADS, D), "rows of both": (PAGES, PAGE, 2, HEADS, D),
             "heads of both": (PAGES, PAGE, HEADS, 2, D)}[layout]
    both = torch.full(store, 7.0, dtype=dtype(type), device="cuda")
    return list(both.unbind(store.index(2))), [both]


@pytest.mark.parametrize("type,layout", itertools.product(("f32", "bf16"), (
    "heads outermost", "rows outermost", "heads in pages", "pages of both", "rows of both", "heads of both")))
def test_layouts(tk, type, layout):
    import torch

    import telmo_amd

    say("cache", type, layout)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    new = [torch.randn(34, HEADS, D, generator=g, device="cuda") for _ in "kv"]
    q = torch.randn(34, HEADS, D, generator=g, device="cuda").to(dtype(type))
    tables, lens, starts = ints([[4, 0, 8], [1, 6, 2]]), ints([21, 16]), ints([0, 20, 34])
    rotary, att = telmo_amd.Rotary(tk, D), telmo_amd.Attention(tk, HEADS, D, right=0)
    results = []
    for form in ("rows", layout):
        (k, v), stores = caches(type, form)
        cache, out = telmo_amd.PagedCache(tk, k, v), torch.zeros_like(q)
        cache.append(*new, tables, lens, q_starts=starts, rotary=rotary)
        att.paged(q, cache, tables, lens, out, q_starts=starts)
        one = torch.zeros_like(q[:2])
        att.paged(q[:2], cache, tables, lens, one)
        tk.synchronize()
        assert sum(int((s != 7.0).sum()) for s in stores) == 2 * 34 * HEADS * D
        results.append([x.clone() for x in (k, v, out, one)])
    for want, got in zip(*results):
        assert torch.equal(want.contiguous(), got.contiguous())
