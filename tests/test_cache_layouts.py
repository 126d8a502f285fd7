"""Which layouts of a paged cache tg_cache_append_device writes, judged without a GPU: a call whose arguments
stand answers that the context is null."""
import itertools

import pytest

from test_attention_refusals import AT, OK, SHAPE, paged, rows

PAGES, PAGE, HEADS, D = 7, 16, 2, 64  # of `paged`


def layout(order, sizes, d, gap=(0, 0, 0)):
    """The steps of pages, rows and heads stored with the axes in this order, the outermost first, gap[i] values
    behind each block of axis i, and the values from the first to behind the last."""
    steps, reach = [0, 0, 0], d
    for axis in reversed(order):
        steps[axis] = reach + gap[axis]
        reach = (sizes[axis] - 1) * steps[axis] + reach
    return steps, reach


def append(k, v, sizes=(PAGES, PAGE, HEADS), d=D):
    """What the call answers for a cache in f16 whose k and v are (address, steps, span)."""
    from telmo_amd import _lib

    a = paged(kv_heads=sizes[2], d=d, pages=sizes[0], page=sizes[1], k=_lib.Rows(k[0], k[2], k[1][1], k[1][2]),
              v=_lib.Rows(v[0], v[2], v[1][1], v[1][2]), k_page=k[1][0], v_page=v[1][0])
    new = [rows(AT * 12 + i, 20, sizes[2], d) for i in (0, AT)]
    return _lib.lib().tg_cache_append_device(None, a, 0, *new, None)


@pytest.mark.parametrize("order,gap", itertools.product(itertools.permutations(range(3)), ((0, 0, 0), (8, 24, 16))))
def test_axes_in_any_order(order, gap):
    steps, span = layout(order, (PAGES, PAGE, HEADS), D, gap)
    assert append((AT * 2, steps, span), (AT * 3, steps, span)) == OK
    for axis in range(3):  # a step that ends inside the blocks below it
        bad = list(steps)
        bad[axis] -= 8 + gap[axis]
        assert append((AT * 2, bad, span), (AT * 3, steps, span)) == SHAPE
        assert append((AT * 2, steps, span), (AT * 3, bad, span)) == SHAPE
