"""Which layouts of a paged cache tg_cache_append_device writes, judged without a GPU: a call whose arguments
stand answers that the context is null."""
import itertools

import numpy as np
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


def places(at, steps, sizes, d):
    """The values that a cache at `at` takes."""
    i = np.indices(sizes).reshape(3, -1)
    return (at + (np.array(steps)[:, None] * i).sum(0)[:, None] + np.arange(d)).ravel()


def test_keys_and_values_that_share_memory():
    """Keys and values at random nested steps in one buffer against their values' places, one by one: none that
    share a value are written, and all are that do not and step alike."""
    rng = np.random.default_rng(6)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        sizes, d = tuple(int(x) for x in rng.integers(1, 4, 3)), 8 * int(rng.integers(1, 3))
        order = rng.permutation(3)
        steps, span = layout(order, sizes, d, 8 * rng.integers(0, 5, 3))
        other, other_span = (steps, span) if rng.random() < 0.7 else layout(rng.permutation(3), sizes, d, 8 * rng.integers(0, 5, 3))
        by = 8 * int(rng.integers(-span // 8 - 2, span // 8 + 3))
        shared = np.intersect1d(places(0, steps, sizes, d), places(by, other, sizes, d)).size > 0
        got = append((AT * 2, steps, span), (AT * 2 + 2 * by, other, other_span), sizes, d)
        if shared:
            assert got == SHAPE, (sizes, d, steps, other, by)
        elif steps == other:
            assert got == OK, (sizes, d, steps, by)
        seen[shared] += 1
    assert min(seen.values()) > 500


def test_keys_and_values_of_one_buffer():
    page = PAGE * HEADS * D
    # A page of keys, then one of values; the values with their heads outermost in the page.
    keys = [2 * page, HEADS * D, D]
    span = (PAGES - 1) * 2 * page + page
    assert append((AT * 2, keys, span), (AT * 2 + 2 * page, keys, span)) == OK
    assert append((AT * 2, keys, span), (AT * 2 + 2 * page, [2 * page, D, PAGE * D], span)) == OK
    assert append((AT * 2, keys, span), (AT * 2 + 2 * page - 16, keys, span)) == SHAPE
    assert append((AT * 2, keys, span), (AT * 2 + 2 * page - 16, [2 * page, D, PAGE * D], span)) == SHAPE
    # Values one page on from the keys, in the same pages.
    whole, span = [page, HEADS * D, D], PAGES * page
    assert append((AT * 2, whole, span), (AT * 2 + 2 * page, whole, span)) == SHAPE
    assert append((AT * 2, whole, span), (AT * 2, whole, span)) == SHAPE
    assert append((AT * 2, whole, span), (AT * 2 + 2 * span, whole, span)) == OK
