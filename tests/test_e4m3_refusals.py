"""The eight-bit entry points without a GPU: what they refuse, through the C ABI (a call whose arguments stand
answers that the context is null)."""
import pytest

from test_attention_refusals import ALIGN, ARG, AT, NULL, OK, SHAPE, UNSUPPORTED, paged, rows


def cached(**kw):
    """A sound description over seven pages of 16 e4m3 rows, and its exponents in blocks of 8 rows."""
    from telmo_amd import _lib

    c = _lib.CacheE4m3(AT * 20, AT * 21, 7 * 4, 7 * 4, 4, 4, 8)
    for name in [n for n in kw if n in dict(_lib.CacheE4m3._fields_) and n not in ("k_page", "v_page")]:
        setattr(c, name, kw.pop(name))
    c.k_page, c.v_page = kw.pop("k_epage", 4), kw.pop("v_epage", 4)
    return paged(**kw), c


CACHE = [
    ({}, OK), (dict(type=3), ARG), (dict(d=56), UNSUPPORTED), (dict(d=24), UNSUPPORTED), (dict(d=264), UNSUPPORTED),
    (dict(block=0), SHAPE), (dict(block=5), SHAPE), (dict(block=32), SHAPE), (dict(block=4), SHAPE),
    (dict(block=4, k_exps_len=56, v_exps_len=56, k_epage=8, v_epage=8), OK), (dict(block=16, k_epage=2, v_epage=2), OK),
    (dict(k_exps=0), NULL), (dict(v_exps=0), NULL), (dict(k_exps_len=27), SHAPE), (dict(v_exps_len=27), SHAPE),
    (dict(k_epage=5), SHAPE), (dict(k_epage=5, k_exps_len=34), OK), (dict(v_epage=1 << 62), SHAPE),
    (dict(k=rows(AT * 2 + 8, 7 * 16, 2, 64)), ALIGN), (dict(v=rows(AT * 3, 7 * 16, 2, 64, ld=136)), ALIGN),
    (dict(k=rows(AT * 2, 7 * 16, 2, 64, ld=144, hs=72)), ALIGN), (dict(k=rows(AT * 2, 7 * 16 - 1, 2, 64)), SHAPE),
    (dict(k_page=16 * 128 - 8), ALIGN), (dict(k=rows(0, 7 * 16, 2, 64)), NULL), (dict(tables=0), NULL), (dict(page=0), UNSUPPORTED),
    (dict(pages=0, k_exps=0, v_exps=0), OK),
]


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(out=rows(AT * 20 - 256, 20, 4, 64)), ARG), (dict(workspace=AT * 21 + 16, workspace_len=64), ARG),
    (dict(out=rows(AT * 2 + 7 * 2048, 20, 4, 64)), OK), (dict(out=rows(AT * 2 + 7 * 2048 - 16, 20, 4, 64)), ARG),
    (dict(heads=3), SHAPE), (dict(scale=0.0), ARG), (dict(q_docs=AT * 7, q_docs_len=20), ARG),
    (dict(rel=AT * 7, rel_len=1 << 20, ldrel=64, rel_span=3, type=0), UNSUPPORTED), (dict(type=0), OK), (dict(type=2), OK),
])
def test_attention_over_e4m3_pages(kw, code):
    from telmo_amd import _lib

    kw = dict(kw)
    if kw.get("type") == 0:  # f32 rows are twice as long
        kw.update(q=rows(AT, 20, 4, 64), out=rows(AT * 5, 20, 4, 64))
    a, c = cached(**kw)
    assert _lib.lib().tg_attention_paged_e4m3_device(None, a, c) == code


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(v=rows(AT * 2, 7 * 16, 2, 64)), SHAPE), (dict(k_exps=AT * 2 + 64), ARG), (dict(v_exps=AT * 20), SHAPE),
    (dict(v_exps=AT * 20 + 4, k_epage=8, v_epage=8, k_exps_len=56, v_exps_len=56), OK),
    (dict(v_exps=AT * 20 + 3, k_epage=8, v_epage=8, k_exps_len=56, v_exps_len=56), SHAPE),
    (dict(k_epage=3, v_epage=4), SHAPE), (dict(new_type=3), ARG), (dict(k_new=rows(AT * 30, 19, 2, 64)), SHAPE),
    (dict(k_new=rows(AT * 30 + 8, 20, 2, 64)), ALIGN), (dict(k_new=rows(AT * 3, 20, 2, 64)), ARG),
    (dict(k_new=rows(AT * 20 - 4096, 20, 2, 64)), ARG),
])
def test_appends_to_e4m3_pages(kw, code):
    from telmo_amd import _lib

    kw = dict(kw)
    new, k_new = kw.pop("new_type", 0), kw.pop("k_new", rows(AT * 30, 20, 2, 64))
    a, c = cached(**kw)
    assert _lib.lib().tg_cache_append_e4m3_device(None, a, c, new, k_new, rows(AT * 31, 20, 2, 64), None) == code


def test_null_caches():
    from telmo_amd import _lib

    a, c = cached()
    assert _lib.lib().tg_attention_paged_e4m3_device(None, a, None) == NULL
    assert _lib.lib().tg_attention_paged_e4m3_device(None, None, c) == NULL
    assert _lib.lib().tg_cache_append_e4m3_device(None, a, None, 0, rows(AT * 30, 20, 2, 64), rows(AT * 31, 20, 2, 64), None) == NULL
