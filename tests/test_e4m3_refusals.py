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


def upload(L, n=200, k=300, values=AT, values_len=None, ldv=300, scales=AT * 2, n_scales=6, out=True, device=True):
    import ctypes

    handle = ctypes.c_void_p()
    f = L.tg_weights_e4m3_upload_device if device else L.tg_weights_e4m3_upload
    return f(None, values, 199 * ldv + k if values_len is None else values_len, ldv, scales, n_scales, n, k,
             ctypes.byref(handle) if out else None)


@pytest.mark.parametrize("device", (True, False))
@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(out=False), NULL), (dict(n=(1 << 24) + 1), UNSUPPORTED), (dict(k=(1 << 24) + 1), UNSUPPORTED), (dict(ldv=299), SHAPE),
    (dict(values_len=199 * 300 + 299), SHAPE), (dict(n_scales=5), SHAPE), (dict(values=0), NULL), (dict(scales=0), NULL),
    (dict(scales=AT + 2), ALIGN), (dict(n=201, ldv=1 << 60), SHAPE),
])
def test_uploads_of_e4m3_weights(kw, code, device):
    from telmo_amd import _lib

    assert upload(_lib.lib(), device=device, **kw) == code


def test_products_without_weights():
    """A product's other refusals need weights, which need a GPU (test_gpu_e4m3_refusals.py)."""
    from telmo_amd import _lib

    L = _lib.lib()
    assert L.tg_linear_e4m3_device(None, 0, AT, 100, 10, 10, None, 0, AT * 2, 100, 10, None, None, 0) == NULL
    L.tg_weights_e4m3_free(None)
    assert L.tg_weights_e4m3_n(None) == L.tg_weights_e4m3_k(None) == L.tg_weights_e4m3_bytes(None) == 0


@pytest.mark.parametrize("m,k,want", ((0, 100, 0), (16, 4096, 0), (17, 128, 2 * 2048 + 2 * 64 + 1024), (33, 640, 3 * 5 * 2048 + 2 * 3 * 64 + 1024),
                                      ((1 << 24) + 1, 128, 0), (128, (1 << 24) + 1, 0)))
def test_workspaces_of_products(m, k, want):
    from telmo_amd import _lib

    assert _lib.lib().tg_linear_e4m3_workspace_bytes(m, k) == want


def test_encoding_refuses_what_is_not_finite_and_wrong_lengths():
    import ctypes

    import numpy as np

    from telmo_amd import TelmoError, _lib, encode_e4m3

    with pytest.raises(TelmoError):
        encode_e4m3(np.array([1.0, np.nan], np.float32), 1, 2)
    with pytest.raises(TelmoError):
        encode_e4m3(np.array([1.0, -np.inf], np.float32), 2, 1)
    with pytest.raises(ValueError):
        encode_e4m3(np.zeros(5, np.float32), 2, 3)
    w, v, s = np.zeros(6, np.float32), np.zeros(6, np.uint8), np.zeros(1, np.float32)
    at = [x.ctypes.data_as(ctypes.c_void_p) for x in (w, v, s)]
    assert _lib.lib().tg_encode_e4m3(at[0], 2, 3, at[1], 5, at[2], 1) == ARG
    assert _lib.lib().tg_encode_e4m3(at[0], 2, 3, at[1], 6, at[2], 2) == ARG
    assert _lib.lib().tg_encode_e4m3(None, 2, 3, at[1], 6, at[2], 1) == NULL


def test_encoding_rounds_to_nearest():
    """Every value of a block, and points between and beside neighbours, against the definition."""
    import numpy as np

    from e4m3_oracle import VALUES, encode
    from telmo_amd import encode_e4m3

    grid = VALUES[:127]
    x = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2, (grid[1:] + grid[:-1]) / 2 * (1 + 2.0**-20), (grid[1:] + grid[:-1]) / 2 * (1 - 2.0**-20)])
    x = np.concatenate([x, -x]).astype(np.float32)
    codes, scales = encode_e4m3(x, 1, x.size)
    for b in range(scales.shape[1]):
        part = x[128 * b:128 * b + 128].astype(np.float64)
        assert np.array_equal(codes[0, 128 * b:128 * b + 128], encode(np.clip(part / float(scales[0, b]), -448, 448)))
    zeros, one = encode_e4m3(np.zeros(130, np.float32), 130, 1)
    assert not zeros.any() and np.all(one == 1.0)
