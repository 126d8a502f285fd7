"""The attention, rotary and append entry points without a GPU: what they refuse, through the C ABI (a call
whose arguments stand answers that the context is null), and what the kernels make of row numbers, lengths
and page numbers that leave the buffers."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT

OK, NULL, SHAPE, ALIGN, UNSUPPORTED, ARG = -1, -1, -2, -3, -5, -7  # OK: only the context is missing
AT = 1 << 20  # an address that no call here reads


def rows(at, n, heads, d, ld=None, hs=None):
    from telmo_amd import _lib

    ld, hs = ld or heads * d, hs or d
    return _lib.Rows(at, (n - 1) * ld + (heads - 1) * hs + d if n else 0, ld, hs)


def desc(**kw):
    """A sound description of 20 rows in two equal sequences, 4 heads of 64 over 2, in f16."""
    from telmo_amd import _lib

    a = _lib.AttentionDesc()
    a.type, a.heads, a.kv_heads, a.d, a.scale, a.left, a.right = 1, 4, 2, 64, 0.125, -1, -1
    a.batch, a.q_rows, a.k_rows = 2, 20, 20
    a.q, a.k, a.v, a.out = (rows(AT * (i + 1), 20, 4 if i in (0, 3) else 2, 64) for i in range(4))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def paged(**kw):
    a = desc(tables=AT * 9, tables_len=10, ldt=5, width=5, lengths=AT * 10, lengths_len=2, pages=7, page=16,
             k_page=16 * 128, v_page=16 * 128, k=rows(AT * 2, 7 * 16, 2, 64), v=rows(AT * 3, 7 * 16, 2, 64))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def call(a, which="tg_attention_device"):
    from telmo_amd import _lib

    return getattr(_lib.lib(), which)(None, a)


@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(type=3), ARG), (dict(type=4), ARG), (dict(type=9), ARG),
    (dict(d=0), UNSUPPORTED), (dict(d=4), UNSUPPORTED), (dict(d=60), UNSUPPORTED), (dict(d=264), UNSUPPORTED),
    (dict(kv_heads=0), UNSUPPORTED), (dict(kv_heads=3), SHAPE), (dict(heads=0), SHAPE), (dict(heads=1 << 20, kv_heads=1), SHAPE),
    (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(softcap=-1.0), ARG), (dict(softcap=float("nan")), ARG), (dict(softcap=float("inf")), ARG),
    (dict(batch=3), SHAPE), (dict(batch=70000), UNSUPPORTED), (dict(q_rows=1 << 31), UNSUPPORTED),
    (dict(k_rows=1 << 31), UNSUPPORTED), (dict(k_rows=21), SHAPE),
    (dict(q_starts=AT * 7, q_starts_len=2), SHAPE), (dict(q_starts=AT * 7, q_starts_len=3), OK),
    (dict(q_starts=AT * 7, q_starts_len=3, k_rows=18), SHAPE),
    (dict(q_starts=AT * 7, q_starts_len=3, k_starts=AT * 8, k_starts_len=3, k_rows=18), OK),
    (dict(q_starts=AT * 7, q_starts_len=3, k_starts=AT * 8, k_starts_len=2, k_rows=18), SHAPE),
    (dict(q=rows(0, 20, 4, 64)), NULL), (dict(out=rows(0, 20, 4, 64)), NULL), (dict(k=rows(0, 20, 2, 64)), NULL),
    (dict(q=rows(AT, 19, 4, 64)), SHAPE), (dict(v=rows(AT * 3, 19, 2, 64)), SHAPE), (dict(out=rows(AT * 4, 19, 4, 64)), SHAPE),
    (dict(q=rows(AT + 8, 20, 4, 64)), ALIGN), (dict(k=rows(AT * 2, 20, 2, 64, ld=132)), ALIGN),
    (dict(v=rows(AT * 3, 20, 2, 64, hs=68)), ALIGN), (dict(q=rows(AT, 20, 4, 64, ld=(1 << 62))), SHAPE),
    (dict(out=rows(AT * 4, 20, 4, 64, ld=128)), SHAPE), (dict(out=rows(AT * 4, 20, 4, 64, hs=32)), SHAPE),
    (dict(out=rows(AT * 4, 20, 4, 64, ld=64, hs=20 * 64)), OK),
    (dict(out=rows(AT, 20, 4, 64)), ARG), (dict(out=rows(AT * 2 + 512, 20, 4, 64)), ARG), (dict(out=rows(AT * 3 - 16, 20, 4, 64)), ARG),
    (dict(slopes=AT * 7, slopes_len=3), SHAPE), (dict(table=AT * 7, table_len=11, table_span=1), SHAPE),
    (dict(table=AT * 7, table_len=12, table_span=1), OK), (dict(table=AT * 7, table_len=12, table_span=1 << 62), SHAPE),
    (dict(rel=AT * 7, rel_len=1 << 20, ldrel=64, rel_span=3), UNSUPPORTED),
    (dict(rel_u=AT * 7, rel_u_len=256), ARG), (dict(rel_v=AT * 7, rel_v_len=256), ARG),
    (dict(prefix=AT * 7, prefix_len=1), SHAPE), (dict(prefix=AT * 7, prefix_len=2), OK),
    (dict(q_docs=AT * 7, q_docs_len=19), SHAPE), (dict(q_docs=AT * 7, q_docs_len=20), OK), (dict(k_docs=AT * 7, k_docs_len=20), ARG),
    (dict(q_docs=AT * 7, q_docs_len=20, k_docs=AT * 8, k_docs_len=19), SHAPE),
    (dict(workspace=AT * 7 + 8, workspace_len=64), ALIGN), (dict(tables=AT * 7), ARG), (dict(lengths=AT * 7), ARG),
    (dict(workspace=AT * 7, workspace_len=64), OK), (dict(workspace=AT - 48, workspace_len=64), ARG), (dict(workspace=AT * 2, workspace_len=64), ARG),
    (dict(workspace=AT * 3 + 4096, workspace_len=64), ARG), (dict(workspace=AT * 4 + 10224, workspace_len=64), ARG),
    (dict(table=AT * 7, table_len=1 << 40, table_span=1 << 30), SHAPE), (dict(table=AT * 7, table_len=1 << 40, table_span=(1 << 30) - 1), OK),
    (dict(q_rows=0, k_rows=0, q=rows(0, 0, 4, 64), out=rows(0, 0, 4, 64)), OK), (dict(k_rows=0, k=rows(0, 0, 2, 64), v=rows(0, 0, 2, 64)), OK)])
def test_attention(kw, code):
    assert call(desc(**kw)) == code


@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(rel_len=7 * 256 - 1), SHAPE), (dict(rel=AT * 7 + 4), ALIGN), (dict(ldrel=257, rel_len=1 << 20), ALIGN),
    (dict(rel_span=4), SHAPE), (dict(hsrel=0), OK), (dict(rel_u=AT * 8, rel_u_len=255), SHAPE),
    (dict(rel_u=AT * 8, rel_u_len=256, rel_v=AT * 9, rel_v_len=256), OK), (dict(rel_span=1 << 40), UNSUPPORTED),
    (dict(rel_span=1 << 30, rel_len=1 << 50), UNSUPPORTED), (dict(rel_span=(1 << 30) - 1, rel_len=1 << 50), OK)])
def test_position_rows(kw, code):
    a = desc(type=0, rel=AT * 7, rel_len=7 * 256, ldrel=256, hsrel=64, rel_span=3)
    for name, value in kw.items():
        setattr(a, name, value)
    assert call(a) == code


@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(tables=0), NULL), (dict(lengths=0), NULL), (dict(page=0), UNSUPPORTED), (dict(pages=1 << 31), UNSUPPORTED),
    (dict(width=1 << 31), UNSUPPORTED), (dict(tables_len=9), SHAPE), (dict(ldt=6), SHAPE), (dict(ldt=1 << 62), SHAPE),
    (dict(lengths_len=1), SHAPE), (dict(pages=8), SHAPE), (dict(k_page=16 * 128 - 4), ALIGN), (dict(v_page=1 << 62), SHAPE),
    (dict(q_docs=AT * 11, q_docs_len=20), ARG), (dict(k_starts=AT * 11, k_starts_len=3), ARG),
    (dict(k=rows(0, 7 * 16, 2, 64)), NULL), (dict(out=rows(AT * 2, 20, 4, 64)), ARG),
    (dict(pages=0, k=rows(0, 0, 2, 64), v=rows(0, 0, 2, 64)), OK)])
def test_paged(kw, code):
    assert call(paged(**kw), "tg_attention_paged_device") == code


def test_null_descriptions():
    from telmo_amd import _lib

    lib = _lib.lib()
    assert lib.tg_attention_device(None, None) == NULL and lib.tg_attention_paged_device(None, None) == NULL
    assert lib.tg_cache_append_device(None, None, 0, rows(AT, 1, 1, 8), rows(AT, 1, 1, 8), None) == NULL


def turned(**kw):
    from telmo_amd import _lib

    r = _lib.RotaryDesc(AT * 20, 32, 64, 0, 1.0)
    for name, value in kw.items():
        setattr(r, name, value)
    return r


@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(type=3), ARG), (dict(out_type=7), ARG), (dict(d=60), UNSUPPORTED), (dict(d=512), UNSUPPORTED),
    (dict(heads=1 << 17), UNSUPPORTED), (dict(rows=1 << 31), UNSUPPORTED), (dict(x=rows(AT, 9, 3, 64)), SHAPE),
    (dict(x=rows(0, 10, 3, 64)), NULL), (dict(x=rows(AT + 4, 10, 3, 64)), ALIGN), (dict(out=rows(AT * 2, 10, 3, 64, hs=16)), SHAPE),
    (dict(out=rows(AT, 10, 3, 64)), OK), (dict(out=rows(AT, 10, 3, 64), out_type=1), ARG), (dict(out=rows(AT + 256, 10, 3, 64)), ARG),
    (dict(positions=AT * 3, positions_len=9), SHAPE), (dict(positions=AT * 3, positions_len=10), OK),
    (dict(rotary=turned(dim=63)), SHAPE), (dict(rotary=turned(dim=66)), SHAPE), (dict(rotary=turned(turns=0)), NULL),
    (dict(rotary=turned(turns_len=31)), SHAPE), (dict(rotary=turned(amplitude=float("inf"))), ARG), (dict(rotary=turned(dim=0)), OK)])
def test_rotary(kw, code):
    from telmo_amd import _lib

    a = dict(type=0, x=rows(AT, 10, 3, 64), out_type=0, out=rows(AT * 2, 10, 3, 64), rows=10, heads=3, d=64, positions=None,
             positions_len=0, start=0, rotary=turned())
    a.update(kw)
    assert _lib.lib().tg_rotary_device(None, *a.values()) == code


@pytest.mark.parametrize("kw,new,code", [
    ({}, {}, OK), (dict(type=3), {}, ARG), ({}, dict(type=3), ARG), ({}, dict(k=rows(AT * 12, 19, 2, 64)), SHAPE),
    ({}, dict(v=rows(0, 20, 2, 64)), NULL), ({}, dict(k=rows(AT * 12 + 2, 20, 2, 64)), ALIGN), ({}, dict(k=rows(AT * 2, 20, 2, 64)), ARG),
    ({}, dict(v=rows(AT * 3 + 64, 20, 2, 64)), ARG), (dict(k_page=15 * 128), {}, SHAPE), (dict(v_page=0), {}, SHAPE),
    (dict(k=rows(AT * 2, 7 * 16, 2, 64, hs=32)), {}, SHAPE), (dict(tables=0), {}, NULL), (dict(pages=8), {}, SHAPE),
    (dict(v=rows(AT * 2, 7 * 16, 2, 64)), {}, SHAPE),
    ({}, dict(rotary=turned(dim=66)), SHAPE)])
def test_append(kw, new, code):
    from telmo_amd import _lib

    a = dict(type=0, k=rows(AT * 12, 20, 2, 64), v=rows(AT * 13, 20, 2, 64), rotary=turned())
    a.update(new)
    assert _lib.lib().tg_cache_append_device(None, paged(**kw), *a.values()) == code


def test_workspace_sizes_of_impossible_calls_are_zero():
    from telmo_amd import _lib

    size = _lib.lib().tg_attention_workspace_bytes
    for args in ((0, 4, 2, 64, 1, 100), (1, 0, 2, 64, 1, 100), (1, 4, 3, 64, 1, 100), (1, 4, 0, 64, 1, 100), (1, 4, 2, 0, 1, 100),
                 (1, 4, 2, 512, 1, 100), (1, 4, 2, 64, 0, 100), (1 << 40, 4, 2, 64, 1, 100), (1, 4, 2, 64, 1 << 20, 100)):
        assert size(*args) == 0, args


@pytest.fixture(scope="module")
def spans(tmp_path_factory):
    from telmo_amd import build

    exe = str(tmp_path_factory.mktemp("spans") / "spans")
    src = os.path.join(ROOT, "tests", "attention_spans.cpp")
    cmd = [build.HIPCC, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", src, "-o", exe]
    subprocess.run(cmd, check=True, capture_output=True)

    def run(text):
        return subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.splitlines()

    return run


def test_row_numbers_lengths_and_pages_are_cut_to_the_buffers(spans):
    rng = np.random.default_rng(4)
    wild = [-2**31, -5, -1, 0, 1, 3, 7, 19, 20, 21, 40, 2**31 - 1]
    for _ in range(200):
        batch, q_rows, k_rows = int(rng.integers(1, 5)), int(rng.integers(0, 21)), int(rng.integers(0, 41))
        width, page, pages = (int(x) for x in rng.integers(1, 6, 3))
        for paged_ in (0, 1):
            ints = rng.choice(wild, 2 * (batch + 1) + batch + batch * width)
            qs, ks = ints[:batch + 1], ints[batch + 1:2 * batch + 2]
            lens, table = ints[2 * batch + 2:3 * batch + 2], ints[3 * batch + 2:].reshape(batch, width)
            lines = spans(" ".join(str(x) for x in [batch, q_rows, k_rows, paged_, width, page, pages, *ints]))
            for b in range(batch):
                q0, nq, k0, nk, *held = (int(x) for x in lines[b].split())
                assert 0 <= q0 <= q0 + nq <= q_rows
                lo = min(max(qs[b], 0), q_rows)
                assert (q0, nq) == (lo, max(min(qs[b + 1], q_rows), lo) - lo)
                if paged_:
                    assert nk == min(max(lens[b], 0), width * page)
                    want = [int(table[b, j // page]) for j in range(nk)]
                    assert held == [p if 0 <= p < pages else -1 for p in want]
                else:
                    assert 0 <= k0 <= k0 + nk <= k_rows


def test_windows_are_cut_to_the_keys(spans):
    got = [tuple(int(x) for x in line.split()[1:]) for line in spans("") if line[0] == "w"]
    assert got == [(0, 10, 0), (3, 6, 0), (0, 0, 0), (10, 10, 10), (0, 10, 0), (0, 0, 3)]


def test_pages_are_found_by_multiplication(spans):
    assert [line for line in spans("") if line[0] == "d"] == ["d 0 1"]


def test_scalings_of_the_frequencies():
    from telmo_amd import rotary_frequencies

    f, a = rotary_frequencies(8, 100.0)
    assert np.allclose(f, [1.0, 100**-0.25, 0.1, 100**-0.75]) and a == 1.0
    g, _ = rotary_frequencies(8, 100.0, "linear", factor=4.0)
    assert np.allclose(g, f / 4)
    g, _ = rotary_frequencies(8, 100.0, "base", factor=4.0)
    assert g[0] == 1.0 and np.isclose(g[-1], f[-1] / 4) and np.all(np.diff(g / f) < 0)
    g, a = rotary_frequencies(128, 10000.0, "parts", factor=8.0, original=4096, slow=1.0, fast=32.0)
    f, _ = rotary_frequencies(128, 10000.0)
    turns = 4096 * f / (2 * np.pi)
    assert np.array_equal(g[turns >= 32], f[turns >= 32]) and np.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    assert np.all((g <= f) & (g >= f / 8 * (1 - 1e-15))) and np.isclose(a, 0.1 * np.log(8) + 1)
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.0), dict(dim=2, scaling="base"),
                dict(dim=8, scaling="parts"), dict(dim=8, scaling="other")):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_tensors_are_refused_by_place_shape_and_type():
    """The wrappers' own checks, on host tensors (get_device gives -1 for those)."""
    import torch

    from telmo_amd import attention

    class Kern:
        device = -1

    class Gpu:
        device = 0

    from telmo_amd import _lib

    into = _lib.Rows()
    x = torch.zeros(5, 3, 64)
    assert attention._rows(Kern, x, 3, 64, "x", into) == 5 and (into.len, into.ld, into.hs) == (960, 192, 64)
    assert attention._rows(Kern, x.view(5, 192), 3, 64, "x", into) == 5 and into.len == 960
    assert attention._rows(Kern, x[:1, :, :].expand(1, 3, 64), 3, 64, "x", into) == 1 and into.ld == 192
    assert attention._rows(Kern, x[:0], 3, 64, "x", into) == 0 and into.len == 0
    assert attention._rows(Kern, x.transpose(0, 1).contiguous().transpose(0, 1), 3, 64, "x", into) == 5
    assert (into.ld, into.hs, into.len) == (64, 320, 960)
    with pytest.raises(TypeError, match="context's GPU"):
        attention._rows(Gpu, x, 3, 64, "x", into)
    with pytest.raises(ValueError, match="must be"):
        attention._rows(Kern, x, 4, 64, "x", into)
    with pytest.raises(ValueError, match="contiguous"):
        attention._rows(Kern, torch.zeros(5, 64, 3).transpose(1, 2), 3, 64, "x", into)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        attention._type(x.double(), "x")
    with pytest.raises(TypeError, match="int32"):
        attention._array(Kern, torch.zeros(3, dtype=torch.int64), "int32", "n", 3)
    with pytest.raises(ValueError, match="hold 4"):
        attention._array(Kern, torch.zeros(3, dtype=torch.int32), "int32", "n", 4)
    with pytest.raises(ValueError, match="contiguous"):
        attention._array(Kern, torch.zeros(6, dtype=torch.int32)[::2], "int32", "n", 3)
    with pytest.raises(ValueError, match="left"):
        attention.Attention(Kern, 2, 64, left=-1)
    with pytest.raises(ValueError, match="table"):
        attention.Attention(Kern, 2, 64, table=torch.zeros(2, 4))
    k = torch.zeros(4, 16, 2, 64)
    cache = attention.PagedCache(Kern, k, k.clone())
    assert (cache._desc.k_page, cache._desc.k.ld, cache._desc.k.hs, cache._desc.k.len) == (2048, 128, 64, 8192)
    one = attention.PagedCache(Kern, k, k)._desc  # values that are the keys
    assert (one.k_page, one.v_page, one.v.ld, one.v.len) == (2048, 2048, 128, 8192)
    rotary = attention.Rotary.__new__(attention.Rotary)
    rotary._kernels = Gpu
    with pytest.raises(TypeError, match="another GPU"):
        cache.append(k[0], k[1], torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), rotary=rotary)
    with pytest.raises(ValueError, match="one type"):
        attention.PagedCache(Kern, k, k.half())
    att, q = attention.Attention(Kern, 4, 64, kv_heads=2), torch.zeros(3, 4, 64)
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="cache's heads"):
        att.paged(q.half(), cache, tables, lens, torch.zeros_like(q.half()))
    with pytest.raises(TypeError, match="tables"):
        att.paged(q, cache, tables.long(), lens, torch.zeros_like(q))
    with pytest.raises(ValueError, match="rows and type"):
        att.paged(q, cache, tables, lens, torch.zeros(2, 4, 64))
    with pytest.raises(ValueError, match="go with rel"):
        att.forward(q, q[:, :2], q[:, 2:], torch.zeros_like(q), rel_u=torch.zeros(4, 64))
    for call in (lambda: att.forward(q, q[:, :2], q[:, 2:], torch.zeros_like(q), longest=-1),
                 lambda: att.paged(q, cache, tables, lens, torch.zeros_like(q), longest=-1)):
        with pytest.raises(ValueError, match="longest"):
            call()


def test_descriptions_are_written_where_their_fields_lie():
    """The neighbouring fields that the wrappers write at once, read back by name."""
    from telmo_amd import _lib, attention

    a = _lib.AttentionDesc()
    attention._ROWS.pack_into(a, attention._AT_Q, 1, 2, 3, 4)
    attention._ROWS.pack_into(a, attention._AT_OUT, 5, 6, 7, 8)
    attention._CACHE.pack_into(a, attention._AT_K, *range(11, 19))
    attention._SEQS.pack_into(a, attention._AT_SEQS, *range(21, 29))
    attention._PAGES.pack_into(a, attention._AT_PAGES, *range(31, 41))
    rows = [(r.p, r.len, r.ld, r.hs) for r in (a.q, a.k, a.v, a.out)]
    assert rows == [(1, 2, 3, 4), (11, 12, 13, 14), (15, 16, 17, 18), (5, 6, 7, 8)]
    assert [getattr(a, n) for n in ("batch", "q_rows", "k_rows", "longest", "q_starts", "k_starts", "q_starts_len",
                                    "k_starts_len")] == list(range(21, 29))
    assert [getattr(a, n) for n in ("tables", "tables_len", "ldt", "width", "lengths", "lengths_len", "pages", "page",
                                    "k_page", "v_page")] == list(range(31, 41))
    assert a.prefix is None and a.workspace is None and a.q_docs is None
