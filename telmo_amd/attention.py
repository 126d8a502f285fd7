"""Attention on the device: the core between a layer's qkv product and its output product, over rows
(``Attention.forward``) or over a paged cache (``Attention.paged``), rotary positions (``Rotary``) and
the cache's writes (``PagedCache.append``).

``Attention.forward`` is what the layers leave to their ``attention`` argument: Parakeet's attention
with relative positions (src/parakeet.rs:1176-1282), Granite's inside blocks of frames
(src/granite.rs:962-1036), a text encoder's with windows and documents; ``Attention.for_layer`` makes
that argument. Rows are GPU tensors [rows, heads, d], or [rows, heads * d] with the heads side by
side, as views at any strides that are whole multiples of 16 bytes; everything is queued on the
context's stream and nothing is allocated but by ``Rotary``'s constructor. Tensors that a call or an object names
must live until the stream has reached the call, in a captured graph as long as that is replayed.
"""
from __future__ import annotations

import math
import struct
from typing import Optional

import numpy as np

from . import _lib
from .kernels import Kernels, Precision, _check

# Neighbouring fields of the descriptions, written at once: a call of a few microseconds is queued for every token.
_ROWS = struct.Struct("@PNNN")  # a tg_rows
_SEQS = struct.Struct("@NNNNPPNN")  # batch to k_starts_len of a tg_attention_desc
_PAGES = struct.Struct("@PNNNPNNNNN")  # its tables to v_page
_CACHE = struct.Struct("@PNNNPNNN")  # its k and v
_AT_SEQS, _AT_Q, _AT_K, _AT_V, _AT_OUT, _AT_PAGES = (getattr(_lib.AttentionDesc, name).offset for name in
                                                     ("batch", "q", "k", "v", "out", "tables"))

_FAR = 1 << 62  # further than any position, and within 64 bits: ctypes cuts what is past them

_TYPES = {}  # torch's types, made on first use
_INT32, _FLOAT32 = "int32", "float32"


def _types():
    if not _TYPES:
        import torch

        _TYPES.update({torch.float32: int(Precision.F32), torch.float16: int(Precision.F16),
                       torch.bfloat16: int(Precision.BF16), _INT32: torch.int32, _FLOAT32: torch.float32})
    return _TYPES


def _on(kern: Kernels, t, name: str) -> None:
    if t.get_device() != kern.device:
        raise TypeError(f"{name} must be a tensor on the context's GPU {kern.device}, not on {t.device}")


def _type(t, name: str) -> int:
    p = _types().get(t.dtype)
    if p is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return p


def _rows(kern: Kernels, t, heads: int, d: int, name: str, into, at: int = 0) -> int:
    """Writes t, [rows, heads, d] or [rows, heads * d], as a tg_rows at byte `at` of `into`; returns the rows."""
    _on(kern, t, name)
    shape, stride = t.shape, t.stride()
    if len(shape) == 3 and shape[1] == heads and shape[2] == d:
        hs = stride[1] if heads > 1 else d
    elif len(shape) == 2 and shape[1] == heads * d:
        hs = d
    else:
        raise ValueError(f"{name} must be [rows, {heads}, {d}] or [rows, {heads * d}], not {list(shape)}")
    if stride[-1] != 1 and d > 1:
        raise ValueError(f"{name}: a head's values must be contiguous")
    rows = shape[0]
    ld = stride[0] if rows > 1 else heads * d
    _ROWS.pack_into(into, at, t.data_ptr(), (rows - 1) * ld + (heads - 1) * hs + d if rows else 0, ld, hs)
    return rows


def _array(kern: Kernels, t, kind: str, name: str, n: int) -> int:
    """The address of at least n values of a contiguous GPU tensor of the kind."""
    if t.dtype != _types()[kind]:
        raise TypeError(f"{name} must be {kind}, not {t.dtype}")
    _on(kern, t, name)
    if not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{name} must be contiguous and hold {n} values")
    return t.data_ptr()


def _count(longest: Optional[int]) -> int:
    """The most rows of a sequence, 0 where any number."""
    if longest is None:
        return 0
    if longest < 0:
        raise ValueError("longest must not be negative")
    return longest


def _begun(desc):
    """A call's own copy of what an object's description holds already: calls from several threads may
    share the object."""
    return type(desc).from_buffer_copy(desc)


class PagedCache:
    """Keys and values of many sequences in pages: k and v are GPU tensors [pages, page, kv_heads, d] of
    one type (views at any strides that are whole multiples of 16 bytes). Key position j of sequence b is
    row j % page of page tables[b, j // page]. The tensors are held, not copied."""

    def __init__(self, kernels: Kernels, k, v):
        self._kernels = kernels
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [pages, page, kv_heads, d] of one type")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("a head's values must be contiguous")
        for t, name in ((k, "k"), (v, "v")):
            _on(kernels, t, name)
        self.k, self.v = k, v
        self.pages, self.page, self.kv_heads, self.d = k.shape
        self.type = _type(k, "k")
        a = self._desc = _lib.AttentionDesc()
        a.type, a.kv_heads, a.d = self.type, self.kv_heads, self.d
        self._k, self._k_page = self._strides(k)
        self._v, self._v_page = self._strides(v)
        a.pages, a.page, a.k_page, a.v_page = self.pages, self.page, self._k_page, self._v_page
        _CACHE.pack_into(a, _AT_K, *self._k, *self._v)

    def _strides(self, t):
        """t's tg_rows, and the values between its pages."""
        (pages, page, heads, d), (ps, ld, hs, _) = t.shape, t.stride()
        ld, hs = ld if page > 1 else heads * d, hs if heads > 1 else d
        ps = ps if pages > 1 else page * heads * d
        span = (pages - 1) * ps + (page - 1) * ld + (heads - 1) * hs + d if t.numel() else 0
        return (t.data_ptr(), span, ld, hs), ps

    def _name_seqs(self, a, rows: int, tables, lengths, q_starts, longest: Optional[int]) -> None:
        """The sequences of `rows` new rows in a: their tables, lengths and first rows."""
        kern = self._kernels
        if tables.dtype != _types()[_INT32] or tables.dim() != 2:
            raise TypeError("tables must be int32 [batch, entries]")
        _on(kern, tables, "tables")
        (batch, width), (ldt, one) = tables.shape, tables.stride()
        if width > 1 and one != 1:
            raise ValueError("a sequence's table must be contiguous")
        ldt = ldt if batch > 1 else width
        _PAGES.pack_into(a, _AT_PAGES, tables.data_ptr(), (batch - 1) * ldt + width if batch else 0, ldt, width,
                         _array(kern, lengths, _INT32, "lengths", batch), batch, self.pages, self.page, self._k_page,
                         self._v_page)
        at, n = (0, 0) if q_starts is None else (_array(kern, q_starts, _INT32, "q_starts", batch + 1), batch + 1)
        _SEQS.pack_into(a, _AT_SEQS, batch, rows, 0, _count(longest), at, 0, n, 0)

    def append(self, k, v, tables, lengths, q_starts=None, longest: Optional[int] = None,
               rotary: Optional["Rotary"] = None) -> None:
        """Writes new rows k and v ([rows, kv_heads, d], in their own type) into the pages
        (tg_cache_append_device): the n rows of sequence b, rows q_starts[b] to q_starts[b + 1] or an
        equal share, at key positions lengths[b] - n to lengths[b] - 1, keys rotated for those positions
        by `rotary`. longest: the most rows of one sequence (default: all)."""
        a, kern = _begun(self._desc), self._kernels
        if rotary is not None and rotary._kernels.device != kern.device:
            raise TypeError("the rotary positions live on another GPU")
        kn, vn = _lib.Rows(), _lib.Rows()
        rows = _rows(kern, k, self.kv_heads, self.d, "k", kn)
        if _rows(kern, v, self.kv_heads, self.d, "v", vn) != rows or v.dtype != k.dtype:
            raise ValueError("k and v must have the same rows and type")
        self._name_seqs(a, rows, tables, lengths, q_starts, longest)
        rc = _lib.lib().tg_cache_append_device(kern._ctx, a, _type(k, "k"), kn, vn,
                                               None if rotary is None else rotary._desc)
        if rc:
            _check(rc, kern._ctx)


class Attention:
    """One kind of attention layer: its heads, its scale and what is done to its scores.

    kv_heads: heads of k and v, shared by heads // kv_heads heads of q each (default: heads). scale: of
    the scores (default 1 / sqrt(head_dim)). softcap: scores become softcap tanh(s / softcap) (0: off).
    left, right: how many positions before and after its own a query is shown (None: all; right=0:
    causal). slopes: float32 GPU tensor [heads], the score's loss per position of distance. table:
    float32 GPU tensor [heads, 2 span + 1], added to the score by the distance key - query, distances
    past the span sharing the last value. Tensors are held, not copied."""

    def __init__(self, kernels: Kernels, heads: int, head_dim: int, kv_heads: Optional[int] = None,
                 scale: Optional[float] = None, softcap: float = 0.0, left: Optional[int] = None,
                 right: Optional[int] = None, slopes=None, table=None):
        self._kernels = kernels
        self.heads, self.head_dim = heads, head_dim
        self.kv_heads = heads if kv_heads is None else kv_heads
        for n, name in ((left, "left"), (right, "right")):
            if n is not None and n < 0:
                raise ValueError(f"{name} must not be negative (None: no limit)")
        a = self._desc = _lib.AttentionDesc()
        a.heads, a.kv_heads, a.d = heads, self.kv_heads, head_dim
        a.scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
        a.softcap = softcap
        a.left, a.right = (-1 if n is None else min(n, _FAR) for n in (left, right))
        if slopes is not None:
            a.slopes, a.slopes_len = _array(kernels, slopes, _FLOAT32, "slopes", heads), slopes.numel()
        if table is not None:
            if table.dim() != 2 or table.shape[0] != heads or table.shape[1] % 2 == 0:
                raise ValueError("table must be [heads, 2 span + 1]")
            a.table, a.table_len = _array(kernels, table, _FLOAT32, "table", table.numel()), table.numel()
            a.table_span = table.shape[1] // 2
        self._keep = (slopes, table)

    def workspace_bytes(self, rows: int, keys: int, batch: int = 1) -> int:
        """Bytes of workspace with which calls of `rows` query rows in `batch` sequences of up to `keys`
        keys split long sequences over the GPU (tg_attention_workspace_bytes). Over pages `keys` is what the tables
        hold, and their width decides the parts: for sequences far shorter, name a narrower view of the tables or a
        smaller workspace."""
        return _lib.lib().tg_attention_workspace_bytes(rows, self.heads, self.kv_heads, self.head_dim, batch, keys)

    def _fill(self, a, q, out, prefix, workspace) -> int:
        kern = self._kernels
        rows = _rows(kern, q, self.heads, self.head_dim, "q", a, _AT_Q)
        if _rows(kern, out, self.heads, self.head_dim, "out", a, _AT_OUT) != rows or out.dtype != q.dtype:
            raise ValueError("out must have q's rows and type")
        if prefix is not None:
            a.prefix, a.prefix_len = _array(kern, prefix, _INT32, "prefix", 1), prefix.numel()
        if workspace is not None:
            _on(kern, workspace, "workspace")
            if not workspace.is_contiguous():
                raise ValueError("workspace must be contiguous")
            a.workspace, a.workspace_len = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        return rows

    def forward(self, q, k, v, out, batch: int = 1, q_starts=None, k_starts=None, longest: Optional[int] = None,
                prefix=None, q_docs=None, k_docs=None, rel=None, rel_u=None, rel_v=None, workspace=None) -> None:
        """out = attention(q, k, v) (tg_attention_device). The rows are `batch` equal-length sequences
        stacked one after another, or sequence b's are rows starts[b] to starts[b + 1] (q_starts, int32
        GPU tensor; k_starts for other lengths of the keys). longest: the most query rows of a sequence
        (default: all); rows past it are left as they were. prefix: int32 GPU tensor [batch], the first
        keys of each sequence that all its queries are shown. q_docs, k_docs: int32 GPU tensors, a
        document's number for each row (negative: none); k_docs defaults to q_docs.

        rel: position rows [2 span + 1, heads * head_dim], or [2 span + 1, head_dim] for all heads alike,
        float32: row span + c adds (q + rel_v) rel to the product of keys at the distance c = key - query
        (distances past the span take the last row); rel_u and rel_v [heads, head_dim] are added to q in
        the two products. workspace: GPU tensor of workspace_bytes(...) bytes, or None."""
        a, kern = _begun(self._desc), self._kernels
        a.type = _type(q, "q")
        rows = self._fill(a, q, out, prefix, workspace)
        keys = _rows(kern, k, self.kv_heads, self.head_dim, "k", a, _AT_K)
        if _rows(kern, v, self.kv_heads, self.head_dim, "v", a, _AT_V) != keys:
            raise ValueError("k and v must have the same rows")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError("q, k and v must have one type")
        q_at = q_n = k_at = k_n = 0
        if q_starts is not None:
            q_at, q_n = _array(kern, q_starts, _INT32, "q_starts", 1), q_starts.numel()
            batch = q_n - 1
        if batch < 0:
            raise ValueError("batch must not be negative")
        if k_starts is not None:
            k_at, k_n = _array(kern, k_starts, _INT32, "k_starts", batch + 1), batch + 1
        _SEQS.pack_into(a, _AT_SEQS, batch, rows, keys, _count(longest), q_at, k_at, q_n, k_n)
        if q_docs is not None:
            a.q_docs, a.q_docs_len = _array(kern, q_docs, _INT32, "q_docs", rows), rows
        if k_docs is not None:
            a.k_docs, a.k_docs_len = _array(kern, k_docs, _INT32, "k_docs", keys), keys
        if rel is not None:
            self._fill_rel(a, rel, rel_u, rel_v)
        elif rel_u is not None or rel_v is not None:
            raise ValueError("rel_u and rel_v go with rel")
        rc = _lib.lib().tg_attention_device(kern._ctx, a)
        if rc:
            _check(rc, kern._ctx)

    def for_layer(self, out, rel=None, **options):
        """The `attention` argument of ConformerLayer.forward and GraniteBlock.forward: a function of a
        layer's qkv rows, and of its projected positions where it has them (rel else), that runs forward
        with these options into the first rows of out and returns those."""
        width, kv_width = self.heads * self.head_dim, self.kv_heads * self.head_dim

        def attention(qkv, positions=None):
            att = out[:qkv.shape[0]]
            q, k, v = qkv.split((width, kv_width, kv_width), dim=1)
            self.forward(q, k, v, att, rel=rel if positions is None else positions, **options)
            return att

        return attention

    def _fill_rel(self, a, rel, rel_u, rel_v) -> None:
        kern, wide = self._kernels, self.heads * self.head_dim
        if rel.dtype != _types()[_FLOAT32] or rel.dim() != 2 or rel.stride(1) != 1:
            raise TypeError("rel must be float32 rows")
        _on(kern, rel, "rel")
        count, width = rel.shape
        if width not in (wide, self.head_dim) or count % 2 == 0:
            raise ValueError(f"rel must be [2 span + 1, {wide}] or [2 span + 1, {self.head_dim}]")
        ld = rel.stride(0) if count > 1 else width
        a.rel, a.rel_len, a.ldrel = rel.data_ptr(), (count - 1) * ld + width, ld
        a.hsrel = self.head_dim if width == wide and self.heads > 1 else 0
        a.rel_span = count // 2
        if rel_u is not None:
            a.rel_u, a.rel_u_len = _array(kern, rel_u, _FLOAT32, "rel_u", wide), wide
        if rel_v is not None:
            a.rel_v, a.rel_v_len = _array(kern, rel_v, _FLOAT32, "rel_v", wide), wide

    def paged(self, q, cache: PagedCache, tables, lengths, out, q_starts=None, longest: Optional[int] = None,
              prefix=None, workspace=None) -> None:
        """out = attention of new rows over the cache (tg_attention_paged_device), which holds their own
        keys and values too: the n rows of sequence b, rows q_starts[b] to q_starts[b + 1] of q or an equal
        share, stand at the last n of its lengths[b] positions. tables: int32 GPU tensor [batch, entries];
        lengths: int32 GPU tensor [batch]. q, out and the cache have one type."""
        a, kern = _begun(self._desc), self._kernels
        if cache.kv_heads != self.kv_heads or cache.d != self.head_dim or cache.type != _type(q, "q"):
            raise ValueError("the cache's heads, head size and type must be the layer's")
        if cache._kernels.device != kern.device:
            raise TypeError("the cache lives on another GPU")
        rows = self._fill(a, q, out, prefix, workspace)
        a.type = cache.type
        _CACHE.pack_into(a, _AT_K, *cache._k, *cache._v)
        cache._name_seqs(a, rows, tables, lengths, q_starts, longest)
        rc = _lib.lib().tg_attention_paged_device(kern._ctx, a)
        if rc:
            _check(rc, kern._ctx)


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original: int = 0, slow: float = 1.0, fast: float = 32.0):
    """Radians per position of each of the dim / 2 pairs, in 64 bits, and the amplitude of the rotated
    values. f_i = base^(-2 i / dim), and for contexts `factor` times as long as the original:

    "linear"  f_i / factor: positions closer together
    "base"    a base larger by factor^(dim / (dim - 2)): the slowest pair turns factor times slower, the
              fastest as before
    "parts"   by how often a pair turns in the `original` context: past `fast` turns as before, below
              `slow` as "linear", between them in proportion; amplitude 0.1 ln(factor) + 1"""
    if dim < 2 or dim % 2:
        raise ValueError("dim must be even and at least 2")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    i = np.arange(dim // 2, dtype=np.float64)
    if scaling == "base":
        if dim == 2:
            raise ValueError("one pair has no slowest one: scaling by the base needs dim > 2")
        return (base * factor ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
    f = float(base) ** (-2.0 * i / dim)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":
        if original < 1 or not fast > slow:
            raise ValueError("scaling by parts needs the original context's length and fast > slow")
        keep = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    raise ValueError("scaling must be none, linear, base or parts")


class Rotary:
    """Rotary positions over the first dim values of each head: pairs (i, i + dim / 2), or (2 i, 2 i + 1)
    when interleaved, with the frequencies of rotary_frequencies. The object itself may go once its calls are queued."""

    def __init__(self, kernels: Kernels, dim: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", **options):
        import torch

        self._kernels = kernels
        self.dim, self.interleaved = dim, interleaved
        f, self.amplitude = rotary_frequencies(dim, base, scaling, **options)
        self.turns = kernels._turns.get(f.tobytes())
        if self.turns is None:
            turns = torch.from_numpy(f / (2.0 * math.pi)).to(f"cuda:{kernels.device}")
            # The upload runs on torch's current stream and the kernels on the context's: wait for it here.
            torch.cuda.current_stream(kernels.device).synchronize()
            # Queued kernels and captured graphs read them after this object is gone, and torch's allocator does not know
            # of them: each set of frequencies, at most 1 KB, stays as long as the context.
            self.turns = kernels._turns.setdefault(f.tobytes(), turns)
        self._desc = _lib.RotaryDesc(self.turns.data_ptr(), dim // 2, dim, int(bool(interleaved)), self.amplitude)

    def apply(self, x, out, positions=None, start: int = 0) -> None:
        """out = x with each head's first dim values rotated (tg_rotary_device): x and out GPU tensors
        [rows, heads, d], out in x's type or another one, or x itself. Row r stands at positions[r] (int32
        GPU tensor), or at start + r."""
        kern = self._kernels
        if x.dim() != 3 or out.shape != x.shape:
            raise ValueError("x and out must be [rows, heads, d]")
        rows, heads, d = x.shape
        if abs(start) > _FAR:
            raise ValueError("start is past 2^62")
        xr, orr = _lib.Rows(), _lib.Rows()
        _rows(kern, x, heads, d, "x", xr)
        _rows(kern, out, heads, d, "out", orr)
        p, n = (None, 0) if positions is None else (_array(kern, positions, _INT32, "positions", rows), rows)
        rc = _lib.lib().tg_rotary_device(kern._ctx, _type(x, "x"), xr, _type(out, "out"), orr, rows, heads, d,
                                         p, n, start, self._desc)
        if rc:
            _check(rc, kern._ctx)
