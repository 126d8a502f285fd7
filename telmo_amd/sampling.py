"""Tokens drawn from logits on the device, where a greedy decode takes the largest (src/parakeet.rs:1412-1513).

Everything is queued on the context's stream and nothing is allocated; tensors that a call or an object names must live
until the stream has reached the call, in a captured graph as long as that is replayed.
"""
from __future__ import annotations

from . import _lib
from .kernels import _ROW_TYPES, Kernels, _check


def _rows_of(kern: Kernels, t, kind: str, name: str, rows: int) -> int:
    """The address of a contiguous GPU tensor of the kind with a value for each row."""
    if str(t.dtype) != "torch." + kind:
        raise TypeError(f"{name} must be {kind}, not {t.dtype}")
    if t.get_device() != kern.device:
        raise TypeError(f"{name} must be a tensor on the context's GPU {kern.device}, not on {t.device}")
    if not t.is_contiguous() or t.numel() < rows:
        raise ValueError(f"{name} must be contiguous and hold {rows} values")
    return t.data_ptr()


class Sampler:
    """How tokens are drawn (tg_sampling): with the tokens in the order of falling logits, the first top_k stay (0: all),
    of those the ones before which less than top_p of the probability lies, of those the ones at least min_p times as
    likely as the first, which always stays. temperature 0 takes the largest logit. Each is a number for all rows, or a
    GPU tensor with a value for each (int32 for top_k, float32 else); tensors are held, not copied."""

    def __init__(self, kernels: Kernels, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        self._kernels = kernels
        o = self._desc = _lib.Sampling(1.0, 0, 1.0, 0.0)
        self._keep = (temperature, top_k, top_p, min_p)
        for value, name, kind in zip(self._keep, ("temperature", "top_k", "top_p", "min_p"), ("float32", "int32", "float32", "float32")):
            if hasattr(value, "data_ptr"):
                setattr(o, name + "s", _rows_of(kernels, value, kind, name, 0))
                setattr(o, name + "s_len", value.numel())
            elif name == "top_k":
                if not 0 <= value < 1 << 31:
                    raise ValueError("top_k must not be negative")
                o.top_k = value
            else:
                setattr(o, name, value)

    def workspace_bytes(self, rows: int, n: int) -> int:
        """Bytes of workspace that a call of `rows` rows of n logits needs (0 for short rows)."""
        return _lib.lib().tg_sample_workspace_bytes(rows, n)

    def sample(self, logits, uniforms, tokens, probs=None, workspace=None) -> None:
        """Writes a token of each row of logits (tg_sample_device), [rows, n] of float32, float16 or bfloat16 at any row
        stride, into tokens (int32 [rows]), and its probability among those that stayed into probs (float32 [rows]).
        uniforms: float32 [rows], a random number from 0 up to 1 for each. workspace: a GPU tensor of
        workspace_bytes(rows, n) bytes."""
        kern = self._kernels
        kind = _ROW_TYPES.get(str(logits.dtype))
        if kind is None or logits.dim() != 2:
            raise TypeError(f"logits must be float32, float16 or bfloat16 [rows, n], not {logits.dtype}")
        if logits.get_device() != kern.device:
            raise TypeError(f"logits must be a tensor on the context's GPU {kern.device}, not on {logits.device}")
        rows, n = logits.shape
        if logits.stride(1) != 1 and n > 1:
            raise ValueError("a row's logits must be contiguous")
        ld = logits.stride(0) if rows > 1 else n
        space, space_len = None, 0
        if workspace is not None:
            if workspace.get_device() != kern.device or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on the context's GPU")
            space, space_len = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        rc = _lib.lib().tg_sample_device(kern._ctx, kind, logits.data_ptr(), (rows - 1) * ld + n if rows else 0, ld, rows, n,
                                         self._desc, _rows_of(kern, uniforms, "float32", "uniforms", rows), rows,
                                         _rows_of(kern, tokens, "int32", "tokens", rows), rows,
                                         None if probs is None else _rows_of(kern, probs, "float32", "probs", rows), rows,
                                         space, space_len)
        if rc:
            _check(rc, kern._ctx)
