"""Operators of a decode step on MI355X (gfx950): what follows the prefill.

The reference prefills a prompt and hands its caches to mlx-lm, which decodes
token by token (``fpv2/generate.py:97-130``).  Here the step's operators are
HIP kernels of the same library (``include/fpv2_decode.h``):

``decode_attention``   one new token per sequence over a paged or contiguous
                       KV cache, optionally with a window and sinks.

All of them run on the current stream of their tensors' device, whichever
device is current, allocate from torch's allocator only (so they can be
captured into a graph) and never synchronise.  None has a backward: tensors
that require a gradient are refused while gradients are recorded.
"""

from __future__ import annotations

import ctypes

import torch

from fpv2 import _lib
from fpv2.kernel import SUPPORTED_HEAD_DIMS

_HALF = (torch.float16, torch.bfloat16)


def _on_device(device: torch.device, call) -> None:
    """``call(stream)`` with ``device`` current."""
    stream = _lib.stream_ptr(device)
    if device.index == torch.cuda.current_device():
        call(stream)
    else:
        with torch.cuda.device(device):
            call(stream)


def _no_grad_needed(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the decode operators have no backward: call them under "
                                   "torch.no_grad() or detach their inputs")


def _count(value, name: str, least: int = 0) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or value < least:
        raise ValueError(f"{name} must be an integer of at least {least}")
    return value


def _row_aligned(t: torch.Tensor) -> bool:
    """16-byte aligned rows: what the kernels read in place."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1))


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor) -> None:
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.ndim != 4:
            raise ValueError(f"{name} must have shape [pages, KV heads, page size, head dim]")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if k_pages.dtype not in _HALF or v_pages.dtype != k_pages.dtype:
        raise ValueError("the caches must share float16 or bfloat16 dtype")
    if k_pages.shape[0] == 0 or k_pages.shape[2] == 0:
        raise ValueError("the caches must hold at least one row")


def decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor | None, lengths: torch.Tensor | int, *,
                     scale: float | None = None, window_tokens: int | None = None,
                     sink_tokens: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached keys.

    ``q`` ``[B, Hq, D]``; ``k_pages``/``v_pages`` ``[P, Hkv, page_size, D]`` with
    any page, head and row strides (``D`` contiguous, rows 16-byte aligned);
    ``page_table`` int32 ``[B, n]``: token ``t`` of sequence ``b`` is row
    ``t % page_size`` of page ``page_table[b, t // page_size]``, or ``None`` where
    sequence ``b``'s whole cache is page ``b`` (contiguous caches); ``lengths``
    int32 ``[B]``, or one integer for all: the keys of each sequence, the new
    token's among them.  With ``window_tokens`` only the last that many keys
    and the first ``sink_tokens`` are visible.  Returns ``[B, Hq, D]`` (``out``
    where given, any strides with ``D`` contiguous).

    Lengths and page ids are read on the device: they are clipped to what the
    table and the pages hold, and a sequence of length 0 gives zeros.  Rows
    behind a sequence's length are never used, whatever they hold.
    """
    if q.ndim != 3:
        raise ValueError("q must have shape [batch, query heads, head dim]")
    _pages(k_pages, v_pages)
    batch, heads, dim = q.shape
    pages, kv_heads, page_size, _ = k_pages.shape
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if dim not in SUPPORTED_HEAD_DIMS or k_pages.shape[3] != dim:
        raise ValueError(f"head dimension must be one of {SUPPORTED_HEAD_DIMS}, the caches' too")
    if q.dtype != k_pages.dtype:
        raise ValueError("q and the caches must share float16 or bfloat16 dtype")
    if not _row_aligned(k_pages) or not _row_aligned(v_pages):
        raise ValueError("the caches' rows must be contiguous and 16-byte aligned")
    tensors = [q, k_pages, v_pages]
    if page_table is not None:
        if page_table.ndim != 2 or page_table.shape[0] != batch or page_table.dtype != torch.int32:
            raise ValueError("page_table must be int32 [batch, pages of a sequence]")
        if page_table.shape[1] == 0 or page_table.stride(1) != 1 and page_table.shape[1] > 1:
            raise ValueError("page_table must have contiguous rows of at least one page")
        tensors.append(page_table)
    elif pages < batch:
        raise ValueError("without a page_table every sequence needs a page")
    uniform = 0
    if isinstance(lengths, torch.Tensor):
        if lengths.shape != (batch,) or lengths.dtype != torch.int32 or not lengths.is_contiguous():
            raise ValueError("lengths must be contiguous int32 [batch], or an integer")
        tensors.append(lengths)
    else:
        uniform, lengths = _count(lengths, "lengths"), None
    window = 0 if window_tokens is None else _count(window_tokens, "window_tokens", 1)
    _count(sink_tokens, "sink_tokens")
    if out is None:
        out = torch.empty((batch, heads, dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or dim > 1 and out.stride(2) != 1:
        raise ValueError("out must be [batch, query heads, head dim] of q's dtype with a "
                         "contiguous last dimension")
    else:
        tensors.append(out)
    _no_grad_needed(*tensors)
    device = _lib.require_device(*tensors)
    if not _row_aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if batch == 0:
        return out
    lib = _lib.load()
    p = _lib.DecodeParams(
        batch, heads, kv_heads, dim, pages, page_size,
        1 if page_table is None else page_table.shape[1],
        0 if page_table is None else page_table.stride(0), uniform, window, sink_tokens,
        dim ** -0.5 if scale is None else scale, *_strides(q), *_strides(k_pages),
        *_strides(v_pages), out.stride(0), out.stride(1))

    def call(stream):
        need = lib.fpv2_decode_attention_workspace_bytes(ctypes.byref(p))
        work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        _lib.check(lib.fpv2_decode_attention(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(page_table),
            _lib.ptr(lengths), out.data_ptr(), _lib.dtype_code(q.dtype), ctypes.byref(p),
            _lib.ptr(work), max(need, 0), stream), "decode_attention")

    _on_device(device, call)
    return out


def _strides(t: torch.Tensor):
    """Strides of all dimensions but the last; 0 where a dimension has one entry
    (torch leaves any value there)."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]
