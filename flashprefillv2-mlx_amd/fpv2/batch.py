"""Operators of serving a batch on MI355X (gfx950), beside the decode step's.

The reference ends where one prompt is prefilled (``fpv2/generate.py:97-130``).
These go on with many sequences of it and with longer caches (HIP kernels of the
same library, ``include/fpv2_batch.h``):

``shared_prefix_attention``     one new token per sequence of a batch that continues
                                one prompt: the prompt's keys are read once for all.
``quantize_to_pages``           keys and values as 8-bit codes into a paged cache of
                                half the bytes,
``dequantize_pages``            back in order, for a prefill that goes on over them,
``quantized_decode_attention``  and one new token per sequence over the codes.
``token_logprobs``              log probabilities of given tokens, entropies and the
                                most likely alternatives.

They keep ``fpv2.decode``'s rules: the current stream of their tensors' device,
torch's allocator only (so they can be captured into a graph), no synchronisation,
no derivative.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple

import torch

from fpv2 import _lib
from fpv2.decode import (_HALF, MAX_VOCAB, _check_apart, _count, _device, _extent, _in_place, _index,
                         _on_device, _overlaps_itself, _page_strides, _pages, _row_strides,
                         _rows_meet, _rows_overlap, _share_memory)
from fpv2.kernel import SUPPORTED_HEAD_DIMS

MAX_SEQUENCES = 0xFFFF       # of an attention call
MAX_QUERY_HEADS = 0xFFFFFF   # of all its sequences together, after a shared prefix


def _table(page_table, rows: int | None, name: str):
    """A page table's width and row stride; ``rows`` ``None``: of one sequence, ``[n]``."""
    ndim, shape = (1, "[pages of the prefix]") if rows is None else (2, "[batch, pages of a sequence]")
    if (page_table.ndim != ndim or page_table.dtype != torch.int32
            or rows is not None and page_table.shape[0] != rows):
        raise ValueError(f"{name} must be int32 {shape}")
    width = page_table.shape[-1]
    if width == 0 or page_table.stride(-1) != 1 and width > 1:
        raise ValueError(f"{name} must have contiguous rows of at least one page")
    return width, page_table.stride(0) if rows is not None else 0


def _lengths(lengths, batch: int, keys: int):
    """Lengths in a tensor of ``batch``, or one number, clipped to ``keys``."""
    if isinstance(lengths, torch.Tensor):
        if lengths.shape != (batch,) or lengths.dtype != torch.int32 or not lengths.is_contiguous():
            raise ValueError("lengths must be contiguous int32 [batch], or an integer")
        return lengths, 0
    return None, min(_count(lengths, "lengths"), keys)


def _queries(q: torch.Tensor, kv_heads: int, page_dim: int):
    if q.ndim != 3:
        raise ValueError("q must have shape [batch, query heads, head dim]")
    batch, heads, dim = q.shape
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if dim not in SUPPORTED_HEAD_DIMS or page_dim != dim:
        raise ValueError(f"head dimension must be one of {SUPPORTED_HEAD_DIMS}, the caches' too")
    return batch, heads, dim


def _attention_out(out: torch.Tensor, q: torch.Tensor, operands: list) -> None:
    """``operands``: what the call reads, ``q`` first."""
    if (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or _overlaps_itself(out)):
        raise ValueError("out must be [batch, query heads, head dim] of q's dtype with a "
                         "contiguous last dimension and no overlap")
    _check_apart(out, *operands[_in_place(out, q):])


@lru_cache(maxsize=256)
def _shared_plan(index: int, own: tuple, *fields):
    """A call's parameters but for its integer lengths, and the bytes of workspace that it
    needs on device ``index`` (the current one)."""
    params = _lib.SharedPrefixParams(_lib.DecodeParams(*own), *fields)
    need = _lib.load().fpv2_shared_prefix_attention_workspace_bytes(ctypes.byref(params))
    return params, ctypes.byref(params), need


def shared_prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                            prefix_table: torch.Tensor | None, prefix_length: torch.Tensor | int,
                            k_pages: torch.Tensor, v_pages: torch.Tensor,
                            page_table: torch.Tensor | None, lengths: torch.Tensor | int, *,
                            scale: float | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over a prefix that all of them share and
    each one's own keys.

    ``q`` ``[B, Hq, D]``.  ``prefix_k``/``prefix_v`` ``[P, Hkv, page_size, D]`` hold the
    prefix: its token ``t`` is row ``t % page_size`` of page ``prefix_table[t //
    page_size]`` (int32 ``[n]``), or with ``None`` of page 0 (the cache of a
    ``ChunkedPrefill``: ``*cp.pages(), None, cp.length``); ``prefix_length`` is an integer or int32
    ``[1]``.  ``k_pages``, ``v_pages``, ``page_table`` and ``lengths`` are the sequences' own
    keys, the new tokens' among them, as ``decode_attention`` takes them; both may lie in one
    pool of pages.  Returns ``[B, Hq, D]`` (``out`` where given, any strides with ``D``
    contiguous; ``q`` itself, or apart from all operands): what ``decode_attention`` gives
    for sequences that hold the prefix and their own keys, reading the prefix once.

    Lengths and page ids are read on the device and clipped to what tables and pages
    hold.  Either part may be empty; a sequence without any key gives zeros.  Rows
    behind a length are never used, whatever they hold.
    """
    pages, kv_heads, page_size, page_dim = _pages(k_pages, v_pages)
    batch, heads, dim = _queries(q, kv_heads, page_dim)
    p_pages, p_heads, p_size, p_dim = _pages(prefix_k, prefix_v)
    if p_heads != kv_heads or p_dim != dim:
        raise ValueError("the prefix must have the KV heads and head dimension of the caches")
    if q.dtype != k_pages.dtype or prefix_k.dtype != q.dtype:
        raise ValueError("q and the caches must share float16 or bfloat16 dtype")
    page_strides = _page_strides(k_pages, v_pages)
    prefix_strides = _page_strides(prefix_k, prefix_v)
    tensors = [q, prefix_k, prefix_v, k_pages, v_pages]
    width, table_stride, p_width = 1, 0, 1
    if page_table is not None:
        width, table_stride = _table(page_table, batch, "page_table")
        tensors.append(page_table)
    elif pages < batch:
        raise ValueError("without a page_table every sequence needs a page")
    if prefix_table is not None:
        p_width, _ = _table(prefix_table, None, "prefix_table")
        tensors.append(prefix_table)
    # (numbers past the caches are all of them: none leaves the parameters' 64 bits)
    lengths, length = _lengths(lengths, batch, width * page_size)
    p_lengths, p_length = None, 0
    if isinstance(prefix_length, torch.Tensor):
        if prefix_length.shape != (1,) or prefix_length.dtype != torch.int32:
            raise ValueError("prefix_length must be int32 [1], or an integer")
        p_lengths = prefix_length
    else:
        p_length = min(_count(prefix_length, "prefix_length"), p_width * p_size)
    tensors += [t for t in (lengths, p_lengths) if t is not None]
    scale = dim ** -0.5 if scale is None else float(scale)
    if out is not None:
        _attention_out(out, q, tensors)
        tensors.append(out)
    index = _device(tensors)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    q_strides = _row_strides(q)
    if q_strides is None:
        q = q.clone(memory_format=torch.contiguous_format)
        q_strides = _row_strides(q)
    if batch == 0:
        return out
    lib = _lib.load()

    def call(stream):
        params, ref, need = _shared_plan(
            index, (batch, heads, kv_heads, dim, pages, page_size, width, table_stride, 0, 0, 0, scale,
                    *q_strides, *page_strides, out.stride(0), out.stride(1)),
            p_pages, p_size, p_width, 0, *prefix_strides)
        if lengths is None or p_lengths is None:
            params = _lib.SharedPrefixParams.from_buffer_copy(params)
            params.own.length, params.prefix_length = length, p_length
            ref = ctypes.byref(params)
        work = torch.empty(max(need, 0), dtype=torch.uint8, device=out.device)
        _lib.check(lib.fpv2_shared_prefix_attention(
            q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), _lib.ptr(prefix_table),
            _lib.ptr(p_lengths), k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(page_table),
            _lib.ptr(lengths), out.data_ptr(), _lib.dtype_code(q.dtype), ref, work.data_ptr(),
            max(need, 0), stream), "shared_prefix_attention")

    _on_device(index, call)
    return out


class _Codes(NamedTuple):
    """A cache of codes as the calls need it."""

    shape: tuple     # (P, Hkv, page_size, D)
    strides: tuple   # of k_codes' and v_codes' first three dimensions
    scales: tuple    # of k_scales and v_scales
    bytes: tuple     # from each tensor's first byte to behind its last
    overlap: bool    # whether rows share memory


@lru_cache(maxsize=256)
def _codes_layout(shape, k_strides, v_strides, ks_strides, vs_strides, *distances) -> _Codes:
    """Of codes ``shape`` and their scales, the latter three tensors ``distances`` bytes behind the
    first one."""
    if 0 in shape[:3]:
        raise ValueError("the caches must hold at least one row")
    if shape[3] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {SUPPORTED_HEAD_DIMS}")
    layouts = []  # (bytes of an element, shape, strides) of k_codes, v_codes, k_scales, v_scales
    for strides in (k_strides, v_strides):
        if strides[3] != 1 or any(s % 16 for s, n in zip(strides, shape[:3]) if n > 1):
            raise ValueError("the codes' rows must be contiguous and 16-byte aligned")
        layouts.append((1, shape, strides))
    layouts += [(4, (*shape[:3], 1), (*strides, 1)) for strides in (ks_strides, vs_strides)]
    overlap = any(_rows_overlap(n, s) for _, n, s in layouts)
    extents = tuple(size * _extent(n, s) for size, n, s in layouts)
    at = (0, *distances)
    for i, a in enumerate(layouts):
        for j, b in enumerate(layouts[:i]):
            if -extents[i] < at[i] - at[j] < extents[j]:
                overlap = overlap or _rows_meet(at[i] - at[j], a, b)
    codes = [s if n > 1 else 0 for strides in (k_strides, v_strides) for s, n in zip(strides, shape[:3])]
    return _Codes(shape, tuple(codes), (*ks_strides, *vs_strides), extents, overlap)


def _code_pages(k_codes, k_scales, v_codes, v_scales) -> _Codes:
    shape = k_codes.shape
    if (k_codes.dtype != torch.int8 or v_codes.dtype != torch.int8 or len(shape) != 4
            or v_codes.shape != shape or k_scales.dtype != torch.float32
            or v_scales.dtype != torch.float32 or k_scales.shape != shape[:3]
            or v_scales.shape != shape[:3]):
        for name, codes, scales in (("k", k_codes, k_scales), ("v", v_codes, v_scales)):
            if codes.ndim != 4 or codes.dtype != torch.int8:
                raise ValueError(f"{name}_codes must be int8 [pages, KV heads, page size, head dim]")
            if codes.shape != shape:
                raise ValueError("k_codes and v_codes must have the same shape")
            if scales.shape != shape[:3] or scales.dtype != torch.float32:
                raise ValueError(f"{name}_scales must be float32 [pages, KV heads, page size]")
    first, second = k_codes.data_ptr(), v_codes.data_ptr()
    if (first | second) & 15:
        raise ValueError("the codes' rows must be contiguous and 16-byte aligned")
    return _codes_layout(shape, k_codes.stride(), v_codes.stride(), k_scales.stride(), v_scales.stride(),
                         second - first, k_scales.data_ptr() - first, v_scales.data_ptr() - first)


@lru_cache(maxsize=256)
def _write_params(codes: _Codes, *fields):
    params = _lib.QuantizeParams(
        _lib.CodePages(codes.shape[1], codes.shape[3], codes.shape[0], codes.shape[2], *codes.strides,
                       *codes.scales), *fields)
    return params, ctypes.byref(params)


@lru_cache(maxsize=256)
def _read_params(codes: _Codes, *fields):
    params = _lib.DequantizeParams(
        _lib.CodePages(codes.shape[1], codes.shape[3], codes.shape[0], codes.shape[2], *codes.strides,
                       *codes.scales), *fields)
    return params, ctypes.byref(params)


def quantize_to_pages(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor | int,
                      k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                      v_scales: torch.Tensor) -> None:
    """Write tokens' keys and values into a paged cache of 8-bit codes.

    ``k``/``v`` ``[T, Hkv, D]`` in float16 or bfloat16, any strides with ``D`` contiguous (rows that
    are not 16-byte aligned are copied first).  ``k_codes``/``v_codes`` int8 ``[P, Hkv,
    page_size, D]`` and ``k_scales``/``v_scales`` float32 ``[P, Hkv, page_size]``, any page,
    head and row strides.  With ``a`` the greatest magnitude of a token's ``D`` values of a
    head, its codes are ``127 x / a`` rounded to whole numbers (half way: the even
    one) and its scale is ``a / 127``: a value is off by at most ``a / 254``.  They go to
    row ``slots[t] % page_size`` of page ``slots[t] // page_size``; ``slots`` as in
    ``rope_to_pages`` (int32 or int64 ``[T]``, or the first one; a token whose slot lies
    outside the pages is padding and not written; slots must be distinct).

    A row with an infinity or a NaN reads back as NaN, a row of zeros as zeros.
    """
    codes = _code_pages(k_codes, k_scales, v_codes, v_scales)
    _, kv_heads, _, dim = codes.shape
    shape, dtype = k.shape, k.dtype
    if (len(shape) != 3 or v.shape != shape or shape[1] != kv_heads or shape[2] != dim
            or dtype not in _HALF or v.dtype != dtype):
        for name, x in (("k", k), ("v", v)):
            if x.ndim != 3 or x.shape[1:] != (kv_heads, dim) or x.shape != shape:
                raise ValueError(f"{name} must be [tokens, KV heads, head dim] of the caches' geometry")
        raise ValueError("k and v must share float16 or bfloat16 dtype")
    tokens = shape[0]
    if codes.overlap:
        raise ValueError("the caches' rows overlap")
    slots, slot_bytes, first_slot = _index(slots, "slots", tokens)
    tensors = [k, v, k_codes, v_codes, k_scales, v_scales]
    if slots is not None:
        tensors.append(slots)
    # (what is read lies apart from what is written)
    firsts = [x.data_ptr() for x in tensors]
    _, _, a, b, c, d = firsts[:6]
    size = codes.bytes
    a_end, b_end, c_end, d_end = a + size[0], b + size[1], c + size[2], d + size[3]
    for x in tensors if slots is None else (k, v, slots):
        if x is k_codes:
            break
        first = x.data_ptr()
        end = first + x.element_size() * _extent(x.shape, x.stride())
        if ((first < a_end and a < end or first < b_end and b < end or first < c_end and c < end
                or first < d_end and d < end) and any(_share_memory(cache, x) for cache in tensors[2:6])):
            raise ValueError("the caches must not share memory with what the call reads")
    index = _device(tensors)
    if tokens == 0:
        return
    k_strides, v_strides = _row_strides(k), _row_strides(v)
    if k_strides is None:
        k = k.clone(memory_format=torch.contiguous_format)
        k_strides = _row_strides(k)
    if v_strides is None:
        v = v.clone(memory_format=torch.contiguous_format)
        v_strides = _row_strides(v)
    params, ref = _write_params(codes, tokens, slot_bytes, 0, *k_strides, *v_strides)
    if first_slot:
        params = _lib.QuantizeParams.from_buffer_copy(params)
        params.first_slot = first_slot
        ref = ctypes.byref(params)

    def call(stream):
        _lib.check(_lib.load().fpv2_quantize_to_pages(
            k.data_ptr(), v.data_ptr(), None if slots is None else firsts[6], firsts[2], firsts[4],
            firsts[3], firsts[5], _lib.dtype_code(dtype), ref, stream), "quantize_to_pages")

    _on_device(index, call)


def dequantize_pages(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                     v_scales: torch.Tensor, page_table: torch.Tensor | None,
                     lengths: torch.Tensor | int, *, tokens: int | None = None,
                     dtype: torch.dtype | None = None,
                     out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Sequences' keys and values ``[B, Hkv, tokens, D]`` from a cache of 8-bit codes.

    The cache as in ``quantize_to_pages``; ``page_table`` and ``lengths`` as in
    ``decode_attention`` (``None`` and an integer: sequence ``b`` is page ``b``, for all
    pages, or for ``out``'s batch).  ``tokens`` rows of each sequence are read (by default as many
    as its pages hold), code times scale rounded once to ``dtype`` (bfloat16 by default, or
    ``out``'s); sequences times heads are at most 65535.  Rows behind a sequence's length are zeros, or left as they are in ``out``, a pair
    of destinations with 16-byte aligned rows, apart from one another and from all operands:
    the caches of a ``ChunkedPrefill`` that goes on are ``out=cp.pages()``.
    """
    codes = _code_pages(k_codes, k_scales, v_codes, v_scales)
    pages, kv_heads, page_size, dim = codes.shape
    width, table_stride = 1, 0
    if page_table is not None:
        batch = page_table.shape[0] if page_table.ndim == 2 else -1
        width, table_stride = _table(page_table, batch, "page_table")
    elif isinstance(lengths, torch.Tensor):
        batch = lengths.numel()
    else:
        batch = pages if out is None else out[0].shape[0]
    if page_table is None and pages < batch:
        raise ValueError("without a page_table every sequence needs a page")
    lengths, length = _lengths(lengths, batch, width * page_size)
    tensors = [k_codes, k_scales, v_codes, v_scales]
    if page_table is not None:
        tensors.append(page_table)
    if lengths is not None:
        tensors.append(lengths)
    if out is None:
        tokens = width * page_size if tokens is None else _count(tokens, "tokens")
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in _HALF:
            raise ValueError("dtype must be float16 or bfloat16")
    else:
        tokens = out[0].shape[2] if tokens is None and out[0].ndim == 4 else tokens
        dtype = out[0].dtype if dtype is None else dtype
        for x in out:
            if (tokens is None or x.shape != (batch, kv_heads, tokens, dim) or x.dtype != dtype
                    or dtype not in _HALF or _row_strides(x) is None or _overlaps_itself(x)):
                raise ValueError("out must be a pair of [batch, KV heads, tokens, head dim] in float16 "
                                 "or bfloat16 with 16-byte aligned rows and no overlap")
            _check_apart(x, *tensors)
        _check_apart(out[0], out[1])
        tensors += out
    index = _device(tensors)
    zero_rest = out is None
    if out is None:
        shape, device = (batch, kv_heads, tokens, dim), k_codes.device
        out = (torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))
        strides = 2 * (kv_heads * tokens * dim, tokens * dim, dim)
    else:
        strides = (*_row_strides(out[0]), *_row_strides(out[1]))
    if batch == 0 or tokens == 0:
        return out
    params, ref = _read_params(codes, batch, width, table_stride, 0, tokens, zero_rest, *strides)
    if length:
        params = _lib.DequantizeParams.from_buffer_copy(params)
        params.length = length
        ref = ctypes.byref(params)

    def call(stream):
        _lib.check(_lib.load().fpv2_dequantize_pages(
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
            _lib.ptr(page_table), _lib.ptr(lengths), out[0].data_ptr(), out[1].data_ptr(),
            _lib.dtype_code(dtype), ref, stream), "dequantize_pages")

    _on_device(index, call)
    return out


@lru_cache(maxsize=256)
def _quantized_plan(index: int, attention: tuple, *fields):
    """A call's parameters but for an integer length, and the bytes of workspace that it
    needs on device ``index`` (the current one)."""
    params = _lib.QuantizedDecodeParams(_lib.DecodeParams(*attention), *fields)
    need = _lib.load().fpv2_quantized_decode_attention_workspace_bytes(ctypes.byref(params))
    return params, ctypes.byref(params), need


def quantized_decode_attention(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                               v_codes: torch.Tensor, v_scales: torch.Tensor,
                               page_table: torch.Tensor | None, lengths: torch.Tensor | int, *,
                               scale: float | None = None, window_tokens: int | None = None,
                               sink_tokens: int = 0,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """``decode_attention`` over a paged cache of 8-bit codes.

    The cache as in ``quantize_to_pages``, all else as in ``decode_attention``.  The
    codes are exact in the products; a query's values below 2^-14 of its greatest one are
    rounded to 2^-25 of it, the weights times the values' scales to float16 of 11 bits (products
    below 2^-111, where the greatest score's weight is 1, may count as 0).
    """
    codes = _code_pages(k_codes, k_scales, v_codes, v_scales)
    pages, kv_heads, page_size, page_dim = codes.shape
    batch, heads, dim = _queries(q, kv_heads, page_dim)
    if q.dtype not in _HALF:
        raise ValueError("q must be float16 or bfloat16")
    tensors = [q, k_codes, k_scales, v_codes, v_scales]
    width, table_stride = 1, 0
    if page_table is not None:
        width, table_stride = _table(page_table, batch, "page_table")
        tensors.append(page_table)
    elif pages < batch:
        raise ValueError("without a page_table every sequence needs a page")
    keys = width * page_size
    lengths, length = _lengths(lengths, batch, keys)
    if lengths is not None:
        tensors.append(lengths)
    window = 0 if window_tokens is None else min(_count(window_tokens, "window_tokens", 1), keys)
    sinks = min(_count(sink_tokens, "sink_tokens"), keys)
    scale = dim ** -0.5 if scale is None else float(scale)
    if out is not None:
        _attention_out(out, q, tensors)
        tensors.append(out)
    index = _device(tensors)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    q_strides = _row_strides(q)
    if q_strides is None:
        q = q.clone(memory_format=torch.contiguous_format)
        q_strides = _row_strides(q)
    if batch == 0:
        return out
    lib = _lib.load()

    def call(stream):
        params, ref, need = _quantized_plan(
            index, (batch, heads, kv_heads, dim, pages, page_size, width, table_stride, 0, window, sinks,
                    scale, *q_strides, *codes.strides, out.stride(0), out.stride(1)), *codes.scales)
        if lengths is None:
            params = _lib.QuantizedDecodeParams.from_buffer_copy(params)
            params.attention.length = length
            ref = ctypes.byref(params)
        work = torch.empty(need, dtype=torch.uint8, device=out.device) if need > 0 else None
        _lib.check(lib.fpv2_quantized_decode_attention(
            q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
            v_scales.data_ptr(), _lib.ptr(page_table), _lib.ptr(lengths), out.data_ptr(),
            _lib.dtype_code(q.dtype), ref, _lib.ptr(work), max(need, 0), stream),
            "quantized_decode_attention")

    _on_device(index, call)
    return out


MAX_TOP = 32  # FPV2_MAX_TOP


class TokenLogprobs(NamedTuple):
    """``token_logprobs``' result."""

    logprobs: torch.Tensor      # float32 [N]: of the given tokens
    entropy: torch.Tensor       # float32 [N]: of the rows' distributions, in nats
    top_tokens: torch.Tensor    # int64 [N, top]: the most likely tokens, in order
    top_logprobs: torch.Tensor  # float32 [N, top]


@lru_cache(maxsize=256)
def _logprobs_plan(index: int, *fields):
    """A call's parameters and the bytes of workspace that it needs on device ``index`` (the
    current one)."""
    ref = ctypes.byref(_lib.LogprobsParams(*fields))
    return ref, _lib.load().fpv2_token_logprobs_workspace_bytes(ref)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` ``[N]`` (int32 or int64), one for each row of ``logits``
    ``[N, V]``, the entropies of the rows' distributions and their ``top`` most likely
    tokens (at most 32), equal logits in the order of their tokens.

    ``logits`` float32, float16 or bfloat16, any strides (rows that are not contiguous
    are copied first).  Sums are in float32.  A token outside the vocabulary (padding, or
    ``sample_tokens``' -1) has -inf.  A NaN logit counts as -inf, magnitudes beyond 2^126 as
    2^126 in the probabilities (alternatives are in the order of the logits as given); a row of nothing but -inf gives -inf, an entropy of 0 and, as for every
    alternative that is missing because fewer tokens are above -inf, token -1 with -inf.
    """
    if logits.ndim != 2 or logits.dtype not in (torch.float32, *_HALF):
        raise ValueError("logits must be [rows, vocabulary] in float32, float16 or bfloat16")
    rows, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {MAX_VOCAB} tokens")
    if (tokens.shape != (rows,) or tokens.dtype not in (torch.int32, torch.int64)
            or not tokens.is_contiguous()):
        raise ValueError("tokens must be contiguous int32 or int64 [rows]")
    if _count(top, "top") > MAX_TOP:
        raise ValueError(f"top must be at most {MAX_TOP}")
    index = _device([logits, tokens])
    if vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    device = logits.device
    res = TokenLogprobs(*(torch.empty(rows, dtype=torch.float32, device=device) for _ in range(2)),
                        torch.empty((rows, top), dtype=torch.int64, device=device),
                        torch.empty((rows, top), dtype=torch.float32, device=device))
    if rows == 0:
        return res

    def call(stream):
        ref, need = _logprobs_plan(index, rows, vocab, logits.stride(0) if rows > 1 else 0,
                                   tokens.element_size(), top)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        _lib.check(_lib.load().fpv2_token_logprobs(
            logits.data_ptr(), tokens.data_ptr(), _lib.dtype_code(logits.dtype), ref,
            res.logprobs.data_ptr(), res.entropy.data_ptr(), res.top_tokens.data_ptr(),
            res.top_logprobs.data_ptr(), _lib.ptr(work), max(need, 0), stream), "token_logprobs")

    _on_device(index, call)
    return res
