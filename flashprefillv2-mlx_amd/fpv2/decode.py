"""Operators of a decode step on MI355X (gfx950): what follows the prefill.

The reference prefills a prompt and hands its caches to mlx-lm, which decodes
token by token (``fpv2/generate.py:97-130``).  Here the step's operators are
HIP kernels of the same library (``include/fpv2_decode.h``):

``decode_attention``   one new token per sequence over a paged or contiguous
                       KV cache, optionally with a window and sinks.
``rope_to_pages``      norms of the query and key heads, the position rotation
                       and the K/V write into a paged cache.
``quantized_linear``   rows times 4-bit weights with group scales and biases
                       (``quantize_weight`` / ``dequantize_weight`` convert).
``sample_tokens``      temperature, top-k, top-p and min-p from given random
                       numbers.

All of them run on the current stream of their tensors' device, whichever
device is current, allocate from torch's allocator only (so they can be
captured into a graph) and never synchronise.  None has a derivative: tensors
that require a gradient are refused while gradients are recorded, and ones with a
forward-mode tangent always.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from fpv2 import _lib
from fpv2.kernel import SUPPORTED_HEAD_DIMS

_HALF = (torch.float16, torch.bfloat16)


def _device(tensors) -> int:
    """The index of the one ROCm device that all tensors are on; raises where there is
    none, or where a gradient would be lost.  (These calls take microseconds on
    the device, so the checks are made in few steps.)"""
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the decode operators have no derivative: their inputs must not "
                           "carry tangents")
    index = tensors[0].get_device()
    if index >= 0:
        for t in tensors:
            if t.requires_grad or t.get_device() != index:
                break
        else:
            return index
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("the decode operators have no backward: call them under "
                           "torch.no_grad() or detach their inputs")
    _lib.require_device(*tensors)
    return index


def _on_device(index: int, call) -> None:
    """``call(stream)`` with device ``index`` current and its current stream."""
    if index == torch._C._cuda_getDevice():
        call(torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            call(torch._C._cuda_getCurrentRawStream(index))


def _count(value, name: str, least: int = 0) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or value < least:
        raise ValueError(f"{name} must be an integer of at least {least}")
    return value


def _row_strides(t: torch.Tensor):
    """The strides of all dimensions but the last (any multiple of 8 where a
    dimension has one entry), or ``None`` where the rows are not contiguous and
    16-byte aligned: what the kernels read in place."""
    if t.data_ptr() & 15:
        return None
    *strides, last = t.stride()
    if last != 1 and t.shape[-1] > 1:
        return None
    union = 0
    for s in strides:
        union |= s
    if union & 7:
        strides = [s if n > 1 else 0 for s, n in zip(strides, t.shape)]
        if any(s & 7 for s in strides):
            return None
    return strides


def _reaches(base: int, spans: list, low: int, high: int) -> bool:
    """Whether ``base`` and a whole number of strides of each of ``spans`` ``[(stride, least,
    most)]`` can add up to a number in ``(low, high)``.  (A search over the strides from the
    greatest on, cut off where the rest cannot reach; layouts that nest take a few
    steps, and one that takes thousands counts as reaching.)"""
    spans = sorted((x for x in spans if x[0] > 0), reverse=True)
    rest = [(0, 0)]
    for s, a, b in reversed(spans):
        rest.append((rest[-1][0] + s * a, rest[-1][1] + s * b))
    rest.reverse()  # of spans[i:]
    budget = 4096

    def search(i, at):
        nonlocal budget
        budget -= 1
        if budget < 0:
            return True
        if i == len(spans):
            return low < at < high
        s, a, b = spans[i]
        below, above = rest[i + 1]
        first = max(a, -((at + above - low - 1) // s))
        last = min(b, (high - 1 - at - below) // s)
        return any(search(i + 1, at + s * n) for n in range(first, last + 1))

    return search(0, base)


@lru_cache(maxsize=256)
def _rows_overlap(shape, strides) -> bool:
    """Whether two rows (of contiguous last dimensions) of a tensor share memory."""
    if 0 in shape:
        return False
    width = shape[-1]
    dims = sorted(((s, n) for n, s in zip(shape[:-1], strides) if n > 1), reverse=True)
    extent = width
    for s, n in reversed(dims):
        if s < extent:
            break
        extent += s * (n - 1)
    else:
        return False  # each dimension steps over all of the next one
    # two rows whose first difference (in this order) is in dimension i
    return any(_reaches(s, [(s, 0, n - 2)] + [(r, 1 - m, m - 1) for r, m in dims[i + 1:]], -width, width)
               for i, (s, n) in enumerate(dims))


def _overlaps_itself(t: torch.Tensor) -> bool:
    return not t.is_contiguous() and _rows_overlap(t.shape, t.stride())


@lru_cache(maxsize=256)
def _extent(shape, strides) -> int:
    """Elements from a tensor's first to behind its last."""
    return 0 if 0 in shape else 1 + sum(s * (n - 1) for s, n in zip(strides, shape))


@lru_cache(maxsize=256)
def _rows_meet(distance: int, *layouts) -> bool:
    """Whether two tensors ``(bytes of an element, shape, strides)`` have a byte in common, the
    first of which starts ``distance`` bytes behind the second."""
    spans: dict = {}
    widths = []
    for sign, (size, shape, strides) in zip((1, -1), layouts):
        dims = [(s * size, n) for s, n in zip(strides, shape) if n > 1]
        widths.append(dims.pop()[1] * size if dims and shape[-1] > 1 and strides[-1] == 1 else size)
        for s, n in dims:
            least, most = spans.get(s, (0, 0))
            spans[s] = (least, most + n - 1) if sign > 0 else (least - n + 1, most)
    return _reaches(distance, [(s, *x) for s, x in spans.items()], -widths[0], widths[1])


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one device have a byte in common."""
    distance = a.data_ptr() - b.data_ptr()
    size, other, layout, other_layout = a.element_size(), b.element_size(), a.stride(), b.stride()
    if (distance >= other * _extent(b.shape, other_layout)
            or -distance >= size * _extent(a.shape, layout)):
        return False
    if a.numel() == 0 or b.numel() == 0:
        return False
    return _rows_meet(distance, (size, a.shape, layout), (other, b.shape, other_layout))


def _in_place(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether ``out`` is ``t``, element for element."""
    return out.data_ptr() == t.data_ptr() and all(
        n == 1 or a == b for n, a, b in zip(out.shape, out.stride(), t.stride()))


def _check_apart(out: torch.Tensor, *operands) -> None:
    first = out.data_ptr()
    end = first + out.element_size() * _extent(out.shape, out.stride())
    for t in operands:
        at = t.data_ptr()
        if (at < end and first < at + t.element_size() * _extent(t.shape, t.stride())
                and _share_memory(out, t)):
            raise ValueError("out must not share memory with what the call reads or writes beside it")


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor):
    """The caches' shape and strides."""
    if k_pages.ndim != 4 or v_pages.ndim != 4:
        name = "v_pages" if k_pages.ndim == 4 else "k_pages"
        raise ValueError(f"{name} must have shape [pages, KV heads, page size, head dim]")
    shape = k_pages.shape
    if shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if k_pages.dtype not in _HALF or v_pages.dtype != k_pages.dtype:
        raise ValueError("the caches must share float16 or bfloat16 dtype")
    if shape[0] == 0 or shape[2] == 0:
        raise ValueError("the caches must hold at least one row")
    return shape


def _page_strides(k_pages: torch.Tensor, v_pages: torch.Tensor):
    a, b, c, last = k_pages.stride()
    d, e, f, other = v_pages.stride()
    if (last == 1 == other and not (a | b | c | d | e | f) & 7
            and not (k_pages.data_ptr() | v_pages.data_ptr()) & 15):
        return a, b, c, d, e, f
    k, v = _row_strides(k_pages), _row_strides(v_pages)
    if k is None or v is None:
        raise ValueError("the caches' rows must be contiguous and 16-byte aligned")
    return *k, *v


@lru_cache(maxsize=256)
def _page_layout(pages, heads, rows, dim, *strides):
    """Whether rows of a cache share memory, and the bytes that each of them spans."""
    shape = (pages, heads, rows, dim)
    k, v = (*strides[:3], 1), (*strides[3:], 1)
    return (_rows_overlap(shape, k) or _rows_overlap(shape, v), 2 * _extent(shape, k),
            2 * _extent(shape, v))


@lru_cache(maxsize=256)
def _decode_plan(index: int, *fields):
    """A call's parameters but for an integer length, which grows from token to token,
    and the bytes of workspace that it needs on device ``index`` (the current one)."""
    params = _lib.DecodeParams(*fields)
    need = _lib.load().fpv2_decode_attention_workspace_bytes(ctypes.byref(params))
    return params, ctypes.byref(params), need


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
    where given, any strides with ``D`` contiguous; ``q`` itself, or apart from all operands).

    Lengths and page ids are read on the device: they are clipped to what the
    table and the pages hold, and a sequence of length 0 gives zeros.  Rows
    behind a sequence's length are never used, whatever they hold.
    """
    if q.ndim != 3:
        raise ValueError("q must have shape [batch, query heads, head dim]")
    pages, kv_heads, page_size, page_dim = _pages(k_pages, v_pages)
    shape, dtype = q.shape, q.dtype
    batch, heads, dim = shape
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if dim not in SUPPORTED_HEAD_DIMS or page_dim != dim:
        raise ValueError(f"head dimension must be one of {SUPPORTED_HEAD_DIMS}, the caches' too")
    if dtype != k_pages.dtype:
        raise ValueError("q and the caches must share float16 or bfloat16 dtype")
    page_strides = _page_strides(k_pages, v_pages)
    tensors = [q, k_pages, v_pages]
    width, table_stride, table_ptr = 1, 0, None
    if page_table is not None:
        if page_table.ndim != 2 or page_table.shape[0] != batch or page_table.dtype != torch.int32:
            raise ValueError("page_table must be int32 [batch, pages of a sequence]")
        width = page_table.shape[1]
        table_stride, last = page_table.stride()
        if width == 0 or last != 1 and width > 1:
            raise ValueError("page_table must have contiguous rows of at least one page")
        table_ptr = page_table.data_ptr()
        tensors.append(page_table)
    elif pages < batch:
        raise ValueError("without a page_table every sequence needs a page")
    uniform, lengths_ptr = 0, None
    if isinstance(lengths, torch.Tensor):
        if lengths.shape != (batch,) or lengths.dtype != torch.int32 or not lengths.is_contiguous():
            raise ValueError("lengths must be contiguous int32 [batch], or an integer")
        lengths_ptr = lengths.data_ptr()
        tensors.append(lengths)
    else:
        uniform = _count(lengths, "lengths")
    # (numbers past the cache are all of it: none leaves the parameters' 64 bits)
    keys = width * page_size
    uniform = min(uniform, keys)
    window = 0 if window_tokens is None else min(_count(window_tokens, "window_tokens", 1), keys)
    sinks = min(_count(sink_tokens, "sink_tokens"), keys)
    # (a number, as it is part of what a plan is kept by)
    scale = dim ** -0.5 if scale is None else float(scale)
    if out is not None:
        if (out.shape != shape or out.dtype != dtype or out.stride(2) != 1
                or _overlaps_itself(out)):
            raise ValueError("out must be [batch, query heads, head dim] of q's dtype with a "
                             "contiguous last dimension and no overlap")
        _check_apart(out, *tensors[_in_place(out, q):3])
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
        params, ref, need = _decode_plan(
            index, batch, heads, kv_heads, dim, pages, page_size, width, table_stride, 0, window,
            sinks, scale, *q_strides, *page_strides, out.stride(0), out.stride(1))
        if lengths_ptr is None:
            params = _lib.DecodeParams.from_buffer_copy(params)
            params.length = uniform
            ref = ctypes.byref(params)
        work = torch.empty(need, dtype=torch.uint8, device=out.device) if need > 0 else None
        _lib.check(lib.fpv2_decode_attention(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table_ptr, lengths_ptr,
            out.data_ptr(), _lib.dtype_code(dtype), ref, _lib.ptr(work), max(need, 0), stream),
            "decode_attention")

    _on_device(index, call)
    return out


_rope_params = lru_cache(maxsize=256)(lambda *fields: _lib.RopePagesParams(*fields))


def _index(value, name: str, tokens: int):
    """Positions or slots: an integer tensor of one per token, or the first one."""
    if isinstance(value, torch.Tensor):
        if (value.shape != (tokens,) or value.dtype not in (torch.int32, torch.int64)
                or not value.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32 or int64 [tokens], or an integer")
        return value, value.element_size(), 0
    if _count(value, name) >= 1 << 62:
        raise ValueError(f"{name} must be below 2^62")
    return None, 0, value


def rope_to_pages(qkv: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                  cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | int,
                  slots: torch.Tensor | int, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                  query_heads: int, eps: float = 1e-6, interleaved: bool = False,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Norm and rotate the heads of fused projection rows; K and V go into pages.

    ``qkv`` ``[T, (Hq + 2 Hkv) D]`` holds each token's query, key and value heads.
    Query and key heads are RMS-normalised with ``q_weight``/``k_weight`` ``[D]``
    (``None``: not normalised) and rotated by row ``positions[t]`` of the float32
    tables ``cos``/``sin`` ``[positions, R]``: pairs ``(j, j + R)``, or ``(2j, 2j +
    1)`` with ``interleaved``, of the first ``2R`` dimensions.  Key and value heads
    are written to row ``slots[t] % page_size`` of page ``slots[t] // page_size``;
    a token whose slot lies outside the pages (say -1) is padding and is not
    written.  ``positions`` and ``slots`` are int32 or int64 ``[T]``, or an
    integer: the first token's, the others following.  Returns the query
    heads ``[T, Hq, D]`` (``out`` where given: the query heads of ``qkv`` themselves, or apart
    from all operands).

    Everything is computed in float32 and rounded once.  Positions are clipped
    to the tables.  Slots must be distinct: of two tokens with one slot,
    either's values may stay.
    """
    if qkv.ndim != 2 or qkv.dtype not in _HALF:
        raise ValueError("qkv must be [tokens, heads * head dim] in float16 or bfloat16")
    pages, kv_heads, page_size, dim = _pages(k_pages, v_pages)
    tokens = qkv.shape[0]
    _count(query_heads, "query_heads", 1)
    if k_pages.dtype != qkv.dtype:
        raise ValueError("qkv and the caches must share a dtype")
    if dim % 16 or not 0 < dim <= 512:
        raise ValueError("head dimension must be a multiple of 16 and at most 512")
    if kv_heads == 0 or qkv.shape[1] != (query_heads + 2 * kv_heads) * dim:
        raise ValueError("qkv rows must hold the query, key and value heads")
    page_strides = _page_strides(k_pages, v_pages)
    overlap, k_bytes, v_bytes = _page_layout(pages, kv_heads, page_size, dim, *page_strides)
    if overlap or (-v_bytes < v_pages.data_ptr() - k_pages.data_ptr() < k_bytes
                   and _share_memory(k_pages, v_pages)):
        raise ValueError("the caches' rows overlap")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and (t.shape != (dim,) or t.dtype != qkv.dtype or t.data_ptr() & 15
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous [head dim] of qkv's dtype, 16-byte aligned")
    if not (cos.ndim == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32
            and cos.is_contiguous() and sin.is_contiguous()
            and not (cos.data_ptr() | sin.data_ptr()) & 15):
        for name, t in (("cos", cos), ("sin", sin)):
            if (t.ndim != 2 or t.shape != cos.shape or t.dtype != torch.float32
                    or not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError(f"{name} must be a contiguous float32 [positions, R] table")
    rows, half = cos.shape
    if rows == 0 or half == 0 or half % 8 or 2 * half > dim:
        raise ValueError("cos and sin must have rows of a multiple of 8 angles, at most half the "
                         "head dimension")
    positions, position_bytes, first_position = _index(positions, "positions", tokens)
    slots, slot_bytes, first_slot = _index(slots, "slots", tokens)
    tensors = [qkv, k_pages, v_pages, cos, sin]
    for t in (q_weight, k_weight, positions, slots):
        if t is not None:
            tensors.append(t)
    if out is not None and (out.shape != (tokens, query_heads, dim) or out.dtype != qkv.dtype
                            or _row_strides(out) is None
                            or _overlaps_itself(out)):
        raise ValueError("out must be [tokens, query heads, head dim] of qkv's dtype with 16-byte "
                         "aligned rows")
    if out is not None:
        here = (out.data_ptr() == qkv.data_ptr() and (tokens <= 1 or out.stride(0) == qkv.stride(0))
                and (query_heads == 1 or out.stride(1) == dim))
        _check_apart(out, *tensors[here:3])
        tensors.append(out)
    index = _device(tensors)
    if out is None:
        out = torch.empty((tokens, query_heads, dim), dtype=qkv.dtype, device=qkv.device)
    qkv_strides = _row_strides(qkv)
    if qkv_strides is None:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        qkv_strides = _row_strides(qkv)
    if tokens == 0:
        return out
    lib = _lib.load()
    p = (_rope_params if position_bytes and slot_bytes else _lib.RopePagesParams)(
        tokens, query_heads, kv_heads, dim, half, rows, bool(interleaved), pages, page_size,
        position_bytes, slot_bytes, first_position, first_slot, *qkv_strides, *_row_strides(out),
        *page_strides, float(eps))

    def call(stream):
        _lib.check(lib.fpv2_rope_to_pages(
            qkv.data_ptr(), _lib.ptr(q_weight), _lib.ptr(k_weight), cos.data_ptr(), sin.data_ptr(),
            _lib.ptr(positions), _lib.ptr(slots), out.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), _lib.dtype_code(qkv.dtype), ctypes.byref(p), stream),
            "rope_to_pages")

    _on_device(index, call)
    return out


GROUP_SIZES = (32, 64, 128)


def quantize_weight(weight: torch.Tensor, *, group_size: int = 64):
    """4-bit weights of ``weight`` ``[N, K]``: ``(packed, scales, biases)``.

    Each group of ``group_size`` weights along ``K`` is cut into 15 equal steps
    from its least to its greatest: ``w ~ scale q + bias``.  ``packed`` is int32
    ``[N, K / 8]`` with weight ``k`` in bits ``4 (k % 8)`` of word ``k // 8``, ``scales``
    and ``biases`` ``[N, K / group_size]`` are of ``weight``'s dtype: the layout of
    MLX's affine quantization.  Runs on any device."""
    if weight.ndim != 2 or not weight.is_floating_point():
        raise ValueError("weight must be [out, in] of a floating type")
    if group_size not in GROUP_SIZES or weight.shape[1] % group_size or weight.shape[1] == 0:
        raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide the columns")
    n, k = weight.shape
    w = weight.detach().float().view(n, k // group_size, group_size)
    low, high = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
    # (a division by a number would be a product with its reciprocal on some
    # devices; the steps are counted with the scale and bias that will be stored)
    scales = ((high - low) / torch.full_like(high, 15)).to(weight.dtype)
    biases = low.to(weight.dtype)
    step = scales.float()
    q = ((w - biases.float()) / torch.where(step == 0, 1.0, step)).round().clamp(0, 15)
    q = q.to(torch.int32).view(n, k // 8, 8)
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=weight.device)
    packed = (q << shifts).sum(-1, dtype=torch.int32)
    return packed, scales[..., 0].contiguous(), biases[..., 0].contiguous()


def dequantize_weight(packed: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *,
                      dtype: torch.dtype | None = None) -> torch.Tensor:
    """``[N, K]`` weights of ``quantize_weight``'s result (float32 arithmetic,
    rounded once to ``dtype``, by default the scales')."""
    group = _group_size(packed, scales, biases)
    n = packed.shape[0]
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=packed.device)
    q = ((packed.view(torch.int32)[..., None] >> shifts) & 15).reshape(n, scales.shape[1], group)
    w = q * scales.float()[..., None] + biases.float()[..., None]
    return w.reshape(n, packed.shape[1] * 8).to(scales.dtype if dtype is None else dtype)


def _group_size(packed, scales, biases) -> int:
    if packed.ndim != 2 or packed.dtype not in (torch.int32, torch.uint32):
        raise ValueError("packed must be int32 [out, in / 8]")
    if scales.ndim != 2 or scales.shape != biases.shape or scales.shape[0] != packed.shape[0]:
        raise ValueError("scales and biases must be [out, groups]")
    groups = scales.shape[1]
    for group in GROUP_SIZES:
        if groups and groups * group == packed.shape[1] * 8:
            return group
    raise ValueError(f"the groups must be of one of {GROUP_SIZES} columns")


def quantized_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
                     biases: torch.Tensor, *, out_dtype: torch.dtype | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w.T`` with the 4-bit weights of ``quantize_weight``.

    ``x`` ``[..., K]`` in float16 or bfloat16, ``scales``/``biases`` of the same
    dtype; returns ``[..., N]`` in that dtype or, with ``out_dtype``, in float32.
    ``out``: optional ``[M, N]`` destination (``x`` ``[M, K]``) with contiguous
    rows, apart from all operands.  Products and sums are in float32 with the weights
    exact; ``x`` must be below 1e34 (an infinite value gives NaN).  Made for the few
    rows of a decode step: the weights are read once for every 32 rows, so a large
    prompt is better served by a product with ``dequantize_weight``'s result."""
    if x.ndim < 1 or x.dtype not in _HALF:
        raise ValueError("x must be [..., in] in float16 or bfloat16")
    group = _group_size(packed, scales, biases)
    n, k = packed.shape[0], packed.shape[1] * 8
    if x.shape[-1] != k:
        raise ValueError("x must have as many columns as the weights")
    if scales.dtype != x.dtype or biases.dtype != x.dtype:
        raise ValueError("x, scales and biases must share a dtype")
    kind = x.dtype if out_dtype is None else out_dtype
    if kind not in (x.dtype, torch.float32):
        raise ValueError("out_dtype must be x's dtype or float32")
    if packed.stride(1) != 1 or (n > 1 and packed.stride(0) % 4) or packed.data_ptr() % 16:
        raise ValueError("packed must have contiguous, 16-byte aligned rows")
    for name, t in (("scales", scales), ("biases", biases)):
        if t.shape[1] > 1 and t.stride(1) != 1 or n > 1 and t.stride(0) != scales.stride(0):
            raise ValueError(f"{name} must have contiguous rows, both with one row stride")
    rows = x if x.ndim == 2 else x.reshape(-1, k)
    m = rows.shape[0]
    tensors = [x, packed, scales, biases]
    out_stride = n
    if out is not None:
        if (x.ndim != 2 or out.shape != (m, n) or out.dtype != kind
                or n > 1 and out.stride(1) != 1 or m > 1 and out.stride(0) < n):
            raise ValueError("out must be [rows, out] of out_dtype with contiguous rows, x [rows, in]")
        out_stride = out.stride(0) if m > 1 else n
        _check_apart(out, x, packed, scales, biases)
        tensors.append(out)
    index = _device(tensors)
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=kind, device=x.device)
    strides = _row_strides(rows)
    if strides is None or m > 1 and strides[0] < k:
        rows = rows.clone(memory_format=torch.contiguous_format)
        strides = _row_strides(rows)
    if m == 0 or n == 0:
        return out
    lib = _lib.load()

    def call(stream):
        _lib.check(lib.fpv2_quantized_linear(
            rows.data_ptr(), packed.data_ptr(), scales.data_ptr(), biases.data_ptr(),
            out.data_ptr(), _lib.dtype_code(x.dtype), _lib.dtype_code(kind), m, n, k, group,
            strides[0] if m > 1 else k, packed.stride(0) if n > 1 else k // 8,
            scales.stride(0) if n > 1 else k // group, out_stride, stream), "quantized_linear")

    _on_device(index, call)
    return out


MAX_VOCAB = 1 << 19  # FPV2_MAX_VOCAB


def _setting(value, name: str, batch: int, dtype: torch.dtype, low, high):
    """A row setting: ``(tensor, number)``, the number where there is no tensor."""
    if isinstance(value, torch.Tensor):
        if value.shape != (batch,) or value.dtype != dtype or not value.is_contiguous():
            raise ValueError(f"{name} must be a number or contiguous "
                             f"{str(dtype).removeprefix('torch.')} [batch]")
        return value, 0
    if dtype == torch.int32:
        return None, _count(value, name)
    if isinstance(value, bool) or not isinstance(value, (int, float)) or not low <= value <= high:
        raise ValueError(f"{name} must be a number in [{low}, {high}] or a tensor")
    return None, value


def _settings(temperature, top_k, top_p, min_p, batch: int):
    inf = float("inf")
    return (_setting(temperature, "temperature", batch, torch.float32, 0, 1e30),
            _setting(top_k, "top_k", batch, torch.int32, 0, inf),
            _setting(top_p, "top_p", batch, torch.float32, 0, 1),
            _setting(min_p, "min_p", batch, torch.float32, 0, 1))


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *,
                  temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0,
                  top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
                  return_logprobs: bool = False):
    """One token per row of ``logits`` ``[B, V]`` by the row's number ``uniform[b]``.

    ``logits`` float32, float16 or bfloat16 with contiguous rows; ``uniform``
    float32 ``[B]`` in ``[0, 1)``.  Each setting is a number, or a tensor ``[B]``
    with one for each row (float32; ``top_k`` int32).  With the weights ``w_i =
    exp((logit_i - max) / temperature)`` and the tokens ordered by logit, equal
    ones by index, the kept ones are the first ``top_k`` (0: all), of these the
    ones whose weight before them is less than ``top_p`` of the weight of all of
    these, and of these the ones with ``w_i >= min_p``; the first always is.
    The token is the first one, in index order, whose running kept weight
    exceeds ``uniform[b]`` times all kept weight.  Temperature 0: the greatest
    logit, of equal ones the first.  (In tensors, temperatures of 0 or less and NaN
    are 0, ``top_k`` of 0 or less and ``top_p`` of 1 or more are no limit, and a
    negative ``min_p`` is 0, one above 1 is 1.)

    Returns int64 tokens ``[B]``, with ``return_logprobs`` also the float32 log of
    each token's share of the kept weight.  The result is the same in every
    call and batch.  A NaN logit counts as -inf; a row of nothing but -inf gives
    token -1 and -inf.
    """
    if logits.ndim != 2 or logits.dtype not in (torch.float32, *_HALF):
        raise ValueError("logits must be [batch, vocabulary] in float32, float16 or bfloat16")
    batch, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {MAX_VOCAB} tokens")
    if uniform.shape != (batch,) or uniform.dtype != torch.float32 or not uniform.is_contiguous():
        raise ValueError("uniform must be contiguous float32 [batch]")
    (t_rows, t), (k_rows, k), (p_rows, p), (m_rows, m) = _settings(
        temperature, top_k, top_p, min_p, batch)
    index = _device([logits, uniform, *(x for x in (t_rows, k_rows, p_rows, m_rows)
                                        if x is not None)])
    device = logits.device
    if vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    tokens = torch.empty(batch, dtype=torch.int64, device=device)
    logprobs = torch.empty(batch, dtype=torch.float32, device=device) if return_logprobs else None
    if batch > 0:
        lib = _lib.load()
        params = _lib.SampleParams(
            batch, vocab, logits.stride(0) if batch > 1 else 0, _lib.ptr(t_rows),
            _lib.ptr(k_rows), _lib.ptr(p_rows), _lib.ptr(m_rows), t, min(k, vocab), p, m)

        def call(stream):
            need = lib.fpv2_sample_tokens_workspace_bytes(ctypes.byref(params))
            work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
            _lib.check(lib.fpv2_sample_tokens(
                logits.data_ptr(), uniform.data_ptr(), _lib.dtype_code(logits.dtype),
                ctypes.byref(params), tokens.data_ptr(), _lib.ptr(logprobs), _lib.ptr(work),
                max(need, 0), stream), "sample_tokens")

        _on_device(index, call)
    return (tokens, logprobs) if return_logprobs else tokens
