"""The cache of 8-bit codes on the GPU: ``fpv2.quantize_to_pages`` and ``fpv2.dequantize_pages``
bit for bit against their definition, ``fpv2.quantized_decode_attention`` against the formula in
float64 over the values that the codes stand for."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from batch_cases import BF16, F16, attention, fill_pages, paged, quantized, rand, tolerance

pytestmark = pytest.mark.gpu


def _cache(cuda, pages, hkv, page, dim, code=99, scale=7.0):
    return [x for _ in "kv" for x in (
        torch.full((pages, hkv, page, dim), code, dtype=torch.int8, device=cuda),
        torch.full((pages, hkv, page), scale, device=cuda))]


def _rows(pages):
    """Rows in slot order ``[slots, Hkv, ...]`` on the CPU."""
    return pages.cpu().transpose(1, 2).flatten(0, 1)


def _same(a, b):
    return torch.equal(a, b) if not a.is_floating_point() else bool(
        ((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("tokens,hkv,page", [(1, 1, 1), (1, 8, 16), (37, 3, 48), (200, 2, 7), (5000, 1, 64)])
def test_write_and_read(cuda, dtype, dim, tokens, hkv, page):
    """Codes, scales and what they read back as; other rows stay as they were."""
    gen = torch.Generator().manual_seed(tokens + dim)
    k = torch.randn((tokens, hkv, dim), generator=gen) * (1 + 3 * (torch.arange(dim) % 29 == 0))
    k, v = k.to(dtype), rand(gen, tokens, hkv, dim, dtype=dtype) * 0.01
    table, total, slots, _ = paged(gen, [tokens], page)
    cache = _cache(cuda, total, hkv, page, dim)
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), slots[0].to(cuda), *cache)
    other = torch.ones(total * page, dtype=torch.bool)
    other[slots[0]] = False
    want = []
    for x, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        q, s = quantized(x)
        assert torch.equal(_rows(codes)[slots[0]], q) and torch.equal(_rows(scales)[slots[0]], s)
        assert bool((_rows(codes)[other] == 99).all()) and bool((_rows(scales)[other] == 7).all())
        want.append((q.float() * s[..., None]).to(dtype).transpose(0, 1))
        # within half a step of what was written, and the rounding of the result
        a = x.float().abs().amax(-1, keepdim=True)
        err = (want[-1].transpose(0, 1).float() - x.float()).abs()
        assert bool((err <= a / 254 + a * torch.finfo(dtype).eps).all())
    got = fpv2.dequantize_pages(*cache, table.to(cuda), tokens, tokens=tokens, dtype=dtype)
    assert all(torch.equal(g[0].cpu(), w) for g, w in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_every_quotient(cuda, dtype):
    """Every greatest value's leading digits with values of 8 digits at 8 exponents, and with
    its own halves; among them are values half way between two codes."""
    digits = 8 if dtype == BF16 else 11
    greatest = torch.arange(2 ** (digits - 1), 2 ** digits, dtype=torch.float64)[:, None]
    rows = []
    for shift in range(8):
        x = (torch.arange(1, 256, dtype=torch.float64) / 2.0 ** shift).expand(len(greatest), 255)
        rows.append(torch.cat([torch.where(x <= greatest, x, 0.0), greatest], 1))
    halves = greatest / 2.0 ** (torch.arange(256, dtype=torch.float64) % 20)
    rows.append(halves * (-1) ** torch.arange(256))
    x = (torch.cat(rows)[:, None] * 2.0 ** -6).to(dtype)
    codes, scales = quantized(x)
    cache = _cache(cuda, 1, 1, len(x), 256)
    fpv2.quantize_to_pages(x.to(cuda), -x.to(cuda), 0, *cache)
    assert torch.equal(cache[0].cpu()[0, 0], codes[:, 0]) and torch.equal(cache[2].cpu()[0, 0], -codes[:, 0])
    assert torch.equal(cache[1].cpu()[0, 0], scales[:, 0]) and torch.equal(cache[3].cpu()[0, 0], scales[:, 0])
    ratio = 127 * x.double() / x.double().abs().amax(-1, keepdim=True)
    assert int(((ratio - 0.5) == (ratio - 0.5).round()).sum()) >= len(greatest)  # half way


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_extreme_rows(cuda, dtype):
    """Zeros, the least and greatest numbers, infinities and NaN."""
    info = torch.finfo(dtype)
    least = info.smallest_normal * info.eps
    x = torch.zeros((9, 1, 64), dtype=dtype)
    x[1, 0, 3] = least
    x[2, 0, ::2], x[2, 0, 1::2] = 100 * least, -31 * least
    x[3, 0, :] = info.max
    x[4, 0, 5], x[4, 0, 6], x[4, 0, 7] = info.max, -info.max / 2, info.max / 254
    x[5, 0, 1], x[5, 0, 2] = math.inf, 1.0
    x[6, 0, 1], x[6, 0, 2] = -math.inf, 1.0
    x[7, 0, 63] = math.nan
    x[8, 0, 0] = -0.0
    codes, scales = quantized(x)
    codes[5:8], scales[5:8] = 0, math.nan
    cache = _cache(cuda, 1, 1, 9, 64)
    fpv2.quantize_to_pages(x.to(cuda), x.to(cuda), 0, *cache)
    for c, s in (cache[:2], cache[2:]):
        assert torch.equal(c.cpu()[0, 0], codes[:, 0]) and _same(s.cpu()[0, 0], scales[:, 0])
    k, v = fpv2.dequantize_pages(*cache, None, 9, dtype=dtype)
    want = (codes[:, 0].float() * scales).to(dtype)
    assert _same(k.cpu()[0, 0], want) and _same(v.cpu()[0, 0], want)
    assert torch.equal(k.cpu()[0, 0, 3], x[3, 0])


@pytest.mark.parametrize("slots", [torch.int32, torch.int64, int])
def test_slots(cuda, slots):
    """Types of slots, padding, and integers that run past the pages."""
    gen = torch.Generator().manual_seed(1)
    k, v = (rand(gen, 10, 2, 64, dtype=BF16) for _ in "kv")
    cache = _cache(cuda, 3, 2, 5, 64)
    if slots is int:
        at, arg = torch.arange(8, 18), 8  # 15 slots: the last three tokens have none
    else:
        at = torch.tensor([3, -1, 14, 15, 0, -2 ** 31, 2 ** 31 - 1, 7, 9, 12])
        arg = at.to(slots).to(cuda)
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), arg, *cache)
    live = (at >= 0) & (at < 15)
    for x, c, s in ((k, *cache[:2]), (v, *cache[2:])):
        codes, scales = torch.full((15, 2, 64), 99, dtype=torch.int8), torch.full((15, 2), 7.0)
        q = quantized(x)
        codes[at[live]], scales[at[live]] = q[0][live], q[1][live]
        assert torch.equal(_rows(c), codes) and torch.equal(_rows(s), scales)


def test_write_strides(cuda):
    """Keys and values as views of projection rows, of a cache with heads outside, off the
    16-byte grid; caches with the heads inside the rows and scales beside them."""
    gen = torch.Generator().manual_seed(2)
    k, v = (rand(gen, 21, 4, 96, dtype=F16) for _ in "kv")
    want = _cache(cuda, 4, 4, 8, 96)
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), 3, *want)
    qkv = torch.cat([k.flatten(1), v.flatten(1)], 1).to(cuda)
    outside = v.transpose(0, 1).contiguous().to(cuda).transpose(0, 1)
    odd = torch.empty(21 * 4 * 97, dtype=F16, device=cuda).view(21, 4, 97)[..., 1:]
    odd.copy_(v)
    for x, y in ((qkv[:, :384].unflatten(1, (4, 96)), qkv[:, 384:].unflatten(1, (4, 96))),
                 (k.to(cuda), outside), (k.to(cuda), odd)):
        codes = torch.full((4, 8, 2, 4, 112), 99, dtype=torch.int8, device=cuda)
        scales = torch.full((4, 8, 4, 2), 7.0, device=cuda)
        cache = [codes[:, :, 0, :, :96].transpose(1, 2), scales[..., 0].transpose(1, 2),
                 codes[:, :, 1, :, :96].transpose(1, 2), scales[..., 1].transpose(1, 2)]
        fpv2.quantize_to_pages(x, y, 3, *cache)
        assert all(torch.equal(a, b) for a, b in zip(cache, want))
        assert bool((codes[..., 96:] == 99).all())


def test_read_lengths_and_out(cuda):
    """Zeros behind the lengths, or what a destination held; page ids and lengths are clipped."""
    gen = torch.Generator().manual_seed(3)
    lengths = [0, 1, 30, 47]
    table, total, slots, _ = paged(gen, lengths, 8)
    cache = _cache(cuda, total, 2, 8, 128)
    k, v = (rand(gen, sum(lengths), 2, 128, dtype=BF16) for _ in "kv")
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), torch.cat(slots).to(cuda), *cache)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    got = fpv2.dequantize_pages(*cache, table.to(cuda), lens)
    assert got[0].shape == (4, 2, 48, 128) and got[0].dtype == BF16
    short = fpv2.dequantize_pages(*cache, table.to(cuda), lens, tokens=31, dtype=BF16)
    out = [torch.full((4, 50, 2, 136), 5.0, dtype=BF16, device=cuda)[..., :128].transpose(1, 2) for _ in "kv"]
    assert fpv2.dequantize_pages(*cache, table.to(cuda), lens, out=tuple(out))[0] is out[0]
    for x, g, s, o in zip((k, v), got, short, out):
        start = 0
        for b, n in enumerate(lengths):
            codes, scales = quantized(x[start:start + n])
            want = (codes.float() * scales[..., None]).to(BF16).transpose(0, 1)
            assert torch.equal(g[b, :, :n].cpu(), want) and not g[b, :, n:].any()
            assert torch.equal(s[b], g[b, :, :31])
            assert torch.equal(o[b, :, :n].cpu(), want) and bool((o[b, :, n:] == 5).all())
            start += n
    clipped = fpv2.dequantize_pages(*cache, torch.tensor([[-3], [10 ** 9]], dtype=torch.int32, device=cuda),
                                    torch.tensor([2 ** 31 - 1, -4], dtype=torch.int32, device=cuda))
    first = fpv2.dequantize_pages(*cache, None, 8)
    assert torch.equal(clipped[0][0], first[0][0]) and not clipped[0][1].any()
    assert first[0].shape[0] == total
    assert all(x.shape == (4, 2, 0, 128) for x in fpv2.dequantize_pages(*cache, table.to(cuda), lens, tokens=0))


def test_read_back_into_a_prefill(cuda):
    """A prompt's cache written as codes and read back into a prefill that goes on."""
    from fpv2 import ChunkedPrefill
    gen = torch.Generator().manual_seed(4)
    k, v = (rand(gen, 2, 300, 64, dtype=BF16).to(cuda) for _ in "kv")
    cache = _cache(cuda, 20, 2, 16, 64)
    fpv2.quantize_to_pages(k.transpose(0, 1), v.transpose(0, 1), 5, *cache)
    prefill = ChunkedPrefill(4, 2, 64, 400, device=cuda)
    prefill.reserve(300)
    pages = torch.arange(20, dtype=torch.int32, device=cuda)[None]
    whole = fpv2.dequantize_pages(*cache, pages, 305)
    rows = [torch.full((1, 2, 305, 64), 3.0, dtype=BF16, device=cuda) for _ in "kv"]
    fpv2.dequantize_pages(*cache, pages, 305, out=tuple(rows))
    for x, w, c in zip(rows, whole, prefill.pages()):
        assert torch.equal(x, w[:, :, :305])
        c[:, :, :300] = x[:, :, 5:]
    q = rand(gen, 4, 1, 64, dtype=BF16).to(cuda)
    got = prefill.decode(q)
    want = fpv2.decode_attention(q.transpose(0, 1), *(x[:, :, 5:305] for x in whole), None, 300)
    assert torch.equal(got[0].transpose(0, 1), want)


def _visible(n, window, sinks):
    t = torch.arange(n)
    return t if window is None else t[(t < sinks) | (t >= n - window)]


def _attend(cuda, seed, lengths, heads, hkv, dim, dtype, page, *, window=None, sinks=0, scale=None,
            spread=1.0, contiguous=False):
    """Codes of every value and scales over ``spread`` powers of two; unused rows hold NaN scales."""
    gen = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    codes = [torch.randint(-127, 128, (hkv, n, dim), generator=gen).to(torch.int8) for _ in "kv"]
    scales = [0.01 * 2 ** (spread * (torch.rand((hkv, n), generator=gen) - 0.5)) for _ in "kv"]
    q = rand(gen, len(lengths), heads, dim, dtype=dtype) * 2
    if contiguous:
        table, page, total = None, max(lengths) + 3, len(lengths)
        slots = [b * page + torch.arange(m) for b, m in enumerate(lengths)]
    else:
        table, total, slots, _ = paged(gen, lengths, page)
    at = torch.cat(slots)
    cache = []
    for c, s in zip(codes, scales):
        cache.append(fill_pages(total, hkv, page, dim, at, c, -77, torch.int8))
        cache.append(fill_pages(total, hkv, page, 1, at, s[..., None], math.nan, torch.float32)[..., 0])
    lens = torch.tensor(lengths, dtype=torch.int32)
    args = [x if x is None else x.to(cuda) for x in (q, *cache, table, lens)]
    got = fpv2.quantized_decode_attention(*args, window_tokens=window, sink_tokens=sinks, scale=scale)
    factor = dim ** -0.5 if scale is None else scale
    start = 0
    for b, m in enumerate(lengths):
        seen = start + _visible(m, window, sinks)
        k, v = (c[:, seen].double() * s[:, seen].double()[..., None] for c, s in zip(codes, scales))
        want, mass, size = attention(q[b], k, v, factor)
        # (float16 weights for both types; the queries' small values to 2^-25 of the greatest, and
        # log2 of a value's scale, of at most 2^5 + spread, in float32)
        least = 2.0 ** -24 * float(q[b].abs().max()) * factor * float(k.abs().sum(-1).max()) if len(seen) else 0
        tol = (tolerance(want, mass, size, len(seen), dim, dtype, F16)
               + (2 * least + 2.0 ** -22 * (32 + spread)) * mass)
        err = (got[b].cpu().double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        start += m
    return got, args


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,hkv", [(4, 1), (6, 6), (14, 2), (24, 1), (32, 2)])
def test_attention_ragged_pages(cuda, dtype, dim, heads, hkv):
    got, _ = _attend(cuda, dim + heads, [0, 1, 33, 129, 700], heads, hkv, dim, dtype, 16)
    assert not got[0].any()


@pytest.mark.parametrize("page", [1, 3, 32, 48, 1000])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (64, 5), (333, 130), (5000, 5000)])
def test_attention_pages_and_windows(cuda, page, window, sinks):
    _attend(cuda, page, [31, 32, 127, 128, 129, 455, 1301], 8, 2, 64, BF16, page, window=window,
            sinks=sinks, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("length", [1, 2, 129, 5000])
def test_attention_contiguous(cuda, dtype, length):
    got, args = _attend(cuda, length, [length] * 3, 8, 2, 128, dtype, 0, contiguous=True)
    assert torch.equal(fpv2.quantized_decode_attention(*args[:-1], length), got)


@pytest.mark.parametrize("spread", [0.0, 20.0, 60.0])
def test_attention_scales_of_many_sizes(cuda, spread):
    """Rows whose values are millions of times smaller than others'."""
    for dtype in (BF16, F16) if spread < 60 else (BF16,):
        scale = None if spread == 0 else 2.0 ** (-spread / 2)
        _attend(cuda, 5, [40, 3000], 8, 2, 128, dtype, 16, spread=spread, scale=scale)


def test_attention_many_sequences(cuda):
    gen = torch.Generator().manual_seed(6)
    lengths = torch.randint(0, 60, (620,), generator=gen).tolist()
    lengths[70], lengths[-1] = 4000, 0
    got, args = _attend(cuda, 6, lengths, 4, 1, 64, F16, 16)
    assert torch.equal(fpv2.quantized_decode_attention(*args), got)


@pytest.mark.parametrize("size", [1e-3, 1.0, 3e4])
def test_attention_sizes_of_queries(cuda, size):
    """Queries of any size and a few far smaller values among them."""
    gen = torch.Generator().manual_seed(7)
    for dtype in (BF16, F16):
        q = rand(gen, 1, 4, 64, dtype=torch.float32) * size * 0.3
        q[..., 3] *= 2.0 ** -9
        q[:, 2] = 0
        q = q.to(dtype)
        codes = torch.randint(-127, 128, (2, 1, 1, 500, 64), generator=gen).to(torch.int8)
        scales = torch.full((1, 1, 500), 0.01)
        got = fpv2.quantized_decode_attention(q.to(cuda), codes[0].to(cuda), scales.to(cuda),
                                              codes[1].to(cuda), scales.to(cuda), None, 500, scale=1 / size)
        k, v = (codes[i, 0].double() * scales[0].double()[..., None] for i in (0, 1))
        want, mass, score = attention(q[0], k, v, 1 / size)
        least = 2.0 ** -24 * float(q.abs().max()) / size * float(k.abs().sum(-1).max())
        tol = tolerance(want, mass, score, 500, 64, dtype, F16) + (2 * least + 2.0 ** -17) * mass
        assert bool(((got[0].cpu().double() - want).abs() <= tol).all())


GAPS = [0.0, 8.0, 12.0, 15.0, 16.875, 17.5, 20.0, 24.0]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("zero", ["codes", "small", "scale"])
@pytest.mark.parametrize("length,at", [(31, 1), (40_000, 0), (40_000, 25_000), (40_000, 39_999)])
def test_attention_keys_far_below_the_greatest(cuda, dtype, zero, length, at):
    """One key far above the rest whose value is nothing, by its codes or its scale, or small.

    Tolerance: a weight is off by half a step of float16, or of its least normal number, which
    is 2^-29 of the greatest product of weight and scale of its 32 keys: where that is the
    greatest key's, the 31 keys beside it are off by 2^-40 of it each.  Scores (three products
    of whole numbers below 2^14, times 2^-10) in float32 are off by less than 2^-14, the
    logarithms by 2^-21, and the exponentials by as much; sums of a lane by 2^-13."""
    gen = torch.Generator().manual_seed(length + at)
    dim = 64
    q = torch.zeros((1, len(GAPS), dim), dtype=dtype)
    q[0, :, 0], q[0, :, 5] = torch.tensor(GAPS), 1.0
    k = torch.zeros((length, dim), dtype=torch.int8)
    k[:, 5] = torch.randint(-32, 33, (length,), generator=gen).to(torch.int8)
    k[at, 0], k[at, 5] = 64, 32
    v = torch.randint(60, 128, (length, dim), generator=gen).to(torch.int8)
    ks, vs = torch.full((length,), 1 / 64), torch.full((length,), 8.0)
    if zero == "codes":
        v[at] = 0
    elif zero == "scale":
        vs[at] = 0
    else:
        v[at] = 1
        vs[at] = 2.0 ** -20
    args = [x.to(cuda) for x in (q, k[None, None], ks[None, None], v[None, None], vs[None, None])]
    got = fpv2.quantized_decode_attention(*args, None, length, scale=1.0)
    value = v.double() * vs.double()[:, None]
    w = torch.softmax(q[0].double() @ (k.double() * ks.double()[:, None]).T, 1)
    want = w @ value
    info = torch.finfo(dtype)
    top = (w * vs.double()).amax(1, keepdim=True)
    tol = (info.eps / 2 * want.abs().clamp(min=info.tiny) + 2.0 ** -11 * want.abs() + 2.0 ** -11 * want.abs()
           + 31 * 2.0 ** -40 * 128 * top)
    err = (got[0].cpu().double() - want).abs()
    assert bool((err <= tol).all()), [float(x) for x in (err / tol).amax(1)]


def test_attention_nan_rows(cuda):
    """A stored infinity or NaN that is visible is NaN, one that is not does nothing."""
    gen = torch.Generator().manual_seed(8)
    k, v = (rand(gen, 100, 1, 64, dtype=BF16) for _ in "kv")
    q = rand(gen, 1, 2, 64, dtype=BF16).to(cuda)
    clean = _cache(cuda, 1, 1, 100, 64)
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), 0, *clean)
    want = fpv2.quantized_decode_attention(q, *clean, None, 90)
    for x in (k, v):
        for bad in (math.inf, math.nan):
            row, x[95, 0, 7] = x[95].clone(), bad
            cache = _cache(cuda, 1, 1, 100, 64)
            fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), 0, *cache)
            assert torch.equal(fpv2.quantized_decode_attention(q, *cache, None, 90), want)
            assert bool(fpv2.quantized_decode_attention(q, *cache, None, 96).isnan().all())
            x[95] = row


def test_attention_strides_and_out(cuda):
    _, args = _attend(cuda, 9, [300, 17], 8, 2, 128, BF16, 32)
    q, kc, ks, vc, vs, table, lens = args
    want = fpv2.quantized_decode_attention(*args)
    pool = torch.zeros((kc.shape[0], 32, 2, 2, 144), dtype=torch.int8, device=cuda)[..., :128]
    pool[:, :, 0], pool[:, :, 1] = kc.transpose(1, 2), vc.transpose(1, 2)
    scales = torch.stack([ks, vs], -1).transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.full((2, 8, 131), 7.0, dtype=BF16, device=cuda)
    shifted = torch.empty(2 * 8 * 128 + 1, dtype=BF16, device=cuda)[1:].view(2, 8, 128)
    shifted.copy_(q)
    for queries in (q, shifted):
        got = fpv2.quantized_decode_attention(queries, pool[:, :, 0].transpose(1, 2), scales[..., 0],
                                              pool[:, :, 1].transpose(1, 2), scales[..., 1], table, lens,
                                              out=out[..., 2:130])
        assert got.data_ptr() == out[..., 2:130].data_ptr() and torch.equal(got, want)
    assert bool((out[..., :2] == 7).all()) and bool((out[..., 130:] == 7).all())
    assert fpv2.quantized_decode_attention(*args, out=q) is q and torch.equal(q, want)


def test_codes_past_32_bits(cuda):
    """A cache of more than 4 GiB of codes: written, attended and read at its end."""
    rows, dim, n = 34_000_000, 128, 70
    gen = torch.Generator().manual_seed(10)
    cache = _cache(cuda, 1, 1, rows, dim, code=0, scale=0.0)
    k, v = (rand(gen, n, 1, dim, dtype=BF16) for _ in "kv")
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), rows - n, *cache)
    q = rand(gen, 1, 4, dim, dtype=BF16)
    got = fpv2.quantized_decode_attention(q.to(cuda), *cache, None, rows, window_tokens=n)
    small = _cache(cuda, 1, 1, n, dim)
    fpv2.quantize_to_pages(k.to(cuda), v.to(cuda), 0, *small)
    assert torch.equal(got, fpv2.quantized_decode_attention(q.to(cuda), *small, None, n))
    assert torch.equal(cache[0][0, 0, -n:], small[0][0, 0]) and not cache[0][0, 0, -n - 1].any()
    whole = fpv2.dequantize_pages(*cache, None, rows)
    want = fpv2.dequantize_pages(*small, None, n)
    assert torch.equal(whole[0][:, :, -n:], want[0]) and torch.equal(whole[1][:, :, -n:], want[1])
    assert not whole[0][:, :, -n - 1].any()


def test_graph_of_a_step(cuda):
    """The write, the attention and the read in one graph, with slots, tables and lengths that
    change between its replays; eager work between them."""
    gen = torch.Generator().manual_seed(11)
    table, total, slots, _ = paged(gen, [90, 40, 70], 16)
    cache = _cache(cuda, total, 2, 16, 64, code=1, scale=0.02)
    k, v = (rand(gen, 3, 2, 64, dtype=BF16).to(cuda) for _ in "kv")
    q = rand(gen, 3, 8, 64, dtype=BF16).to(cuda)
    table, lens = table.to(cuda), torch.tensor([10, 20, 30], dtype=torch.int32, device=cuda)
    at = torch.tensor([int(s[n - 1]) for s, n in zip(slots, (10, 20, 30))], device=cuda)

    def step(cache):
        fpv2.quantize_to_pages(k, v, at, *cache)
        return (fpv2.quantized_decode_attention(q, *cache, table, lens),
                *fpv2.dequantize_pages(*cache, table, lens))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step([x.clone() for x in cache])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache)
    mirror = [x.clone() for x in cache]
    for i in range(4):
        for x in (k, v, q):
            x.mul_(-1.1)
        lens.add_(1)
        at.copy_(torch.tensor([int(s[n + i]) for s, n in zip(slots, (10, 20, 30))]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(mirror)):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(cache, mirror))


def test_run_on_the_current_stream(cuda):
    gen = torch.Generator().manual_seed(12)
    k, v = (rand(gen, 500, 2, 64, dtype=BF16).to(cuda) for _ in "kv")
    q = rand(gen, 1, 8, 64, dtype=BF16).to(cuda)

    def run(k):
        cache = _cache(cuda, 1, 2, 500, 64)
        fpv2.quantize_to_pages(k, v, 0, *cache)
        return [fpv2.quantized_decode_attention(q, *cache, None, 500), *fpv2.dequantize_pages(*cache, None, 500)]

    want = run(k)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(k)
        torch.cuda._sleep(20_000_000)
        late.copy_(k)
        got = run(late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
