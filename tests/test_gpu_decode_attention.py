"""``fpv2.decode_attention`` against the formula in float64 on the CPU.

Tolerance, per element: the weights are rounded once to the storage type before
the product with V (half a step of sum_t w_t |v_t|) and the result once (half a
step of |o|); a float32 score is off by at most (D + 8) 2^-24 scale sum |q k|,
which scales its weight by as much, and sums of n float32 terms by n 2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _rand(gen, *shape, dtype):
    return torch.randn(shape, generator=gen).to(dtype)


def _visible(n, window, sinks):
    return [t for t in range(n) if window is None or t < sinks or t >= n - window]


def _reference(q, k, v, table, lengths, scale, window, sinks):
    """float64 result and tolerance; q, k, v on the CPU."""
    batch, heads, dim = q.shape
    page, hkv = k.shape[2], k.shape[1]
    group = heads // hkv
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros((batch, heads, dim), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(batch):
        t = torch.tensor(_visible(int(lengths[b]), window, sinks), dtype=torch.long)
        if not len(t):
            continue
        pages = torch.full_like(t, b) if table is None else table[b].long()[t // page]
        for h in range(hkv):
            rows = slice(h * group, (h + 1) * group)
            kk, vv = k[pages, h, t % page].double(), v[pages, h, t % page].double()
            s = q[b, rows].double() @ kk.T * scale
            size = (q[b, rows].double().abs() @ kk.abs().T * abs(scale)).amax(1, keepdim=True)
            w = torch.softmax(s, 1)
            out[b, rows] = w @ vv
            mass = w @ vv.abs()
            tol[b, rows] = (half * (mass + out[b, rows].abs())
                            + (2 * (dim + 8) * size + 2 * len(t) + 64) * 2.0 ** -24 * mass)
    return out, tol


def _check(cuda, q, k, v, table, lengths, *, scale=None, window=None, sinks=0, **kwargs):
    dev = [x if x is None else x.to(cuda) for x in (q, k, v, table)]
    got = fpv2.decode_attention(*dev, torch.as_tensor(lengths, dtype=torch.int32).to(cuda),
                                scale=scale, window_tokens=window, sink_tokens=sinks, **kwargs)
    want, tol = _reference(q, k, v, table, lengths, q.shape[-1] ** -0.5 if scale is None else scale,
                           window, sinks)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())
    return got


def _paged(gen, lengths, hkv, page, dim, dtype, fill=math.nan, spare=2):
    """Pages in random order; rows behind the lengths and spare pages hold ``fill``."""
    counts = [-(-n // page) for n in lengths]
    width, total = max(1, *counts), sum(counts) + spare
    perm = torch.randperm(total, generator=gen)
    k = torch.full((total, hkv, page, dim), fill, dtype=dtype)
    v = torch.full_like(k, fill)
    table = torch.full((len(lengths), width), int(perm[-1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            rows = min(page, n - i * page)
            table[b, i] = perm[at]
            k[perm[at], :, :rows] = _rand(gen, hkv, rows, dim, dtype=dtype)
            v[perm[at], :, :rows] = _rand(gen, hkv, rows, dim, dtype=dtype)
            at += 1
    return k, v, table


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,hkv", [(4, 1), (6, 6), (14, 2), (24, 1), (80, 2), (32, 2)])
def test_ragged_pages(cuda, dtype, dim, heads, hkv):
    gen = torch.Generator().manual_seed(dim + heads)
    lengths = [0, 1, 33, 129, 700]
    k, v, table = _paged(gen, lengths, hkv, 16, dim, dtype)
    q = _rand(gen, len(lengths), heads, dim, dtype=dtype) * 2
    got = _check(cuda, q, k, v, table, lengths)
    assert not got[0].any()


@pytest.mark.parametrize("heads,hkv,dim", [(8, 8, 64), (24, 1, 96), (12, 4, 128)])
@pytest.mark.parametrize("longest", [1, 40, 400])
def test_more_items_than_workgroups(cuda, heads, hkv, dim, longest):
    """Hundreds of short sequences: a workgroup has several, and one in two at most."""
    gen = torch.Generator().manual_seed(heads + longest)
    batch = 1200 // hkv + 7 if hkv > 1 else 611
    lengths = torch.randint(0, longest + 1, (batch,), generator=gen).tolist()
    lengths[3], lengths[-1] = 5 * longest, longest
    k, v, table = _paged(gen, lengths, hkv, 16, dim, BF16)
    q = _rand(gen, batch, heads, dim, dtype=BF16) * 2
    _check(cuda, q, k, v, table, lengths)
    _check(cuda, q, k, v, table, lengths, window=30, sinks=3)


@pytest.mark.parametrize("batch", [63, 64, 65, 128, 129, 300])
def test_batches_past_a_wave(cuda, batch):
    """More sequences than lanes, fewer items than workgroups, long ones among short ones."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 300, (batch,), generator=gen).tolist()
    lengths[0], lengths[batch // 2], lengths[-1], lengths[5] = 2500, 3001, 1999, 0
    k, v, table = _paged(gen, lengths, 1, 32, 64, F16)
    _check(cuda, _rand(gen, batch, 5, 64, dtype=F16) * 2, k, v, table, lengths)


@pytest.mark.parametrize("page", [1, 3, 7, 32, 48, 128, 1000])
@pytest.mark.parametrize("window,sinks", [(None, 0), (None, 9), (1, 0), (100, 0), (64, 5), (333, 130),
                                          (5000, 5000)])
def test_page_sizes_and_windows(cuda, page, window, sinks):
    gen = torch.Generator().manual_seed(page)
    lengths = [31, 32, 127, 128, 129, 455, 1301]
    k, v, table = _paged(gen, lengths, 2, page, 64, BF16)
    q = _rand(gen, len(lengths), 8, 64, dtype=BF16) * 2
    _check(cuda, q, k, v, table, lengths, window=window, sinks=sinks, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("length", [1, 2, 129, 5000])
def test_contiguous_caches(cuda, dtype, length):
    gen = torch.Generator().manual_seed(length)
    k, v = (_rand(gen, 3, 2, 5003, 128, dtype=dtype) for _ in "kv")
    k[:, :, length:] = math.nan
    v[:, :, length:] = math.inf
    q = _rand(gen, 3, 8, 128, dtype=dtype)
    got = _check(cuda, q, k, v, None, [length] * 3)
    one = fpv2.decode_attention(q.to(cuda), k.to(cuda), v.to(cuda), None, length)
    assert torch.equal(got, one)  # one length for all, as an integer


def test_many_sequences(cuda):
    """More sequences than a wave has lanes; some longer than the rest together."""
    gen = torch.Generator().manual_seed(5)
    lengths = [int(x) for x in torch.randint(0, 40, (150,), generator=gen)]
    lengths[70], lengths[149] = 6000, 1500
    k, v, table = _paged(gen, lengths, 1, 16, 64, F16)
    q = _rand(gen, 150, 4, 64, dtype=F16)
    got = _check(cuda, q, k, v, table, lengths)
    again = fpv2.decode_attention(*(x.to(cuda) for x in (q, k, v, table)),
                                  torch.tensor(lengths, dtype=torch.int32, device=cuda))
    assert torch.equal(got, again)


def test_strides_and_out(cuda):
    """Pages of one K/V pool with the heads inside the rows, strided q and out, wide table."""
    gen = torch.Generator().manual_seed(6)
    lengths = [300, 17]
    k, v, table = _paged(gen, lengths, 2, 32, 128, BF16)
    pool = torch.empty((k.shape[0], 32, 2, 2, 128), dtype=BF16, device=cuda)
    pool[:, :, 0] = k.transpose(1, 2).to(cuda)
    pool[:, :, 1] = v.transpose(1, 2).to(cuda)
    kp, vp = (pool[:, :, i].transpose(1, 2) for i in (0, 1))
    wide = torch.full((2, table.shape[1] + 5), 10 ** 6, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = _rand(gen, 8, 2, 136, dtype=BF16)[..., :128].transpose(0, 1)
    out = torch.full((2, 8, 131), 7.0, dtype=BF16, device=cuda)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    got = fpv2.decode_attention(q.to(cuda), kp, vp, wide.to(cuda)[:, :table.shape[1]], lens,
                                out=out[..., 2:130])
    want, tol = _reference(q, k, v, table, lengths, 128 ** -0.5, None, 0)
    assert got.data_ptr() == out[..., 2:130].data_ptr()
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert bool((out[..., :2] == 7).all()) and bool((out[..., 130:] == 7).all())
    # q off a 16-byte boundary
    shifted = torch.empty(2 * 8 * 128 + 1, dtype=BF16, device=cuda)[1:].view(2, 8, 128)
    shifted.copy_(q)
    assert torch.equal(fpv2.decode_attention(shifted, kp, vp, table.to(cuda), lens), got)


def test_out_of_range_lengths_and_pages_are_clipped(cuda):
    gen = torch.Generator().manual_seed(7)
    k, v = (_rand(gen, 4, 1, 16, 64, dtype=BF16) for _ in "kv")
    q = _rand(gen, 3, 4, 64, dtype=BF16)
    table = torch.tensor([[-5, 1], [99, 2], [0, 3]], dtype=torch.int32)
    lengths = torch.tensor([20, 32, 2 ** 31 - 1], dtype=torch.int32)
    got = fpv2.decode_attention(*(x.to(cuda) for x in (q, k, v, table, lengths)))
    want, tol = _reference(q, k, v, table.clamp(0, 3), [20, 32, 32], 0.125, None, 0)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    below = fpv2.decode_attention(*(x.to(cuda) for x in (q, k, v, table)),
                                  torch.full((3,), -3, dtype=torch.int32, device=cuda))
    assert not below.any()


def test_infinite_and_nan_values(cuda):
    """What is visible counts as the formula has it, what is masked does not."""
    gen = torch.Generator().manual_seed(8)
    k, v = (_rand(gen, 4, 1, 300, 64, dtype=BF16) for _ in "kv")
    q = _rand(gen, 4, 2, 64, dtype=BF16)
    q[1].abs_()
    v[0, 0, 7, 3] = math.inf       # one infinite value
    k[1, 0, 11] = -math.inf        # a key of score -inf: no weight
    k[2, 0, :, 0] = math.nan       # every score NaN
    k[3, 0, :] = -math.inf         # nothing but scores of -inf
    q[3].abs_()
    lengths = [200, 200, 200, 200]
    k[:, :, 200:], v[:, :, 200:] = math.nan, math.nan
    got = fpv2.decode_attention(*(x.to(cuda) for x in (q, k, v)), None, 200).cpu().double()
    want, tol = _reference(q, k, v, None, lengths, 0.125, None, 0)
    assert bool((got[0, :, 3] == math.inf).all())
    assert bool(torch.isnan(got[2:]).all()) and bool(torch.isnan(want[2:]).all())
    fine = torch.isfinite(want[:2])
    assert torch.equal(fine, torch.isfinite(got[:2]))
    assert bool(((got[:2] - want[:2]).abs() <= tol[:2])[fine].all())


def test_cache_past_32_bits(cuda):
    """A contiguous cache whose last rows lie behind 4 GiB (and 2^31 elements)."""
    rows, window, sinks, dim = 17_000_000, 100, 50, 128
    gen = torch.Generator().manual_seed(9)
    k = torch.empty((1, 1, rows, dim), dtype=BF16, device=cuda)
    v = torch.empty_like(k)
    small = [_rand(gen, 1, 1, window + sinks, dim, dtype=BF16) for _ in "kv"]
    length = rows - 3
    for big, part in zip((k, v), small):
        big[:, :, :sinks] = part[:, :, :sinks].to(cuda)
        big[:, :, length - window:length] = part[:, :, sinks:].to(cuda)
    q = _rand(gen, 1, 4, dim, dtype=BF16)
    got = fpv2.decode_attention(q.to(cuda), k, v, None, length, window_tokens=window,
                                sink_tokens=sinks)
    want, tol = _reference(q, *small, None, [window + sinks], dim ** -0.5, None, 0)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


def test_graph_replays_follow_lengths_and_tables(cuda):
    """Two captured calls of different sizes and eager calls between their replays."""
    gen = torch.Generator().manual_seed(10)
    cases = []
    for lengths, page in (([900, 40, 0], 16), ([3000], 64)):
        k, v, table = _paged(gen, lengths, 2, page, 64, BF16, fill=0.0)
        q = _rand(gen, len(lengths), 8, 64, dtype=BF16)
        cases.append([x.to(cuda) for x in (q, k, v, table,
                                           torch.tensor(lengths, dtype=torch.int32))])
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for args in cases:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            fpv2.decode_attention(*args)  # warm-up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fpv2.decode_attention(*args))
        graphs.append(graph)
    for step in range(4):
        for args in cases:
            args[0].mul_(1.1)
            args[4].sub_(13)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, args in zip(outs, cases):
            assert torch.equal(out, fpv2.decode_attention(*args))


def test_runs_on_the_current_stream(cuda):
    gen = torch.Generator().manual_seed(11)
    k, v = (_rand(gen, 2, 2, 4000, 128, dtype=BF16).to(cuda) for _ in "kv")
    q = _rand(gen, 2, 8, 128, dtype=BF16).to(cuda)
    want = fpv2.decode_attention(q, k, v, None, 4000)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        got = fpv2.decode_attention(late, k, v, None, 4000)
    side.synchronize()
    assert torch.equal(got, want)


def test_windows_past_any_cache(cuda):
    """Windows and sinks of the largest integers see everything."""
    gen = torch.Generator().manual_seed(12)
    k, v, table = _paged(gen, [700, 90], 2, 16, 64, BF16)
    q = _rand(gen, 2, 4, 64, dtype=BF16)
    want = _check(cuda, q, k, v, table, [700, 90])
    for window, sinks in ((2 ** 62, 2 ** 62), (2 ** 63 - 1, 2 ** 63 - 1), (1, 2 ** 63 - 1), (2 ** 62, 0)):
        got = fpv2.decode_attention(q.to(cuda), k.to(cuda), v.to(cuda), table.to(cuda),
                                    torch.tensor([700, 90], dtype=torch.int32, device=cuda),
                                    window_tokens=window, sink_tokens=sinks)
        assert torch.equal(got, want)


def test_small_float16_values(cuda):
    """Subnormal keys and values count."""
    gen = torch.Generator().manual_seed(13)
    k, v = (_rand(gen, 1, 1, 200, 64, dtype=torch.float32) * 2e-6 for _ in "kv")
    k, v = (x.to(F16) for x in (k, v))
    q = _rand(gen, 1, 4, 64, dtype=F16) * 30
    got = fpv2.decode_attention(q.to(cuda), k.to(cuda), v.to(cuda), None, 200, scale=1000.0)
    want, tol = _reference(q, k, v, None, [200], 1000.0, None, 0)
    # (a result this small is rounded to a multiple of 2^-24)
    assert bool(((got.cpu().double() - want).abs() <= tol + 2.0 ** -25).all())
    assert float(want.abs().max()) > 2.0 ** -22
