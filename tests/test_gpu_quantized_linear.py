"""``fpv2.quantized_linear`` against float64 products of the same 4-bit weights.

Tolerance, per element: P = sum (16 + q) x and X = sum x of a group are float32
sums of at most 128 terms, c = b - 16 s is rounded once, and the groups' s P + c X
are added over K / 128 steps and 8 waves: below (160 + K / 128) 2^-23 of
sum |s| (16 + q) |x| + |c| |x|.  A 16-bit result is rounded once more.
"""

from __future__ import annotations

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _weights(gen, n, k, group, dtype):
    packed = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=gen).to(torch.int32)
    scales = (0.01 * (0.2 + torch.rand((n, k // group), generator=gen))).to(dtype)
    biases = (-7.5 * scales.float() * (1 + 0.3 * torch.randn(scales.shape, generator=gen))).to(dtype)
    return packed, scales, biases


def _reference(x, packed, scales, biases):
    n, k = packed.shape[0], packed.shape[1] * 8
    group = k // scales.shape[1]
    q = torch.stack([(packed.long() >> (4 * i)) & 15 for i in range(8)], -1).view(n, -1, group)
    s, b = scales.double()[..., None], biases.double()[..., None]
    w = (q * s + b).view(n, k)
    size = (s.abs() * (16 + q) + (b - 16 * s).abs()).view(n, k)
    xd = x.double()
    return xd @ w.T, (160 + k / 128) * 2.0 ** -23 * (xd.abs() @ size.T)


def _check(cuda, x, weights, out_dtype=None):
    got = fpv2.quantized_linear(x.to(cuda), *(t.to(cuda) for t in weights), out_dtype=out_dtype)
    want, tol = _reference(x, *weights)
    if got.dtype != F32:
        info = torch.finfo(got.dtype)
        tol = tol * (1 + info.eps) + info.eps / 2 * want.abs().clamp(min=info.tiny)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 17, 33, 70])
def test_rows_and_groups(cuda, dtype, group, rows):
    gen = torch.Generator().manual_seed(rows + group)
    weights = _weights(gen, 83, 640, group, dtype)
    x = torch.randn((rows, 640), generator=gen).to(dtype)
    _check(cuda, x, weights)
    _check(cuda, x, weights, F32)


@pytest.mark.parametrize("group,cols", [(32, 32), (32, 96), (32, 1056), (64, 64), (64, 192),
                                        (64, 2496), (128, 128), (128, 1152), (64, 9728)])
@pytest.mark.parametrize("out", [1, 15, 16, 17, 300])
def test_column_counts(cuda, group, cols, out):
    """Columns that end inside a step of 128, odd numbers of outputs."""
    gen = torch.Generator().manual_seed(cols + out)
    weights = _weights(gen, out, cols, group, BF16)
    for rows in (1, 6):
        _check(cuda, torch.randn((rows, cols), generator=gen).to(BF16), weights, F32)


@pytest.mark.parametrize("group,cols", [(32, 2592), (64, 5184), (128, 5376), (64, 10304), (128, 20608)])
@pytest.mark.parametrize("rows", [4, 5, 16, 19, 64])
def test_rows_of_several_panels(cuda, group, cols, rows):
    """More columns of x than lie in LDS at a time, the last panel short or of a part of a step."""
    gen = torch.Generator().manual_seed(cols + rows)
    weights = _weights(gen, 35, cols, group, F16 if rows % 2 else BF16)
    x = torch.randn((rows, cols), generator=gen).to(weights[1].dtype)
    _check(cuda, x, weights, F32)


@pytest.mark.parametrize("rows", [6, 20])
def test_panels_of_workgroups_that_share_a_cu(cuda, rows):
    gen = torch.Generator().manual_seed(rows)
    weights = _weights(gen, 17003, 2624, 64, BF16)
    _check(cuda, torch.randn((rows, 2624), generator=gen).to(BF16), weights)


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_many_outputs(cuda, rows):
    """Enough outputs for the wide tiles; two calls agree to the bit."""
    gen = torch.Generator().manual_seed(rows)
    weights = _weights(gen, 20011, 256, 64, BF16)
    x = torch.randn((rows, 256), generator=gen).to(BF16)
    got = _check(cuda, x, weights)
    dev = [t.to(cuda) for t in weights]
    assert torch.equal(got, fpv2.quantized_linear(x.to(cuda), *dev))


def test_large_values_and_special_groups(cuda):
    """Activations near the largest, groups of scale zero and of one step."""
    gen = torch.Generator().manual_seed(1)
    packed, scales, biases = _weights(gen, 40, 512, 64, BF16)
    scales[::3] = 0
    biases[1::3] = 0
    packed[5] = -1
    packed[6] = 0
    x = (torch.randn((3, 512), generator=gen) * 1e30).to(BF16)
    _check(cuda, x, (packed, scales, biases), F32)
    _check(cuda, torch.zeros((3, 512), dtype=BF16), (packed, scales, biases), F32)


def test_nan_rows_stay_in_their_rows(cuda):
    gen = torch.Generator().manual_seed(2)
    weights = [t.to(cuda) for t in _weights(gen, 50, 256, 32, F16)]
    x = torch.randn((6, 256), generator=gen).to(F16).to(cuda)
    clean = fpv2.quantized_linear(x, *weights)
    x[4, 100] = float("nan")
    got = fpv2.quantized_linear(x, *weights)
    assert bool(got[4].isnan().all())
    assert torch.equal(got[[0, 1, 2, 3, 5]], clean[[0, 1, 2, 3, 5]])


def test_strides_and_shapes(cuda):
    gen = torch.Generator().manual_seed(3)
    packed, scales, biases = _weights(gen, 37, 384, 64, BF16)
    wide = torch.full((37, 56), 123, dtype=torch.int32)
    wide[:, 4:52] = packed
    sb = torch.full((37, 14), float("nan"), dtype=BF16)
    sb[:, :6], sb[:, 7:13] = scales, biases
    dev = wide.to(cuda)[:, 4:52], sb.to(cuda)[:, :6], sb.to(cuda)[:, 7:13]
    x = torch.randn((5, 400), generator=gen).to(BF16).to(cuda)
    want = fpv2.quantized_linear(x[:, :384].contiguous(), packed.to(cuda), scales.to(cuda),
                                 biases.to(cuda))
    assert torch.equal(fpv2.quantized_linear(x[:, :384], *dev), want)
    assert torch.equal(fpv2.quantized_linear(x[:, None, :384], *dev)[:, 0], want)
    off = torch.empty(5 * 384 + 1, dtype=BF16, device=cuda)[1:].view(5, 384)
    off.copy_(x[:, :384])
    assert torch.equal(fpv2.quantized_linear(off, *dev), want)
    assert torch.equal(fpv2.quantized_linear(x[0, :384], *dev), fpv2.quantized_linear(x[:1, :384], *dev)[0])
    assert torch.equal(fpv2.quantized_linear(x[:1, :384].expand(5, 384), *dev),
                       fpv2.quantized_linear(x[:1, :384].repeat(5, 1), *dev))
    out = torch.full((5, 50), 9.0, dtype=BF16, device=cuda)
    assert fpv2.quantized_linear(x[:, :384], *dev, out=out[:, 3:40]).data_ptr() == out[:, 3:40].data_ptr()
    assert torch.equal(out[:, 3:40], want)
    assert bool((out[:, :3] == 9).all()) and bool((out[:, 40:] == 9).all())
    assert fpv2.quantized_linear(x[:0, :384], *dev).shape == (0, 37)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_weights_are_near_the_weights(cuda, dtype, group):
    """Off by at most half a step, the stored bias' rounding, the range that the
    stored scale's rounding loses and the result's own rounding."""
    gen = torch.Generator().manual_seed(group)
    w = torch.randn((20, 256), generator=gen).to(dtype)
    w[3] = 0.5
    w[4, :group] = 0
    packed, scales, biases = fpv2.quantize_weight(w.to(cuda), group_size=group)
    back = fpv2.dequantize_weight(packed, scales, biases).cpu().double()
    half = torch.finfo(dtype).eps / 2
    g = w.double().view(20, -1, group)
    spread = (g.amax(-1) - g.amin(-1))[..., None]
    tol = (spread / 30 * (1 + 2 * half) + 2 * half * g.amin(-1).abs()[..., None] + 2 * half * spread
           + half * g.abs() + 2.0 ** -20).expand(g.shape).reshape(20, 256)
    assert bool(((back - w.double()).abs() <= tol).all())
    cpu = fpv2.quantize_weight(w, group_size=group)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((packed, scales, biases), cpu))
    if dtype != F32:
        x = torch.randn((3, 256), generator=gen).to(dtype)
        _check(cuda, x, (packed.cpu(), scales.cpu(), biases.cpu()))


def test_captured_and_streams(cuda):
    gen = torch.Generator().manual_seed(4)
    weights = [t.to(cuda) for t in _weights(gen, 2560, 1024, 64, BF16)]
    x = torch.randn((2, 1024), generator=gen).to(BF16).to(cuda)
    fpv2.quantized_linear(x, *weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fpv2.quantized_linear(x, *weights)
    for step in range(3):
        x.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fpv2.quantized_linear(x, *weights))


def test_small_float16_values(cuda):
    """Subnormal activations and scales count."""
    gen = torch.Generator().manual_seed(5)
    packed, scales, biases = _weights(gen, 40, 256, 64, F16)
    x = (torch.randn((3, 256), generator=gen) * 3e-6).to(F16)
    _check(cuda, x, (packed, scales, biases), F32)
    small = ((scales.float() * 1e-3).to(F16), (biases.float() * 1e-3).to(F16))
    _check(cuda, (x.float() * 1e4).to(F16), (packed, *small), F32)
