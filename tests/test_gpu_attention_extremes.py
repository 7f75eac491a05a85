"""Attention of single tokens where scores, scales or values are as great as their types allow,
against the formula in float64 on the CPU.

Scores here are powers of two and whole numbers of steps beside them, exact in float32, so that
a weight is 2 to the power of an exact difference whatever the scores' size."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from batch_cases import BF16, F16, attention, tolerance

pytestmark = pytest.mark.gpu

LN2 = math.log(2)  # a scale of ln 2: scores are exponents of two


def _great_scores(exponent, dtype, dim, heads, n, sign):
    """Queries ``[heads, dim]``, keys ``[n, dim]`` and the exponents ``[heads, n]``: 2^exponent and
    whole steps beside it, of 4 or of a float32 number's, which grow (``sign`` 1) or fall (-1) by one from
    each 128 keys to the next and by one more for a key of each 32."""
    step = max(4.0, 2.0 ** (exponent - 23))
    t = torch.arange(n)
    steps = sign * (t // 128 + (t % 32 == 5).long())
    q, k = torch.zeros((heads, dim), dtype=dtype), torch.zeros((n, dim), dtype=dtype)
    q[:, 0], k[:, 0] = 2.0 ** 14, 2.0 ** (exponent - 14)
    q[:, 3], k[:, 3] = step * (torch.arange(heads) % 3), steps.to(dtype)
    s = q.double() @ k.double().T
    assert torch.equal(s, s.float().double())
    return q, k, s


def _great_result(s, v, dtype):
    """The result and its tolerance: the weights are powers of two, exact where they are 2^-24 of their 32
    keys' greatest and more, else off by 2^-25 of it; v_exp_f32 by 2^-22, sums of n terms by n 2^-24."""
    w = torch.exp2(s - s.amax(1, keepdim=True))
    w = w / w.sum(1, keepdim=True)
    want, mass = w @ v.double(), w @ v.double().abs()
    tol = (torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * mass
           + 2 * len(v) * (2.0 ** -24 * mass + 2.0 ** -25 * float(v.abs().max())))
    return want, tol


EXPONENTS = [14, 20, 21, 22, 23, 24, 25, 26, 27, 28]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("exponent", EXPONENTS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [2, 5])
def test_shared_prefix_great_scores(cuda, dtype, exponent, dim, batch):
    """In the prefix, up to 16 rows a KV head and more, and among the own keys."""
    for sign in (1, -1):
        n = 600
        q, k, s = _great_scores(exponent, dtype, dim, 6, n, sign)
        v = torch.randn((n, dim), generator=torch.Generator().manual_seed(exponent)).to(dtype)
        want, tol = _great_result(s, v, dtype)
        kd, vd = k.to(cuda), v.to(cuda)
        for prefix in (n, 320, 0):
            own = [x[prefix:].expand(batch, 1, n - prefix, dim).contiguous() if prefix < n
                   else torch.zeros((batch, 1, 1, dim), dtype=dtype, device=cuda) for x in (kd, vd)]
            got = fpv2.shared_prefix_attention(
                q.expand(batch, 6, dim).to(cuda), kd[None, None], vd[None, None], None, prefix, *own, None,
                n - prefix, scale=LN2)
            err = (got.cpu().double() - want).abs()
            assert bool((err <= tol).all()), (sign, prefix, float((err / tol).amax()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("exponent", EXPONENTS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_great_scores(cuda, dtype, exponent, dim):
    for sign in (1, -1):
        for n in (1, 600):
            q, k, s = _great_scores(exponent, dtype, dim, 6, n, sign)
            v = torch.randn((n, dim), generator=torch.Generator().manual_seed(exponent)).to(dtype)
            want, tol = _great_result(s, v, dtype)
            got = fpv2.decode_attention(q[None].to(cuda), k[None, None].to(cuda), v[None, None].to(cuda), None, n,
                                        scale=LN2)
            err = (got[0].cpu().double() - want).abs()
            assert bool((err <= tol).all()), (sign, n, float((err / tol).amax()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("exponent", EXPONENTS)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_quantized_decode_great_scores(cuda, dtype, exponent, dim):
    """The values' scales are of any size beside the scores'.

    Tolerance: weight times scale is rounded once to float16 (half a step of the mass), where it is
    below 2^-29 of its 32 keys' greatest by 2^-40 of that; the scale's logarithm, of at most 8, is off by 2^-22
    and the weight's exponent by 2^-20 when it is added; sums as above."""
    for sign in (1, -1):
        for n in (1, 600):
            gen = torch.Generator().manual_seed(exponent)
            step = max(4.0, 2.0 ** (exponent - 23))
            t = torch.arange(n)
            steps = sign * (t // 128 + (t % 32 == 5).long())
            q = torch.zeros((6, dim), dtype=dtype)
            k = torch.zeros((n, dim), dtype=torch.int8)
            ks = torch.full((n,), 2.0 ** (exponent - 20))
            q[:, 0], k[:, 0] = 2.0 ** 14, 64
            q[:, 3], k[:, 3] = step * 2.0 ** (20 - exponent) * (torch.arange(6) % 3), steps.to(torch.int8)
            v = torch.randint(-127, 128, (n, dim), generator=gen).to(torch.int8)
            vs = 2.0 ** (12 * torch.rand(n, generator=gen) - 6)
            got = fpv2.quantized_decode_attention(
                *(x.to(cuda) for x in (q[None], k[None, None], ks[None, None], v[None, None], vs[None, None])),
                None, n, scale=LN2)
            s = q.double() @ (k.double() * ks.double()[:, None]).T
            assert torch.equal(s, s.float().double())
            value = v.double() * vs.double()[:, None]
            w = torch.exp2(s - s.amax(1, keepdim=True))
            w = w / w.sum(1, keepdim=True)
            want, mass = w @ value, w @ value.abs()
            greatest = (w * vs.double()).amax(1, keepdim=True)
            tol = (torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -19) * mass
                   + 2 * n * (2.0 ** -24 * mass + 2.0 ** -40 * 127 * greatest))
            err = (got[0].cpu().double() - want).abs()
            assert bool((err <= tol).all()), (sign, n, float((err / tol).amax()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch", [2, 9])
@pytest.mark.parametrize("prefix", [300, 0])
def test_scale_that_is_no_number(cuda, dtype, batch, prefix):
    """As the formula and the other attentions have it: NaN wherever a key is visible."""
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=gen).to(dtype).to(cuda)
               for s in ((batch, 4, 64), (batch, 1, 300, 64), (batch, 1, 300, 64)))
    got = fpv2.shared_prefix_attention(q, k[:1], v[:1], None, prefix, k, v, None, 40, scale=math.nan)
    assert bool(got.isnan().all())
    assert bool(fpv2.decode_attention(q, k, v, None, 40, scale=math.nan).isnan().all())
    got = fpv2.shared_prefix_attention(q, k[:1], v[:1], None, 0, k, v, None, 0, scale=math.nan)
    assert not got.any()


@pytest.mark.parametrize("batch", [2, 9])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -120, -2.0 ** -110, 0.0])
def test_scales_far_below_one(cuda, batch, scale):
    """Great queries and keys under a tiny scale have ordinary scores; a scale of zero has equal
    weights."""
    gen = torch.Generator().manual_seed(2)
    dim, n, prefix = 64, 500, 300
    size = 2.0 ** round(-math.log2(abs(scale)) / 2) if scale else 1.0
    q = (torch.randn((batch, 4, dim), generator=gen) * size).to(BF16)
    k = (torch.randn((n, dim), generator=gen) * size / 2).to(BF16)
    v = torch.randn((n, dim), generator=gen).to(BF16)
    kd, vd = k.to(cuda), v.to(cuda)
    own = [x[prefix:].expand(batch, 1, n - prefix, dim).contiguous() for x in (kd, vd)]
    got = fpv2.shared_prefix_attention(q.to(cuda), kd[None, None], vd[None, None], None, prefix, *own, None,
                                       n - prefix, scale=scale)
    for b in range(batch):
        want, mass, most = attention(q[b], k[None], v[None], scale)
        tol = tolerance(want, mass, most, n, dim, BF16, BF16)
        err = (got[b].cpu().double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))


@pytest.mark.parametrize("batch", [2, 9])
@pytest.mark.parametrize("prefix", [400, 200, 0])
@pytest.mark.parametrize("gap", [0.0, 3.0, 7.5, 8.0, 8.5])
def test_values_near_the_greatest(cuda, batch, prefix, gap):
    """One key ``gap`` bits above the ones before it, whose value is next to bfloat16's greatest
    number, as the result is: no weight leaves more room above a value than ``decode_attention``'s do."""
    n, dim, at = 400, 64, 390
    q, k, v = torch.zeros((batch, 4, dim), dtype=BF16), torch.zeros((n, dim), dtype=BF16), torch.zeros((n, dim))
    q[:, :, 0], k[at, 0] = 1.0, gap
    v = v.to(BF16)
    v[at] = 2.0 ** 127 * 1.875
    kd, vd = k.to(cuda), v.to(cuda)
    own = [x[prefix:].expand(batch, 1, n - prefix, dim).contiguous() if prefix < n
           else torch.zeros((batch, 1, 1, dim), dtype=BF16, device=cuda) for x in (kd, vd)]
    got = fpv2.shared_prefix_attention(q.to(cuda), kd[None, None], vd[None, None], None, prefix, *own, None,
                                       n - prefix, scale=LN2)
    want, mass, most = attention(q[0], k[None], v[None], LN2)
    assert bool(fpv2.decode_attention(q[:1].to(cuda), kd[None, None], vd[None, None], None, n, scale=LN2)
                .isfinite().all())
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tolerance(want, mass, most, n, dim, BF16, BF16)).all())


@pytest.mark.parametrize("batch", [2, 9])
@pytest.mark.parametrize("prefix", [100, 0])
def test_scores_near_the_lowest(cuda, batch, prefix):
    """Every score next to float32's lowest number: equal weights."""
    dim = 64
    q, k = torch.zeros((batch, 4, dim), dtype=BF16), torch.zeros((1, 1, 100, dim), dtype=BF16)
    q[:, :, 0], k[..., 0] = -1.984375 * 2.0 ** 64, 2.0 ** 63
    v = torch.randn((1, 1, 100, dim), generator=torch.Generator().manual_seed(3)).to(BF16)
    own = [x.expand(batch, 1, 100, dim).contiguous().to(cuda) for x in (k, v)]
    got = fpv2.shared_prefix_attention(q.to(cuda), k.to(cuda), v.to(cuda), None, prefix, *own, None,
                                       100 if prefix == 0 else 0, scale=LN2)
    want, mass = v[0, 0].double().mean(0), v[0, 0].double().abs().mean(0)
    # (equal weights of at most 2^7: exact in bfloat16; sums of 100 terms)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 300 * 2.0 ** -24 * mass).all())
