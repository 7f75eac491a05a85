"""``fpv2.rope_to_pages`` against the formula in float64 on the CPU.

Tolerance, per element: one rounding to the storage type (half a step of the
value, or of the least normal number), and float32 arithmetic whose relative
error is below (D + 16) 2^-24 of each rotated term (a sum of D squares, the root,
three products and a sum).
"""

from __future__ import annotations

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
EPS = 1e-6


def _tables(limit, half):
    inv = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = torch.arange(limit, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _rotated(x, weight, cos, sin, interleaved):
    """x [T, H, D] -> float64 values and the sizes of the rotated terms."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    half = cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    out, size = x.clone(), x.abs()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return out, size


def _close(got, want, size):
    info = torch.finfo(got.dtype)
    tol = (info.eps / 2 * want.abs().clamp(min=info.tiny)
           + (want.shape[-1] + 16) * 2.0 ** -24 * (1 + info.eps) * size)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _case(gen, tokens, heads, hkv, dim, half, dtype, page, limit=5000):
    qkv = (torch.randn((tokens, (heads + 2 * hkv) * dim), generator=gen) * 2).to(dtype)
    weights = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) for _ in "qk"]
    cos, sin = _tables(limit, half)
    pages = -(-tokens // page) + 2
    pools = [torch.randn((pages, hkv, page, dim), generator=gen).to(dtype) for _ in "kv"]
    positions = torch.randint(0, limit, (tokens,), generator=gen)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    return qkv, weights, cos, sin, pools, positions, slots


def _run(cuda, qkv, weights, cos, sin, pools, positions, slots, heads, **kwargs):
    dev = [None if x is None else x.to(cuda) if isinstance(x, torch.Tensor) else x
           for x in (qkv, *weights, cos, sin, positions, slots)]
    kp, vp = (p.to(cuda) for p in pools)
    q = fpv2.rope_to_pages(dev[0], dev[1], dev[2], dev[3], dev[4], dev[5], dev[6], kp, vp,
                           query_heads=heads, eps=EPS, **kwargs)
    return q, kp, vp


def _check(q, kp, vp, qkv, weights, cos, sin, pools, positions, slots, heads, interleaved=False):
    hkv, page, dim = pools[0].shape[1:]
    x = qkv.view(qkv.shape[0], -1, dim)
    pos = positions.long().clamp(0, cos.shape[0] - 1)
    want, size = _rotated(x[:, :heads], weights[0], cos[pos], sin[pos], interleaved)
    _close(q, want, size)
    want, size = _rotated(x[:, heads:heads + hkv], weights[1], cos[pos], sin[pos], interleaved)
    kept = (slots >= 0) & (slots < pools[0].shape[0] * page)
    at = slots[kept].long()
    _close(kp.cpu()[at // page, :, at % page], want[kept], size[kept])
    vwant = pools[1].clone()
    vwant[at // page, :, at % page] = x[kept, heads + hkv:]
    assert torch.equal(vp.cpu(), vwant)
    other = torch.ones(pools[0].shape[0] * page, dtype=torch.bool)
    other[at] = False
    same = kp.cpu().transpose(1, 2).flatten(0, 1)[other]
    assert torch.equal(same, pools[0].transpose(1, 2).flatten(0, 1)[other])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(128, 64), (64, 32), (96, 48), (96, 24), (256, 128), (128, 32),
                                      (16, 8), (80, 40), (112, 8), (512, 256), (320, 80)])
def test_heads_and_rotations(cuda, dtype, interleaved, dim, half):
    gen = torch.Generator().manual_seed(dim + half)
    case = _case(gen, 21, 5, 3, dim, half, dtype, 16)
    got = _run(cuda, *case, 5, interleaved=interleaved)
    _check(*got, *case, 5, interleaved)


@pytest.mark.parametrize("tokens,page", [(1, 16), (3, 1), (200, 7), (2500, 48)])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_token_counts(cuda, tokens, page, ids):
    """A token, and more than a wave takes at a time; padding and clipped positions."""
    gen = torch.Generator().manual_seed(tokens)
    qkv, weights, cos, sin, pools, positions, slots = _case(gen, tokens, 32, 8, 128, 64, BF16, page)
    if tokens > 2:
        slots[::5] = -1
        slots[1] = pools[0].shape[0] * page
        slots[2] = 2 ** 31 - 1
        positions[0], positions[1] = -4, 5000
    case = (qkv, weights, cos, sin, pools, positions.to(ids), slots.to(ids))
    _check(*_run(cuda, *case, 32), *case, 32)


def test_integer_positions_and_slots_and_no_norm(cuda):
    gen = torch.Generator().manual_seed(3)
    qkv, weights, cos, sin, pools, _, _ = _case(gen, 19, 4, 2, 64, 32, F16, 16)
    t = torch.arange(19)
    for w in (weights, (None, weights[1]), (weights[0], None), (None, None)):
        got = _run(cuda, qkv, w, cos, sin, pools, 4990, 13, 4)
        _check(*got, qkv, w, cos, sin, pools, t + 4990, t + 13, 4)


def test_strided_caches_and_out(cuda):
    """The cache of a chunked prefill as one page, q into a projection's layout."""
    gen = torch.Generator().manual_seed(4)
    qkv, weights, cos, sin, _, positions, _ = _case(gen, 9, 4, 2, 128, 64, BF16, 16)
    kv = torch.randn((2, 2, 1000, 136), generator=gen).to(BF16)
    caches = kv.to(cuda)
    kp, vp = (caches[i, None, :, :, :128] for i in (0, 1))
    wide = torch.full((9, 4 * 128 + 8), 5.0, dtype=BF16, device=cuda)
    out = wide[:, :512].view(9, 4, 128)
    slots = torch.arange(700, 709)
    # qkv off a 16-byte boundary
    shifted = torch.empty(qkv.numel() + 1, dtype=BF16, device=cuda)[1:].view(qkv.shape)
    shifted.copy_(qkv)
    q = fpv2.rope_to_pages(shifted, weights[0].to(cuda), weights[1].to(cuda), cos.to(cuda),
                           sin.to(cuda), positions.to(cuda), 700, kp, vp, query_heads=4, eps=EPS,
                           out=out)
    assert q.data_ptr() == wide.data_ptr()
    pools = [kv[i, None, :, :, :128] for i in (0, 1)]
    _check(q, kp, vp, qkv, weights, cos, sin, [p.contiguous() for p in pools], positions, slots, 4)
    assert bool((wide[:, 512:] == 5).all())
    assert torch.equal(caches[..., 128:].cpu(), kv[..., 128:])


def test_values_and_rounding_agree_with_the_contiguous_kernel(cuda):
    """The prefill's own norm and rotation, which rounds the norm's output too,
    writes the same rows to within that rounding."""
    from fpv2.prefill_harness import DecoderShape, _qk_norm_rope, rope_tables
    gen = torch.Generator().manual_seed(5)
    shape = DecoderShape(query_heads=4, kv_heads=2, head_dim=128)
    qkv = torch.randn((33, 8 * 128), generator=gen).to(BF16).to(cuda)
    w = [(1 + 0.1 * torch.randn(128, generator=gen)).to(BF16).to(cuda) for _ in "qk"]
    cos, sin = rope_tables(shape, torch.arange(40, 73, device=cuda))
    q0, k0 = _qk_norm_rope(qkv, *w, cos, sin, shape)
    pages = [torch.zeros((1, 2, 40, 128), dtype=BF16, device=cuda) for _ in "kv"]
    q1 = fpv2.rope_to_pages(qkv, *w, cos[:, :64].contiguous(), sin[:, :64].contiguous(), 0, 4,
                            *pages, query_heads=4, eps=shape.rms_eps)
    torch.testing.assert_close(q1.transpose(0, 1).float(), q0.float(), rtol=2 ** -6, atol=2 ** -6)
    torch.testing.assert_close(pages[0][0, :, 4:37].float(), k0.float(), rtol=2 ** -6, atol=2 ** -6)


def test_infinite_and_nan_rows_stay_in_their_rows(cuda):
    gen = torch.Generator().manual_seed(6)
    case = _case(gen, 7, 4, 2, 64, 32, BF16, 16)
    clean = _run(cuda, *case, 4)
    dirty = case[0].clone()
    dirty[3] = float("nan")
    got = _run(cuda, dirty, *case[1:], 4)
    keep = [0, 1, 2, 4, 5, 6]
    assert torch.equal(got[0][keep], clean[0][keep]) and bool(got[0][3].isnan().all())


def test_captured(cuda):
    gen = torch.Generator().manual_seed(7)
    qkv, weights, cos, sin, pools, positions, slots = (
        x.to(cuda) if isinstance(x, torch.Tensor) else [y.to(cuda) for y in x]
        for x in _case(gen, 5, 4, 2, 64, 32, BF16, 16))
    def call(kp, vp):
        return fpv2.rope_to_pages(qkv, *weights, cos, sin, positions, slots, kp, vp, query_heads=4)
    call(*pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(*pools)
    for step in range(3):
        positions.add_(17)
        slots.copy_((slots + 11) % (pools[0].shape[0] * 16))
        want = [p.clone() for p in pools]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, call(*want))
        assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_pages_past_32_bits(cuda):
    """Slots whose rows lie behind 4 GiB."""
    gen = torch.Generator().manual_seed(8)
    qkv, weights, cos, sin, _, positions, _ = _case(gen, 4, 2, 1, 256, 128, BF16, 16)
    page, pages = 64, 150_000
    kp, vp = (torch.empty((pages, 1, page, 256), dtype=BF16, device=cuda) for _ in "kv")
    slots = torch.tensor([pages * page - 1, 9_000_000, -(2 ** 40), 2 ** 33])
    q = fpv2.rope_to_pages(qkv.to(cuda), *(w.to(cuda) for w in weights), cos.to(cuda), sin.to(cuda),
                           positions.to(cuda), slots.to(cuda), kp, vp, query_heads=2, eps=EPS)
    x = qkv.view(4, -1, 256)
    want, size = _rotated(x[:, 2:3], weights[1], cos[positions], sin[positions], False)
    at = slots[:2].to(cuda)
    _close(kp[at // page, :, at % page], want[:2], size[:2])
    assert torch.equal(vp[at // page, :, at % page].cpu(), x[:2, 3:])
    assert q.shape == (4, 2, 256)
