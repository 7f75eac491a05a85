"""Corners of a decode step's operators on the GPU: scores far below a sequence's
greatest, infinities beside a rotation, numbers past 64 bits, side streams.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from fpv2 import ChunkedPrefill
from fpv2.prefill_harness import ChunkedPrefillRunner, DecoderShape, RandomDecoder

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16

# Of heads that share their keys: how far the other keys are below the greatest, in nats.
GAPS = [0.0, 8.0, 12.0, 15.0, 16.875, 17.5, 20.0, 24.0]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,batch,at", [(31, 1, 0), (200, 1, 199), (200, 600, 0), (200, 600, 77),
                                             (700, 600, 300), (40_000, 1, 0), (40_000, 1, 25_000),
                                             (40_000, 1, 39_999)])
def test_keys_far_below_the_greatest(cuda, dtype, dim, length, batch, at):
    """One key far above the rest whose value is zero, so that the rest are the result; in
    items of one workgroup (600 sequences of one table row) and of many.

    Tolerance: every weight and the result are off by half a step of the storage type, or
    of its least normal number, of which a weight's is 2^-29 of the greatest of its 32 keys,
    so that the 31 keys beside the greatest are off by 2^-40 each.  Scores are sums of three
    terms of at most 2^5 in float32 times log2 e: off by less than 8 * 2^-19, and the
    exponential by as much relative to its value; sums of n terms by n 2^-24, which for
    partial sums of a lane are fewer than 2^11."""
    gen = torch.Generator().manual_seed(length + at)
    heads, page = len(GAPS), 64
    q = torch.zeros((1, heads, dim), dtype=dtype)
    k = torch.zeros((1, 1, length, dim), dtype=dtype)
    q[0, :, 0], q[0, :, 5] = torch.tensor(GAPS), 1.0
    k[0, 0, at, 0] = 1.0
    k[0, 0, :, 5] = torch.randint(-32, 33, (length,), generator=gen) / 64
    k[0, 0, at, 5] = 0.5
    v = (1000 * (0.5 + torch.rand((1, 1, length, dim), generator=gen))).to(dtype)
    v[0, 0, at] = 0
    pages = -(-length // page)
    kp, vp = (torch.zeros((pages * page, dim), dtype=dtype) for _ in "kv")
    kp[:length], vp[:length] = k[0, 0], v[0, 0]
    kp, vp = (x.view(pages, page, 1, dim).transpose(1, 2).to(cuda) for x in (kp, vp))
    table = torch.arange(pages, dtype=torch.int32, device=cuda).expand(batch, pages)
    got = fpv2.decode_attention(q.expand(batch, heads, dim).to(cuda), kp, vp, table, length, scale=1.0)
    s = q[0].double() @ k[0, 0].double().T
    w = torch.softmax(s, 1)
    want = w @ v[0, 0].double()
    info = torch.finfo(dtype)
    top = w.amax(1, keepdim=True)
    tol = (info.eps / 2 * (2 * want.abs()).clamp(min=info.tiny) + 2.0 ** -12 * want.abs()
           + (31 * 2.0 ** -40 * 1500 * top if dtype == F16 else 0))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), [float(x) for x in (err / tol).amax((0, 2))]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half,tokens", [(96, 24, 3), (128, 8, 2500), (256, 64, 1)])
def test_dimensions_behind_the_rotation_are_copied(cuda, dtype, interleaved, dim, half, tokens):
    """Heads without a norm: what is not rotated stays as it is, bit for bit, beside infinities
    and NaN too."""
    gen = torch.Generator().manual_seed(dim)
    heads, hkv, page = 5, 2, 16
    x = torch.randn((tokens, heads + 2 * hkv, dim), generator=gen).to(dtype)
    x[:, :, 2 * half + 2] = math.inf
    x[:, 1::2, 2 * half + 5] = -math.inf
    x[:, ::2, dim - 1] = math.nan
    x[:, :, dim - 4] = -0.0
    angle = torch.rand((50, half), generator=gen) * 6
    kp, vp = (torch.zeros((-(-tokens // page), hkv, page, dim), dtype=dtype, device=cuda) for _ in "kv")
    q = fpv2.rope_to_pages(x.view(tokens, -1).to(cuda), None, None, angle.cos().to(cuda),
                           angle.sin().to(cuda), 7, 0, kp, vp, query_heads=heads, interleaved=interleaved)
    k = kp.transpose(1, 2).flatten(0, 1)[:tokens]
    for got, want in ((q.cpu(), x[:, :heads]), (k.cpu(), x[:, heads:heads + hkv])):
        got, want = got[..., 2 * half:], want[..., 2 * half:]
        nan = want.isnan()
        assert torch.equal(got.isnan(), nan)
        assert torch.equal(got.view(torch.int16)[~nan], want.contiguous().view(torch.int16)[~nan])


def _decode_case(cuda, lengths=(700, 90)):
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((48, 2, 16, 64), generator=gen).to(BF16).to(cuda) for _ in "kv")
    q = torch.randn((2, 4, 64), generator=gen).to(BF16).to(cuda)
    table = torch.arange(48, dtype=torch.int32).expand(2, 48).contiguous().to(cuda)
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("past", [2 ** 63, 2 ** 64, 2 ** 64 + 5, 2 ** 70 + 17])
def test_integers_past_64_bits(cuda, past):
    """Windows, sinks and lengths past any cache are the whole of it."""
    q, k, v, table, lengths = _decode_case(cuda)
    want = fpv2.decode_attention(q, k, v, table, lengths)
    for kwargs in (dict(window_tokens=past), dict(window_tokens=past, sink_tokens=past),
                   dict(window_tokens=3, sink_tokens=past), dict(sink_tokens=past)):
        assert torch.equal(fpv2.decode_attention(q, k, v, table, lengths, **kwargs), want)
    assert torch.equal(fpv2.decode_attention(q, k, v, table, past),
                       fpv2.decode_attention(q, k, v, table, 768))


def test_numbers_given_as_tensors_are_read_in_each_call(cuda):
    """A scale or eps in a tensor of one element that changes between two calls."""
    q, k, v, table, lengths = _decode_case(cuda)
    scale = torch.tensor(0.125)
    for x in (0.125, 0.5, 0.25):
        scale.fill_(x)
        assert torch.equal(fpv2.decode_attention(q, k, v, table, lengths, scale=scale),
                           fpv2.decode_attention(q, k, v, table, lengths, scale=x))
    ones, eps = torch.ones(64, dtype=BF16, device=cuda), torch.tensor(1e-6)
    angle = torch.rand((9, 32), device=cuda)
    at = torch.arange(2, device=cuda)

    def rope(e):
        return fpv2.rope_to_pages(q.flatten(1).repeat(1, 2), ones, ones, angle, angle, at, at, k, v,
                                  query_heads=4, eps=e)

    for x in (1e-6, 0.5, 3.0):
        eps.fill_(x)
        assert torch.equal(rope(eps), rope(float(eps)))


def test_growing_lengths_share_a_plan(cuda):
    """An integer length is no part of what is kept for calls of one form."""
    from fpv2.decode import _decode_plan
    q, k, v, table, _ = _decode_case(cuda)
    fpv2.decode_attention(q, k, v, table, 1)
    size = _decode_plan.cache_info().currsize
    got = [fpv2.decode_attention(q, k, v, table, n) for n in range(2, 60)]
    assert _decode_plan.cache_info().currsize == size
    for n, x in zip(range(2, 60), got):
        both = torch.full((2,), n, dtype=torch.int32, device=cuda)
        assert torch.equal(x, fpv2.decode_attention(q, k, v, table, both))


SHAPE = DecoderShape(layers=2, hidden=256, query_heads=8, kv_heads=2, head_dim=64,
                     intermediate=512, vocab=1000)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("token", [-1, -1000, 1000, 2 ** 40])
def test_a_token_outside_the_vocabulary_has_no_logits(cuda, quantized, token):
    model = RandomDecoder(SHAPE, device=cuda, seed=1)
    if quantized:
        model.quantize(32)
    runner = ChunkedPrefillRunner(model, 64)
    prompt = torch.arange(20, device=cuda)
    runner.prefill(prompt, 64)
    want = runner.decode(torch.tensor([999], device=cuda))
    runner.reset()
    runner.prefill(prompt, 64)
    assert torch.equal(runner.decode(torch.tensor(999, dtype=torch.int32, device=cuda)), want)
    assert bool(want.isfinite().all())
    bad = runner.decode(torch.tensor([token], device=cuda))
    assert bool(bad.isnan().all())
    after = runner.decode(torch.tensor([5], device=cuda))  # attends to it
    assert int(fpv2.sample_tokens(after[None], torch.zeros(1, device=cuda))) == -1


def test_generate_ends_with_the_first_row_of_nothing(cuda):
    """A row without a token: all tokens after it are -1 as well."""
    runner = ChunkedPrefillRunner(RandomDecoder(SHAPE, device=cuda, seed=2), 64)
    prompt = torch.arange(20, device=cuda)
    free = runner.generate(prompt, 64, 6, temperature=0.0)
    assert bool((free >= 0).all())
    runner.reset()
    step, calls = runner.decode, []

    def decode(token):
        logits = step(token)
        calls.append(int(token))
        return torch.full_like(logits, -math.inf) if len(calls) == 2 else logits

    runner.decode = decode
    assert runner.generate(prompt, 64, 6, temperature=0.0).tolist() == free[:2].tolist() + [-1] * 4


@pytest.mark.parametrize("heads,hkv", [(8, 2), (40, 1)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("batch,length", [(1, 9000), (3, 1), (700, 90)])
def test_attention_in_the_queries_place(cuda, heads, hkv, dim, batch, length):
    """``out`` may be ``q``: items of one workgroup, of many, and of more heads than a tile."""
    gen = torch.Generator(device=cuda).manual_seed(length)
    q = torch.randn((batch, heads, dim), generator=gen, device=cuda).to(BF16)
    k, v = (torch.randn((40, hkv, 256, dim), generator=gen, device=cuda).to(BF16) for _ in "kv")
    table = torch.randint(0, 40, (batch, 36), generator=gen, device=cuda, dtype=torch.int32)
    want = fpv2.decode_attention(q, k, v, table, length)
    assert fpv2.decode_attention(q, k, v, table, length, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("tokens", [1, 9, 2500])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_in_the_projections_place(cuda, tokens, interleaved):
    """``out`` may be the query heads of the rows themselves."""
    gen = torch.Generator(device=cuda).manual_seed(tokens)
    qkv = torch.randn((tokens, 12 * 128), generator=gen, device=cuda).to(BF16)
    weight = torch.rand(128, generator=gen, device=cuda).to(BF16)
    angle = torch.rand((tokens, 32), generator=gen, device=cuda)
    pages = [torch.zeros((-(-tokens // 16), 2, 16, 128), dtype=BF16, device=cuda) for _ in "kvkv"]

    def call(kp, vp, out):
        return fpv2.rope_to_pages(qkv, weight, weight, angle, angle, 0, 0, kp, vp, query_heads=8,
                                  interleaved=interleaved, out=out)

    rest = qkv[:, 1024:].clone()
    want = call(*pages[:2], None)
    got = call(*pages[2:], qkv[:, :1024].unflatten(1, (8, 128)))
    assert got.data_ptr() == qkv.data_ptr() and torch.equal(got, want)
    assert torch.equal(pages[0], pages[2]) and torch.equal(pages[1], pages[3])
    assert torch.equal(qkv[:, 1024:], rest)


def test_a_cache_as_destination_is_refused_before_the_append(cuda):
    cache = ChunkedPrefill(4, 2, 64, 8, device=cuda)
    q, k = (torch.ones((h, 1, 64), dtype=BF16, device=cuda) for h in (4, 2))
    for out in (cache.k.view(-1)[:256].view(4, 1, 64), cache.v.view(-1)[512:768].view(4, 1, 64)):
        with pytest.raises(ValueError, match="share memory"):
            cache.decode(q, k, k, out=out)
        assert cache.length == 0
    want = cache.decode(q, k, k)
    cache.reset()
    assert torch.equal(cache.decode(q, k, k, out=q), want) and torch.equal(q[None], want)


def test_generate_refuses_before_the_prefill(cuda):
    """What the sampling of the first token would refuse is refused with empty caches."""
    runner = ChunkedPrefillRunner(RandomDecoder(SHAPE, device=cuda, seed=2), 64)
    prompt = torch.arange(20, device=cuda)
    for error, bad in ((RuntimeError, dict(temperature=torch.ones(1))),
                       (RuntimeError, dict(top_k=torch.ones(1, dtype=torch.int32))),
                       (RuntimeError, dict(uniform=torch.rand(2, device=cuda).requires_grad_())),
                       (RuntimeError, dict(top_p=torch.ones(1, device=cuda, requires_grad=True))),
                       (ValueError, dict(chunk=0)), (ValueError, dict(chunk=-3)),
                       (ValueError, dict(tokens=prompt[:0]))):
        with pytest.raises(error):
            runner.generate(**{"tokens": prompt, "chunk": 64, "new_tokens": 2, **bad})
        assert all(cache.length == 0 for cache in runner.caches)
    assert runner.generate(prompt, 64, 2).shape == (2,)
    wide = DecoderShape(layers=1, hidden=64, query_heads=2, kv_heads=1, head_dim=64,
                        intermediate=64, vocab=(1 << 19) + 1)
    runner = ChunkedPrefillRunner(RandomDecoder(wide, device=cuda, seed=2), 64)
    with pytest.raises(ValueError, match="vocabulary"):
        runner.generate(prompt, 64, 2)
    assert runner.caches[0].length == 0


def _late(tensor):
    """A copy of a tensor that is there only after a while, on the current stream."""
    late = torch.zeros_like(tensor)
    torch.cuda._sleep(20_000_000)
    late.copy_(tensor)
    return late


def test_every_operator_runs_on_the_current_stream(cuda):
    """The input of a call on a side stream comes late: a launch elsewhere reads zeros."""
    gen = torch.Generator().manual_seed(4)
    weights = [t.to(cuda) for t in fpv2.quantize_weight(torch.randn((2560, 1024), generator=gen).to(BF16))]
    x = torch.randn((6, 1024), generator=gen).to(BF16).to(cuda)
    logits = torch.randn((3, 40_009), generator=gen).to(cuda)
    short = logits[:, :300].contiguous()
    u = torch.rand(3, generator=gen).to(cuda)
    qkv = torch.randn((5, 8 * 64), generator=gen).to(BF16).to(cuda)
    angle = torch.rand((9, 32), generator=gen).to(cuda)
    pages = [torch.zeros((2, 2, 16, 64), dtype=BF16, device=cuda) for _ in "kv"]

    def rope(rows):
        q = fpv2.rope_to_pages(rows, None, None, angle, angle, 2, 3, *pages, query_heads=4)
        return [q, *(p.clone() for p in pages)]

    cases = [(x, lambda t: [fpv2.quantized_linear(t, *weights)]),
             (x[:1], lambda t: [fpv2.quantized_linear(t, *weights, out_dtype=torch.float32)]),
             (qkv, rope)]
    for rows in (logits, short):
        for kwargs in (dict(), dict(temperature=0.0), dict(top_k=60, top_p=0.9), dict(top_p=0.9),
                       dict(min_p=0.1)):
            cases.append((rows, lambda t, kwargs=kwargs: list(
                fpv2.sample_tokens(t, u, return_logprobs=True, **kwargs))))
    side = torch.cuda.Stream()
    for tensor, call in cases:
        want = call(tensor)
        for page in pages:
            page.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = call(_late(tensor))
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_scale_that_is_no_number_leaves_the_cache(cuda):
    cache = ChunkedPrefill(4, 2, 64, 8, device=cuda)
    q, k = (torch.ones((h, 1, 64), dtype=BF16, device=cuda) for h in (4, 2))
    for bad in ("wide", [0.1], torch.ones(2)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            cache.decode(q, k, k, scale=bad)
        assert cache.length == 0
    cache.decode(q, k, k, scale=0.5)
    assert cache.length == 1


def test_a_step_that_fails_takes_its_token_back(cuda):
    """A refusal inside a later layer leaves every layer's cache as it was."""
    model = RandomDecoder(SHAPE, device=cuda, seed=3)
    runner = ChunkedPrefillRunner(model, 64)
    prompt, token = torch.arange(20, device=cuda), torch.tensor([7], device=cuda)
    runner.prefill(prompt, 64)
    want = runner.decode(token)
    runner.reset()
    runner.prefill(prompt, 64)
    model.layers[1]["qkv"].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        runner.decode(token)
    assert [cache.length for cache in runner.caches] == [20, 20]
    with torch.no_grad():
        model.final_norm, norm = model.final_norm.float(), model.final_norm
        with pytest.raises(ValueError, match="weight"):
            runner.decode(token)
        assert [cache.length for cache in runner.caches] == [20, 20]
        model.final_norm = norm
        assert torch.equal(runner.decode(token), want)
