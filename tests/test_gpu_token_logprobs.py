"""``fpv2.token_logprobs`` against the formulas in float64 on the CPU.

Tolerance: an exponent is one float32 rounding of at most 2^-24 of its size and log2 e is off by
2^-26 of it, which scales the logits; a weight by 2^-22 more; a thread sums at most n / 256 + 32
weights, and their joins are six and more.  So with spread = max - (the smallest logit that weighs
2^-30 or is given), the logarithm of the sum is off by (n / 256 + 64) 2^-24 + 2^-22 + spread
2^-23, a log probability by as much and the roundings of its own size, and the entropy by as much
times 1 + the mean distance from the greatest logit."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _reference(logits, tokens, top):
    """On the CPU: log probabilities, entropies, alternatives, and the tolerances of the first two."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=2.0 ** 126)
    x = torch.where(x == -math.inf, x, x.clamp(min=-2.0 ** 126))
    greatest = x.amax(1, keepdim=True)
    none = greatest == -math.inf
    shifted = torch.where(none, -math.inf, x - torch.where(none, 0.0, greatest))
    p = shifted.exp()
    total = p.sum(1, keepdim=True)
    logs = shifted - total.log()
    p = p / total
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    given = logs.gather(1, torch.where(inside, tokens, 0).long()[:, None])[:, 0]
    given = torch.where(inside & ~none[:, 0], given, -math.inf)
    order = torch.argsort(torch.where(logits.isnan(), -math.inf, logits.float()), dim=1, descending=True,
                          stable=True)[:, :top]
    best = logs.gather(1, order)
    missing = (x.gather(1, order) == -math.inf)
    order, best = torch.where(missing, -1, order), torch.where(missing, -math.inf, best)
    if order.shape[1] < top:
        more = top - order.shape[1]
        order = torch.nn.functional.pad(order, (0, more), value=-1)
        best = torch.nn.functional.pad(best, (0, more), value=-math.inf)
    distance = torch.where(p > 0, -p * shifted, 0.0).sum(1)
    base = (x.shape[1] / 256 + 64) * 2.0 ** -24 + 2.0 ** -22 + 21 * 2.0 ** -23
    return (given, torch.where(none[:, 0], 0.0, entropy), order, best,
            base, base * (1 + distance + entropy))


def _check(cuda, logits, tokens, top):
    got = fpv2.token_logprobs(logits.to(cuda), tokens.to(cuda), top=top)
    given, entropy, order, best, base, entropy_tol = _reference(logits.cpu(), tokens, top)
    assert got.logprobs.dtype == torch.float32 and got.top_tokens.dtype == torch.int64
    assert got.top_tokens.shape == got.top_logprobs.shape == (logits.shape[0], top)
    assert torch.equal(got.top_tokens.cpu(), order)
    for a, b in ((got.logprobs.cpu(), given), (got.top_logprobs.cpu(), best)):
        a, inf = a.double(), b == -math.inf
        assert torch.equal(a == -math.inf, inf)
        assert bool(((a - b).abs() <= base + b.abs() * 2.0 ** -22)[~inf].all())
    err = (got.entropy.cpu().double() - entropy).abs()
    none = entropy_tol.isnan()
    assert bool((err <= entropy_tol)[~none].all()) and not got.entropy.cpu()[none].any()
    return got


def _logits(gen, rows, vocab, dtype):
    x = 2.5 * torch.randn((rows, vocab), generator=gen)
    likely = torch.randint(0, vocab, (rows, 5), generator=gen)
    x.scatter_(1, likely, 5 + 8 * torch.rand(likely.shape, generator=gen))
    return x.to(dtype), torch.where(torch.arange(rows) % 2 == 0, likely[:, 0],
                                    torch.randint(0, vocab, (rows,), generator=gen))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 255, 1000, 8191, 8192, 8193, 50001, 151936])
@pytest.mark.parametrize("rows,top", [(1, 20), (3, 0), (5, 32)])
def test_sizes(cuda, dtype, vocab, rows, top):
    gen = torch.Generator().manual_seed(vocab + rows)
    _check(cuda, *_logits(gen, rows, vocab, dtype), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 300, 1100])
@pytest.mark.parametrize("top", [0, 1, 5])
def test_many_rows(cuda, dtype, rows, top):
    """Rows of several workgroups, and a workgroup a row."""
    gen = torch.Generator().manual_seed(rows)
    _check(cuda, *_logits(gen, rows, 20_011, dtype), top)


@pytest.mark.parametrize("top", [1, 2, 3, 8, 17, 31, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 30_000), (600, 3001)])
def test_ties(cuda, top, rows, vocab):
    """Few different values: equal logits in the order of their tokens; and rows in rising and
    falling order, of which every logit or none enters the list."""
    gen = torch.Generator().manual_seed(top)
    x = torch.randint(0, 12, (rows, vocab), generator=gen).float()
    tokens = torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32)
    _check(cuda, x, tokens, top)
    ramp = torch.arange(vocab).float().expand(rows, vocab) / 1000
    _check(cuda, ramp.contiguous(), tokens, top)
    _check(cuda, -ramp, tokens, top)
    _check(cuda, torch.zeros((rows, vocab), dtype=torch.bfloat16), tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [100, 40_000])
def test_masked_and_extreme_logits(cuda, dtype, vocab):
    """Rows of nothing, of one token, of the type's lowest value, infinities, NaN, large offsets."""
    gen = torch.Generator().manual_seed(vocab)
    x, tokens = _logits(gen, 14, vocab, torch.float32)
    low = torch.finfo(dtype).min
    x = x.to(dtype)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 77] = -3.0
    x[2] = low                        # one value for all: a uniform distribution
    x[3, ::2] = low
    x[4, ::3] = -math.inf
    x[5, 5:9] = math.inf
    x[6, 3] = math.nan
    x[7] = math.nan
    x[8] = (x[8].float() + 3e4).to(dtype)
    x[9] = (x[9].float() - 3e4).to(dtype)
    x[10] = torch.finfo(dtype).max
    x[11] = -math.inf
    x[11, 20], x[11, 10] = math.inf, low
    x[12, :50] = math.nan
    x[13] = math.inf
    tokens[0], tokens[1], tokens[4], tokens[5], tokens[6], tokens[11] = 3, 77, 3, 6, 3, 10
    got = _check(cuda, x, tokens, 20)
    assert float(got.logprobs[1]) == 0 and got.top_tokens[1].tolist() == [77] + [-1] * 19
    assert got.top_tokens[7].tolist() == [-1] * 20
    _check(cuda, x, tokens, 0)


def test_tokens_outside_the_vocabulary(cuda):
    gen = torch.Generator().manual_seed(1)
    x, _ = _logits(gen, 6, 1000, torch.float32)
    for dtype, far in ((torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 62)):
        tokens = torch.tensor([-1, 1000, far, -far, 0, 999], dtype=dtype)
        got = _check(cuda, x, tokens, 1)
        assert bool((got.logprobs[:4] == -math.inf).all()) and bool(got.logprobs[4:].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 1100])
def test_strides(cuda, dtype, rows):
    """Rows off the 16-byte grid, padded, broadcast and not contiguous; what lies around a row
    does not count."""
    gen = torch.Generator().manual_seed(rows)
    x, tokens = _logits(gen, rows, 1003, dtype)
    want = _check(cuda, x, tokens, 6)
    wide = torch.full((rows, 1021), math.inf, dtype=dtype, device=cuda)
    for first in range(0, 9):
        view = wide[:, first:first + 1003]
        view.copy_(x)
        got = fpv2.token_logprobs(view, tokens.to(cuda), top=6)
        # (a row's threads take other logits where it starts elsewhere: sums in another order)
        assert torch.equal(got.top_tokens, want.top_tokens)
        for a, b in zip(got, want):
            assert bool(((a - b).abs() <= 2e-5 * (1 + b.abs())).all())
        view.fill_(math.inf)
    turned = x.t().contiguous().to(cuda).t()
    for a, b in zip(fpv2.token_logprobs(turned, tokens.to(cuda), top=6), want):
        assert torch.equal(a, b)
    one = x[:1].to(cuda).expand(rows, -1)
    got = fpv2.token_logprobs(one, tokens[:1].to(cuda).expand(rows).contiguous(), top=6)
    assert bool((got.top_tokens == want.top_tokens[:1]).all())


def test_rows_past_32_bits(cuda):
    """Rows whose first logits lie behind 2^31 elements."""
    vocab, rows = 400_000, 5600
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=cuda)
    x[-1, 399_999], x[-2, 7] = 30.0, 20.0
    tokens = torch.full((rows,), 399_999, device=cuda)
    got = fpv2.token_logprobs(x, tokens, top=2)
    assert got.top_tokens[-1].tolist() == [399_999, 0] and got.top_tokens[-2].tolist() == [7, 0]
    assert abs(float(got.logprobs[-1])) < 1e-6 and abs(float(got.logprobs[-3]) + math.log(vocab)) < 1e-4
    assert bool((got.logprobs[:-2] == got.logprobs[0]).all())


def test_same_in_every_batch(cuda):
    """A row alone, among few and among many: the same alternatives, and sums within rounding."""
    gen = torch.Generator().manual_seed(2)
    x, tokens = _logits(gen, 1, 151936, torch.float32)
    alone = fpv2.token_logprobs(x.to(cuda), tokens.to(cuda), top=20)
    many = fpv2.token_logprobs(x.expand(1300, -1).contiguous().to(cuda), tokens.expand(1300).contiguous().to(cuda),
                               top=20)
    assert bool((many.top_tokens == alone.top_tokens).all())
    assert bool((many.logprobs == many.logprobs[0]).all())
    assert abs(float(many.logprobs[0] - alone.logprobs[0])) < 1e-4
    again = fpv2.token_logprobs(x.to(cuda), tokens.to(cuda), top=20)
    assert all(torch.equal(a, b) for a, b in zip(alone, again))


def test_graph_replays(cuda):
    gen = torch.Generator().manual_seed(3)
    cases = [[t.to(cuda) for t in _logits(gen, rows, 30_011, torch.float32)] for rows in (2, 1100)]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for args in cases:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            fpv2.token_logprobs(*args, top=9)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fpv2.token_logprobs(*args, top=9))
        graphs.append(graph)
    for _ in range(4):
        for x, tokens in cases:
            x.mul_(0.9)
            tokens.add_(1)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, args in zip(outs, cases):
            assert all(torch.equal(a, b) for a, b in zip(out, fpv2.token_logprobs(*args, top=9)))


def test_runs_on_the_current_stream(cuda):
    gen = torch.Generator().manual_seed(4)
    for rows in (2, 1100):
        x, tokens = (t.to(cuda) for t in _logits(gen, rows, 9000, torch.float32))
        want = fpv2.token_logprobs(x, tokens, top=4)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            late = torch.zeros_like(x)
            torch.cuda._sleep(20_000_000)
            late.copy_(x)
            got = fpv2.token_logprobs(late, tokens, top=4)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
