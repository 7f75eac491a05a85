"""``fpv2.sample_tokens`` against the rule in float64 on the CPU.

Tokens must be equal.  The kernel rounds each weight to 2^-44 of the greatest;
the reference's weights are doubles, so a token could differ only where a border
or a number falls within V 2^-45 of a running weight.  The reference finds such rows,
and with these seeds there are none.

A logprob is a float32 of a float64 difference: half a step, and 2^-44 V of
relative error in the kept weight.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _reference(row, u, temperature, top_k, top_p, min_p):
    """(token, logprob, near): one row (CPU) by the rule, in float64."""
    x = torch.where(torch.isnan(row), -math.inf, row.double())
    top = x.max()
    if top == -math.inf:
        return -1, -math.inf, False
    if temperature <= 0:
        return int((x == top).nonzero()[0]), 0.0, False
    w = torch.where(x == top, 1.0, torch.exp((x - top) / temperature))
    order = torch.sort(x, descending=True, stable=True).indices
    n = x.numel() if top_k <= 0 else min(int(top_k), x.numel())
    run = w[order].cumsum(0)
    slack = x.numel() * 2.0 ** -45
    near = False
    if top_p < 1:
        share = top_p * run[n - 1]
        near |= bool(((run[:n] - share).abs() <= slack).any()) and not bool((run[:n] == share).any())
        n = min(n, 1 + int((run[:n] < share).sum()))
    n = max(1, min(n, int((w[order][:n] >= min(min_p, 1.0)).sum())))
    kept = torch.zeros_like(w)
    kept[order[:n]] = w[order[:n]]
    run = kept.cumsum(0)
    target = min(max(float(u), 0.0), 1.0) * run[-1]
    # (equal is not near: sums of weights of 1 are exact on both sides)
    near |= bool((((run - target).abs() <= slack) & (run != target) & (kept > 2 * slack)).any()) and 0 < u < 1
    token = int((run <= target).sum())
    if token >= x.numel():
        token = int((kept > 2.0 ** -45).nonzero()[-1])
    return token, float(torch.log(w[token] / run[-1])), near


def _check(cuda, logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    dev = lambda x: x.to(cuda) if isinstance(x, torch.Tensor) else x  # noqa: E731
    tokens, logprobs = fpv2.sample_tokens(
        dev(logits), dev(uniform), temperature=dev(temperature), top_k=dev(top_k),
        top_p=dev(top_p), min_p=dev(min_p), return_logprobs=True)
    at = lambda x, b: float(x[b]) if isinstance(x, torch.Tensor) else x  # noqa: E731
    tokens, logprobs = tokens.cpu(), logprobs.cpu()
    for b in range(logits.shape[0]):
        want, logp, near = _reference(logits[b].float(), uniform[b], at(temperature, b), at(top_k, b),
                                      at(top_p, b), at(min_p, b))
        assert not near, f"row {b}: choose another seed"
        assert int(tokens[b]) == want, f"row {b}"
        if math.isinf(logp):
            assert float(logprobs[b]) == logp
        else:
            assert abs(float(logprobs[b]) - logp) <= 2.0 ** -23 * abs(logp) + logits.shape[1] * 2.0 ** -43
    return tokens


def _logits(gen, batch, vocab, dtype, spread=2.5):
    x = spread * torch.randn((batch, vocab), generator=gen)
    x[:, :: max(1, vocab // 7)] += 6
    return x.to(dtype)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9),
            dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=0.0),
            dict(top_k=50, top_p=0.95, temperature=0.8), dict(top_k=5000, top_p=0.99),
            dict(top_k=300, min_p=0.01, top_p=0.5, temperature=1.7), dict(temperature=30.0, top_p=0.7),
            dict(temperature=1e-4, top_k=3), dict(temperature=1e30, top_p=0.4)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 32003, 151936])
def test_settings(cuda, dtype, vocab):
    gen = torch.Generator().manual_seed(vocab)
    logits = _logits(gen, 4, vocab, dtype)
    for setting in SETTINGS:
        _check(cuda, logits, torch.rand(4, generator=gen), **setting)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_settings_of_each_row(cuda, dtype):
    gen = torch.Generator().manual_seed(1)
    n = len(SETTINGS)
    rows = {name: torch.tensor([s.get(name, default) for s in SETTINGS],
                               dtype=torch.int32 if name == "top_k" else F32)
            for name, default in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    logits = _logits(gen, n, 20011, dtype)
    uniform = torch.rand(n, generator=gen)
    tokens = _check(cuda, logits, uniform, **rows)
    for b in (0, 4, 9, 11):  # a row alone
        one = fpv2.sample_tokens(logits[b:b + 1].to(cuda), uniform[b:b + 1].to(cuda),
                                 **{k: v[b:b + 1].to(cuda) for k, v in rows.items()})
        assert int(one[0]) == int(tokens[b])


@pytest.mark.parametrize("vocab", [7, 4096, 100_003])
def test_equal_logits(cuda, vocab):
    """Ties go to the lowest index, also where they are all there is."""
    gen = torch.Generator().manual_seed(vocab)
    flat = torch.full((4, vocab), -3.25)
    u = torch.tensor([0.0, 0.37, 0.8125, 0.999])
    for setting in SETTINGS:
        _check(cuda, flat, u, **setting)
    # exact borders: half of the weight, a quarter of the tokens
    _check(cuda, flat, torch.full((4,), 0.5), top_p=0.5, top_k=max(1, vocab // 4))
    steps = torch.randint(0, 3, (4, vocab), generator=gen).float()
    for setting in SETTINGS:
        _check(cuda, steps, u, **setting)


def test_masked_infinite_and_nan_logits(cuda):
    gen = torch.Generator().manual_seed(2)
    logits = _logits(gen, 8, 5003, F32)
    logits[0] = -math.inf                        # nothing left
    logits[1, 1:] = -math.inf                    # one token
    logits[2, :5000] = -math.inf                 # three tokens, fewer than top-k
    logits[3, 100] = math.nan                    # NaN counts as -inf
    logits[4] = math.nan
    logits[5, 17] = logits[5, 4000] = math.inf   # two infinite ones share the weight
    logits[6] = torch.finfo(F32).min             # masks of the lowest value
    logits[7, 50:] = torch.finfo(F32).min
    for setting in SETTINGS:
        tokens = _check(cuda, logits, torch.rand(8, generator=gen), **setting)
        assert int(tokens[0]) == -1 and int(tokens[4]) == -1


def test_uniform_numbers_at_their_ends(cuda):
    gen = torch.Generator().manual_seed(3)
    logits = _logits(gen, 6, 3001, BF16)
    logits[:, 0] = logits[:, -1] = -math.inf
    u = torch.tensor([0.0, 1.0, 2.0 ** -126, 1 - 2.0 ** -24, -5.0, 9.0])
    for setting in SETTINGS:
        _check(cuda, logits, u, **setting)


def test_tiny_weights_at_the_end_of_the_order(cuda):
    """Logits over 80 units: weights below 2^-45 are never chosen."""
    logits = torch.linspace(40, -40, 2000)[None].repeat(3, 1)
    _check(cuda, logits, torch.tensor([0.0, 0.6, 0.9999]))
    _check(cuda, logits, torch.tensor([0.0, 0.6, 0.9999]), top_k=1999, top_p=0.9999)


def test_strides(cuda):
    gen = torch.Generator().manual_seed(4)
    logits = _logits(gen, 3, 1003, F16).to(cuda)
    u = torch.rand(3, generator=gen).to(cuda)
    want = fpv2.sample_tokens(logits, u, top_p=0.9)
    wide = torch.full((3, 1111), 50.0, dtype=F16, device=cuda)
    wide[:, 5:1008] = logits
    assert torch.equal(fpv2.sample_tokens(wide[:, 5:1008], u, top_p=0.9), want)
    assert torch.equal(fpv2.sample_tokens(logits.T.contiguous().T, u, top_p=0.9), want)
    assert torch.equal(fpv2.sample_tokens(logits[:1].expand(3, -1), u, top_p=0.9),
                       fpv2.sample_tokens(logits[:1].repeat(3, 1), u, top_p=0.9))
    assert fpv2.sample_tokens(logits[:0], u[:0]).shape == (0,)


def test_shares_follow_the_weights(cuda):
    """Evenly spaced numbers draw each token as often as its weight says, within one."""
    gen = torch.Generator().manual_seed(5)
    row, n = torch.randn(40, generator=gen), 4096
    u = (torch.arange(n) + 0.5) / n
    tokens = fpv2.sample_tokens(row.expand(n, 40).contiguous().to(cuda), u.to(cuda), temperature=0.9)
    share = torch.softmax(row.double() / 0.9, 0) * n
    assert bool(((torch.bincount(tokens.cpu(), minlength=40) - share).abs() <= 1).all())


def test_captured(cuda):
    gen = torch.Generator().manual_seed(6)
    logits, u = _logits(gen, 5, 30011, F32).to(cuda), torch.rand(5, generator=gen).to(cuda)
    def call():
        return fpv2.sample_tokens(logits, u, top_k=60, top_p=0.9, return_logprobs=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for step in range(4):
        u.copy_(torch.rand(5, generator=gen))
        logits.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def test_settings_out_of_range_in_tensors(cuda):
    """NaN and negative temperatures are greedy, other settings out of range no limit."""
    gen = torch.Generator().manual_seed(7)
    logits, u = _logits(gen, 4, 5003, F32), torch.rand(4, generator=gen)
    dev = logits.to(cuda)
    t = torch.tensor([math.nan, -1.0, 0.0, -math.inf], device=cuda)
    assert torch.equal(fpv2.sample_tokens(dev, u.to(cuda), temperature=t).cpu(), logits.argmax(1))
    want = fpv2.sample_tokens(dev, u.to(cuda))
    got = fpv2.sample_tokens(dev, u.to(cuda), top_k=torch.tensor([-5, 0, 5003, 2 ** 31 - 1], device=cuda,
                                                                 dtype=torch.int32),
                             top_p=torch.tensor([1.0, 7.0, math.inf, math.nan], device=cuda),
                             min_p=torch.tensor([-1.0, math.nan, 0.0, -math.inf], device=cuda))
    assert torch.equal(got, want)
    hot = fpv2.sample_tokens(dev, u.to(cuda), temperature=torch.full((4,), math.inf, device=cuda))
    assert torch.equal(hot, fpv2.sample_tokens(dev, u.to(cuda), temperature=1e30))
    top = fpv2.sample_tokens(dev, u.to(cuda), min_p=torch.full((4,), 9.0, device=cuda))
    assert torch.equal(top.cpu(), logits.argmax(1))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_borders_of_each_kind(cuda, dtype):
    """Long rows whose borders have few tokens above them, many above and few next to
    them, hundreds and thousands next to them."""
    gen = torch.Generator().manual_seed(8)
    vocab = 40_009
    logits = 0.5 * torch.randn((6, vocab), generator=gen) - 30
    at = torch.randperm(vocab, generator=gen)
    logits[:, at[:5]] = 9 + torch.rand((6, 5), generator=gen)
    logits[:, at[5:1005]] = 2 + 4 * torch.rand((6, 1000), generator=gen)
    logits[:, at[1005:1705]] = 1 + 0.01 * torch.rand((6, 700), generator=gen)
    logits[:, at[1705:7705]] = -1 + 0.01 * torch.rand((6, 6000), generator=gen)
    logits = logits.to(dtype)
    u = torch.tensor([0.0, 1.0, 0.25, 0.5, 0.75, 0.9375])
    for top_p in (0.01, 0.2, 0.6, 0.9, 0.955, 0.975, 0.985, 0.99, 0.998, 0.9999):
        _check(cuda, logits, u, top_p=top_p)
        _check(cuda, logits, u, top_p=top_p, top_k=900, min_p=1e-6)
    for top_k in (3, 31, 33, 64, 127, 129, 255, 256, 257, 300, 1300, 1705, 4000, 30_000):
        _check(cuda, logits, u, top_k=top_k)
        _check(cuda, logits, u, top_k=top_k, top_p=0.97, temperature=1.5)
