"""The batch operators together, as a server uses them: many samples of one prompt, a text's
scores, and a prompt that leaves the cache in 8 bits and comes back."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from batch_cases import attention, tolerance
from fpv2 import ChunkedPrefill, prefill_harness
from fpv2.prefill_harness import ChunkedPrefillRunner, DecoderShape, RandomDecoder, rope_tables

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SHAPE = DecoderShape(layers=2, hidden=256, query_heads=8, kv_heads=2, head_dim=64,
                     intermediate=512, vocab=1000)


def _model(cuda, quantized=False):
    """(With a tied head the last token's own logit is about 256 * 0.02 = 5, the others' spread
    a third of one.)"""
    model = RandomDecoder(SHAPE, device=cuda, seed=5)
    if quantized:
        model.quantize(32)
    return model


def _prompt(cuda, n, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, SHAPE.vocab, (n,), generator=gen).to(cuda)


def _forced(runner, tokens, chunk, given):
    """Logits of each of the given tokens, one decode step after the other."""
    runner.reset()
    logits = [runner.prefill(tokens, chunk)]
    for token in given[:-1]:
        logits.append(runner.decode(token))
    return torch.stack(logits)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("samples,n", [(1, 20), (5, 300), (40, 130)])
def test_samples_of_one_prompt(cuda, quantized, samples, n):
    """Each sample's log probabilities are those of one sequence that decodes the same tokens.

    Two runs whose rows differ in bfloat16 roundings here and there: each of 2 layers rounds a
    dozen times by 2^-9 of values about as large as the residual stream, so that the logits
    (|x| <= 6) differ by about 6 sqrt(24) 2^-9 / 4 < 2^-6.6; a log probability by twice that,
    and 8 times that is allowed."""
    runner = ChunkedPrefillRunner(_model(cuda, quantized), n + 8)
    prompt = _prompt(cuda, n)
    uniform = torch.rand((samples, 6), generator=torch.Generator().manual_seed(1)).to(cuda)
    tokens, logprobs = runner.generate_many(prompt, 64, 6, samples, uniform=uniform, top_k=200)
    assert tokens.shape == logprobs.shape == (samples, 6) and bool((tokens >= 0).all())
    assert all(cache.length == n for cache in runner.caches)  # the prompt alone
    assert samples == 1 or len({tuple(x) for x in tokens.tolist()}) > 1
    for b in (0, samples // 2, samples - 1):
        logits = _forced(runner, prompt, 64, tokens[b])
        want = torch.log_softmax(logits.double(), 1).gather(1, tokens[b][:, None])[:, 0]
        assert bool(((logprobs[b] - want).abs() <= 8 * 2.0 ** -5.6).all())
    runner.reset()
    again, scores = runner.generate_many(prompt, 64, 6, samples, uniform=uniform, top_k=200)
    assert torch.equal(again, tokens) and torch.equal(scores, logprobs)


def test_samples_with_settings_of_their_own(cuda):
    """Greedy samples follow the greatest logit; the others take what their numbers say."""
    runner = ChunkedPrefillRunner(_model(cuda), 64)
    prompt = _prompt(cuda, 30)
    temperature = torch.tensor([0.0, 1.0, 0.0, 3.0], device=cuda)
    tokens, logprobs = runner.generate_many(prompt, 64, 5, 4, temperature=temperature)
    assert torch.equal(tokens[0], tokens[2]) and torch.equal(logprobs[0], logprobs[2])
    first = _forced(runner, prompt, 64, tokens[0][:1])[0]
    assert int(tokens[0, 0]) == int(first.argmax())
    for bad in (dict(samples=0), dict(new_tokens=True), dict(chunk=0), dict(tokens=prompt[:0]),
                dict(uniform=torch.rand(4, 4, device=cuda)), dict(temperature=temperature[:3])):
        runner.reset()
        with pytest.raises(ValueError):
            runner.generate_many(**{**dict(tokens=prompt, chunk=64, new_tokens=5, samples=4), **bad})
        assert all(cache.length == 0 for cache in runner.caches)
    with pytest.raises(RuntimeError):
        runner.generate_many(prompt, 64, 5, 4, temperature=temperature.cpu())
    runner.prefill(prompt, 64)
    with pytest.raises(ValueError, match="empty caches"):
        runner.generate_many(prompt, 64, 5, 4)


def test_samples_past_the_capacity(cuda):
    """The prompt fills the caches; the new tokens lie in pages of their own."""
    runner = ChunkedPrefillRunner(_model(cuda), 50)
    tokens, _ = runner.generate_many(_prompt(cuda, 50), 64, 7, 3)
    assert tokens.shape == (3, 7) and bool((tokens >= 0).all())


@pytest.mark.parametrize("n,chunk", [(1, 8), (2, 8), (65, 64), (700, 128), (1300, 1024)])
def test_scores_of_a_text(cuda, n, chunk):
    """The log probabilities of a text's tokens: those of its prefixes' last logits.

    Tolerance: as above; the prefix's chunks end elsewhere, the rows are the same."""
    runner = ChunkedPrefillRunner(_model(cuda), 1300, attention="dense")
    text = _prompt(cuda, n, seed=n)
    scores = runner.score(text, chunk)
    assert scores.shape == (n - 1,) and scores.dtype == torch.float32
    assert bool((scores < 0).all())
    for i in {1, 2, n // 2, n - 1} & set(range(1, n)):
        runner.reset()
        logits = runner.prefill(text[:i], chunk).double()
        want = torch.log_softmax(logits, 0)[text[i]]
        assert abs(float(scores[i - 1] - want)) <= 8 * 2.0 ** -5.6
    runner.reset()
    with pytest.raises(ValueError):
        runner.score(text, 0)
    with pytest.raises(ValueError):
        runner.score(text[:0], 4)
    runner.prefill(text, chunk)
    with pytest.raises(ValueError, match="empty caches"):
        runner.score(text, chunk)


def test_a_prompt_leaves_in_8_bits_and_comes_back(cuda):
    """A prefilled prompt's keys and values in 8-bit pages: single tokens attend there, and a
    prefill that goes on reads them back.

    Tolerance: a key is off by at most a 254th of its row's greatest value, which moves a score
    by scale sum |q| a / 254 at most, and a weight by twice that share; a value by its row's
    254th.  All else is far below (bfloat16's 2^-9 of the result and of the weights)."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    heads, hkv, dim, n, page = 8, 2, 128, 900, 16
    prefill = ChunkedPrefill(heads, hkv, dim, 1200, device=cuda)
    q, k, v = (torch.randn((h, n, dim), generator=gen, device=cuda).to(BF16) for h in (heads, hkv, hkv))
    prefill.step(q, k, v)
    pages = -(-1000 // page)
    cache = [x for _ in "kv" for x in (torch.zeros((pages, hkv, page, dim), dtype=torch.int8, device=cuda),
                                       torch.zeros((pages, hkv, page), device=cuda))]
    order = torch.randperm(pages, generator=gen, device=cuda)
    t = torch.arange(1000, device=cuda)
    slots = order[t // page] * page + t % page
    fpv2.quantize_to_pages(prefill.k[:, :n].transpose(0, 1), prefill.v[:, :n].transpose(0, 1), slots[:n], *cache)
    table = order[None].to(torch.int32)
    # three tokens go on over the codes, and over the cache as it was
    for i in range(3):
        q, k, v = (torch.randn((h, 1, dim), generator=gen, device=cuda).to(BF16) for h in (heads, hkv, hkv))
        want = prefill.decode(q, k, v)[0].transpose(0, 1).double()
        fpv2.quantize_to_pages(k.transpose(0, 1), v.transpose(0, 1), slots[n + i:n + i + 1], *cache)
        got = fpv2.quantized_decode_attention(q.transpose(0, 1), *cache, table, n + i + 1).double()
        size = float(prefill.k[:, :n + i + 1].abs().max()) / 254
        score = float(q.abs().float().sum(-1).max()) * size * dim ** -0.5
        greatest = float(prefill.v[:, :n + i + 1].abs().max())
        assert bool(((got - want).abs() <= 2 * score * greatest + greatest / 254 + 2.0 ** -7 * greatest).all())
        assert float((got - want).abs().mean()) <= 0.01  # (the values of 900 keys: about 0.05)
    # the conversation comes back into a prefill that goes on
    later = ChunkedPrefill(heads, hkv, dim, 1200, device=cuda)
    rows = fpv2.dequantize_pages(*cache, table, n + 3, tokens=n + 3)
    later.append(rows[0][0], rows[1][0])
    for x, y in ((later.k, prefill.k), (later.v, prefill.v)):
        x, y = x[:, :n + 3].float(), y[:, :n + 3].float()
        assert bool(((x - y).abs() <= y.abs().amax(-1, keepdim=True) * (1 / 254 + 2.0 ** -8)).all())
    chunk = [torch.randn((h, 200, dim), generator=gen, device=cuda).to(BF16) for h in (heads, hkv, hkv)]
    a, b = later.step(*chunk).float(), prefill.step(*chunk).float()
    assert float((a - b).abs().mean()) <= 0.01


def test_scores_of_samples_and_alternatives(cuda):
    """Sampled tokens, their log probabilities and the alternatives agree with one another."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    logits = 3 * torch.randn((33, 50_003), generator=gen, device=cuda)
    logits[:, ::7] = -math.inf
    logits[4] = -math.inf
    tokens, kept = fpv2.sample_tokens(logits, torch.rand(33, generator=gen, device=cuda), return_logprobs=True)
    res = fpv2.token_logprobs(logits, tokens, top=4)
    assert int(tokens[4]) == -1 and float(res.logprobs[4]) == -math.inf and float(res.entropy[4]) == 0
    live = tokens >= 0
    assert bool(((res.logprobs - kept).abs() <= 1e-4)[live].all())  # (no filter: the same shares)
    greedy = fpv2.sample_tokens(logits, torch.zeros(33, device=cuda), temperature=0.0)
    assert torch.equal(res.top_tokens[:, 0], greedy)
    assert bool((res.top_logprobs.diff(dim=1)[live] <= 0).all())


def test_refused_before_the_prompt_is_prefilled(cuda):
    """What ``score`` and ``generate_many`` cannot do leaves the caches empty."""
    runner = ChunkedPrefillRunner(_model(cuda), 64)
    text = _prompt(cuda, 40)
    for bad, error in ((text.cpu(), RuntimeError), (text.to(torch.uint8), ValueError),
                       (text.float(), ValueError), (text[None], ValueError)):
        with pytest.raises(error):
            runner.score(bad, 16)
        assert all(cache.length == 0 for cache in runner.caches)
    heads = DecoderShape(layers=1, hidden=64, query_heads=512, kv_heads=32, head_dim=64, intermediate=64, vocab=100)
    for shape, samples in ((SHAPE, 65_536), (heads, 32_768)):
        many = ChunkedPrefillRunner(RandomDecoder(shape, device=cuda, seed=1), 64)
        with pytest.raises(ValueError, match="samples must be at most"):
            many.generate_many(text % 100, 16, 2, samples)
        assert all(cache.length == 0 for cache in many.caches)
    runner.model.embed = torch.zeros(((1 << 19) + 1, SHAPE.hidden), dtype=BF16, device=cuda)
    with pytest.raises(ValueError, match="vocabulary"):
        runner.score(text, 16)
    assert all(cache.length == 0 for cache in runner.caches)


def test_angles_of_the_decode_step_stay(cuda):
    """Samples past the capacity take angles of their own: a captured ``decode`` reads the runner's."""
    runner = ChunkedPrefillRunner(_model(cuda), 50)
    prompt = _prompt(cuda, 40)
    runner.prefill(prompt, 64)
    runner.decode(prompt[:1])
    kept = [x.data_ptr() for x in runner._tables]
    runner.reset()
    tokens, _ = runner.generate_many(prompt, 64, 30, 2, temperature=0.0)
    assert [x.data_ptr() for x in runner._tables] == kept
    wide = ChunkedPrefillRunner(runner.model, 70)
    assert torch.equal(wide.generate_many(prompt, 64, 30, 2, temperature=0.0)[0], tokens)


def _later(k, by):
    """Rotated keys ``[Hkv, n, D]`` as they would be ``by`` positions later."""
    cos, sin = (x.cpu().double() for x in rope_tables(SHAPE, torch.tensor([by])))
    half = k.shape[-1] // 2
    return k * cos + torch.cat([-k[..., half:], k[..., :half]], -1) * sin


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("samples,n", [(1, 20), (3, 3), (5, 300), (40, 130)])
def test_steps_of_samples(cuda, monkeypatch, quantized, samples, n):
    """Every attention call of every step sees the prompt and the sample's own tokens, each at its
    position, and its result is theirs; the logits are those of a sequence that decodes the same tokens.

    Tolerances.  Keys and values against the other run's: rows of a projection differ by a rounding to
    bfloat16 on either side (2^-8 of an element), a key's norm by as much, its rotation mixes two
    elements: 6 2^-8 < 2^-5 of the row's greatest.  In the second layer the streams differ by some 12 roundings
    of 2^-9 / sqrt(3) (0.4 %), which change a projection by as much of its deviation, five times that at
    most among these rows: still below 2^-5 of the greatest, more than twice the deviation.  Attention: of the
    call's own operands, as ``batch_cases`` derives it.  Logits: 24 roundings are 0.6 % of a stream
    of deviation 1, times 16 rows of 0.02: a deviation of 0.002, and 2^-5.6 is ten of them.

    What these see, planted in the reference: a key one position off in every call, the prompt's last
    key or the last own one left out in some."""
    layers, new = SHAPE.layers, 6
    calls, logits = [], []

    def attend(q, *args):
        out = fpv2.shared_prefix_attention(q, *args)
        calls.append([x.cpu() if isinstance(x, torch.Tensor) else x for x in (q, *args, out)])
        return out

    def score(rows, tokens):
        logits.append(rows)
        return fpv2.token_logprobs(rows, tokens)

    monkeypatch.setattr(prefill_harness, "shared_prefix_attention", attend)
    monkeypatch.setattr(prefill_harness, "token_logprobs", score)
    model = _model(cuda, quantized)
    runner = ChunkedPrefillRunner(model, n + 8)
    prompt = _prompt(cuda, n)
    uniform = torch.rand((samples, new), generator=torch.Generator().manual_seed(1)).to(cuda)
    tokens, logprobs = runner.generate_many(prompt, 64, new, samples, uniform=uniform, top_k=200)
    assert len(calls) == layers * (new - 1) and len(logits) == new
    seen = [0, 0]
    for b in {0, samples // 2, samples - 1}:
        other = ChunkedPrefillRunner(model, n + 8)
        want = _forced(other, prompt, 64, tokens[b])
        got = torch.stack([rows[b] for rows in logits])
        assert bool(((got - want).abs() <= 2.0 ** -5.6).all())
        given = torch.log_softmax(got.double(), 1).gather(1, tokens[b][:, None])[:, 0]
        assert bool(((logprobs[b] - given).abs() <= 1e-5).all())
        for c, (q, pk, pv, table, prefix, k, v, own_table, own, out) in enumerate(calls):
            step, cache = c // layers, other.caches[c % layers]
            assert table is None and own_table is None and prefix == n and own == step + 1
            held = [torch.cat([x[0, :, :prefix], y[b, :, :own]], 1).double() for x, y in ((pk, k), (pv, v))]
            for x, y in zip(held, (cache.k, cache.v)):
                y = y[:, :n + own].cpu().double()
                assert torch.equal(x[:, :n], y[:, :n])
                bound = 2.0 ** -5 * y.abs().amax(-1, keepdim=True)
                assert bool(((x - y).abs() <= bound).all())
            for by in (-1, 1):
                wrong = _later(held[0], by)
                assert bool(((wrong - held[0]).abs() > bound).any(-1).all())
            result, mass, size = attention(q[b], *held, 0.125)
            tol = tolerance(result, mass, size, n + own, 64, BF16, BF16)
            assert bool(((out[b].double() - result).abs() <= tol).all())
            for i, gone in enumerate((n - 1, n + own - 1)):
                keep = torch.arange(n + own) != gone
                wrong = attention(q[b], *(x[:, keep] for x in held), 0.125)[0]
                seen[i] += int(((wrong - result).abs() > 2 * tol).any())
    assert min(seen) > 0, seen


@pytest.mark.parametrize("n,chunk", [(2, 8), (65, 64), (700, 128), (1300, 1024)])
def test_scores_are_of_the_next_tokens(cuda, n, chunk):
    """Each row's log probability of the token behind it, from the same chunks' last rows.

    Tolerance: a logit is a float32 sum of 256 products, off by 256 2^-24 of their size; the
    log probability by twice the largest of these and 2^-16 (sums of 1000 weights).  Planted in the reference:
    rows or tokens one off."""
    model = _model(cuda)
    text = _prompt(cuda, n, seed=n)
    scores = ChunkedPrefillRunner(model, n, attention="dense").score(text, chunk).cpu().double()
    rows = [prefill_harness._add_rms_norm(x, delta, model.final_norm, SHAPE.rms_eps).cpu().double()
            for x, delta, _ in ChunkedPrefillRunner(model, n, attention="dense")._chunks(text, chunk)]
    rows, embed, text = torch.cat(rows), model.embed.cpu().double(), text.cpu()
    tol = 2 * 256 * 2.0 ** -24 * float((rows.abs() @ embed.abs().T).max()) + 2.0 ** -16
    logs = torch.log_softmax(rows @ embed.T, 1)
    want = logs[:-1].gather(1, text[1:, None])[:, 0]
    assert bool(((scores - want).abs() <= tol).all())
    for wrong in (logs[1:].gather(1, text[1:, None])[:, 0], logs[:-1].gather(1, text[:-1, None])[:, 0]):
        assert bool(((want - wrong).abs() > 2 * tol)[:n - 1].any())
