"""A decode step's operators together: over the caches of a chunked prefill
(``ChunkedPrefill.decode``, ``ChunkedPrefillRunner.decode`` / ``generate``) and over a
paged batch, against float64 on the CPU.

The model's steps are compared with a float64 decoder on the same (dequantized)
weights.  Each layer rounds about a dozen bf16 results, each off by at most 2^-8 of
its size, whose errors add up like independent ones: the logits of a few layers
are within 2^-5 of their norm, and tokens are sampled from the step's own logits.
"""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from fpv2 import ChunkedPrefill, FPV2Config
from fpv2.prefill_harness import ChunkedPrefillRunner, DecoderShape, RandomDecoder

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SHAPE = DecoderShape(layers=2, hidden=256, query_heads=8, kv_heads=2, head_dim=64,
                     intermediate=512, vocab=1000)


def _attention64(q, k, v, scale):
    group = q.shape[0] // k.shape[0]
    k, v = (x.double().repeat_interleave(group, 0) for x in (k, v))
    return torch.softmax(q.double() @ k.transpose(1, 2) * scale, -1) @ v


def _model64(model, tokens):
    """Logits of the last position by the decoder in float64 (exact attention)."""
    s = model.shape

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + s.rms_eps).sqrt() * w.cpu().double()

    n = tokens.numel()
    half = s.head_dim // 2
    inv = s.rope_theta ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * inv
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def rope(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = model.embed.cpu().double()[tokens.cpu()]
    for p in model.layers:
        w = {name: t.cpu().double() for name, t in p.items()}
        qkv = (norm(x, p["attn_norm"]) @ w["qkv"].T).view(n, -1, s.head_dim)
        q, k, v = qkv.split([s.query_heads, s.kv_heads, s.kv_heads], 1)
        q, k = rope(norm(q, p["q_norm"])), rope(norm(k, p["k_norm"]))
        group = s.query_heads // s.kv_heads
        k, v = (t.repeat_interleave(group, 1) for t in (k, v))
        scores = torch.einsum("qhd,khd->hqk", q, k) * s.head_dim ** -0.5
        scores = scores.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf)
        attn = torch.einsum("hqk,khd->qhd", torch.softmax(scores, -1), v).reshape(n, -1)
        x = x + attn @ w["o"].T
        gate, up = (norm(x, p["mlp_norm"]) @ w["gate_up"].T).split(s.intermediate, 1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].T
    return (norm(x[-1:], model.final_norm) @ model.embed.cpu().double().T)[0]


@pytest.mark.parametrize("quantized", [False, True])
def test_decode_follows_the_prefill(cuda, quantized):
    model = RandomDecoder(SHAPE, device=cuda, seed=1)
    if quantized:
        model.quantize(32)
    gen = torch.Generator(device=cuda).manual_seed(2)
    tokens = torch.randint(0, SHAPE.vocab, (330,), generator=gen, device=cuda)
    runner = ChunkedPrefillRunner(model, 340)
    runner.prefill(tokens[:321], 128)
    for n in range(321, 330):
        got = runner.decode(tokens[n:n + 1]).cpu().double()
        want = _model64(model, tokens[:n + 1])
        assert float((got - want).norm() / want.norm()) < 2 ** -5
    assert all(c.length == 330 for c in runner.caches)
    # the prefill of the whole prompt gives the same logits, to its own rounding
    runner.reset()
    again = runner.prefill(tokens, 128).cpu().double()
    assert float((again - got).norm() / got.norm()) < 2 ** -5


@pytest.mark.parametrize("quantized", [False, True])
def test_generate(cuda, quantized):
    model = RandomDecoder(SHAPE, device=cuda, seed=3)
    if quantized:
        model.quantize(64)
    gen = torch.Generator(device=cuda).manual_seed(4)
    prompt = torch.randint(0, SHAPE.vocab, (200,), generator=gen, device=cuda)
    runner = ChunkedPrefillRunner(model, 207)
    uniform = torch.rand(8, generator=gen, device=cuda)
    settings = dict(temperature=0.05, top_k=20, top_p=0.9, min_p=0.01)
    out = runner.generate(prompt, 64, 8, uniform=uniform, **settings)
    assert out.shape == (8,) and out.dtype == torch.int64
    runner.reset()
    assert torch.equal(runner.generate(prompt, 64, 8, uniform=uniform, **settings), out)
    with pytest.raises(ValueError, match="reset"):
        runner.generate(prompt, 64, 2)
    # step by step
    runner.reset()
    logits = runner.prefill(prompt, 64)
    for i in range(8):
        token = fpv2.sample_tokens(logits[None], uniform[i:i + 1], **settings)
        assert int(token) == int(out[i])
        if i < 7:
            logits = runner.decode(token)
    with pytest.raises(ValueError, match="capacity"):
        runner.decode(out[:1])
    runner.reset()
    with pytest.raises(ValueError, match="capacity"):
        runner.generate(prompt, 64, 9)
    greedy = runner.generate(prompt, 64, 3, temperature=0.0)
    runner.reset()
    assert int(greedy[0]) == int(runner.prefill(prompt, 64).argmax())


def test_decode_refusals(cuda):
    model = RandomDecoder(SHAPE, device=cuda, seed=5)
    runner = ChunkedPrefillRunner(model, 64)
    token = torch.zeros(1, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="prefilled"):
        runner.decode(token)
    with pytest.raises(ValueError, match="new_tokens"):
        runner.generate(token, 64, 0)
    with pytest.raises(ValueError, match="uniform"):
        runner.generate(token, 64, 2, uniform=torch.rand(3, device=cuda))
    runner.prefill(token.repeat(5), 64)
    with pytest.raises(ValueError, match="one element"):
        runner.decode(token.repeat(2))
    with pytest.raises(ValueError, match="'fpv2' or 'dense'"):
        ChunkedPrefillRunner(model, 64, attention="sdpa").decode(token)


def test_refused_calls_leave_the_caches(cuda):
    """What is refused is refused before a token is appended or a prompt prefilled."""
    cache = ChunkedPrefill(4, 2, 64, 8, device=cuda)
    q, k = (torch.zeros((h, 1, 64), dtype=BF16, device=cuda) for h in (4, 2))
    wide = torch.zeros((4, 64, 2), dtype=BF16, device=cuda)
    for error, bad in ((ValueError, dict(out=wide[..., :1].transpose(1, 2))),
                       (ValueError, dict(out=q[:1].expand(4, 1, 64))),
                       (RuntimeError, dict(out=q.cpu())), (RuntimeError, dict(v=k.cpu())),
                       (RuntimeError, dict(k=k.clone().requires_grad_())),
                       (RuntimeError, dict(q=q.clone().requires_grad_()))):
        with pytest.raises(error):
            cache.decode(**{"q": q, "k": k, "v": k, **bad})
        assert cache.length == 0 and not cache.k.requires_grad
    cache.decode(q, k, k)
    assert cache.length == 1

    model = RandomDecoder(SHAPE, device=cuda, seed=7)
    runner = ChunkedPrefillRunner(model, 64)
    prompt = torch.zeros(5, dtype=torch.int64, device=cuda)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(min_p=math.nan),
                dict(uniform=torch.rand(2)),
                dict(uniform=torch.rand(2, device=cuda, dtype=torch.float64))):
        with pytest.raises(ValueError):
            runner.generate(prompt, 64, 2, **bad)
        assert runner.caches[0].length == 0
    stock = ChunkedPrefillRunner(model, 64, attention="sdpa")
    with pytest.raises(ValueError, match="'fpv2' or 'dense'"):
        stock.generate(prompt, 64, 1)
    assert runner.generate(prompt, 64, 2).shape == (2,)


def test_single_tokens_between_chunks(cuda):
    """Decoded rows count for the chunks after them: the cache equals one that had
    them from the start, and later chunks' results too."""
    gen = torch.Generator().manual_seed(6)
    n, hq, hkv, d = 700, 8, 2, 128
    q = torch.randn((hq, n, d), generator=gen).to(BF16).to(cuda)
    k, v = (torch.randn((hkv, n, d), generator=gen).to(BF16).to(cuda) for _ in "kv")
    config = FPV2Config(alpha=0.05, sink_tokens=128)
    one, two = (ChunkedPrefill(hq, hkv, d, n, config=config, min_tokens=256, device=cuda)
                for _ in range(2))
    one.step(q[:, :300], k[:, :300], v[:, :300])
    for t in range(300, 395):
        row = slice(t, t + 1)
        if t % 2:
            got = one.decode(q[:, row], k[:, row], v[:, row])
        else:
            for pages, new in zip(one.pages(), (k, v)):
                pages[0, :, t] = new[:, t]
            one.reserve(1)
            got = torch.empty((1, hq, d), dtype=BF16, device=cuda).transpose(0, 1)
            assert one.decode(q[None, :, row], out=got).data_ptr() == got.data_ptr()
        if t in (300, 301, 394):
            want = _attention64(q[:, row].cpu(), k[:, :t + 1].cpu(), v[:, :t + 1].cpu(), d ** -0.5)
            # two roundings of half a step each, of weights that sum to 1 over |v| < 5
            assert float((got.view(hq, 1, d).cpu().double() - want).abs().max()) < 2 ** -7 * 5
    two.append(k[:, :395], v[:, :395])
    a = one.step(q[:, 395:], k[:, 395:], v[:, 395:])
    b = two.step(q[:, 395:], k[:, 395:], v[:, 395:])
    assert torch.equal(a, b) and torch.equal(one.pooled_k, two.pooled_k)
    with pytest.raises(ValueError, match="capacity"):
        one.decode(q[:, :1], k[:, :1], v[:, :1])
    for bad in (dict(q=q[:, :2]), dict(q=q[:4, :1]), dict(q=q[:, :1].float()),
                dict(q=q[:, :1], k=k[:, :1]), dict(q=q[:, :1], k=k[:, :2], v=v[:, :2]),
                dict(q=q[:, :1], out=q[:, :2])):
        with pytest.raises(ValueError):
            two.decode(**bad)
    with pytest.raises(ValueError, match="query length"):
        ChunkedPrefill(hq, hkv, d, 8, device=cuda).decode(q[:, :1])


def test_paged_batch_steps_in_a_graph(cuda):
    """A batch of sequences in shared pages: projection, rotation into pages, attention,
    4-bit output product and sampling, captured once and replayed for each token."""
    gen = torch.Generator().manual_seed(7)
    batch, hq, hkv, d, page, vocab = 5, 8, 2, 64, 16, 700
    start = [0, 1, 15, 16, 60]
    steps = 20
    width = 6
    pages = batch * width
    table = torch.randperm(pages, generator=gen).view(batch, width).to(torch.int32)
    kp, vp = (torch.randn((pages, hkv, page, d), generator=gen).to(BF16) for _ in "kv")
    w = [fpv2.quantize_weight((torch.randn(shape, generator=gen) * 0.1).to(BF16), group_size=64)
         for shape in (((hq + 2 * hkv) * d, 128), (128, hq * d), (vocab, 128))]
    inv = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    angle = torch.arange(200, dtype=torch.float64)[:, None] * inv
    cos, sin = angle.cos().float(), angle.sin().float()
    x = torch.randn((steps, batch, 128), generator=gen).to(BF16)
    u = torch.rand((steps, batch), generator=gen)
    ones = torch.ones(d, dtype=BF16)

    dev = {name: t.to(cuda) for name, t in dict(table=table, kp=kp, vp=vp, cos=cos, sin=sin,
                                                ones=ones, x=x[0], u=u[0]).items()}
    lengths = torch.tensor(start, dtype=torch.int32, device=cuda)
    wd = [[t.to(cuda) for t in ws] for ws in w]

    def step():
        positions = lengths.clone()
        slots = (dev["table"].gather(1, (positions // page).long()[:, None])[:, 0] * page
                 + positions % page)
        lengths.add_(1)
        qkv = fpv2.quantized_linear(dev["x"], *wd[0])
        q = fpv2.rope_to_pages(qkv, dev["ones"], dev["ones"], dev["cos"], dev["sin"], positions,
                               slots, dev["kp"], dev["vp"], query_heads=hq)
        attn = fpv2.decode_attention(q, dev["kp"], dev["vp"], dev["table"], lengths)
        h = fpv2.quantized_linear(attn.view(batch, -1), *wd[1])
        logits = fpv2.quantized_linear(h, *wd[2], out_dtype=torch.float32)
        return q, attn, logits, fpv2.sample_tokens(logits, dev["u"], top_k=30, top_p=0.9)

    step()  # warm-up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step()
    lengths.copy_(torch.tensor(start, dtype=torch.int32))
    dev["kp"].copy_(kp)
    dev["vp"].copy_(vp)
    for i in range(steps):
        dev["x"].copy_(x[i])
        dev["u"].copy_(u[i])
        graph.replay()
        torch.cuda.synchronize()
        q, attn, logits, tokens = (t.cpu() for t in outputs)
        kc, vc = dev["kp"].cpu(), dev["vp"].cpu()
        for b in range(batch):
            n = start[b] + i + 1
            t = torch.arange(n)
            rows = table[b].long()[t // page]
            keys, values = (c[rows, :, t % page].transpose(0, 1) for c in (kc, vc))
            want = _attention64(q[b][:, None], keys, values, d ** -0.5)[:, 0]
            assert float((attn[b].double() - want).abs().max()) < 2 ** -7 * 6
        again = fpv2.sample_tokens(outputs[2], dev["u"], top_k=30, top_p=0.9)
        assert torch.equal(again.cpu(), tokens)
