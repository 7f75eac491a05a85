"""Corners of what a decode step's operators refuse (no GPU needed): destinations whose
rows share memory, tangents, weights of odd layouts."""

from __future__ import annotations

import random

import pytest
import torch

import fpv2
from fpv2 import decode

BF16 = torch.bfloat16


def _strided(shape, strides):
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return torch.zeros(size, dtype=BF16).as_strided(shape, strides)


def _addresses(t):
    """Element numbers of a tensor's storage, of every element."""
    at = torch.tensor([t.storage_offset()])
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + s * torch.arange(n)).flatten()
    return at


def test_rows_that_share_memory_are_found():
    """Against all addresses, over small shapes of strides that nest, interleave and overlap."""
    rng = random.Random(1)
    found = 0
    for _ in range(4000):
        shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(rng.choice([1, 2, 3]))] + [rng.choice([1, 4, 8])]
        strides = [rng.choice([0, 1, 2, 3, 4, 5, 8, 9, 12, 16, 24, 40, 41, 120]) for _ in shape[:-1]] + [1]
        t = _strided(shape, strides)
        at = _addresses(t)
        want = len(at.unique()) < len(at)
        assert decode._overlaps_itself(t) == want, (shape, strides)
        found += want
    assert 500 < found < 3500


def _shared(t):
    at = _addresses(t)
    return len(at.unique()) < len(at)


def _calls(**change):
    """Calls that get as far as to ask for a ROCm device, if nothing is refused."""
    pages = [torch.zeros(3, 2, 16, 64, dtype=BF16) for _ in "kv"]
    attention = dict(q=torch.zeros(2, 8, 64, dtype=BF16), k_pages=pages[0], v_pages=pages[1],
                     page_table=None, lengths=3)
    rope = dict(qkv=torch.zeros(2, 12 * 64, dtype=BF16), q_weight=None, k_weight=None,
                cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=0, slots=0,
                k_pages=pages[0], v_pages=pages[1], query_heads=8)
    return [(fpv2.decode_attention, {**attention, **change}), (fpv2.rope_to_pages, {**rope, **change})]


@pytest.mark.parametrize("strides,shared", [
    ((64, 64), True), ((128, 72), True), ((512, 8), True), ((448, 64), True), ((64, 72), True),
    ((0, 64), True), ((512, 0), True), ((64, 128), False), ((512, 64), False), ((1000, 72), False),
    ((192, 128), False), ((160, 128), True), ((64, 1024), False)])
def test_destinations_of_one_row_for_two_are_refused(strides, shared):
    """Two heads, or heads of two sequences, in one place."""
    out = _strided((2, 8, 64), (*strides, 1))
    assert _shared(out) == shared
    for call, kwargs in _calls(out=out):
        with pytest.raises(ValueError if shared else RuntimeError,
                           match="out must be" if shared else "ROCm"):
            call(**kwargs)


@pytest.mark.parametrize("strides,shared", [
    ((64, 64, 64), True), ((1024, 64, 64), True), ((2048, 512, 64), True), ((1024, 2048, 72), True),
    ((64, 1024, 128), True), ((2048, 1024, 56), True), ((2048, 0, 64), True), ((2048, 64, 128), False),
    ((64, 4096, 192), False), ((2304, 1152, 72), False), ((1024, 4096, 64), False)])
def test_caches_of_one_row_for_two_are_refused(strides, shared):
    """Two pages, heads or tokens in one place; the attention only reads them."""
    pages = _strided((3, 2, 16, 64), (*strides, 1))
    assert _shared(pages) == shared
    for name in ("k_pages", "v_pages"):
        (read, read_args), (write, write_args) = _calls(**{name: pages})
        with pytest.raises(ValueError if shared else RuntimeError,
                           match="overlap" if shared else "ROCm"):
            write(**write_args)
        with pytest.raises(RuntimeError, match="ROCm"):
            read(**read_args)


def test_shared_memory_is_found():
    """Against all bytes, over pairs of small views of one storage and of two types."""
    rng = random.Random(2)
    store = torch.zeros(4096, dtype=torch.uint8)
    found = 0
    for _ in range(4000):
        pair, taken = [], []
        for _ in "ab":
            size = rng.choice([2, 4])
            shape = [rng.choice([1, 2, 3, 5]) for _ in range(rng.choice([1, 2]))] + [rng.choice([1, 4, 8])]
            strides = [rng.choice([0, 1, 2, 3, 4, 8, 12, 16, 24, 32, 48, 60]) for _ in shape[:-1]]
            strides.append(rng.choice([1, 1, 1, 1, 2]))
            typed = store.view(BF16 if size == 2 else torch.float32)
            t = typed.as_strided(shape, strides, rng.choice([0, 3, 8, 16, 40, 61, 200, 400]) * 4 // size)
            pair.append(t)
            at = _addresses(t) * size
            taken.append({int(x) + i for x in at for i in range(size)})
        want = not taken[0].isdisjoint(taken[1])
        assert decode._share_memory(*pair) == want, [(t.shape, t.stride(), t.storage_offset()) for t in pair]
        found += want
    assert 500 < found < 3500


def test_keys_and_values_in_one_place_are_refused():
    pool = torch.zeros(6, 2, 16, 128, dtype=BF16)
    flat = pool.view(-1)
    shape = (3, 2, 16, 64)
    fine = [(pool[:3, ..., :64], pool[:3, ..., 64:]), (pool[::2, ..., :64], pool[1::2, ..., :64]),
            (pool[:3, :, :, 64:], pool[3:, :, :, 64:]),
            # K of whole pages, V with the heads inside the rows, page by page
            (flat.as_strided(shape, (4096, 1024, 64, 1)), flat[2048:].as_strided(shape, (4096, 64, 128, 1)))]
    bad = [(pool[:3, ..., :64], pool[:3, ..., :64]), (pool[:3, ..., :64], pool[:3, ..., 32:96]),
           (pool[:3, ..., :64], pool[2:5, ..., :64]),
           (flat.as_strided(shape, (4096, 1024, 64, 1)), flat[2040:].as_strided(shape, (4096, 64, 128, 1)))]
    for pairs, error, message in ((fine, RuntimeError, "ROCm"), (bad, ValueError, "overlap")):
        for k, v in pairs + [(v, k) for k, v in pairs]:
            (_, _), (rope, args) = _calls(k_pages=k, v_pages=v)
            with pytest.raises(error, match=message):
                rope(**args)


def test_out_in_the_memory_of_other_operands_is_refused():
    """But for the queries' own place, a destination is apart from what the call reads and writes."""
    (attention, args), (rope, rope_args) = _calls()
    pool = torch.zeros(3200, dtype=BF16)
    q, qkv = pool[:1024].view(2, 8, 64), pool[:2 * 12 * 64].view(2, 12 * 64)
    heads = qkv[:, :512].unflatten(1, (8, 64))
    wide = torch.zeros(2, 8, 2, 64, dtype=BF16)
    for out, fine in ((q, True), (pool[1024:2048].view(2, 8, 64), True),
                      (pool[8:1032].view(2, 8, 64), False)):
        with pytest.raises(RuntimeError if fine else ValueError, match="ROCm" if fine else "share memory"):
            attention(**{**args, "q": q, "out": out})
    swapped = pool[:1024].as_strided((2, 8, 64), (64, 128, 1))  # q's memory in another order
    for bad in (dict(q=q, out=swapped), dict(out=args["k_pages"][0, 0, :16].view(2, 8, 64)),
                dict(out=args["v_pages"][1].view(2, -1)[:, :512].unflatten(1, (8, 64)))):
        with pytest.raises(ValueError, match="share memory"):
            attention(**{**args, **bad})
    for out, fine in ((heads, True), (wide[:, :, 0], True), (q, False),
                      (qkv[:, 256:768].unflatten(1, (8, 64)), False), (pool[1024:2048].view(2, 8, 64), False),
                      (pool[1536:2560].view(2, 8, 64), True)):
        with pytest.raises(RuntimeError if fine else ValueError, match="ROCm" if fine else "share memory"):
            rope(**{**rope_args, "qkv": qkv, "out": out})
    for name in ("k_pages", "v_pages"):
        with pytest.raises(ValueError, match="share memory"):
            rope(**{**rope_args, "out": rope_args[name][1].view(2, -1)[:, :512].unflatten(1, (8, 64))})
    weights = fpv2.quantize_weight(torch.zeros(128, 128, dtype=BF16))
    x = torch.zeros(6, 128, dtype=BF16)
    for out, fine in ((torch.zeros(3, 128, dtype=BF16), True), (x[3:], True), (x[:3], False),
                      (x[2:5], False), (weights[0].view(BF16).view(-1)[:384].view(3, 128), False),
                      (weights[1].view(-1)[:128].view(1, 128), False)):
        rows = x[:out.shape[0]]
        with pytest.raises(RuntimeError if fine else ValueError, match="ROCm" if fine else "share memory"):
            fpv2.quantized_linear(rows, *weights, out=out)


def test_tangents_are_refused():
    """They would be lost without a word, under no_grad too."""
    weights = fpv2.quantize_weight(torch.zeros(128, 128, dtype=BF16))
    (attention, args), (rope, rope_args) = _calls()
    calls = [(attention, args, "q"), (attention, args, "v_pages"), (rope, rope_args, "qkv"),
             (rope, {**rope_args, "k_weight": torch.ones(64, dtype=BF16)}, "k_weight"),
             (fpv2.quantized_linear, dict(x=torch.zeros(3, 128, dtype=BF16), packed=weights[0],
                                          scales=weights[1], biases=weights[2]), "x"),
             (fpv2.sample_tokens, dict(logits=torch.zeros(3, 50), uniform=torch.zeros(3)), "logits")]
    with torch.autograd.forward_ad.dual_level():
        for call, kwargs, name in calls:
            with pytest.raises(RuntimeError, match="ROCm"):
                call(**kwargs)  # a level alone is nothing to refuse
            dual = torch.autograd.forward_ad.make_dual(kwargs[name], torch.ones_like(kwargs[name]))
            with pytest.raises(RuntimeError, match="tangents"):
                call(**{**kwargs, name: dual})
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangents"):
                call(**{**kwargs, name: dual})


@pytest.mark.parametrize("rows,group", [(0, 64), (1, 32), (10, 128)])
def test_weights_of_any_layout_are_read_back(rows, group):
    """No rows, rows in columns, every other row or column."""
    gen = torch.Generator().manual_seed(rows)
    w = torch.randn((rows, 256), generator=gen)
    packed, scales, biases = fpv2.quantize_weight(w, group_size=group)
    want = fpv2.dequantize_weight(packed, scales, biases)
    assert want.shape == (rows, 256) and want.is_contiguous()
    for layout in (lambda t: t.t().contiguous().t(), lambda t: t.repeat_interleave(2, 1)[:, ::2],
                   lambda t: t.repeat_interleave(2, 0)[::2]):
        again = fpv2.dequantize_weight(*(layout(t) for t in (packed, scales, biases)))
        assert torch.equal(again, want)
        parts = fpv2.quantize_weight(layout(w), group_size=group)
        assert all(torch.equal(a, b) and a.is_contiguous() for a, b in zip(parts, (packed, scales, biases)))


@pytest.mark.parametrize("group,intermediate", [(64, 288), (128, 448), (48, 288), (32, 272)])
def test_a_model_is_cut_to_4_bits_as_a_whole_or_not_at_all(group, intermediate):
    """Groups that the last projection's columns do not hold leave the first ones as they were."""
    from fpv2.prefill_harness import DecoderShape, RandomDecoder
    model = RandomDecoder(DecoderShape(layers=2, hidden=256, query_heads=8, kv_heads=2, head_dim=64,
                                       intermediate=intermediate, vocab=100), device="cpu")
    before = [{name: t.clone() for name, t in layer.items()} for layer in model.layers]
    with pytest.raises(ValueError, match="group_size"):
        model.quantize(group)
    assert model.packed is None and model.packed_embed is None
    for layer, old in zip(model.layers, before):
        assert all(torch.equal(layer[name], old[name]) for name in old)
