"""Cases of the batch-serving operators for timing and for comparing results.

``listed`` names them, ``draw`` gives more of the same ranges, ``prepare``
makes what a program holds before the call, ``run`` is one pass (the plain
form in torch, or with ``own`` the framework's calls), ``work`` what a pass
cannot do without and ``exact`` the result in float64, written apart.

Kinds of cases:

``shared``    ``fpv2.shared_prefix_attention``: one new token per sequence of a
              batch that continues one prompt: attention over the prompt's
              keys, which are stored once, and the sequence's own.
``cache``     ``fpv2.quantize_to_pages`` and ``fpv2.dequantize_pages``: keys and
              values written into 8-bit pages, and read back in order.
``attention`` ``fpv2.quantize_to_pages`` and ``fpv2.quantized_decode_attention``:
              a decode step over 8-bit pages: the new tokens' keys and values
              are written, then each sequence's new query attends.
``logprobs``  ``fpv2.token_logprobs``: log probabilities of given tokens, the
              distributions' entropies and the most likely alternatives.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _shared(name, batch, prefix, shortest, longest, page, *, heads=32, kv_heads=8, dim=128,
            dtype="bf16"):
    return {"name": name, "kind": "shared", "batch": batch, "prefix": prefix,
            "shortest": shortest, "longest": longest, "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _cache(name, batch, shortest, longest, page, *, kv_heads=8, dim=128, dtype="bf16"):
    return {"name": name, "kind": "cache", "batch": batch, "shortest": shortest,
            "longest": longest, "page": page, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _attention(name, batch, shortest, longest, page, *, heads=32, kv_heads=8, dim=128,
               dtype="bf16", window=0, sinks=0):
    return {"name": name, "kind": "attention", "batch": batch, "shortest": shortest,
            "longest": longest, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "window": window, "sinks": sinks}


def _logprobs(name, rows, vocab, dtype, top, masked=False):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype,
            "top": top, "masked": masked}


def listed():
    return [
        # four candidates of one short prompt: launches and latency
        _shared("shared_4x1000", 4, 1000, 1, 37, 16),
        # a batch of users over one long document, in pages
        _shared("shared_40x32k", 40, 32768, 20, 700, 64),
        # many samples of one prompt on the prefill's own contiguous cache, float16
        _shared("shared_128x8k_f16", 128, 8191, 5, 300, 0, dtype="f16"),
        # large heads, pages that are no power of two, an odd batch
        _shared("shared_21x20k_d256", 21, 20011, 9, 1500, 48, heads=16, kv_heads=4, dim=256),
        # a few short prompts into the 8-bit cache and back
        _cache("cache_3_short", 3, 7, 61, 16),
        # ragged prompts, for prefills that go on over what was stored
        _cache("cache_6_ragged_f16", 6, 1001, 30011, 48, dtype="f16"),
        # one user's short chat
        _attention("q8_attention_1x1000", 1, 1000, 1000, 16),
        # a token after a 128k prompt, one page for each sequence
        _attention("q8_attention_1x128k", 1, 131072, 131072, 0),
        # a serving batch of short and long sequences
        _attention("q8_attention_32_ragged_f16", 32, 61, 16001, 64, dtype="f16"),
        # the sampled token of one user, with what else was likely
        _logprobs("logprobs_1_top20", 1, 151936, "f32", 20),
        # a chunk of a prompt that is scored
        _logprobs("logprobs_1536_bf16", 1536, 151936, "bf16", 0),
        # a batch with alternatives over an odd, smaller vocabulary, tokens ruled out
        _logprobs("logprobs_160_top5_f16", 160, 50001, "f16", 5, masked=True),
    ]


def _spread(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_GROUPS = [(32, 8), (32, 8), (16, 2), (16, 16), (8, 1), (4, 1), (28, 4), (24, 1)]


def draw(rng):
    kind = rng.choice(["shared"] * 4 + ["cache"] * 2 + ["attention"] * 3 + ["logprobs"] * 3)
    heads, kv_heads = rng.choice(_GROUPS)
    dim = rng.choice([64, 96, 128, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    page = rng.choice([0, 16, 32, 48, 64, 128, 256])
    if kind == "shared":
        batch = _spread(rng, 1, 160)
        # (at most the products of the largest listed case, its prefix's bytes and the bytes of its
        # sequences' own keys)
        longest = min(_spread(rng, 1, 1500), (128 * 300 * 1024) // (batch * kv_heads * dim))
        most = min((40 * 32 * 33000 * 128) // (batch * heads * dim), (32768 * 1024) // (kv_heads * dim))
        case = _shared("", batch, max(1, min(_spread(rng, 100, 65536), most - longest)),
                       rng.randrange(1, longest + 1), longest, page, heads=heads,
                       kv_heads=kv_heads, dim=dim, dtype=dtype)
    elif kind == "cache":
        batch = _spread(rng, 1, 24)
        longest = min(_spread(rng, 1, 30000), (1 << 26) // (batch * kv_heads * dim))
        case = _cache("", batch, rng.randrange(1, longest + 1), longest, page or 64,
                      kv_heads=kv_heads, dim=dim, dtype=dtype)
    elif kind == "attention":
        batch = _spread(rng, 1, 48)
        # (at most the largest listed case's bytes of K and V)
        longest = min(_spread(rng, 100, 131072), (1 << 28) // (batch * kv_heads * dim * 2))
        window, sinks = (_spread(rng, 64, 8192), rng.randrange(0, 300)) if rng.random() < 0.3 else (0, 0)
        case = _attention("", batch, rng.randrange(1, longest + 1), longest, page, heads=heads,
                          kv_heads=kv_heads, dim=dim, dtype=dtype, window=window, sinks=sinks)
    else:
        vocab = _spread(rng, 500, 151936)
        rows = min(_spread(rng, 1, 1536), (1 << 26) // vocab)
        case = _logprobs("", rows, vocab, rng.choice(["f32", "bf16", "f16"]),
                         rng.choice([0, 0, 1, 5, 20, 32]), masked=rng.random() < 0.4)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# What a program holds before the call
# ---------------------------------------------------------------------------


def _lengths(case):
    """The sequences' lengths, spread over the logarithm of [shortest, longest]."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    if n == 1:
        return [hi]
    return [round(lo * (hi / lo) ** (i / (n - 1))) for i in range(n)]


def _tables(case, gen, first_pages=0):
    """Each sequence's length and its pages, in an order of their own, of a pool that
    holds ``first_pages`` more; the latter's ids too."""
    batch, page = case["batch"], case["page"]
    lengths = torch.tensor(_lengths(case), device=DEVICE)
    lengths = lengths[torch.randperm(batch, generator=gen, device=DEVICE)]
    if not page:
        return lengths, None, None, case["longest"], batch
    used = (lengths + page - 1) // page
    width = -(-case["longest"] // page)
    total = sum(-(-n // page) for n in _lengths(case)) + first_pages
    pool = torch.randperm(total, generator=gen, device=DEVICE)
    first = used.cumsum(0) - used + first_pages
    column = torch.arange(width, device=DEVICE)
    # (entries behind a sequence's last page hold a page of someone else)
    table = pool[(first[:, None] + column).clamp(max=total - 1)].to(torch.int32)
    return lengths, table, pool[:first_pages].to(torch.int32), page, total


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"shared": _prepare_shared, "cache": _prepare_cache, "attention": _prepare_attention,
            "logprobs": _prepare_logprobs}[case["kind"]](case, gen)


def _normal(gen, *shape, dtype, std=1.0):
    x = torch.empty(shape, dtype=dtype, device=DEVICE)
    return x.normal_(std=std, generator=gen)


def _prepare_shared(case, gen):
    batch, hkv, dim, dtype = case["batch"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    page, prefix = case["page"], case["prefix"]
    lengths, table, prefix_table, rows, total = _tables(case, gen, -(-prefix // page) if page else 0)
    k, v = (_normal(gen, total, hkv, rows, dim, dtype=dtype) for _ in "kv")
    state = {"case": case, "k": k, "v": v, "table": table, "lengths": lengths.to(torch.int32),
             "prefix_table": prefix_table, "scale": dim ** -0.5,
             # (wider queries than keys: uneven weights)
             "q": _normal(gen, batch, case["heads"], dim, dtype=dtype, std=1.6)}
    if page:  # one pool; the length where a captured step reads it
        state["prefix_k"], state["prefix_v"] = k, v
        state["prefix_length"] = torch.tensor([prefix], dtype=torch.int32, device=DEVICE)
    else:  # the prefill's cache, with room behind the prompt
        state["prefix_k"], state["prefix_v"] = (
            _normal(gen, 1, hkv, prefix + 129, dim, dtype=dtype) for _ in "kv")
        state["prefix_length"] = prefix
    return state


def _empty_cache(total, hkv, rows, dim):
    codes = [torch.zeros((total, hkv, rows, dim), dtype=torch.int8, device=DEVICE) for _ in "kv"]
    scales = [torch.zeros((total, hkv, rows), device=DEVICE) for _ in "kv"]
    return {"k": codes[0], "v": codes[1], "k_scales": scales[0], "v_scales": scales[1]}


def _new_rows(gen, tokens, hkv, dim, dtype):
    """Keys with a few large channels, as rotated keys of trained models have, and values."""
    k = torch.randn((tokens, hkv, dim), generator=gen, device=DEVICE)
    k[..., ::29] *= 4
    v = torch.randn((tokens, hkv, dim), generator=gen, device=DEVICE)
    return k.to(dtype), v.to(dtype)


def _prepare_cache(case, gen):
    batch, hkv, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    lengths, table, _, rows, total = _tables(case, gen)
    # each token's slot, sequence by sequence
    at = torch.arange(case["longest"], device=DEVICE)
    seen = at < lengths[:, None]
    slots = (table.long()[:, at // page] * page + at % page)[seen]
    k, v = _new_rows(gen, slots.numel(), hkv, dim, DTYPES[case["dtype"]])
    return {"case": case, "new_k": k, "new_v": v, "slots": slots, "table": table,
            "lengths": lengths.to(torch.int32), **_empty_cache(total, hkv, rows, dim)}


def _prepare_attention(case, gen):
    batch, hkv, dim, dtype = case["batch"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    lengths, table, _, rows, total = _tables(case, gen)
    cache = _empty_cache(total, hkv, rows, dim)
    for name in "kv":
        cache[name].copy_(torch.randint(-127, 128, cache[name].shape, generator=gen, device=DEVICE,
                                        dtype=torch.int8))
        # (codes spread evenly have 73 of 127 as their deviation)
        scales = cache[name + "_scales"]
        scales.uniform_(0.008, 0.022, generator=gen)
    last = lengths - 1
    owner = torch.arange(batch, device=DEVICE)
    slots = owner * rows + last if table is None else (
        table.long()[owner, last // rows] * rows + last % rows)
    k, v = _new_rows(gen, batch, hkv, dim, dtype)
    return {"case": case, "q": _normal(gen, batch, case["heads"], dim, dtype=dtype, std=1.6),
            "new_k": k, "new_v": v, "slots": slots, "table": table,
            "lengths": lengths.to(torch.int32), "scale": dim ** -0.5, **cache}


def _prepare_logprobs(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    logits = _normal(gen, rows, vocab, dtype=torch.float32, std=2.5)
    # (one in each 24th part of the vocabulary: no token twice)
    part = vocab // 24
    likely = torch.randint(0, part, (rows, 24), generator=gen, device=DEVICE)
    likely += part * torch.arange(24, device=DEVICE)
    logits.scatter_(1, likely, 6 + 8 * torch.rand(likely.shape, generator=gen, device=DEVICE))
    row = torch.arange(rows, device=DEVICE)
    tokens = likely[row, row % 24]
    # (not all of the given tokens are likely ones)
    tokens = torch.where(row % 5 == 3, (tokens * 7 + row) % vocab, tokens)
    if case["masked"]:  # a grammar that rules tokens out
        given = logits.gather(1, tokens[:, None])
        logits[row % 4 == 1, ::3] = -math.inf
        logits.scatter_(1, tokens[:, None], given)
    return {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "tokens": tokens}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

_package = None


def _framework():
    global _package
    if _package is None:
        path = str(Path(__file__).resolve().parents[1] / "flashprefillv2-mlx_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import fpv2
        _package = fpv2
    return _package


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](_framework(), state)
    return _PLAIN[kind](state)


def _own_shared(fpv2, s):
    return fpv2.shared_prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["prefix_table"],
                                        s["prefix_length"], s["k"], s["v"], s["table"],
                                        s["lengths"], scale=s["scale"])


def _own_cache(fpv2, s):
    fpv2.quantize_to_pages(s["new_k"], s["new_v"], s["slots"], s["k"], s["k_scales"], s["v"],
                           s["v_scales"])
    k, v = fpv2.dequantize_pages(s["k"], s["k_scales"], s["v"], s["v_scales"], s["table"],
                                 s["lengths"], tokens=s["case"]["longest"], dtype=s["new_k"].dtype)
    return {"k": k, "v": v}


def _own_attention(fpv2, s):
    case = s["case"]
    fpv2.quantize_to_pages(s["new_k"], s["new_v"], s["slots"], s["k"], s["k_scales"], s["v"],
                           s["v_scales"])
    return fpv2.quantized_decode_attention(s["q"], s["k"], s["k_scales"], s["v"], s["v_scales"],
                                           s["table"], s["lengths"], scale=s["scale"],
                                           window_tokens=case["window"] or None,
                                           sink_tokens=case["sinks"])


def _own_logprobs(fpv2, s):
    res = fpv2.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return {"logprobs": res.logprobs, "entropy": res.entropy, "top_tokens": res.top_tokens,
            "top_logprobs": res.top_logprobs}


def _gather(pages, table):
    """The sequences' rows in order ``[B, Hkv, L, ...]``."""
    if table is None:
        return pages
    rows = pages[table.long()].transpose(1, 2)
    return rows.flatten(2, 3)


def _plain_shared(s):
    case, q = s["case"], s["q"]
    batch, hq, dim = q.shape
    hkv = case["kv_heads"]
    group = hq // hkv
    n = case["prefix"]
    if s["prefix_table"] is None:
        pk, pv = s["prefix_k"][0, :, :n].float(), s["prefix_v"][0, :, :n].float()
    else:
        pk, pv = (_gather(s[name], s["prefix_table"][None])[0, :, :n].float()
                  for name in ("prefix_k", "prefix_v"))
    k, v = (_gather(s[name], s["table"]).float() for name in "kv")
    rows = q.float().view(batch, hkv, group, dim)
    # the shared keys' scores for the rows of all sequences in one product
    packed = rows.transpose(0, 1).reshape(hkv, batch * group, dim)
    first = (packed @ pk.transpose(1, 2).contiguous()) * s["scale"]
    scores = (rows @ k.transpose(2, 3).contiguous()) * s["scale"]
    seen = torch.arange(k.shape[2], device=q.device) < s["lengths"][:, None]
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    first = first.view(hkv, batch, group, n).transpose(0, 1)
    top = torch.maximum(first.amax(-1, keepdim=True), scores.amax(-1, keepdim=True))
    p, w = (first - top).exp(), (scores - top).exp()
    shared = p.transpose(0, 1).reshape(hkv, batch * group, n) @ pv
    shared = shared.view(hkv, batch, group, dim).transpose(0, 1)
    out = (shared + w @ v) / (p.sum(-1, keepdim=True) + w.sum(-1, keepdim=True))
    return out.reshape(batch, hq, dim).to(q.dtype)


def _plain_write(s):
    page = s["k"].shape[2]
    at, row = s["slots"] // page, s["slots"] % page
    for name in "kv":
        x = s["new_" + name]
        # (127 x / max in float64: whether a value is half way between two codes is exact)
        top = x.double().abs().amax(-1, keepdim=True)
        codes = (x.double() * 127 / torch.where(top == 0, 1.0, top)).round()
        s[name][at, :, row] = codes.to(torch.int8)
        s[name + "_scales"][at, :, row] = (top[..., 0] / 127).float()


def _plain_cache(s):
    _plain_write(s)
    longest = s["case"]["longest"]
    seen = torch.arange(longest, device=s["k"].device) < s["lengths"][:, None]
    out = {}
    for name in "kv":
        codes = _gather(s[name], s["table"])[:, :, :longest]
        scales = _gather(s[name + "_scales"], s["table"])[:, :, :longest]
        values = codes.float() * scales[..., None]
        out[name] = torch.where(seen[:, None, :, None], values, 0.0).to(s["new_k"].dtype)
    return out


def _plain_attention(s):
    _plain_write(s)
    case, q = s["case"], s["q"]
    batch, hq, dim = q.shape
    hkv = case["kv_heads"]
    k, v = (_gather(s[name], s["table"]).float() * _gather(s[name + "_scales"], s["table"])[..., None]
            for name in "kv")
    scores = (q.float().view(batch, hkv, hq // hkv, dim) @ k.transpose(2, 3).contiguous()) * s["scale"]
    t = torch.arange(k.shape[2], device=q.device)
    length = s["lengths"][:, None]
    seen = t < length
    if case["window"]:
        seen &= (t >= length - case["window"]) | (t < case["sinks"])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.view(batch, hq, dim).to(q.dtype)


def _plain_logprobs(s):
    logits, top = s["logits"].float(), s["case"]["top"]
    greatest = logits.amax(1, keepdim=True)
    shifted = logits - greatest
    p = shifted.exp()
    total = p.sum(1, keepdim=True)
    norm = total.log()
    # (a weight of zero times -inf is nothing)
    mean = torch.where(p > 0, p * shifted, 0.0).sum(1, keepdim=True) / total
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top] if top else (
        torch.empty((logits.shape[0], 0), dtype=torch.int64, device=logits.device))
    return {"logprobs": (shifted.gather(1, s["tokens"][:, None]) - norm)[:, 0],
            "entropy": (norm - mean)[:, 0], "top_tokens": order,
            "top_logprobs": shifted.gather(1, order) - norm}


_OWN = {"shared": _own_shared, "cache": _own_cache, "attention": _own_attention,
        "logprobs": _own_logprobs}
_PLAIN = {"shared": _plain_shared, "cache": _plain_cache, "attention": _plain_attention,
          "logprobs": _plain_logprobs}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "shared":
        tokens, keys = sum(_lengths(case)), case["prefix"] + sum(_lengths(case))
        b = 4 * keys * case["kv_heads"] * case["dim"] + 4 * case["batch"] * case["heads"] * case["dim"]
        f = 4 * (case["batch"] * case["prefix"] + tokens) * case["heads"] * case["dim"]
    elif kind == "cache":
        # values in, codes and scales out and in again, values out (zeros behind the lengths too)
        rows = sum(_lengths(case)) * case["kv_heads"] * 2
        b = rows * (4 * case["dim"] + 8) + 4 * case["batch"] * case["longest"] * case["kv_heads"] * case["dim"]
        f = rows * case["dim"] * 4
    elif kind == "attention":
        keys = sum(_lengths(case))
        if case["window"]:
            keys = sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"])))
                       for n in _lengths(case))
        b = (keys * case["kv_heads"] * 2 * (case["dim"] + 4)
             + 4 * case["batch"] * (case["heads"] + case["kv_heads"]) * case["dim"])
        f = 4 * keys * case["heads"] * case["dim"]
    else:
        size = 4 if case["dtype"] == "f32" else 2
        b = case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"])
        f = case["rows"] * case["vocab"] * 5
    return {"bytes": int(b), "flops": int(f)}


# ---------------------------------------------------------------------------
# The result in float64, sequence by sequence and row by row
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "cache": _exact_cache, "attention": _exact_attention,
            "logprobs": _exact_logprobs}[case["kind"]](case, s)


def _exact_shared(case, s):
    hq, hkv, n, group = case["heads"], case["kv_heads"], case["prefix"], case["heads"] // case["kv_heads"]
    out = torch.zeros((case["batch"], hq, case["dim"]), dtype=torch.float64, device=DEVICE)
    t = torch.arange(n, device=DEVICE)
    rows = s["prefix_k"].shape[2]
    pages = torch.zeros_like(t) if s["prefix_table"] is None else s["prefix_table"].long()[t // rows]
    lengths = s["lengths"].tolist()
    for h in range(hkv):
        heads = slice(h * group, (h + 1) * group)
        pk, pv = (s[name][pages, h, t % rows].double() for name in ("prefix_k", "prefix_v"))
        for b, m in enumerate(lengths):
            u = torch.arange(m, device=DEVICE)
            page = s["k"].shape[2]
            mine = u // page + b if s["table"] is None else s["table"][b].long()[u // page]
            keys = torch.cat([pk, s["k"][mine, h, u % page].double()])
            values = torch.cat([pv, s["v"][mine, h, u % page].double()])
            logits = torch.mm(s["q"][b, heads].double(), keys.T) * s["scale"]
            out[b, heads] = torch.mm(torch.softmax(logits, 1), values)
    return out


def _stored(x):
    """What the cache holds of rows ``x``: multiples of the greatest's 127th part."""
    x = x.double()
    step = x.abs().max(-1, keepdim=True).values / 127
    whole = torch.round(x / torch.where(step > 0, step, 1.0))
    # half way between two multiples (127 x is exact, and so is the comparison): the even one
    top = step * 127
    ratio = 254 * x.abs() / torch.where(top > 0, x.abs().max(-1, keepdim=True).values, 1.0)
    odd = torch.round(ratio)
    half = (ratio == odd) & (odd % 2 == 1)
    even = torch.sign(x) * 2 * torch.round((odd / 2) / 2)
    return torch.where(half, even, whole) * step


def _exact_cache(case, s):
    k, v = _stored(s["new_k"]), _stored(s["new_v"])
    shape = (case["batch"], case["longest"], case["kv_heads"], case["dim"])
    out = {}
    for name, x in (("k", k), ("v", v)):
        dense = torch.zeros(shape, dtype=torch.float64, device=DEVICE)
        start = 0
        for b, n in enumerate(s["lengths"].tolist()):
            dense[b, :n] = x[start:start + n]
            start += n
        out[name] = dense.transpose(1, 2)
    return out


def _exact_attention(case, s):
    hq, hkv, group = case["heads"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros((case["batch"], hq, case["dim"]), dtype=torch.float64, device=DEVICE)
    new = {"k": _stored(s["new_k"]), "v": _stored(s["new_v"])}
    page = s["k"].shape[2]
    for b, n in enumerate(s["lengths"].tolist()):
        t = torch.arange(n, device=DEVICE)
        if case["window"] and n > case["window"]:
            t = torch.cat([t[:min(case["sinks"], n - case["window"])], t[n - case["window"]:]])
        pages = t // page + b if s["table"] is None else s["table"][b].long()[t // page]
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            rows = {}
            for name in "kv":
                rows[name] = (s[name][pages, h, t % page].double()
                              * s[name + "_scales"][pages, h, t % page].double()[:, None])
                rows[name][-1] = new[name][b, h]
            logits = torch.mm(s["q"][b, heads].double(), rows["k"].T) * s["scale"]
            out[b, heads] = torch.mm(torch.softmax(logits, 1), rows["v"])
    return out


def _exact_logprobs(case, s):
    logprobs, entropy, tokens, best = [], [], [], []
    for b in range(case["rows"]):
        row = s["logits"][b].double()
        logs = torch.log_softmax(row, 0)
        logprobs.append(logs[s["tokens"][b]])
        entropy.append(-torch.special.xlogy(logs.exp(), logs.exp()).sum())
        order = torch.argsort(-row, stable=True)[:case["top"]] if case["top"] else (
            torch.empty(0, dtype=torch.int64, device=DEVICE))
        tokens.append(order)
        best.append(logs[order])
    return {"logprobs": torch.stack(logprobs), "entropy": torch.stack(entropy),
            "top_tokens": torch.stack(tokens), "top_logprobs": torch.stack(best)}
