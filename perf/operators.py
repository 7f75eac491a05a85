"""Cases of the decode step's operators for timing and for comparing results.

``listed`` names them, ``draw`` gives more of the same ranges, ``prepare``
makes what a program holds before the call, ``run`` is one pass (the plain
form in torch, or with ``own`` the framework's call), ``work`` what a pass
cannot do without and ``exact`` the result in float64, written apart.

Kinds of cases:

``attention``  ``fpv2.decode_attention``: one new token per sequence over a
               paged (``page``) or contiguous (``page`` 0) KV cache, the
               sequences' lengths spread between ``shortest`` and ``longest``,
               optionally with a window and first tokens that stay visible.
``rope``       ``fpv2.rope_to_pages``: norms of the query and key heads, the
               position rotation and the K/V write into pages.
``linear``     ``fpv2.quantized_linear``: rows times 4-bit weights with group
               scales and biases.
``sample``     ``fpv2.sample_tokens``: temperature, top-k, top-p and min-p from
               given random numbers.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def _attention(name, batch, shortest, longest, page, *, heads=32, kv_heads=8, dim=128,
               dtype="bf16", window=0, sinks=0):
    return {"name": name, "kind": "attention", "batch": batch, "shortest": shortest,
            "longest": longest, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "window": window, "sinks": sinks}


def _rope(name, tokens, page, *, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16",
          interleaved=False, padding=0):
    return {"name": name, "kind": "rope", "tokens": tokens, "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "dtype": dtype,
            "interleaved": interleaved, "padding": padding}


def _linear(name, rows, out, cols, group, dtype="bf16", out_dtype=None):
    return {"name": name, "kind": "linear", "rows": rows, "out": out, "cols": cols,
            "group": group, "dtype": dtype, "out_dtype": out_dtype or dtype}


def _sample(name, batch, vocab, dtype, *, mixed, top_k=0, top_p=1.0, min_p=0.0, temperature=1.0):
    return {"name": name, "kind": "sample", "batch": batch, "vocab": vocab, "dtype": dtype,
            "mixed": mixed, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "temperature": temperature}


def listed():
    return [
        # one user's short chat: launches and latency
        _attention("attention_1x1000", 1, 1000, 1000, 16),
        # the first token after the 128k prompt, the prefill's own contiguous cache
        _attention("attention_1x128k", 1, 131072, 131072, 0),
        # a serving batch of short and long sequences over 64-token pages
        _attention("attention_24_ragged_f16", 24, 61, 16001, 64, dtype="f16"),
        # large heads, a sliding window with sinks, pages that are no power of two
        _attention("attention_8_window_d256", 8, 20011, 30011, 48, heads=16, kv_heads=4, dim=256,
                   window=4096, sinks=128),
        # a decode step of a few sequences
        _rope("rope_5", 5, 16),
        # a prefill chunk straight into pages, padded at its end
        _rope("rope_8192_f16", 8192, 64, dtype="f16", padding=37),
        # the down projection of one token
        _linear("linear_down_1", 1, 2560, 9728, 64),
        # the gate and up projections of a small batch, fine groups, float16
        _linear("linear_gate_up_12_f16", 12, 19456, 2560, 32, dtype="f16"),
        # the head of three tokens, logits in float32
        _linear("linear_head_3", 3, 151936, 2560, 128, out_dtype="f32"),
        # one user's next token, the usual filters
        _sample("sample_1", 1, 151936, "f32", mixed=False, top_k=50, top_p=0.95, temperature=0.8),
        # a batch of users with settings of their own, bfloat16 logits (many ties), masked tokens
        _sample("sample_48_mixed_bf16", 48, 151936, "bf16", mixed=True),
        # a large batch over an odd, smaller vocabulary
        _sample("sample_160_min_p", 160, 50001, "f32", mixed=False, min_p=0.02, temperature=1.3),
    ]


def _spread(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_GROUPS = [(32, 8), (32, 8), (16, 2), (16, 16), (8, 1), (4, 1), (28, 4), (24, 1)]


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["rope"] * 2 + ["linear"] * 3 + ["sample"] * 3)
    heads, kv_heads = rng.choice(_GROUPS)
    dim = rng.choice([64, 96, 128, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "attention":
        batch = _spread(rng, 1, 48)
        # (at most the K and V bytes of the largest listed case)
        longest = min(_spread(rng, 100, 131072), (1 << 29) // (batch * kv_heads * dim * 4))
        window, sinks = (_spread(rng, 64, 8192), rng.randrange(0, 300)) if rng.random() < 0.3 else (0, 0)
        case = _attention("", batch, rng.randrange(1, longest + 1), longest,
                          rng.choice([0, 16, 32, 48, 64, 128, 256]), heads=heads,
                          kv_heads=kv_heads, dim=dim, dtype=dtype, window=window, sinks=sinks)
    elif kind == "rope":
        case = _rope("", _spread(rng, 1, 8192), rng.choice([16, 48, 64, 256]), heads=heads,
                     kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2]),
                     dtype=dtype, interleaved=rng.random() < 0.3)
        case["padding"] = rng.choice([0, 0, case["tokens"] // 9])
    elif kind == "linear":
        group = rng.choice([32, 64, 128])
        case = _linear("", _spread(rng, 1, 64), _spread(rng, 100, 24000),
                       group * max(1, _spread(rng, 256, 10240) // group), group, dtype,
                       rng.choice([None, "f32"]))
    else:
        mixed = rng.random() < 0.4
        case = _sample("", _spread(rng, 1, 96), _spread(rng, 500, 151936),
                       rng.choice(["f32", "bf16", "f16"]), mixed=mixed,
                       top_k=rng.choice([0, 0, 20, _spread(rng, 1, 400)]),
                       top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                       min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 4)]),
                       temperature=round(rng.uniform(0.4, 1.6), 2))
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


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"attention": _prepare_attention, "rope": _prepare_rope, "linear": _prepare_linear,
            "sample": _prepare_sample}[case["kind"]](case, gen)


def _prepare_attention(case, gen):
    batch, hkv, dim, dtype = case["batch"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    lengths = torch.tensor(_lengths(case), device=DEVICE)
    lengths = lengths[torch.randperm(batch, generator=gen, device=DEVICE)]
    if case["page"]:
        page = case["page"]
        used = (lengths + page - 1) // page
        width = -(-case["longest"] // page)
        total = sum(-(-n // page) for n in _lengths(case))
        pool = torch.randperm(total, generator=gen, device=DEVICE)
        first = used.cumsum(0) - used
        column = torch.arange(width, device=DEVICE)
        # (entries behind a sequence's last page hold a page of someone else)
        table = pool[(first[:, None] + column).clamp(max=total - 1)].to(torch.int32)
    else:
        page, total, table = case["longest"], batch, None
    k = torch.empty((total, hkv, page, dim), dtype=dtype, device=DEVICE)
    v = torch.empty_like(k)
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    # (wider queries than keys: uneven weights)
    q = torch.empty((batch, case["heads"], dim), dtype=dtype, device=DEVICE)
    q.normal_(std=1.6, generator=gen)
    return {"case": case, "q": q, "k": k, "v": v, "table": table,
            "lengths": lengths.to(torch.int32), "scale": dim ** -0.5}


def _prepare_rope(case, gen):
    tokens, page, dim, dtype = case["tokens"], case["page"], case["dim"], DTYPES[case["dtype"]]
    heads, hkv = case["heads"], case["kv_heads"]
    limit, half = 32768, case["rotary"] // 2
    inv = 1e6 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    angle = torch.arange(limit, device=DEVICE, dtype=torch.float64)[:, None] * inv
    pages = -(-tokens // page) + 3
    qkv = torch.empty((tokens, (heads + 2 * hkv) * dim), dtype=dtype, device=DEVICE)
    qkv.normal_(std=2.0, generator=gen)
    weight = [(1 + 0.2 * torch.randn(dim, generator=gen, device=DEVICE)).to(dtype) for _ in "qk"]
    order = torch.randperm(pages, generator=gen, device=DEVICE)
    t = torch.arange(tokens, device=DEVICE)
    slots = order[t // page] * page + t % page
    if case["padding"]:
        slots[-case["padding"]:] = -1
    start = torch.randint(0, limit - tokens + 1, (1,), generator=gen, device=DEVICE)
    pool = torch.randn((2, pages, hkv, page, dim), generator=gen, device=DEVICE).to(dtype)
    return {"case": case, "qkv": qkv, "qw": weight[0], "kw": weight[1],
            "cos": angle.cos().float(), "sin": angle.sin().float(), "positions": t + start,
            "slots": slots, "k": pool[0], "v": pool[1]}


def _prepare_linear(case, gen):
    rows, out, cols, group = case["rows"], case["out"], case["cols"], case["group"]
    dtype = DTYPES[case["dtype"]]
    x = torch.randn((rows, cols), generator=gen, device=DEVICE)
    x[:, ::97] *= 6  # a few channels are larger, as in trained models
    packed = torch.randint(-2 ** 31, 2 ** 31, (out, cols // 8), generator=gen, device=DEVICE,
                           dtype=torch.int64).to(torch.int32)
    scales = 0.004 * (0.5 + torch.rand((out, cols // group), generator=gen, device=DEVICE))
    biases = -scales * (7.5 + torch.randn(scales.shape, generator=gen, device=DEVICE))
    return {"case": case, "x": x.to(dtype), "packed": packed, "scales": scales.to(dtype),
            "biases": biases.to(dtype)}


def _prepare_sample(case, gen):
    batch, vocab = case["batch"], case["vocab"]
    logits = 2.5 * torch.randn((batch, vocab), generator=gen, device=DEVICE)
    top = torch.randint(0, vocab, (batch, 24), generator=gen, device=DEVICE)
    logits.scatter_(1, top, 6 + 8 * torch.rand(top.shape, generator=gen, device=DEVICE))
    state = {"case": case, "uniform": torch.rand(batch, generator=gen, device=DEVICE)}
    if case["mixed"]:
        # users with settings of their own: greedy, unfiltered, each filter, all of them
        row = torch.arange(batch, device=DEVICE)
        logits[row % 4 == 1, ::3] = -math.inf  # a grammar that rules tokens out
        rand = torch.rand((3, batch), generator=gen, device=DEVICE)
        state["temperature"] = torch.where(row % 6 == 0, 0.0, 0.3 + rand[0])
        state["top_k"] = torch.where(row % 3 == 1, 5 + 7 * row, 0).to(torch.int32)
        state["top_p"] = torch.where(row % 2 == 1, 0.5 + 0.45 * rand[1], 1.0)
        state["min_p"] = torch.where(row % 5 == 2, 0.1 * rand[2], 0.0)
    else:
        for name in ("temperature", "top_k", "top_p", "min_p"):
            state[name] = case[name]
    state["logits"] = logits.to(DTYPES[case["dtype"]])
    return state


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


def _own_attention(fpv2, s):
    case = s["case"]
    return fpv2.decode_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale=s["scale"],
                                 window_tokens=case["window"] or None, sink_tokens=case["sinks"])


def _own_rope(fpv2, s):
    case = s["case"]
    q = fpv2.rope_to_pages(s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], s["positions"],
                           s["slots"], s["k"], s["v"], query_heads=case["heads"], eps=EPS,
                           interleaved=case["interleaved"])
    return {"q": q, "k": s["k"], "v": s["v"]}


def _own_linear(fpv2, s):
    return fpv2.quantized_linear(s["x"], s["packed"], s["scales"], s["biases"],
                                 out_dtype=DTYPES[s["case"]["out_dtype"]])


def _own_sample(fpv2, s):
    tokens, logprobs = fpv2.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"],
                                          top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                          return_logprobs=True)
    return {"tokens": tokens, "logprobs": logprobs}


def _plain_attention(s):
    case, q = s["case"], s["q"]
    batch, hq, dim = q.shape
    hkv = s["k"].shape[1]
    k, v = s["k"], s["v"]
    if s["table"] is not None:
        table = s["table"].long()
        k, v = (x[table].transpose(1, 2).reshape(batch, hkv, -1, dim) for x in (k, v))
    k, v = k.float(), v.float()
    scores = (q.float().view(batch, hkv, hq // hkv, dim) @ k.transpose(2, 3)) * s["scale"]
    t = torch.arange(k.shape[2], device=q.device)
    length = s["lengths"][:, None]
    seen = t < length
    if case["window"]:
        seen &= (t >= length - case["window"]) | (t < case["sinks"])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.view(batch, hq, dim).to(q.dtype)


def _plain_rope(s):
    case, qkv = s["case"], s["qkv"]
    heads, hkv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = qkv.float().view(qkv.shape[0], -1, dim)
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    half = cos.shape[-1]
    out = []
    for part, weight in ((x[:, :heads], s["qw"]), (x[:, heads:heads + hkv], s["kw"])):
        n = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + EPS) * weight.float()
        if case["interleaved"]:
            a, b = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = n[..., :half], n[..., half:2 * half]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, n[..., 2 * half:]], -1).to(qkv.dtype))
    k, v, slots = out[1], x[:, heads + hkv:].to(qkv.dtype), s["slots"]
    if case["padding"]:
        kept = slots >= 0
        k, v, slots = k[kept], v[kept], slots[kept]
    s["k"][slots // page, :, slots % page] = k
    s["v"][slots // page, :, slots % page] = v
    return {"q": out[0], "k": s["k"], "v": s["v"]}


def _plain_linear(s):
    case, packed = s["case"], s["packed"]
    shifts = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
    nibbles = ((packed[..., None] >> shifts) & 15).view(packed.shape[0], -1, case["group"])
    w = nibbles * s["scales"].float()[..., None] + s["biases"].float()[..., None]
    return (s["x"].float() @ w.flatten(1).T).to(DTYPES[case["out_dtype"]])


def _plain_sample(s):
    logits = s["logits"].float()
    batch, vocab = logits.shape
    temperature, top_k, top_p, min_p = (
        torch.as_tensor(s[name], device=logits.device).expand(batch)[:, None].double()
        for name in ("temperature", "top_k", "top_p", "min_p"))
    if not s["case"]["mixed"]:  # (a number is meant as it is, not as its float32 in float64)
        top_p, min_p, temperature = (torch.full_like(top_p, s[name])
                                     for name in ("top_p", "min_p", "temperature"))
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    x = order.values.double()
    greedy = temperature == 0
    w = ((x - x[:, :1]) / torch.where(greedy, 1.0, temperature)).exp()
    rank = torch.arange(vocab, device=logits.device)
    kept = (rank < top_k) | (top_k <= 0)
    before = w.cumsum(1) - w
    total = torch.where(kept, w, 0.0).sum(1, keepdim=True)
    kept &= (before < top_p * total) | (top_p >= 1)
    kept &= w >= min_p
    kept &= ~greedy
    kept |= rank == 0
    w = torch.where(kept, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order.indices, w)  # back to the tokens' order
    running = w.cumsum(1)
    target = s["uniform"].double()[:, None] * running[:, -1:]
    tokens = (running <= target).sum(1).clamp(max=vocab - 1)
    chosen = w.gather(1, tokens[:, None]) / running[:, -1:]
    return {"tokens": tokens, "logprobs": chosen[:, 0].log().float()}


_OWN = {"attention": _own_attention, "rope": _own_rope, "linear": _own_linear,
        "sample": _own_sample}
_PLAIN = {"attention": _plain_attention, "rope": _plain_rope, "linear": _plain_linear,
          "sample": _plain_sample}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "attention":
        keys = sum(_lengths(case))
        if case["window"]:
            keys = sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"])))
                       for n in _lengths(case))
        b = 4 * keys * case["kv_heads"] * case["dim"] + 4 * case["batch"] * case["heads"] * case["dim"]
        f = 4 * keys * case["heads"] * case["dim"]
    elif kind == "rope":
        hq, hkv, n = case["heads"], case["kv_heads"], case["tokens"]
        stored = n - case["padding"]
        b = (2 * case["dim"] * (n * hq * 2 + stored * hkv * 4) + 4 * n * case["rotary"] + 16 * n)
        f = n * (hq + hkv) * case["dim"] * 8
    elif kind == "linear":
        m, n, k, g = case["rows"], case["out"], case["cols"], case["group"]
        b = n * k // 2 + 4 * n * (k // g) + 2 * m * k + m * n * (4 if case["out_dtype"] == "f32" else 2)
        f = 2 * m * n * k
    else:
        size = 4 if case["dtype"] == "f32" else 2
        b = case["batch"] * (case["vocab"] * size + 16)
        f = case["batch"] * case["vocab"] * 4
    return {"bytes": int(b), "flops": int(f)}


# ---------------------------------------------------------------------------
# The result in float64, sequence by sequence and row by row
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rope": _exact_rope, "linear": _exact_linear,
            "sample": _exact_sample}[case["kind"]](case, s)


def _exact_attention(case, s):
    hq, hkv, dim, page = case["heads"], case["kv_heads"], case["dim"], s["k"].shape[2]
    out = torch.zeros((case["batch"], hq, dim), dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(s["lengths"].tolist()):
        t = torch.arange(n, device=DEVICE)
        if case["window"] and n > case["window"]:
            t = torch.cat([t[:min(case["sinks"], n - case["window"])], t[n - case["window"]:]])
        pages = t // page + b if s["table"] is None else s["table"][b].long()[t // page]
        for h in range(hkv):
            group = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            keys = s["k"][pages, h, t % page].double()
            logits = torch.mm(s["q"][b, group].double(), keys.T) * s["scale"]
            out[b, group] = torch.mm(torch.softmax(logits, 1), s["v"][pages, h, t % page].double())
    return out


def _exact_rope(case, s):
    heads, hkv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows = s["qkv"].double().unflatten(1, (-1, dim))
    half = case["rotary"] // 2
    if case["interleaved"]:
        first = torch.arange(0, 2 * half, 2, device=DEVICE)
        second = first + 1
    else:
        first = torch.arange(half, device=DEVICE)
        second = first + half
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]

    def turned(x, weight):
        x = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q, k, v = rows.split([heads, hkv, hkv], 1)
    q, k = turned(q, s["qw"]), turned(k, s["kw"])
    pools = []
    for pool, new in ((s["k"], k), (s["v"], v)):
        # slot-major rows, the padding's in one more row behind them
        flat = torch.cat([pool.double().transpose(1, 2).flatten(0, 1),
                          torch.zeros((1, hkv, dim), dtype=torch.float64, device=DEVICE)])
        flat[s["slots"]] = new
        pools.append(flat[:-1].unflatten(0, (-1, page)).transpose(1, 2))
    return {"q": q, "k": pools[0], "v": pools[1]}


def _exact_linear(case, s):
    x, group = s["x"].double(), case["group"]
    out = torch.zeros((case["rows"], case["out"]), dtype=torch.float64, device=DEVICE)
    for g in range(case["cols"] // group):
        words = s["packed"][:, g * group // 8:(g + 1) * group // 8].long()
        part = x[:, g * group:(g + 1) * group]
        dot = torch.zeros_like(out)
        for i in range(8):
            dot += part[:, i::8] @ ((words // 16 ** i) % 16).double().T
        out += dot * s["scales"][:, g].double() + part.sum(1, keepdim=True) * s["biases"][:, g].double()
    return out


def _exact_sample(case, s):
    tokens, logprobs = [], []
    for b in range(case["batch"]):
        t, k, p, m = (float(s[name][b]) if case["mixed"] else float(case[name])
                      for name in ("temperature", "top_k", "top_p", "min_p"))
        row = s["logits"][b].double()
        if t == 0:
            tokens.append(int(row.argmax()))
            logprobs.append(0.0)
            continue
        weight = torch.exp((row - row.max()) / t)
        order = torch.argsort(-row, stable=True)[:int(k) if k > 0 else None]
        sorted_weight = weight[order]
        count = order.numel()
        if p < 1:
            ends = torch.cumsum(sorted_weight, 0)
            count = 1 + int(torch.searchsorted(ends, ends[-1:] * p)[0])
        if m > 0:
            count = min(count, int((sorted_weight >= m).sum()))
        chosen = torch.sort(order[:max(1, count)]).values
        ends = torch.cumsum(weight[chosen], 0)
        at = torch.searchsorted(ends, ends[-1:] * float(s["uniform"][b]), right=True)
        at = int(at[0].clamp(max=chosen.numel() - 1))
        tokens.append(int(chosen[at]))
        logprobs.append(float(torch.log(weight[chosen[at]] / ends[-1])))
    return {"tokens": torch.tensor(tokens, device=DEVICE),
            "logprobs": torch.tensor(logprobs, dtype=torch.float64, device=DEVICE)}
