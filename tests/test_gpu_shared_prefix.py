"""``fpv2.shared_prefix_attention`` against the formula in float64 on the CPU (tolerances:
``batch_cases.tolerance``), and against ``decode_attention`` over caches that hold both parts."""

from __future__ import annotations

import math

import pytest
import torch

import fpv2
from batch_cases import BF16, F16, attention, fill_pages, paged, rand, tolerance

pytestmark = pytest.mark.gpu


def _case(seed, prefix, lengths, heads, hkv, dim, dtype, page, prefix_page, *, fill=math.nan, pool=False):
    """Inputs on the CPU; unused rows hold ``fill``.  ``pool``: one pool of pages for both."""
    gen = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    pk, pv = (rand(gen, hkv, prefix, dim, dtype=dtype) for _ in "kv")
    own = [[rand(gen, hkv, n, dim, dtype=dtype) for _ in "kv"] for n in lengths]
    first = -(-prefix // page) if pool else 0
    table, total, slots, shared = paged(gen, lengths, page, first=first)
    at = torch.cat(slots)
    c = {"q": rand(gen, batch, heads, dim, dtype=dtype) * 2, "table": table,
         "lengths": torch.tensor(lengths, dtype=torch.int32),
         "prefix_length": torch.tensor([prefix], dtype=torch.int32)}
    rows = [torch.cat([x[i] for x in own], 1) for i in (0, 1)]
    if pool:
        t = torch.arange(prefix)
        at = torch.cat([at, shared[t // page] * page + t % page])
        rows = [torch.cat([x, p], 1) for x, p in zip(rows, (pk, pv))]
    c["k"], c["v"] = (fill_pages(total, hkv, page, dim, at, x, fill, dtype) for x in rows)
    if pool:
        c["prefix_k"], c["prefix_v"], c["prefix_table"] = c["k"], c["v"], shared.to(torch.int32)
        if first == 0:
            c["prefix_table"] = torch.zeros(1, dtype=torch.int32)
    elif prefix_page:
        ptable, ptotal, pslots, _ = paged(gen, [prefix], prefix_page)
        c["prefix_k"], c["prefix_v"] = (
            fill_pages(ptotal, hkv, prefix_page, dim, pslots[0], x, fill, dtype) for x in (pk, pv))
        c["prefix_table"] = ptable[0].contiguous()
    else:  # the cache of a prefill, with room behind the prompt
        room = torch.full((hkv, 37, dim), fill, dtype=dtype)
        c["prefix_k"], c["prefix_v"] = (torch.cat([x, room], 1)[None] for x in (pk, pv))
        c["prefix_table"] = None
    c["dense"] = [[torch.cat([p, x], 1) for p, x in zip((pk, pv), xs)] for xs in own]
    return c


NAMES = ("q", "prefix_k", "prefix_v", "prefix_table", "prefix_length", "k", "v", "table", "lengths")


def _args(c, cuda, **change):
    return [x.to(cuda) if isinstance(x, torch.Tensor) else x for x in ({**c, **change}[n] for n in NAMES)]


def _check(c, cuda, scale=None, **change):
    got = fpv2.shared_prefix_attention(*_args(c, cuda, **change), scale=scale)
    q = c["q"]
    for b, (k, v) in enumerate(c["dense"]):
        want, mass, size = attention(q[b], k, v, q.shape[2] ** -0.5 if scale is None else scale)
        tol = tolerance(want, mass, size, k.shape[1], q.shape[2], q.dtype, q.dtype)
        err = (got[b].cpu().double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,hkv", [(4, 1), (6, 6), (14, 2), (24, 1), (40, 2)])
def test_heads(cuda, dtype, dim, heads, hkv):
    c = _case(dim + heads, 515, [0, 1, 33, 130, 7], heads, hkv, dim, dtype, 16, 48)
    _check(c, cuda)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [1, 2, 4, 5, 8, 9, 16, 17, 31, 33, 64, 100])
def test_batches(cuda, dtype, dim, batch):
    """Few rows of a KV head to hundreds: every tile of rows, and its border."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 60, (batch,), generator=gen).tolist()
    c = _case(batch, 700, lengths, 8, 2, dim, dtype, 16, 0)
    _check(c, cuda)


@pytest.mark.parametrize("batch", [3, 20, 70])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 1000, 4099])
def test_prefix_lengths(cuda, batch, prefix):
    c = _case(prefix, prefix, [5] * batch, 8, 2, 64, BF16, 16, 32)
    _check(c, cuda)


@pytest.mark.parametrize("page,prefix_page", [(1, 1), (3, 7), (48, 48), (16, 128), (128, 1000), (1000, 3)])
@pytest.mark.parametrize("batch", [2, 40])
def test_page_sizes(cuda, page, prefix_page, batch):
    c = _case(page, 901, [31, 200] * (batch // 2), 8, 2, 64, F16, page, prefix_page)
    _check(c, cuda, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_pool_equals_decode_attention(cuda, dtype):
    """Both parts in one pool; the same keys as one sequence each give the same within rounding."""
    lengths = [0, 3, 61, 500]
    c = _case(4, 1500, lengths, 8, 2, 128, dtype, 16, 0, pool=True)
    got = _check(c, cuda)
    k, v = (torch.stack([torch.nn.functional.pad(x[i], (0, 0, 0, 2000 - x[i].shape[1])) for x in c["dense"]])
            for i in (0, 1))
    whole = fpv2.decode_attention(c["q"].to(cuda), k.to(cuda), v.to(cuda), None,
                                  torch.tensor([1500 + n for n in lengths], dtype=torch.int32, device=cuda))
    for b, (kk, vv) in enumerate(c["dense"]):
        want, mass, size = attention(c["q"][b], kk, vv, 128 ** -0.5)
        tol = 2 * tolerance(want, mass, size, kk.shape[1], 128, dtype, dtype)
        assert bool(((got[b] - whole[b]).cpu().double().abs() <= tol).all())


def test_nothing_visible(cuda):
    """No prefix and no key of its own: zeros; one of both: the other part alone."""
    c = _case(5, 0, [0, 4, 0], 8, 2, 64, BF16, 16, 16)
    got = _check(c, cuda)
    assert not got[0].any() and not got[2].any() and got[1].any()
    got = _check(c, cuda, prefix_length=0)
    assert not got[0].any()


def test_integer_lengths_and_clipping(cuda):
    c = _case(6, 300, [20, 20, 20], 8, 2, 64, BF16, 16, 16)
    want = _check(c, cuda)
    args = _args(c, cuda, prefix_length=300, lengths=20)
    assert torch.equal(fpv2.shared_prefix_attention(*args), want)
    # past the tables: all that they hold; pages outside the caches: the nearest
    for big in (2 ** 31 - 1, 2 ** 70):
        full = _args(c, cuda, prefix_length=big, lengths=big, k=torch.zeros_like(c["k"]),
                     v=torch.ones_like(c["v"]), prefix_k=torch.zeros_like(c["prefix_k"]),
                     prefix_v=torch.ones_like(c["prefix_v"]), table=c["table"] + 10 ** 6,
                     prefix_table=c["prefix_table"] - 10 ** 6)
        assert bool((fpv2.shared_prefix_attention(*full) == 1).all())
    low = _args(c, cuda, prefix_length=torch.tensor([-5], dtype=torch.int32),
                lengths=torch.full((3,), -9, dtype=torch.int32))
    assert not fpv2.shared_prefix_attention(*low).any()


def test_strides_and_out(cuda):
    """Heads inside the rows of a pool, strided queries and destination, the queries' own place."""
    c = _case(7, 400, [300, 17, 40], 8, 2, 128, BF16, 32, 32)
    want = _check(c, cuda)
    change = {}
    for a, b in (("k", "v"), ("prefix_k", "prefix_v")):
        pages, hkv, page, dim = c[a].shape
        pool = torch.empty((pages, page, 2, hkv, dim + 8), dtype=BF16)[..., :dim]
        pool[:, :, 0], pool[:, :, 1] = c[a].transpose(1, 2), c[b].transpose(1, 2)
        pool = pool.to(cuda)
        change[a], change[b] = pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2)
    wide = torch.empty((8, 3, 136), dtype=BF16, device=cuda)[..., :128].transpose(0, 1)
    wide.copy_(c["q"])
    out = torch.full((3, 8, 131), 7.0, dtype=BF16, device=cuda)
    args = _args(c, cuda, **change)
    got = fpv2.shared_prefix_attention(wide, *args[1:], out=out[..., 2:130])
    assert got.data_ptr() == out[..., 2:130].data_ptr() and torch.equal(got, want)
    assert bool((out[..., :2] == 7).all()) and bool((out[..., 130:] == 7).all())
    shifted = torch.empty(3 * 8 * 128 + 1, dtype=BF16, device=cuda)[1:].view(3, 8, 128)
    shifted.copy_(c["q"])
    assert torch.equal(fpv2.shared_prefix_attention(shifted, *args[1:]), want)
    assert fpv2.shared_prefix_attention(args[0], *args[1:], out=args[0]) is args[0]
    assert torch.equal(args[0], want)


@pytest.mark.parametrize("batch", [2, 30])
def test_infinite_and_nan_values(cuda, batch):
    """What is visible counts as the formula has it."""
    c = _case(8, 200, [10] * batch, 2, 1, 64, BF16, 16, 0)
    c["q"].abs_()
    c["prefix_v"][0, 0, 7, 3] = math.inf
    c["prefix_k"][0, 0, 11] = -math.inf  # a key of score -inf: no weight
    for k, v in c["dense"]:
        v[0, 7, 3], k[0, 11] = math.inf, -math.inf
    got = fpv2.shared_prefix_attention(*_args(c, cuda)).cpu().double()
    assert bool((got[:, :, 3] == math.inf).all())
    for b, (k, v) in enumerate(c["dense"]):
        keep = torch.arange(210) != 11
        vv = v.clone()
        vv[0, :, 3] = 0
        want, mass, size = attention(c["q"][b], k[:, keep], vv[:, keep], 0.125)
        tol = tolerance(want, mass, size, 210, 64, BF16, BF16)
        fine = torch.arange(64) != 3
        assert bool(((got[b] - want).abs() <= tol)[:, fine].all())
    c["prefix_k"][0, 0, 12, 0] = math.nan
    assert bool(fpv2.shared_prefix_attention(*_args(c, cuda)).isnan().all())


# how far the other keys are below the greatest, in nats, one for each head
GAPS = [0.0, 8.0, 12.0, 15.0, 16.875, 17.5, 20.0, 24.0]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [1, 4, 40])
@pytest.mark.parametrize("at", [0, 20_000, 29_999, 30_003])
def test_keys_far_below_the_greatest(cuda, dtype, dim, batch, at):
    """One key far above the rest, in the prefix or behind it, whose value is zero, so that the
    rest are the result.

    Tolerance: every weight and the result are off by half a step of the storage type, or
    of its least normal number.  In float16 a tile's greatest weight is 2^5 to 2^15.9, so the rest of it may lie below the least normal number 2^-14 and be off by half
    a step, 2^-25.  Here it is 2^12 where the rest is so far below: the greatest key's tile is the
    first, or exceeds 2^15.9 and moves the reference to 2^-12 of it, as the rest (within 1 / ln 2
    bits) had 2^10 to 2^14 before.  So its 31 neighbours are off by 2^-37 of it each.  Scores are sums of three
    terms of at most 2^5 in float32 times log2 e: off by less than 8 * 2^-19, and the
    exponential by as much relative to its value; sums of a lane's terms, at most 2^11, by
    2^-13."""
    gen = torch.Generator().manual_seed(at)
    prefix, own = 30_000, 10
    length = prefix + own
    q = torch.zeros((batch, len(GAPS), dim), dtype=dtype)
    k = torch.zeros((length, dim), dtype=dtype)
    q[:, :, 0], q[:, :, 5] = torch.tensor(GAPS), 1.0
    k[at, 0] = 1.0
    k[:, 5] = torch.randint(-32, 33, (length,), generator=gen) / 64
    k[at, 5] = 0.5
    v = (1000 * (0.5 + torch.rand((length, dim), generator=gen))).to(dtype)
    v[at] = 0
    kd, vd = k.to(cuda), v.to(cuda)
    own_k, own_v = (x[prefix:].expand(batch, 1, own, dim).contiguous() for x in (kd, vd))
    got = fpv2.shared_prefix_attention(q.to(cuda), kd[None, None, :prefix], vd[None, None, :prefix], None,
                                       prefix, own_k, own_v, None, own, scale=1.0)
    s = q[0].double() @ k.double().T
    w = torch.softmax(s, 1)
    want = w @ v.double()
    info = torch.finfo(dtype)
    top = w.amax(1, keepdim=True)
    tol = (info.eps / 2 * (2 * want.abs()).clamp(min=info.tiny) + 2.0 ** -12 * want.abs()
           + (31 * 2.0 ** -37 * 1500 * top if dtype == F16 else 0))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), [float(x) for x in (err / tol).amax((0, 2))]


def test_many_short_own_parts(cuda):
    """More own items than workgroups, beside a short prefix."""
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 50, (700,), generator=gen).tolist()
    lengths[3], lengths[-1] = 900, 0
    c = _case(3, 45, lengths, 4, 2, 64, BF16, 16, 16)
    _check(c, cuda)


@pytest.mark.parametrize("lengths", [[9, 1, 0, 33] * 10, [900, 5] * 20], ids=["few", "many"])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_prefix_of_many_rows(cuda, dim, lengths):
    """Own keys before a long prefix's workgroups, and beside them."""
    _check(_case(4, 25_000, lengths, 32, 8, dim, BF16, 16, 64), cuda)


@pytest.mark.parametrize("dim", [64, 256])
def test_more_rows_than_workgroups(cuda, dim):
    """Every workgroup's place taken by one part of the prefix."""
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 40, (2100,), generator=gen).tolist()
    _check(_case(5, 70, lengths, 32, 8, dim, F16, 16, 16), cuda)


@pytest.mark.parametrize("batch,heads,hkv", [(2, 4, 2), (40, 12, 3), (150, 8, 1)])
@pytest.mark.parametrize("prefix,length", [(0, 0), (3, 1), (0, 600), (5000, 0), (5000, 600), (9000, 3)])
def test_caches_wider_than_what_they_hold(cuda, batch, heads, hkv, prefix, length):
    """The launch goes by the caches' size, the work by the lengths on the device."""
    gen = torch.Generator().manual_seed(6)
    dim, page = 64, 16
    k, v = (rand(gen, 700, hkv, page, dim, dtype=BF16) for _ in "kv")
    c = {"q": rand(gen, batch, heads, dim, dtype=BF16) * 2, "k": k, "v": v, "prefix_k": k, "prefix_v": v,
         "prefix_table": torch.randint(0, 700, (600,), generator=gen, dtype=torch.int32),
         "table": torch.randint(0, 700, (batch, 40), generator=gen, dtype=torch.int32),
         "prefix_length": torch.tensor([prefix], dtype=torch.int32),
         "lengths": torch.tensor([max(0, length - b % 3) for b in range(batch)], dtype=torch.int32)}
    rows = [x.transpose(1, 2).reshape(-1, hkv, dim) for x in (k, v)]
    t = torch.arange(page)

    def held(table, n):
        at = (table.long()[:, None] * page + t).view(-1)[:n]
        return [x[at].transpose(0, 1) for x in rows]

    shared = held(c["prefix_table"], prefix)
    c["dense"] = [[torch.cat(x, 1) for x in zip(shared, held(c["table"][b], int(c["lengths"][b])))]
                  for b in range(batch)]
    _check(c, cuda)


def test_prefix_past_32_bits(cuda):
    """A contiguous prefix whose last rows lie behind 4 GiB (and 2^31 elements): values of ones
    there, of zeros before, and scores that make only the last rows count."""
    rows, dim, last = 17_000_000, 128, 96
    k = torch.zeros((1, 1, rows, dim), dtype=BF16, device=cuda)
    v = torch.zeros_like(k)
    length = rows - 5
    k[0, 0, length - last:, 0] = 60.0
    v[0, 0, length - last:length] = 1.0
    k[0, 0, length:], v[0, 0, length:] = math.nan, math.nan
    own = torch.zeros((9, 1, 4, dim), dtype=BF16, device=cuda)
    for batch in (2, 9):
        q = torch.ones((batch, 4, dim), dtype=BF16, device=cuda)
        got = fpv2.shared_prefix_attention(q, k, v, None, length, own[:batch], own[:batch], None, 4, scale=1.0)
        # (the rest weighs 17e6 e^-60; weights of one are exact)
        assert bool((got == 1).all())


@pytest.mark.parametrize("batch", [2, 20])
def test_rows_far_apart(cuda, batch):
    """Rows of the prefix whose distance times 16 leaves 31 bits of bytes."""
    c = _case(7, 39, [5 + b % 7 for b in range(batch)], 4, 1, 64, BF16, 16, 0)
    far = torch.empty(39 * 2 ** 26 + 128, dtype=BF16, device=cuda)
    for name, at in (("prefix_k", 0), ("prefix_v", 64)):
        rows = far.as_strided((1, 1, 39, 64), (0, 0, 2 ** 26, 1), at)
        rows.copy_(c[name][:, :, :39])
        c[name] = rows
    _check(c, cuda)


def test_graph_replays_follow_lengths_and_tables(cuda):
    """Two captured calls of different sizes and eager calls between their replays."""
    cases = [_case(9, 600, [90, 40, 0], 8, 2, 64, BF16, 16, 16, fill=0.0),
             _case(10, 3000, [17] * 40, 8, 2, 128, F16, 16, 64, fill=0.0)]
    cases = [_args(c, cuda) for c in cases]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for args in cases:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            fpv2.shared_prefix_attention(*args)  # warm-up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fpv2.shared_prefix_attention(*args))
        graphs.append(graph)
    for step in range(4):
        for args in cases:
            args[0].mul_(1.1)
            args[4].sub_(130)
            args[8].sub_(3)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, args in zip(outs, cases):
            assert torch.equal(out, fpv2.shared_prefix_attention(*args))


def test_runs_on_the_current_stream(cuda):
    for batch in (2, 40):
        args = _args(_case(11, 2000, [30] * batch, 8, 2, 128, BF16, 16, 0), cuda)
        want = fpv2.shared_prefix_attention(*args)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            late = torch.zeros_like(args[0])
            torch.cuda._sleep(20_000_000)
            late.copy_(args[0])
            got = fpv2.shared_prefix_attention(late, *args[1:])
        side.synchronize()
        assert torch.equal(got, want)
