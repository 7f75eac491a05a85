"""Cases and references shared by the tests of ``fpv2.batch`` (CPU, float64)."""

from __future__ import annotations

import math

import torch

BF16, F16 = torch.bfloat16, torch.float16


def rand(gen, *shape, dtype):
    return torch.randn(shape, generator=gen).to(dtype)


def quantized(x):
    """Codes and scales of rows ``x`` by the definition, with every step exact: ``127 x`` and
    the quotients that lie half way between two codes are whole in float64."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    codes = (127 * x / torch.where(a == 0, 1.0, a)).round()
    return codes.to(torch.int8), (a[..., 0] / 127).float()


def paged(gen, lengths, page, *, spare=2, first=0):
    """Pages in random order: a table for ``lengths`` (unused entries hold a spare page), the
    number of pages, each sequence's tokens' slots, and ``first`` pages more."""
    counts = [-(-n // page) for n in lengths]
    width, total = max(1, *counts), sum(counts) + spare + first
    perm = torch.randperm(total, generator=gen)
    table = torch.full((len(lengths), width), int(perm[-1]), dtype=torch.int32)
    at, slots = first, []
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            table[b, i] = perm[at + i]
        t = torch.arange(n)
        slots.append(perm[at + t // page] * page + t % page if n else t)
        at += counts[b]
    return table, total, slots, perm[:first]


def fill_pages(total, hkv, page, dim, slots, rows, fill, dtype):
    """Pages ``[total, hkv, page, dim]`` of ``fill`` with ``rows`` ``[hkv, n, dim]`` at ``slots``."""
    pages = torch.full((total, page, hkv, dim), fill, dtype=dtype)
    pages.view(total * page, hkv, dim)[slots] = rows.transpose(0, 1).to(dtype)
    return pages.transpose(1, 2).contiguous()


def attention(q, keys, values, scale):
    """float64 result of one sequence's queries ``[Hq, D]`` over ``[Hkv, n, D]``, with the
    weighted mass ``sum w |v|`` and the largest ``scale sum |q k|``."""
    hkv, n, dim = keys.shape
    group = q.shape[0] // hkv
    if n == 0:
        zero = torch.zeros(q.shape, dtype=torch.float64)
        return zero, zero, torch.zeros((q.shape[0], 1), dtype=torch.float64)
    qq = q.double().view(hkv, group, dim)
    k, v = keys.double(), values.double()
    w = torch.softmax(qq @ k.transpose(1, 2) * scale, -1)
    size = (qq.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
    return ((w @ v).view(-1, dim), (w @ v.abs()).view(-1, dim), size.view(-1, 1))


def tolerance(out, mass, size, n, dim, storage, weights):
    """Per element: the weights are rounded once to ``weights`` before their product with V
    (half a step of ``mass``) and the result once to ``storage``; a float32 score is off by at most
    (D + 16) 2^-24 of ``size``, its exponential by as much and by 2^-22, partial sums of n terms
    and their joins by n 2^-24."""
    return (torch.finfo(storage).eps / 2 * out.abs() + torch.finfo(weights).eps / 2 * mass
            + (2 * (dim + 16) * size + 2 * n + 64) * 2.0 ** -24 * mass
            + torch.finfo(storage).smallest_normal * torch.finfo(storage).eps)
