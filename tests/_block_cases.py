"""Caches whose blocks of tokens carry scales, for the tests of their operators: tables and pools on the CPU."""

from __future__ import annotations

import torch

from oracle import blocks as ob

FMTS = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tokens(g, *shape):
    """Normal elements, each token (all but the last axis) at a size of its own."""
    size = torch.exp(0.6 * torch.randn(*shape[:-1], 1, generator=g))
    return torch.randn(*shape, generator=g) * size


def table_of(g, lens, P, extra=0):
    """(table [R, W] int32 of pages at random places from 1 on, -1 past a row's; the pool's pages)."""
    need = [-(-n // P) for n in lens]
    W = max(1, max(need)) + extra
    ids = (torch.randperm(sum(need), generator=g) + 1).tolist()
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(need) + 1


def garbage(cache, scale=None):
    """Every byte of a cache a NaN (int8: -128), every scale NaN: what a pool may hold where nothing was stored."""
    if cache.dtype == torch.bfloat16:
        cache.fill_(float("nan"))
    elif cache.dtype == torch.int8:
        cache.fill_(-128)
    else:
        cache.view(torch.uint8).fill_(0x7F)
    if scale is not None:
        scale.fill_(float("nan"))


def pool(g, nb, G, P, d, bt, fmt):
    """(cache, scale or None) of random codes."""
    x = tokens(g, nb, G, P, d)
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    dt = FMTS[fmt]
    s = x.reshape(nb, G, P // bt, bt * d).abs().amax(-1) / ob.top_of(dt)
    return ob.round_codes(x / s.repeat_interleave(bt, 2).unsqueeze(-1), dt), s


def hide_unstored(cache, scale, table, lens, P):
    """Garbage in every place of the pool that no row's first lens[r] tokens take, scales of wholly unused blocks included."""
    nb, G = cache.shape[:2]
    live = torch.zeros(nb, P, dtype=torch.bool)
    for r, n in enumerate(lens):
        for j in range(n):
            if j // P < table.shape[1] and 0 <= int(table[r, j // P]) < nb:
                live[int(table[r, j // P]), j % P] = True
    bad = torch.empty_like(cache[:1, :1, :1])
    garbage(bad)
    raw, b = (cache.view(torch.uint8), bad.view(torch.uint8)) if cache.dtype == ob.FP8 else (cache, bad)
    raw.copy_(torch.where(live[:, None, :, None], raw, b))
    if scale is not None:
        used = live.view(nb, scale.shape[2], -1).any(-1)
        scale.copy_(torch.where(used[:, None, :], scale, float("nan")))


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    if a.dtype == ob.FP8:
        return torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return torch.equal(a, b)


def to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]
