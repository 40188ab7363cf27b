"""The attention weight of cached keys, the selection and compaction of an eviction, and the multi-axis rotary writer, from
their definitions in 64 bits (CPU). These operators have no reference counterpart; the attention they go by is the
oracle's (attention.segmented_prefill)."""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
from torch import Tensor


def page_rows(cache: Tensor, table_row: Tensor, n: int, g: int) -> tuple[Tensor, Tensor]:
    """(KV head g's rows [n, d] float64 of a row's first n tokens, [n] bool: the token lies on a valid page)."""
    nb, _, P, d = cache.shape
    rows = torch.zeros(n, d, dtype=torch.float64)
    ok = torch.zeros(n, dtype=torch.bool)
    for j in range(n):
        col = j // P
        page = int(table_row[col]) if col < table_row.numel() else -1
        if 0 <= page < nb:
            rows[j] = cache[page, g, j % P].double()
            ok[j] = True
    return rows, ok


def attention_weights(q: Tensor, k_cache: Tensor, table: Tensor, q_start: Sequence[int], prior: Sequence[int], width: int,
                      *, sm_scale: float, k_scale: Optional[Tensor] = None, multiply: bool = False, window: int = 0,
                      sinks: Optional[Tensor] = None) -> tuple[Tensor, float]:
    """([R, G, width] float64 weights, the largest sm_scale * sum |q k| of a visible pair, which bounds what rounding the
    scores can do)."""
    H, d = q.shape[1:]
    nb, G, P, _ = k_cache.shape
    grp, R = H // G, len(prior)
    out = torch.zeros(R, G, width, dtype=torch.float64)
    reach = 0.0
    for r in range(R):
        count = q_start[r + 1] - q_start[r]
        n = min(max(prior[r] + count, 0), table.shape[1] * P)
        if count <= 0 or n <= 0:
            continue
        for g in range(G):
            k, ok = page_rows(k_cache, table[r], n, g)
            if k_scale is not None:
                k = k / k_scale[g].double() if multiply else k * k_scale[g].double()
            for i in range(count):
                pos = prior[r] + i
                j = torch.arange(n)
                seen = ok & (j <= pos)
                if window > 0:
                    seen &= j > pos - window
                if not bool(seen.any()):
                    continue
                for h in range(g * grp, (g + 1) * grp):
                    qr = q[q_start[r] + i, h].double()
                    z = (k[seen] @ qr) * sm_scale
                    reach = max(reach, float((k[seen].abs() @ qr.abs()).max()) * sm_scale)
                    total = torch.logsumexp(z, 0)
                    if sinks is not None:
                        total = torch.logaddexp(total, sinks[h].double())
                    at = j[seen]
                    inside = at < width
                    out[r, g, at[inside]] += torch.exp(z - total)[inside]
    return out, reach


def select_tokens(weights: Tensor, lens: Sequence[int], keep: int, first: int, recent: int) -> tuple[Tensor, list[int]]:
    """(kept [R, G, keep] int32, new lengths), row by row: Python's stable sort on (NaN first, then the value)."""
    R, G, N = weights.shape
    kept = torch.full((R, G, keep), -1, dtype=torch.int32)
    new = []
    for r in range(R):
        L = min(max(int(lens[r]), 0), N)
        new.append(min(L, keep))
        for g in range(G):
            if L <= keep:
                at = list(range(L))
            else:
                w = weights[r, g].tolist()
                mid = sorted(range(first, L - recent), key=lambda i: (0, 0.0) if math.isnan(w[i]) else (1, -w[i]))
                at = sorted(list(range(first)) + mid[:keep - first - recent] + list(range(L - recent, L)))
            kept[r, g, :len(at)] = torch.tensor(at, dtype=torch.int32)
    return kept, new


def compact_tokens(cache: Tensor, table: Tensor, kept: Tensor, dst: Optional[Tensor] = None) -> Tensor:
    """The cache after the move: every kept token's row as it was before, at position i of the target's pages."""
    nb, G, P, _ = cache.shape
    dst = table if dst is None else dst
    out = cache.clone()
    for r in range(kept.shape[0]):
        for g in range(G):
            for i, j in enumerate(kept[r, g].tolist()):
                if j < 0 or j // P >= table.shape[1] or i // P >= dst.shape[1]:
                    continue
                a, b = int(table[r, j // P]), int(dst[r, i // P])
                if 0 <= a < nb and 0 <= b < nb:
                    out[b, g, i % P] = cache[a, g, j % P]
    return out


def mrope_rows(qkv: Tensor, positions: Tensor, inv_freq: Tensor, axes: Sequence[int], Hq: int, Hkv: int, d: int,
               q_norm: Optional[Tensor], k_norm: Optional[Tensor], eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(Q [T, Hq, d], K [T, Hkv, d], V [T, Hkv, d]) float64 of the writer, unrounded, and [T, Hq + Hkv, d] the size
    |x c| + |y s| that a rotated element's rounding errors are relative to (|x| where nothing is rotated)."""
    T, half = qkv.shape[0], inv_freq.numel()
    x = qkv.double().reshape(T, Hq + 2 * Hkv, d).clone()
    qk = x[:, :Hq + Hkv].clone()
    if q_norm is not None:
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + eps)
        qk = torch.cat([qk[:, :Hq] * q_norm.double(), qk[:, Hq:] * k_norm.double()], 1)
    size = qk.abs()
    y = qk.clone()
    for i in range(half):
        angle = (positions[axes[i]].double() * inv_freq[i].double())[:, None]
        c, s = torch.cos(angle), torch.sin(angle)
        a, b = qk[..., i], qk[..., i + half]
        y[..., i], y[..., i + half] = a * c - b * s, b * c + a * s
        size[..., i] = size[..., i + half] = a.abs() + b.abs()
    return y[:, :Hq], y[:, Hq:], x[:, Hq + Hkv:], size
