"""A cache whose blocks of tokens carry scales, its key bounds, and attention over it, from their definitions (CPU). These
operators have no reference counterpart. Scales and codes are stated in 32 bits operation by operation, as a code is exact or
wrong; attention and scores are in 64 bits."""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
from torch import Tensor

FP8 = torch.float8_e4m3fn
LEAST_SCALE = 2.0 ** -100
# What a prompt's query element over int8 codes is off by, of its row's largest: half a step of 32600, the quotient 32600 / largest
# and its product with the element rounded (2^-24 each, of up to 32600 steps), the step's size rounded (2^-24).
INT8_QUERY_OFF = (0.5 + 32600 * 2.0 ** -23) / 32600 + 2.0 ** -24


def top_of(dtype: torch.dtype) -> float:
    return 448.0 if dtype == FP8 else 127.0


def round_codes(y: Tensor, dtype: torch.dtype) -> Tensor:
    """Codes of quotients y (fp32): clamped, to nearest even."""
    if dtype == FP8:
        return y.clamp(-448, 448).to(FP8)
    return torch.nan_to_num(y).clamp(-127, 127).round().to(torch.int8)


def append(cache: Tensor, scale: Optional[Tensor], new: Tensor, table: Tensor, q_start: Sequence[int], prior: Sequence[int],
           bounds: Optional[Tensor] = None, max_q_len: int = 1 << 30) -> None:
    """``new`` [T, G, d] bf16 joined, in place, to a cache [blocks, G, P, d] with scales [blocks, G, n] (None: bf16), block
    by block; bounds [blocks, G, 2, d] of the tokens, when given."""
    nb, G, P, d = cache.shape
    bt = P if scale is None else P // scale.shape[2]
    raw = cache.view(torch.uint8) if cache.dtype == FP8 else cache
    for r in range(len(prior)):
        n = min(q_start[r + 1] - q_start[r], max_q_len)
        at, end = prior[r], prior[r] + n
        while at < end:
            stop = min(end, (at // bt + 1) * bt)
            x = new[q_start[r] + at - prior[r]:q_start[r] + stop - prior[r]].transpose(0, 1)  # [G, n, d]
            col, lo = at // P, at % P
            page = int(table[r, col]) if col < table.shape[1] else -1
            first = at % bt == 0
            fresh_page = lo == 0
            here, at = at, stop
            if not 0 <= page < nb:
                continue
            if bounds is not None:
                f = x.float()
                low = torch.where(f.isnan(), math.inf, f).amin(1)
                high = torch.where(f.isnan(), -math.inf, f).amax(1)
                if not fresh_page:
                    low, high = torch.minimum(low, bounds[page, :, 0].float()), torch.maximum(high, bounds[page, :, 1].float())
                bounds[page, :, 0], bounds[page, :, 1] = low.to(bounds.dtype), high.to(bounds.dtype)
            if scale is None:
                cache[page, :, lo:lo + stop - here] = x
                continue
            u, head = lo // bt, lo - lo % bt
            f = x.float()
            most = torch.where(f.isinf(), 0.0, f.abs()).amax((1, 2))  # (a NaN makes it NaN)
            now = (most * (torch.ones(()) / top_of(cache.dtype))).clamp(min=LEAST_SCALE)
            if not first:
                had = scale[page, :, u].clone()
                now = torch.maximum(now, had)
                old = cache[page, :, head:lo]
                again = round_codes(old.float() * had.view(-1, 1, 1) / now.view(-1, 1, 1), cache.dtype)
                grew = (now > had).view(-1, 1, 1)
                raw[page, :, head:lo] = torch.where(grew, again.view(raw.dtype), raw[page, :, head:lo])
            scale[page, :, u] = now
            raw[page, :, lo:lo + stop - here] = round_codes(f / now.view(-1, 1, 1), cache.dtype).view(raw.dtype)


def rows_of(cache: Tensor, scale: Optional[Tensor], pages: Sequence[int], g: int) -> Tensor:
    """[len(pages) * P, d] float64 values of KV head g on the pages."""
    nb, _, P, d = cache.shape
    at = torch.tensor(list(pages), dtype=torch.long)
    x = cache[at, g].double()
    if scale is not None:
        x = x * scale[at, g].double().repeat_interleave(P // scale.shape[2], 1).unsqueeze(-1)
    return x.reshape(-1, d)


def attend(q: Tensor, k: Tensor, v: Tensor, sm_scale: float, sinks: Optional[Tensor],
           q_off: float = 0.0) -> tuple[Tensor, Tensor]:
    """(out [grp, d], its error bound [grp, d]) of one query's heads q [grp, d] over keys k, v [n, d] (float64) with sinks
    [grp]. The bound is for a kernel that holds scores, statistics and sums in 32 bits, rounds probabilities and the output to
    bf16, each by at most 2^-8 of itself, sums the probabilities as it rounded them, and takes a query element to within q_off
    of its row's largest."""
    grp, d = q.shape
    if k.shape[0] == 0:
        return torch.zeros(grp, d, dtype=torch.float64), torch.zeros(grp, d, dtype=torch.float64)
    z = (q.double() @ k.t()) * sm_scale
    total = torch.logsumexp(z, -1, keepdim=True)
    if sinks is not None:
        total = torch.logaddexp(total, sinks.double().view(-1, 1))
    p = torch.exp(z - total)
    out = p @ v
    reach = (q.double().abs() @ k.abs().t()).amax(-1, keepdim=True) * sm_scale
    # a score is off by at most (d + 4) 2^-24 reach and the exponential by 2^-20 (its argument's rounding among it, under
    # reach 2^-22), so a weight, over its sum, by twice that; the sums by n 2^-24
    q_err = q_off * q.double().abs().amax(-1, keepdim=True) * k.abs().sum(-1).amax() * sm_scale
    rel = 2.0 ** -8 + torch.expm1(2 * q_err) + 2 * ((d + 8) * 2.0 ** -24 * reach + 2.0 ** -20) + k.shape[0] * 2.0 ** -23
    # sum p_j (1 + e_j) v_j / sum p_j (1 + e_j) - out = sum p_j e_j (v_j - out) / sum p_j (1 + e_j), with |e_j| <= 2^-8 at most
    # 2^-8 (sum p_j |v_j| + |out|) / (1 - 2^-8); the output's own rounding is 2^-8 |out| more
    return out, 2.0 ** -8 * (2 + 2.0 ** -7) * out.abs() + rel * (1 + 2.0 ** -7) * (p @ v.abs())


def decode(q: Tensor, k_cache: Tensor, v_cache: Tensor, table: Tensor, lens: Sequence[int], *, sm_scale: float,
           k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None, sinks: Optional[Tensor] = None, window: int = 0,
           rows: Optional[Sequence[int]] = None, blocks: Optional[Tensor] = None,
           q_off: float = 0.0) -> tuple[Tensor, Tensor]:
    """([T, H, d] float64, its error bound) of single queries over their rows, or over the columns that blocks [T, G, n]
    names."""
    T, H, d = q.shape
    nb, G, P, _ = k_cache.shape
    grp, W = H // G, table.shape[1]
    out, off = torch.zeros(T, H, d, dtype=torch.float64), torch.zeros(T, H, d, dtype=torch.float64)
    for t in range(T):
        r = t if rows is None else int(rows[t])
        if not 0 <= r < table.shape[0]:
            continue
        L = int(lens[t])
        for g in range(G):
            cols = range(W) if blocks is None else [int(c) for c in blocks[t, g] if 0 <= int(c) < W]
            cols = [c for c in cols if c * P < L and 0 <= int(table[r, c]) < nb]
            key = (torch.tensor(cols, dtype=torch.long).view(-1, 1) * P + torch.arange(P)).reshape(-1)
            seen = key < L
            if window > 0:
                seen &= key >= L - window
            pages = [int(table[r, c]) for c in cols]
            k, v = rows_of(k_cache, k_scale, pages, g)[seen], rows_of(v_cache, v_scale, pages, g)[seen]
            h = slice(g * grp, (g + 1) * grp)
            out[t, h], off[t, h] = attend(q[t, h], k, v, sm_scale, None if sinks is None else sinks[h],
                                           q_off)
    return out, off


def prefill(q: Tensor, k_cache: Tensor, v_cache: Tensor, table: Tensor, q_start: Sequence[int], prior: Sequence[int],
            **kw) -> tuple[Tensor, Tensor]:
    """The same for chunks: query i of request r sees the keys up to position prior[r] + i."""
    rows, lens = [], []
    for r in range(len(prior)):
        for i in range(q_start[r + 1] - q_start[r]):
            rows.append(r)
            lens.append(prior[r] + i + 1)
    return decode(q, k_cache, v_cache, table, lens, rows=rows, **kw)


def scores(q: Tensor, bounds: Tensor, table: Tensor, lens: Sequence[int], P: int,
           rows: Optional[Sequence[int]] = None) -> tuple[Tensor, Tensor, list[int]]:
    """([T, G, W] float64 scores, the sums of magnitudes that their rounding errors are relative to, the rows' pages). A product
    with a query element of 0 is 0, whatever the bounds; a head whose sum is NaN counts only where all of them are."""
    T, H, d = q.shape
    nb, G = bounds.shape[:2]
    grp, W = H // G, table.shape[1]
    out = torch.full((T, G, W), -math.inf, dtype=torch.float64)
    size = torch.zeros(T, G, W, dtype=torch.float64)
    counts = [-(-max(int(n), 0) // P) for n in lens]
    for t in range(T):
        r = t if rows is None else int(rows[t])
        if not 0 <= r < table.shape[0]:
            continue
        for c in range(min(W, counts[t])):
            page = int(table[r, c])
            if not 0 <= page < nb:
                continue
            for g in range(G):
                x = q[t, g * grp:(g + 1) * grp].double()
                lo, hi = bounds[page, g, 0].double(), bounds[page, g, 1].double()
                each = torch.where(x == 0, 0.0, torch.maximum(x * lo, x * hi))
                heads = each.sum(-1)
                out[t, g, c] = heads.max() if bool(heads.isnan().all()) else heads[~heads.isnan()].max()
                size[t, g, c] = each.abs().sum(-1).max()
    return out, size, counts
