"""Performance cases of a KV cache whose blocks of tokens carry a scale of their own (e4m3fn or int8, or bf16 without
scales): the writer that appends tokens to it, attention of single tokens and of prompt chunks over it, the score of each
page for a query from the bounds of the page's keys, and attention over the pages that a query selects. Each case runs the
package's entry points, or the same operators in plain torch operations.

A case is a dict of plain values; ``op`` names the operator, ``P`` is the page and ``bt`` the tokens that share a scale. A
batch's lengths are spread over ``lo`` .. ``hi`` (so the work does not depend on the seed) and dealt to its rows at random;
pages lie at random places of the pool.
"""

from __future__ import annotations

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DEV = "cuda"
LEAST_SCALE = 2.0 ** -100
TOP = {"fp8": 448.0, "int8": 127.0}

# head shapes: (query heads, KV heads, head dim)
QWEN3_8B = dict(H=32, G=8, d=128)
QWEN3_06B = dict(H=16, G=8, d=128)
GPT_OSS_SHARE = dict(H=8, G=1, d=64)  # one of eight ranks' heads


def listed():
    return [
        # the new token of each row of a small batch joins its block: the shortest call
        dict(name="store-step-8-int8", op="store", R=8, q_lo=1, q_hi=1, lo=128, hi=1024, **QWEN3_06B, P=16, bt=16,
             fmt="int8", bounds=False),
        # a prefill batch's chunks: four requests, each 2048 tokens after an odd prompt, with the pages' key bounds kept
        dict(name="store-chunk-4x2048-fp8", op="store", R=4, q_lo=2048, q_hi=2048, lo=2049, hi=4077, **QWEN3_8B, P=64,
             bt=32, fmt="fp8", bounds=True),
        # one decode step of a small model's batch: launches and latency
        dict(name="decode-b8-int8", op="decode", R=8, q=1, lo=128, hi=1024, **QWEN3_06B, P=16, bt=16, fmt="int8",
             window=0, sinks=False),
        # a full serving batch at 4k context
        dict(name="decode-b64-fp8", op="decode", R=64, q=1, lo=4096, hi=4096, **QWEN3_8B, P=16, bt=16, fmt="fp8", window=0,
             sinks=False),
        # a ragged batch of wide groups with sinks: one rank's share of the heads
        dict(name="decode-b128-sinks-int8", op="decode", R=128, q=1, lo=2048, hi=8192, **GPT_OSS_SHARE, P=32, bt=32,
             fmt="int8", window=0, sinks=True),
        # one very long document
        dict(name="decode-131071-int8", op="decode", R=1, q=1, lo=131071, hi=131071, **QWEN3_8B, P=128, bt=32, fmt="int8",
             window=0, sinks=False),
        # a prefill batch in chunks: four requests, each 2048 tokens after 2048
        dict(name="chunk-4x2048-fp8", op="chunk", R=4, q_lo=2048, q_hi=2048, lo=4096, hi=4096, **QWEN3_8B, P=16, bt=16,
             fmt="fp8", window=0, sinks=False),
        # odd chunks of a model with a sliding window and sinks
        dict(name="chunk-3x635-int8", op="chunk", R=3, q_lo=101, q_hi=635, lo=777, hi=2270, H=24, G=4, d=64, P=32, bt=16,
             fmt="int8", window=1000, sinks=True),
        # a serving batch scores the pages of 16k tokens at each step
        dict(name="scores-b64", op="scores", R=64, q=1, lo=16384, hi=16384, **QWEN3_8B, P=64),
        # one very long document in small pages
        dict(name="scores-131071", op="scores", R=1, q=1, lo=131071, hi=131071, **QWEN3_8B, P=32),
        # a step over 2048 selected keys of up to 32768 a row
        dict(name="selected-b32-fp8", op="selected", R=32, q=1, lo=9001, hi=32768, **QWEN3_8B, P=64, bt=64, fmt="fp8",
             n=32, sinks=False),
        # the last 256 queries of two prompts, each with pages of its own choice
        dict(name="selected-2x256-bf16", op="selected", R=2, q=256, lo=8191, hi=16384, **QWEN3_06B, P=64, bt=64,
             fmt="bf16", n=16, sinks=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "store", "decode", "decode", "decode", "chunk", "chunk", "scores", "selected", "selected"])
    heads = dict(rng.choice([QWEN3_8B, QWEN3_06B, GPT_OSS_SHARE, dict(H=12, G=4, d=128), dict(H=20, G=4, d=64)]))
    P = rng.choice([16, 32, 48, 64, 128])
    bt = rng.choice([b for b in (16, 32, 48, 64, 128) if P % b == 0])
    fmt = rng.choice(["fp8", "fp8", "int8", "int8", "bf16"])
    es = 2 if fmt == "bf16" else 1
    G, d, H = heads["G"], heads["d"], heads["H"]
    if op == "store":
        R, q = _log_int(rng, 1, 128), _log_int(rng, 1, 4096) if rng.random() < 0.6 else 1
        while R * q > 8192:
            R = max(1, R // 2)
        hi = q + _log_int(rng, 1, 4096)
        while R * hi * G * d > 4 * 4096 * 8 * 128 * 4:
            hi = q + (hi - q) // 2
        lo = max(q, int(hi * rng.uniform(0.3, 1.0)))
        return dict(op=op, R=R, q_lo=max(1, int(q * rng.uniform(0.2, 1.0))), q_hi=q, lo=lo, hi=hi, **heads, P=P, bt=bt,
                    fmt=fmt, bounds=rng.random() < 0.5)
    if op == "chunk":
        R, hi, q = _log_int(rng, 1, 8), _log_int(rng, 64, 131072), _log_int(rng, 1, 4096)
        while R * min(q, hi) * hi * H > 7.0e8 or R * min(q, hi) > 8192 or R * hi * G * d * es > 64 * 4096 * 8 * 128:
            hi, q, R = max(64, hi * 3 // 4), max(1, q * 3 // 4), max(1, R - 1)
        q = min(q, hi)
        return dict(op=op, R=R, q_lo=max(1, int(q * rng.uniform(0.2, 1.0))), q_hi=q, lo=max(q, int(hi * rng.uniform(0.3, 1.0))),
                    hi=hi, **heads, P=P, bt=bt, fmt=fmt, window=rng.choice([0, 0, 0, 128, 1000]), sinks=rng.random() < 0.4)
    R, hi, q = _log_int(rng, 1, 128), _log_int(rng, 16, 131072), rng.choice([1, 1, 1, 1, 3])
    if op == "scores":
        while R * -(-hi // P) * G * d > 64 * 256 * 8 * 128:
            hi = max(1, hi * 2 // 3)
        return dict(op=op, R=R, q=min(q, hi), lo=max(min(q, hi), int(hi * rng.uniform(0.1, 1.0))), hi=hi, **heads, P=P)
    if op == "selected":
        q = rng.choice([1, 1, 1, 3, _log_int(rng, 1, 256)])
        n = _log_int(rng, 1, 64)
        while R * q * n * P * G * d * es > 32 * 2048 * 8 * 128 * 2:
            R, q, n = max(1, R * 2 // 3), max(1, q * 2 // 3), max(1, n * 3 // 4)
        while R * hi * G * d * es > 32 * 32768 * 8 * 128:
            hi = max(1, hi * 2 // 3)
        q = min(q, hi)
        return dict(op=op, R=R, q=q, lo=max(q, int(hi * rng.uniform(0.1, 1.0))), hi=hi, **heads, P=P, bt=bt, fmt=fmt, n=n,
                    sinks=rng.random() < 0.4)
    while R * hi * G * d * es > 64 * 4096 * 8 * 128:
        hi = max(1, hi * 2 // 3)
    q = min(q, hi)
    return dict(op=op, R=R, q=q, lo=max(q, int(hi * rng.uniform(0.1, 1.0))), hi=hi, **heads, P=P, bt=bt, fmt=fmt,
                window=rng.choice([0, 0, 0, 128, 1000]), sinks=rng.random() < 0.4)


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _spread(lo, hi, n):
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _tokens(g, *shape):
    """Normal elements, each token (all but the last axis) at a size of its own, as keys and values have it."""
    return _randn(g, *shape) * torch.exp(0.4 * _randn(g, *shape[:-1], 1))


def _pool(g, blocks, G, P, d, bt, fmt):
    x = _tokens(g, blocks, G, P, d)
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    s = x.view(blocks, G, P // bt, bt * d).abs().amax(-1) / TOP[fmt]
    y = x / s.repeat_interleave(bt, 2).unsqueeze(-1)
    return (y.clamp(-448, 448).to(FP8) if fmt == "fp8" else y.round().clamp(-127, 127).to(torch.int8)), s


def _table(g, lens, P):
    """[R, width] int32 pages at random places from page 1 on, -1 past a row's."""
    need = torch.tensor([-(-n // P) for n in lens], device=DEV)
    W, count = max(1, -(-max(lens) // P)), sum(-(-n // P) for n in lens)
    live = torch.arange(W, device=DEV)[None, :] < need[:, None]
    table = torch.full((len(lens), W), -1, dtype=torch.int32, device=DEV)
    table[live] = (torch.randperm(count, generator=g, device=DEV) + 1).to(torch.int32)
    return table, count


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    op, R, H, G, d, P = case["op"], case["R"], case["H"], case["G"], case["d"], case["P"]
    deal = torch.randperm(R, generator=g, device=DEV).tolist()
    lens = [_spread(case["lo"], case["hi"], R)[i] for i in deal]
    table, count = _table(g, lens, P)
    s = dict(op=op, H=H, G=G, d=d, P=P, table=table)
    if op != "scores":
        s.update(bt=case["bt"], fmt=case["fmt"])
        s["k"], s["k_scale"] = _pool(g, count + 1, G, P, d, case["bt"], case["fmt"])
        s["v"], s["v_scale"] = _pool(g, count + 1, G, P, d, case["bt"], case["fmt"])
    if op in ("store", "chunk"):
        qs = [_spread(case["q_lo"], case["q_hi"], R)[i] for i in deal]
        qs = [min(q, n) for q, n in zip(qs, lens)]
        start = [sum(qs[:r]) for r in range(R + 1)]
        s.update(max_q=max(qs), prior=_i32([n - q for n, q in zip(lens, qs)]),
                 q_start=None if op == "store" and max(qs) == 1 else _i32(start))
        T = start[-1]
        if op == "store":
            s["new_k"], s["new_v"] = _tokens(g, T, G, d).to(torch.bfloat16), _tokens(g, T, G, d).to(torch.bfloat16)
            s["bounds"] = None
            if case["bounds"]:
                x = _tokens(g, count + 1, G, 4, d)
                s["bounds"] = torch.stack([x.amin(2), x.amax(2)], 2).to(torch.bfloat16)
            return s
    else:  # the last q queries of each row, each seeing what lies before it
        q = case["q"]
        T = R * q
        s.update(rows=None if q == 1 else _i32([r for r in range(R) for _ in range(q)]),
                 lens=_i32([n - q + 1 + i for n in lens for i in range(q)]))
    s["q"] = _randn(g, T, H, d).to(torch.bfloat16)
    if op == "scores":
        x = _tokens(g, count + 1, G, 8, d)
        s["bounds"] = torch.stack([x.amin(2), x.amax(2)], 2).to(torch.bfloat16)
        return s
    s.update(sm_scale=1.0 / math.sqrt(d), window=case.get("window", 0), sinks=_randn(g, H) if case["sinks"] else None)
    if op == "selected":  # each query and KV head: the first and the last page and others at random, in order
        n, W = case["n"], table.shape[1]
        pages = (s["lens"] + P - 1) // P
        c = torch.arange(W, device=DEV)
        rank = torch.rand(T, G, W, generator=g, device=DEV)
        rank = torch.where((c == 0) | (c == pages.view(T, 1, 1) - 1), 2.0, rank)
        rank = torch.where(c < pages.view(T, 1, 1), rank, -1.0)
        top = rank.topk(min(n, W), -1)
        at = torch.where(top.values >= 0, top.indices, W).sort(-1).values
        s["blocks"] = torch.where(at < W, at, -1).to(torch.int32).contiguous()
    return s


# ---- one pass ----

def run(s):
    if own:
        return _run_own(s)
    return {"store": _plain_store, "decode": _plain_decode, "chunk": _plain_chunk, "scores": _plain_scores,
            "selected": _plain_decode}[s["op"]](s)


def _run_own(s):
    from sglang_neuron_amd import ops

    if s["op"] == "store":
        ops.kv_store_blocks(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["prior"], q_start=s["q_start"],
                            max_q_len=s["max_q"], k_scale=s["k_scale"], v_scale=s["v_scale"], k_bounds=s["bounds"])
        return [x for x in (s["k"], s["v"], s["k_scale"], s["v_scale"], s["bounds"]) if x is not None]
    if s["op"] == "scores":
        return ops.block_scores(s["q"], s["bounds"], s["table"], s["lens"], page_size=s["P"], rows=s["rows"])
    if s["op"] == "chunk":
        return ops.prefill_attention_blocks(s["q"], s["k"], s["v"], s["table"], s["q_start"], s["prior"],
                                            max_q_len=s["max_q"], sm_scale=s["sm_scale"], k_scale=s["k_scale"],
                                            v_scale=s["v_scale"], sinks=s["sinks"], window=s["window"])
    if s["op"] == "selected":
        return ops.paged_decode_selected(s["q"], s["k"], s["v"], s["table"], s["lens"], s["blocks"], sm_scale=s["sm_scale"],
                                         k_scale=s["k_scale"], v_scale=s["v_scale"], sinks=s["sinks"], rows=s["rows"])
    return ops.paged_decode_blocks(s["q"], s["k"], s["v"], s["table"], s["lens"], sm_scale=s["sm_scale"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], sinks=s["sinks"], window=s["window"],
                                   rows=s["rows"])


def _plain_store(s):
    """Tokens joined to their blocks: a block's scale is its largest element's over the type's top, kept where it was
    larger (unless the block starts anew); where it grows, the block's earlier tokens are rounded again."""
    R, P = s["prior"].shape[0], s["P"]
    t = torch.arange(s["new_k"].shape[0], device=DEV)
    if s["q_start"] is None:
        req, i = t, 0
    else:
        req = torch.searchsorted(s["q_start"][1:].contiguous(), t.to(torch.int32), right=True)
        i = t - s["q_start"][req]
    pos = s["prior"][req].long() + i
    page, off = s["table"][req, pos // P].long(), pos % P
    _plain_append(s["k"], s["k_scale"], s["new_k"], page, off, s["bt"], s["fmt"])
    _plain_append(s["v"], s["v_scale"], s["new_v"], page, off, s["bt"], s["fmt"])
    if s["bounds"] is not None:
        nb, G, _, d = s["bounds"].shape
        first = torch.full((nb,), P, device=DEV).scatter_reduce_(0, page, off, "amin")
        b = torch.where((first == 0).view(nb, 1, 1, 1), _i32([1, -1]).view(1, 1, 2, 1) * math.inf, s["bounds"].float())
        x = s["new_k"].float()
        at = page.view(-1, 1, 1).expand_as(x)
        b[:, :, 0] = b[:, :, 0].scatter_reduce(0, at, x, "amin")
        b[:, :, 1] = b[:, :, 1].scatter_reduce(0, at, x, "amax")
        s["bounds"].copy_(b)
    return [x for x in (s["k"], s["v"], s["k_scale"], s["v_scale"], s["bounds"]) if x is not None]


def _plain_append(cache, scale, new, page, off, bt, fmt):
    nb, G, P, d = cache.shape
    if fmt == "bf16":
        cache[page, :, off] = new
        return
    x, n = new.float(), P // bt
    blk = page * n + off // bt
    first = torch.full((nb * n,), bt, device=DEV).scatter_reduce_(0, blk, off % bt, "amin").view(nb, 1, n)
    most = torch.zeros(nb * n, G, device=DEV).scatter_reduce_(0, blk.view(-1, 1).expand(-1, G), x.abs().amax(-1), "amax")
    fresh = (most / TOP[fmt]).clamp(min=LEAST_SCALE).view(nb, n, G).transpose(1, 2)
    grown = torch.where(first < bt, torch.where(first == 0, fresh, torch.maximum(fresh, scale)), scale)
    b, h, u = torch.nonzero((first > 0) & (first < bt) & (grown > scale), as_tuple=True)
    blocks = _codes(cache).view(nb, G, n, bt, d)
    old = blocks[b, h, u]
    again = _rounded(_values(old, fmt) * scale[b, h, u].view(-1, 1, 1) / grown[b, h, u].view(-1, 1, 1), fmt)
    before = torch.arange(bt, device=DEV).view(1, bt, 1) < first[b, 0, u].view(-1, 1, 1)
    blocks[b, h, u] = torch.where(before, _codes(again), old)
    scale.copy_(grown)
    _codes(cache)[page, :, off] = _codes(_rounded(x / scale[page, :, off // bt].unsqueeze(-1), fmt))


def _codes(c):
    return c.view(torch.uint8) if c.dtype == FP8 else c


def _values(codes, fmt):
    return codes.view(FP8).float() if fmt == "fp8" else codes.float()


def _rounded(y, fmt):
    return y.clamp(-448, 448).to(FP8) if fmt == "fp8" else y.round().clamp(-127, 127).to(torch.int8)


def _plain_values(cache, scale, pages, h):
    """[..., P, d] fp32 values of the (page, KV head) pairs."""
    x = cache[pages, h].float()
    if scale is not None:
        x = x * scale[pages, h].repeat_interleave(x.shape[-2] // scale.shape[2], -1).unsqueeze(-1)
    return x


def _plain_softmax(scores, seen, sinks):
    """Probabilities of [.., G, grp, keys]; a row that sees nothing has none."""
    top = torch.where(seen, scores, -1.0e30).amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    e = torch.where(seen, torch.exp(scores - top), 0.0)
    den = e.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + torch.exp(sinks - top)
    return e / torch.where(den > 0, den, 1.0)


def _plain_decode(s):
    """[T, H, d]: each query over the keys of its row, or of the pages in its list."""
    H, G, d, P, table = s["H"], s["G"], s["d"], s["P"], s["table"]
    T, W, grp = s["q"].shape[0], table.shape[1], s["H"] // s["G"]
    c = torch.arange(W, device=DEV).view(1, 1, W).expand(T, G, W) if s["op"] == "decode" else s["blocks"].long()
    row = torch.arange(T, device=DEV) if s["rows"] is None else s["rows"].long()
    pages = table[row.view(T, 1, 1), c.clamp(min=0)].long()
    ok = (c >= 0) & (pages >= 0)
    pages, h = pages.clamp(min=0), torch.arange(G, device=DEV).view(1, G, 1).expand_as(pages)
    n = c.shape[2] * P
    keys = _plain_values(s["k"], s["k_scale"], pages, h).reshape(T * G, n, d)
    scores = torch.bmm(s["q"].float().view(T * G, grp, d), keys.transpose(1, 2).contiguous()).view(T, G, grp, n) * s["sm_scale"]
    key = (c.unsqueeze(-1) * P + torch.arange(P, device=DEV)).reshape(T, G, 1, n)
    last = s["lens"].view(T, 1, 1, 1)
    seen = ok.repeat_interleave(P, 2).unsqueeze(2) & (key < last)
    if s["window"] > 0:
        seen &= key >= last - s["window"]
    p = _plain_softmax(scores, seen, None if s["sinks"] is None else s["sinks"].view(1, G, grp, 1))
    del keys, scores
    values = _plain_values(s["v"], s["v_scale"], pages, h).reshape(T * G, n, d)
    return torch.bmm(p.view(T * G, grp, n), values).view(T, H, d).to(torch.bfloat16)


def _plain_chunk(s):
    H, G, d, P, table = s["H"], s["G"], s["d"], s["P"], s["table"]
    R, W, grp, S = table.shape[0], table.shape[1], s["H"] // s["G"], s["max_q"]
    i = torch.arange(S, device=DEV)
    live = i[None, :] < (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    at = (s["q_start"][:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    pages = table.clamp(min=0).long()[:, None, :].expand(R, G, W)
    h = torch.arange(G, device=DEV).view(1, G, 1).expand_as(pages)
    keys = _plain_values(s["k"], s["k_scale"], pages, h).reshape(R * G, W * P, d)
    q = s["q"][at].float().view(R, S, G, grp, d).transpose(1, 2).reshape(R * G, S * grp, d)
    scores = (torch.bmm(q, keys.transpose(1, 2).contiguous()) * s["sm_scale"]).view(R, G, S, grp, W * P)
    j, pos = torch.arange(W * P, device=DEV), s["prior"][:, None].long() + i[None, :]
    seen = (j <= pos[:, :, None]) & live[:, :, None] & (table >= 0).repeat_interleave(P, 1)[:, None, :]
    if s["window"] > 0:
        seen &= j > pos[:, :, None] - s["window"]
    p = _plain_softmax(scores, seen[:, None, :, None, :], None if s["sinks"] is None else s["sinks"].view(1, G, 1, grp, 1))
    del scores
    values = _plain_values(s["v"], s["v_scale"], pages, h).reshape(R * G, W * P, d)
    o = torch.bmm(p.view(R * G, S * grp, W * P), values).view(R, G, S, grp, d).transpose(1, 2).reshape(R, S, H, d)
    return o[live].to(torch.bfloat16)


def _plain_scores(s):
    """[T, G, W]: the most that any key inside a page's bounds can give one of the group's heads, -inf past the row's
    pages; [T] the rows' pages."""
    H, G, d, P, table = s["H"], s["G"], s["d"], s["P"], s["table"]
    T, W, grp = s["q"].shape[0], table.shape[1], s["H"] // s["G"]
    row = torch.arange(T, device=DEV) if s["rows"] is None else s["rows"].long()
    pages = table[row].long()
    b = s["bounds"][pages.clamp(min=0)].float()  # [T, W, G, 2, d]
    b = b.permute(0, 2, 3, 4, 1).reshape(T * G, 2 * d, W)
    q = s["q"].float().view(T * G, grp, d)
    best = torch.bmm(torch.cat([q.clamp(max=0), q.clamp(min=0)], -1), b).view(T, G, grp, W).amax(2)
    count = (s["lens"] + P - 1) // P
    seen = (torch.arange(W, device=DEV)[None, :] < count[:, None]) & (pages >= 0)
    return torch.where(seen[:, None, :], best, -math.inf), count


# ---- what a pass cannot do without ----

def _pairs(n, q, window):
    """(query, key) pairs that a request of n keys and q queries (its last ones) sees."""
    if window <= 0:
        return q * (n - q) + q * (q + 1) // 2
    short = max(0, min(q, window - 1 - (n - q)))  # the queries whose window reaches the first key
    return short * (n - q) + short * (short + 1) // 2 + (q - short) * window


def work(case):
    op, R, H, G, d, P = case["op"], case["R"], case["H"], case["G"], case["d"], case["P"]
    lens = _spread(case["lo"], case["hi"], R)
    pages = sum(-(-n // P) for n in lens)
    if op == "scores":
        T = R * case["q"]
        out = T * (max(-(-n // P) for n in lens) * G * 4 + 4)
        return dict(bytes=pages * G * 2 * d * 2 + T * H * d * 2 + out + pages * 4, flops=pages * case["q"] * H * 4 * d)
    es = 2 if case["fmt"] == "bf16" else 1
    token = G * 2 * (d * es + (0 if es == 2 else 4 / case["bt"]))  # a cached token's bytes, its share of the scales among them
    if op == "store":
        qs = [min(q, n) for q, n in zip(_spread(case["q_lo"], case["q_hi"], R), lens)]
        T = sum(qs)
        touched = sum(-(-n // P) - (n - q) // P for n, q in zip(lens, qs))
        return dict(bytes=T * (G * d * 4 + token) + touched * (4 + (G * d * 4 if case["bounds"] else 0)), flops=T * G * d * 4)
    if op == "chunk":
        qs = [min(q, n) for q, n in zip(_spread(case["q_lo"], case["q_hi"], R), lens)]
        win = case["window"]
        keys = sum(n if win <= 0 else min(n, win + q - 1) for n, q in zip(lens, qs))
        pairs = sum(_pairs(n, q, win) for n, q in zip(lens, qs)) * H
        return dict(bytes=keys * token + sum(qs) * H * d * 4 + pages * 4, flops=pairs * 4 * d)
    q = case["q"]
    if op == "decode":
        win = case["window"]
        keys = sum(n if win <= 0 else min(n, win + q - 1) for n in lens)
        pairs = sum(_pairs(n, q, win) for n in lens) * H
        return dict(bytes=keys * token + R * q * H * d * 4 + pages * 4, flops=pairs * 4 * d)
    # each query's pages are its own; those of one row's queries are counted once, up to the whole row
    n = case["n"]
    keys = sum(min(L, q * n * P) for L in lens)
    pairs = sum(min(L, n * P) for L in lens) * q * H
    lists = R * q * G * min(n, max(-(-L // P) for L in lens)) * 4
    return dict(bytes=keys * token + R * q * H * d * 4 + lists, flops=pairs * 4 * d)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "decode": _exact_rows, "chunk": _exact_chunk, "scores": _exact_scores,
            "selected": _exact_rows}[s["op"]](s)


def _exact_store(s):
    """Request by request: scales as they are defined, e4m3fn elements before their last rounding, int8 codes not at all."""
    P, bt, fmt = s["P"], s["bt"], s["fmt"]
    R = s["prior"].shape[0]
    start = list(range(R + 1)) if s["q_start"] is None else s["q_start"].tolist()
    prior, table = s["prior"].tolist(), s["table"].tolist()
    caches, scales = [], []
    for new, cache, scale in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        x = new.double()
        c = cache.double()
        z = None if scale is None else scale.double()
        for r in range(R):
            at, end = prior[r], prior[r] + start[r + 1] - start[r]
            while at < end:  # one block of tokens at a time
                stop = min(end, (at // bt + 1) * bt)
                page, lo = table[r][at // P], at % P
                part = x[start[r] + at - prior[r]:start[r] + stop - prior[r]].transpose(0, 1)  # [G, n, d]
                if fmt != "bf16":
                    u, head = lo // bt, lo - lo % bt
                    top = (part.abs().amax((1, 2)) / TOP[fmt]).clamp(min=LEAST_SCALE)
                    if lo > head:
                        top = torch.maximum(top, z[page, :, u])
                        c[page, :, head:lo] *= (z[page, :, u] / top).view(-1, 1, 1)
                    z[page, :, u] = top
                    part = part / top.view(-1, 1, 1)
                c[page, :, lo:lo + part.shape[1]] = part
                at = stop
        caches.append(None if fmt == "int8" else c)
        scales.append(z)
    out = [caches[0], caches[1]]
    if fmt != "bf16":
        out += scales
    if s["bounds"] is not None:
        b = s["bounds"].double()
        for r in range(R):
            at, end = prior[r], prior[r] + start[r + 1] - start[r]
            while at < end:
                stop = min(end, (at // P + 1) * P)
                page = table[r][at // P]
                part = s["new_k"][start[r] + at - prior[r]:start[r] + stop - prior[r]].double()
                lo, hi = part.amin(0), part.amax(0)
                if at % P:
                    lo, hi = torch.minimum(lo, b[page, :, 0]), torch.maximum(hi, b[page, :, 1])
                b[page, :, 0], b[page, :, 1] = lo, hi
                at = stop
        out.append(b)
    return out


def _exact_tokens(s, name, pages, g):
    x = s[name][pages, g].double()
    scale = s[name + "_scale"]
    if scale is not None:
        z = scale[pages, g].double()
        x = (x.view(z.shape[0], z.shape[1], -1) * z.unsqueeze(-1)).view_as(x)
    return x.reshape(-1, s["d"])


def _exact_mix(z, values, sinks):
    """Softmax of z [.., grp, n] (-inf hidden) over the keys and, where given, the heads' sinks, times values."""
    total = torch.logsumexp(z, -1, keepdim=True)
    if sinks is not None:
        total = torch.logaddexp(total, sinks.double().view(-1, 1).expand_as(total))
    return torch.exp(z - total) @ values


def _exact_rows(s):
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    T, grp = s["q"].shape[0], H // G
    out = torch.zeros(T, H, d, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    rows = list(range(T)) if s["rows"] is None else s["rows"].tolist()
    lists = s["blocks"].cpu() if s["op"] == "selected" else None
    for t, n in enumerate(lens):
        for g in range(G):
            if lists is None:
                cols = torch.arange(-(-n // P), device=DEV)
            else:
                cols = lists[t, g][lists[t, g] >= 0].long().to(DEV)
            pages = s["table"][rows[t]][cols].long()
            key = (cols[:, None] * P + torch.arange(P, device=DEV)).reshape(-1)
            hide = key >= n
            if s["window"] > 0:
                hide |= key < n - s["window"]
            k, v = _exact_tokens(s, "k", pages, g), _exact_tokens(s, "v", pages, g)
            z = (s["q"][t, g * grp:(g + 1) * grp].double() @ k.t()) * s["sm_scale"]
            out[t, g * grp:(g + 1) * grp] = _exact_mix(z.masked_fill(hide, -math.inf), v,
                                                       None if s["sinks"] is None else s["sinks"][g * grp:(g + 1) * grp])
    return out


def _exact_chunk(s):
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    grp = H // G
    out = torch.zeros(s["q"].shape[0], H, d, dtype=torch.float64, device=DEV)
    start, prior = s["q_start"].tolist(), s["prior"].tolist()
    for r in range(len(prior)):
        count = start[r + 1] - start[r]
        n = prior[r] + count
        pages = s["table"][r, :-(-n // P)].long()
        key = torch.arange(n, device=DEV)
        for g in range(G):
            k, v = _exact_tokens(s, "k", pages, g)[:n], _exact_tokens(s, "v", pages, g)[:n]
            step = max(1, (1 << 27) // (n * grp))
            for t0 in range(0, count, step):
                q = s["q"][start[r] + t0:min(start[r] + t0 + step, start[r + 1]), g * grp:(g + 1) * grp].double()
                at = prior[r] + t0 + torch.arange(q.shape[0], device=DEV)
                hide = key[None, :] > at[:, None]
                if s["window"] > 0:
                    hide |= key[None, :] <= at[:, None] - s["window"]
                z = (q.reshape(-1, d) @ k.t()).view(-1, grp, n) * s["sm_scale"]
                o = _exact_mix(z.masked_fill(hide[:, None, :], -math.inf), v,
                               None if s["sinks"] is None else s["sinks"][g * grp:(g + 1) * grp])
                out[start[r] + t0:start[r] + t0 + q.shape[0], g * grp:(g + 1) * grp] = o
    return out


def _exact_scores(s):
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    T, W, grp = s["q"].shape[0], s["table"].shape[1], H // G
    out = torch.full((T, G, W), -math.inf, dtype=torch.float64, device=DEV)
    rows = list(range(T)) if s["rows"] is None else s["rows"].tolist()
    for t, n in enumerate(s["lens"].tolist()):
        count = -(-n // P)
        b = s["bounds"][s["table"][rows[t], :count].long()].double()  # [count, G, 2, d]
        for g in range(G):
            q = s["q"][t, g * grp:(g + 1) * grp].double()
            step = max(1, (1 << 26) // (grp * d))
            for c0 in range(0, count, step):
                part = b[c0:c0 + step, g].unsqueeze(1)  # [c, 1, 2, d]
                most = torch.maximum(part[:, :, 0] * q, part[:, :, 1] * q).sum(-1)  # [c, grp]
                out[t, g, c0:c0 + step] = most.amax(1)
    return out, torch.tensor([-(-n // P) for n in s["lens"].tolist()], dtype=torch.int32)
