"""Performance cases of the operators around a long prompt's cache: the attention weight that cached keys receive (for a
prompt's queries and for a decode step), the eviction of the keys that receive least, and the QKV writer for positions
with several axes. Each case runs the package's entry points, or the same operators in plain torch operations.

A case is a dict of plain values; ``op`` names the operator. A batch's lengths are spread over ``lo`` .. ``hi`` (so the
work does not depend on the seed) and dealt to its rows at random; pages lie at random places of the pool.
"""

from __future__ import annotations

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DEV = "cuda"

# head shapes: (query heads, KV heads, head dim)
QWEN3_8B = dict(H=32, G=8, d=128)
QWEN3_06B = dict(H=16, G=8, d=128)
GPT_OSS_SHARE = dict(H=8, G=1, d=64)  # one of eight ranks' heads


def listed():
    return [
        # one decode step of a small model's batch: the shortest call, where launches and latency are everything
        dict(name="step-b8-bf16", op="step", R=8, lo=128, hi=1024, **QWEN3_06B, P=16, fp8=False, window=0, sinks=False),
        # a full serving batch at 4k context over an FP8 pool, its keys weighed at every step
        dict(name="step-b64-fp8", op="step", R=64, lo=4096, hi=4096, **QWEN3_8B, P=16, fp8=True, window=0, sinks=False),
        # a ragged batch of wide groups with sinks: one rank's share of the heads
        dict(name="step-b128-sinks", op="step", R=128, lo=2048, hi=8192, **GPT_OSS_SHARE, P=16, fp8=True, window=0,
             sinks=True),
        # the last 32 tokens of four prompts weigh the whole of them, after the prompts' last chunk
        dict(name="observe-4x32-fp8", op="prompt", R=4, q_lo=32, q_hi=32, lo=3001, hi=16384, **QWEN3_8B, P=16, fp8=True,
             window=0, sinks=False),
        # one very long prompt, weighed by its last 64 tokens before most of it is dropped
        dict(name="observe-131071", op="prompt", R=1, q_lo=64, q_hi=64, lo=131071, hi=131071, **QWEN3_8B, P=64,
             fp8=False, window=0, sinks=False),
        # every query of a prefill batch in chunks counts: four requests, each 2048 tokens after 2048
        dict(name="accumulate-4x2048", op="prompt", R=4, q_lo=2048, q_hi=2048, lo=4096, hi=4096, **QWEN3_8B, P=16,
             fp8=True, window=0, sinks=False),
        # one short conversation thinned to 256 tokens
        dict(name="evict-b1-short", op="evict", R=1, lo=1000, hi=1000, keep=256, first=4, recent=32, **QWEN3_06B, P=16,
             fp8=False),
        # a batch of prompts thinned to 1024 tokens after their prefill; one row is short and stays whole
        dict(name="evict-b32", op="evict", R=32, lo=900, hi=8192, keep=1024, first=4, recent=64, **QWEN3_8B, P=16,
             fp8=True),
        # long documents thinned sixteenfold
        dict(name="evict-4x131072", op="evict", R=4, lo=50001, hi=131072, keep=8192, first=16, recent=512, **QWEN3_8B,
             P=64, fp8=False),
        # the writer of one decode step
        dict(name="mrope-step-8", op="mrope", T=8, **QWEN3_06B, P=16, fp8=False, norm=True, rot=128,
             sections="24,20,20", interleaved=True),
        # the writer of a prefill chunk that holds images, FP8 pool
        dict(name="mrope-chunk-8192", op="mrope", T=8192, **QWEN3_8B, P=16, fp8=True, norm=True, rot=128,
             sections="16,24,24", interleaved=False),
        # an odd chunk at head dim 64, half of it rotated, two axes, no norm
        dict(name="mrope-chunk-1531", op="mrope", T=1531, H=24, G=4, d=64, P=32, fp8=False, norm=False, rot=32,
             sections="8,8", interleaved=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "step", "prompt", "prompt", "evict", "evict", "mrope"])
    heads = dict(rng.choice([QWEN3_8B, QWEN3_06B, GPT_OSS_SHARE, dict(H=12, G=4, d=128), dict(H=20, G=4, d=64)]))
    P = rng.choice([16, 32, 64, 128])
    fp8 = rng.random() < 0.5
    if op == "mrope":
        rot = rng.choice([heads["d"], heads["d"], heads["d"] // 2])
        a = rng.choice([2, 3, 3, 4])
        cut = sorted(rng.sample(range(1, rot // 2), a - 1))
        parts = [y - x for x, y in zip([0] + cut, cut + [rot // 2])]
        return dict(op=op, T=_log_int(rng, 1, 8192), **heads, P=P, fp8=fp8, norm=rng.random() < 0.6, rot=rot,
                    sections=",".join(str(p) for p in parts), interleaved=False)
    if op == "evict":
        c = dict(op=op, R=_log_int(rng, 1, 48), hi=_log_int(rng, 200, 131072), **heads, P=P, fp8=fp8)
        while c["R"] * c["hi"] * c["G"] > 4 * 90000 * 8:
            c["hi"] = c["hi"] * 2 // 3
        c["lo"] = max(1, int(c["hi"] * rng.uniform(0.2, 1.0)))
        c["keep"] = max(16, int(c["hi"] * rng.uniform(0.06, 0.5)))
        while c["R"] * c["keep"] * c["G"] * c["d"] * (1 if fp8 else 2) > 4 * 8192 * 8 * 256:
            c["keep"] = c["keep"] * 2 // 3
        c["first"] = rng.choice([0, 4, min(16, c["keep"] // 4)])
        c["recent"] = min(c["keep"] // 2, _log_int(rng, 1, 512))
        return c
    window = rng.choice([0, 0, 0, 128, 1000])
    c = dict(op=op, R=_log_int(rng, 1, 128 if op == "step" else 8), **heads, P=P, fp8=fp8, window=window,
             sinks=rng.random() < 0.4)
    hi = _log_int(rng, 64, 131072)
    if op == "step":
        while c["R"] * hi * c["G"] * c["d"] * (1 if fp8 else 2) > 260e6:
            hi = hi * 2 // 3
        c.update(hi=max(hi, 1), lo=max(1, int(hi * rng.uniform(0.1, 1.0))))
        return c
    q = _log_int(rng, 1, 4096)
    while c["R"] * min(q, hi) * hi * c["H"] > 1.0e9 or c["R"] * min(q, hi) > 8192:
        hi, q, c["R"] = max(64, hi * 3 // 4), max(1, q * 3 // 4), max(1, c["R"] - 1)
    q = min(q, hi)
    c.update(hi=hi, lo=max(q, int(hi * rng.uniform(0.3, 1.0))), q_hi=q, q_lo=max(1, int(q * rng.uniform(0.2, 1.0))))
    return c


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _spread(lo, hi, n):
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sections(case):
    return [int(x) for x in case["sections"].split(",")]


def _axes(case):
    """The axis of each rotated pair: the sections one after another, or dealt in turn (pair i to axis i mod A while
    that axis has pairs left among the first A * its section, else to axis 0)."""
    sec = _sections(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    A = len(sec)
    return [i % A if i % A > 0 and i < A * sec[i % A] else 0 for i in range(sum(sec))]


def _pool(g, blocks, G, P, d, fp8):
    x = torch.randn(blocks, G, P, d, generator=g, device=DEV, dtype=torch.float32)
    if not fp8:
        return x.to(torch.bfloat16), None
    s = x.abs().amax((0, 2, 3)) / 448
    return (x / s.view(1, G, 1, 1)).clamp_(-448, 448).to(FP8), s


def _table(g, lens, P, first_page, width=0):
    """[R, width] int32 pages at random places from ``first_page`` on, -1 past a row's."""
    R = len(lens)
    need = torch.tensor([-(-n // P) for n in lens], device=DEV)
    W = max(width, 1, max(-(-n // P) for n in lens))
    live = torch.arange(W, device=DEV)[None, :] < need[:, None]
    count = sum(-(-n // P) for n in lens)
    table = torch.full((R, W), -1, dtype=torch.int32, device=DEV)
    table[live] = (torch.randperm(count, generator=g, device=DEV) + first_page).to(torch.int32)
    return table, count


def prepare(case, seed):
    g = _gen(seed)
    H, G, d, P, fp8 = case["H"], case["G"], case["d"], case["P"], case["fp8"]
    if case["op"] == "mrope":
        return _prepare_mrope(case, g)
    R = case["R"]
    deal = torch.randperm(R, generator=g, device=DEV).tolist()
    lens = [_spread(case["lo"], case["hi"], R)[i] for i in deal]
    table, count = _table(g, lens, P, 1)
    s = dict(op=case["op"], fp8=fp8, H=H, G=G, d=d, P=P, table=table,
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if case["op"] == "evict":
        keep = case["keep"]
        dst, more = _table(g, [min(n, keep) for n in lens], P, 1 + count, -(-keep // P))
        s["k"], _ = _pool(g, 1 + count + more, G, P, d, fp8)
        s["v"], _ = _pool(g, 1 + count + more, G, P, d, fp8)
        N = max(lens)
        w = torch.exp(2.5 * torch.randn(R, G, N, generator=g, device=DEV) - 4)  # heavy tails, as summed softmax rows have
        w[torch.rand(R, G, N, generator=g, device=DEV) < 0.02] = 0  # keys that underflowed: ties
        s.update(dst=dst, weights=w, weights_out=torch.empty(R, G, keep, dtype=torch.float32, device=DEV), keep=keep,
                 first=case["first"], recent=case["recent"])
        return s
    s["k"], s["k_scale"] = _pool(g, 1 + count, G, P, d, fp8)
    s.update(window=case["window"], sm_scale=1.0 / math.sqrt(d),
             sinks=torch.randn(H, generator=g, device=DEV) if case["sinks"] else None)
    if case["op"] == "step":
        s["q"] = torch.randn(R, H, d, generator=g, device=DEV).to(torch.bfloat16)
        s["lens_host"] = lens
        return s
    qs = [_spread(case["q_lo"], case["q_hi"], R)[i] for i in deal]
    start = [0]
    for n in qs:
        start.append(start[-1] + n)
    s["q"] = torch.randn(start[-1], H, d, generator=g, device=DEV).to(torch.bfloat16)
    s.update(q_start=torch.tensor(start, dtype=torch.int32, device=DEV), max_q=max(qs),
             prior=torch.tensor([n - q for n, q in zip(lens, qs)], dtype=torch.int32, device=DEV))
    return s


def _prepare_mrope(case, g):
    H, G, d, P, fp8, T = case["H"], case["G"], case["d"], case["P"], case["fp8"], case["T"]
    A, half = len(_sections(case)), case["rot"] // 2
    blocks = -(-T // P) + 3
    k, ks = _pool(g, blocks, G, P, d, fp8)
    v, vs = _pool(g, blocks, G, P, d, fp8)
    # text, an image's grid, text again: the axes are equal outside the image and differ inside
    at = torch.arange(T, device=DEV)
    base = int(torch.randint(0, 200000, (1,), generator=g, device=DEV))
    lo, hi = T // 4, T // 4 + T // 2
    inside = (at >= lo) & (at < hi)
    pos = [torch.where(inside, lo + (at - lo) // 1000, at)]
    for a in range(1, A):
        pos.append(torch.where(inside, lo + ((at - lo) // 37 if a == 1 else (at - lo)) % 37, at))
    inv = 1.0e6 ** (-torch.arange(half, device=DEV, dtype=torch.float32) / half)
    slots = torch.randperm((blocks - 1) * P, generator=g, device=DEV)[:T] + P
    gamma = [(1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2)]
    return dict(op="mrope", fp8=fp8, H=H, G=G, d=d, P=P, k=k, v=v, k_scale=ks, v_scale=vs, axes=_axes(case),
                axis=torch.tensor(_axes(case), device=DEV), positions=(torch.stack(pos) + base).contiguous(), inv_freq=inv,
                slots=slots, qkv=torch.randn(T, (H + 2 * G) * d, generator=g, device=DEV).to(torch.bfloat16),
                q_norm=gamma[0] if case["norm"] else None, k_norm=gamma[1] if case["norm"] else None,
                q_out=torch.empty(T, H, d, dtype=torch.bfloat16, device=DEV))


# ---- one pass ----

def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "evict":
        return _plain_evict(s)
    if s["op"] == "mrope":
        return _plain_mrope(s)
    return _plain_weights(s)


def _run_own(s):
    from sglang_neuron_amd import ops

    if s["op"] == "step":
        return ops.decode_attention_weights(s["q"], s["k"], s["table"], s["lens"], sm_scale=s["sm_scale"],
                                            k_scale=s["k_scale"], sinks=s["sinks"], window=s["window"])
    if s["op"] == "prompt":
        return ops.prefill_attention_weights(s["q"], s["k"], s["table"], s["q_start"], s["prior"], max_q_len=s["max_q"],
                                             sm_scale=s["sm_scale"], k_scale=s["k_scale"], sinks=s["sinks"],
                                             window=s["window"])
    if s["op"] == "evict":
        kept, lens = ops.evict_tokens(s["k"], s["v"], s["table"], s["lens"], s["weights"], keep=s["keep"],
                                      first=s["first"], recent=s["recent"], dst_table=s["dst"],
                                      weights_out=s["weights_out"])
        return kept, lens, s["weights_out"], s["k"], s["v"]
    q = ops.qkv_norm_mrope_store(s["qkv"], positions=s["positions"], inv_freq=s["inv_freq"], axes=s["axes"],
                                 num_q_heads=s["H"], num_kv_heads=s["G"], d_head=s["d"], k_cache=s["k"], v_cache=s["v"],
                                 slot_mapping=s["slots"], q_norm=s["q_norm"], k_norm=s["k_norm"], norm_eps=1e-6,
                                 k_scale=s["k_scale"], v_scale=s["v_scale"], q_out=s["q_out"])
    return q, s["k"], s["v"]


def _plain_weights(s):
    """[R, G, W * P] fp32: the queries' softmax probabilities summed over queries and the heads of a group."""
    H, G, d, P, table, window = s["H"], s["G"], s["d"], s["P"], s["table"], s["window"]
    R, W = table.shape
    if s["op"] == "step":
        Q, pos, live = s["q"][:, None], (s["lens"] - 1)[:, None].long(), torch.ones(R, 1, dtype=torch.bool, device=DEV)
    else:
        i = torch.arange(s["max_q"], device=DEV)
        live = i[None, :] < (s["q_start"][1:] - s["q_start"][:-1])[:, None]
        Q = s["q"][(s["q_start"][:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)]
        pos = s["prior"][:, None].long() + i[None, :]
    S, grp = Q.shape[1], H // G
    keys = s["k"][table.clamp(min=0).long()].float()  # [R, W, G, P, d]
    if s["fp8"]:
        keys = keys * s["k_scale"].view(1, 1, G, 1, 1)
    keys = keys.permute(0, 2, 1, 3, 4).reshape(R * G, W * P, d)
    Q = Q.float().view(R, S, G, grp, d).permute(0, 2, 1, 3, 4).reshape(R * G, S * grp, d)
    scores = torch.bmm(Q, keys.transpose(1, 2).contiguous()) * s["sm_scale"]
    scores = scores.view(R, G, S, grp, W * P)
    j = torch.arange(W * P, device=DEV)
    seen = (j[None, None, :] <= pos[:, :, None]) & live[:, :, None] & (table >= 0).repeat_interleave(P, 1)[:, None, :]
    if window > 0:
        seen &= j[None, None, :] > pos[:, :, None] - window
    seen = seen[:, None, :, None, :]
    top = torch.where(seen, scores, -1.0e30).amax(-1, keepdim=True)
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].view(1, G, 1, grp, 1))
    e = torch.where(seen, torch.exp(scores - top), 0.0)
    den = e.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        den = den + torch.exp(s["sinks"].view(1, G, 1, grp, 1) - top)
    return (e / torch.where(den > 0, den, 1.0)).sum((2, 3))


def _plain_evict(s):
    R, G, N = s["weights"].shape
    keep, P, L = s["keep"], s["P"], s["lens"].long().view(R, 1, 1)
    j = torch.arange(N, device=DEV).view(1, 1, N)
    inside = j < L
    forced = inside & ((j < s["first"]) | (j >= L - s["recent"]) | (L <= keep))
    rank = torch.where(forced, math.inf, torch.where(inside, s["weights"], -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    if N < keep:
        order = torch.cat([order, torch.full((R, G, keep - N), N, device=DEV)], -1)
    order = torch.where(order < L, order, 1 << 40).sort(-1).values
    live = order < (1 << 40)
    src = torch.where(live, order, 0)
    kept = torch.where(live, order, -1).to(torch.int32)
    s["weights_out"].copy_(torch.where(live, torch.gather(s["weights"], 2, src), 0.0))
    i = torch.arange(keep, device=DEV).view(1, 1, keep).expand(R, G, keep)
    r = torch.arange(R, device=DEV).view(R, 1, 1).expand(R, G, keep)[live]
    h = torch.arange(G, device=DEV).view(1, G, 1).expand(R, G, keep)[live]
    src, i = src[live], i[live]
    at = s["table"][r, src // P].long()
    to = s["dst"][r, i // P].long()
    for c in (s["k"], s["v"]):
        c.view(torch.int8)[to, h, i % P] = c.view(torch.int8)[at, h, src % P]
    return kept, torch.clamp(s["lens"], max=keep), s["weights_out"], s["k"], s["v"]


def _plain_mrope(s):
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    T, half = s["qkv"].shape[0], s["inv_freq"].numel()
    x = s["qkv"].float().view(T, H + 2 * G, d)
    angle = s["positions"][s["axis"]].t().double() * s["inv_freq"].double()  # far positions: 64 bits
    c, n = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    qk = x[:, :H + G]
    if s["q_norm"] is not None:
        gamma = torch.cat([s["q_norm"].float().expand(H, d), s["k_norm"].float().expand(G, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * gamma
    a, b = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat([a * c - b * n, b * c + a * n, qk[..., 2 * half:]], -1)
    s["q_out"].copy_(qk[:, :H])
    k, v = qk[:, H:], x[:, H + G:]
    page, off = s["slots"] // P, s["slots"] % P
    if s["fp8"]:
        k = (k / s["k_scale"].view(1, G, 1)).clamp(-448, 448).to(FP8).view(torch.uint8)
        v = (v / s["v_scale"].view(1, G, 1)).clamp(-448, 448).to(FP8).view(torch.uint8)
        s["k"].view(torch.uint8)[page, :, off] = k
        s["v"].view(torch.uint8)[page, :, off] = v
    else:
        s["k"][page, :, off] = k.to(torch.bfloat16)
        s["v"][page, :, off] = v.to(torch.bfloat16)
    return s["q_out"], s["k"], s["v"]


# ---- what a pass cannot do without ----

def _pairs(n, q, window):
    """(query, key) pairs that a request of n keys and q queries (its last ones) sees."""
    if window <= 0:
        return q * (n - q) + q * (q + 1) // 2
    short = max(0, min(q, window - 1 - (n - q)))  # the queries whose window reaches the first key
    return sum((short * (n - q) + short * (short + 1) // 2, (q - short) * window))


def work(case):
    H, G, d, P, es = case["H"], case["G"], case["d"], case["P"], 1 if case["fp8"] else 2
    if case["op"] == "mrope":
        T, half = case["T"], case["rot"] // 2
        io = T * (H + 2 * G) * d * 2 + T * H * d * 2 + T * 2 * G * d * es
        return dict(bytes=io + T * 8 * (len(_sections(case)) + 1), flops=T * (H + G) * (6 * half + (4 * d if case["norm"] else 0)))
    lens = _spread(case["lo"], case["hi"], case["R"])
    pages = sum(-(-n // P) for n in lens)
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return dict(bytes=sum(lens) * G * 4 + kept * G * (4 * d * es + 4) + case["R"] * G * case["keep"] * 4 + pages * 4,
                    flops=sum(lens) * G)
    qs = [1] * case["R"] if case["op"] == "step" else _spread(case["q_lo"], case["q_hi"], case["R"])
    win = case["window"]
    keys = sum(n if win <= 0 else min(n, win + q - 1) for n, q in zip(lens, qs))
    W = max(-(-n // P) for n in lens)
    pairs = sum(_pairs(n, q, win) for n, q in zip(lens, qs)) * H
    return dict(bytes=keys * G * d * es + sum(qs) * H * d * 2 + case["R"] * G * W * P * 4 + pages * 4,
                flops=pairs * (2 * d + 3))


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "evict":
        return _exact_evict(s)
    if s["op"] == "mrope":
        return _exact_mrope(s)
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    table, grp = s["table"], s["H"] // s["G"]
    out = torch.zeros(table.shape[0], G, table.shape[1] * P, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for r, n in enumerate(lens):
        if s["op"] == "step":
            rows = s["q"][r:r + 1]
        else:
            rows = s["q"][int(s["q_start"][r]):int(s["q_start"][r + 1])]
        count = rows.shape[0]
        pages = table[r, :-(-n // P)].long()
        for g in range(G):
            k = s["k"][pages, g].reshape(-1, d)[:n].double()
            if s["fp8"]:
                k = k * s["k_scale"][g].double()
            step = max(1, (1 << 27) // (n * grp))
            for t0 in range(0, count, step):
                q = rows[t0:t0 + step, g * grp:(g + 1) * grp].double()
                at = n - count + t0 + torch.arange(q.shape[0], device=DEV)
                z = (q.reshape(-1, d) @ k.t()).view(-1, grp, n) * s["sm_scale"]
                key = torch.arange(n, device=DEV)
                hide = key[None, :] > at[:, None]
                if s["window"] > 0:
                    hide |= key[None, :] <= at[:, None] - s["window"]
                z = z.masked_fill(hide[:, None, :], -math.inf)
                total = torch.logsumexp(z, -1, keepdim=True)
                if s["sinks"] is not None:
                    total = torch.logaddexp(total, s["sinks"][g * grp:(g + 1) * grp].double().view(1, grp, 1).expand_as(total))
                out[r, g, :n] += torch.exp(z - total).sum((0, 1))
    return out


def _exact_evict(s):
    """Kept positions, lengths and weights by sorting each row alone; the moved rows are copies, checked as such."""
    R, G, _ = s["weights"].shape
    kept = torch.full((R, G, s["keep"]), -1, dtype=torch.int32)
    out = torch.zeros(R, G, s["keep"], dtype=torch.float64)
    lens = s["lens"].tolist()
    w = s["weights"].cpu()
    for r, n in enumerate(lens):
        for g in range(G):
            if n <= s["keep"]:
                at = torch.arange(n)
            else:
                mid = torch.arange(s["first"], n - s["recent"])
                by = torch.sort(w[r, g, mid].double(), descending=True, stable=True).indices
                best = mid[by[:s["keep"] - s["first"] - s["recent"]]]
                at = torch.cat([torch.arange(s["first"]), best.sort().values, torch.arange(n - s["recent"], n)])
            kept[r, g, :at.numel()] = at.to(torch.int32)
            out[r, g, :at.numel()] = w[r, g, at].double()
    return kept, torch.tensor([min(n, s["keep"]) for n in lens], dtype=torch.int32), out, None, None


def _exact_mrope(s):
    H, G, d, P = s["H"], s["G"], s["d"], s["P"]
    T, half = s["qkv"].shape[0], s["inv_freq"].numel()
    x = s["qkv"].double().view(T, H + 2 * G, d)
    if s["q_norm"] is not None:
        size = (x.square().sum(-1, keepdim=True) / d + 1e-6).sqrt()
        x = torch.cat([x[:, :H] / size[:, :H] * s["q_norm"].double(), x[:, H:H + G] / size[:, H:H + G] * s["k_norm"].double(),
                       x[:, H + G:]], 1)
    y = x.clone()
    for i in range(half):
        turn = s["positions"][s["axes"][i]].double() * s["inv_freq"][i].double()
        c, n = turn.cos()[:, None], turn.sin()[:, None]
        y[:, :H + G, i] = x[:, :H + G, i] * c - x[:, :H + G, i + half] * n
        y[:, :H + G, i + half] = x[:, :H + G, i + half] * c + x[:, :H + G, i] * n
    caches = []
    for c, part, scale in ((s["k"], y[:, H:H + G], s["k_scale"]), (s["v"], y[:, H + G:], s["v_scale"])):
        c = c.double()
        c[s["slots"] // P, :, s["slots"] % P] = part if scale is None else (part / scale.double().view(1, G, 1)).clamp(-448, 448)
        caches.append(c)
    return y[:, :H], caches[0], caches[1]
