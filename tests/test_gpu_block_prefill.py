"""ops.prefill_attention_blocks against its definition in 64 bits, on pools that hold garbage wherever nothing was stored. The
bounds are oracle.blocks.attend's; over int8 codes a query element is off by up to 2^-16 of its row's largest."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import blocks as ob
from sglang_neuron_amd import _lib, ops
from tests._block_cases import FMTS, gen, hide_unstored, pool, table_of, to, tokens
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _case(seed, priors, counts, H, G, d, P, bt, fmt, extra=0, hide=True):
    g = gen(seed)
    lens = [p + n for p, n in zip(priors, counts)]
    table, nb = table_of(g, lens, P, extra)
    kc, ks = pool(g, nb + 1, G, P, d, bt, fmt)
    vc, vs = pool(g, nb + 1, G, P, d, bt, fmt)
    if hide:
        for c, s in ((kc, ks), (vc, vs)):
            hide_unstored(c, s, table, lens, P)
    start = [sum(counts[:r]) for r in range(len(counts) + 1)]
    return torch.randn(start[-1], H, d, generator=g).to(torch.bfloat16), kc, vc, ks, vs, table, start


def _run(q, kc, vc, ks, vs, table, start, priors, max_q=None, **kw):
    q, kc, vc, ks, vs, table = to(DEV, q, kc, vc, ks, vs, table)
    kw = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    most = max(b - a for a, b in zip(start, start[1:]))
    return ops.prefill_attention_blocks(q, kc, vc, table, _i32(start).to(DEV), _i32(priors).to(DEV), max_q_len=max_q or most,
                                        k_scale=ks, v_scale=vs, host_q_start=start, **kw)


def _check(args, priors, fmt, rows=None, **kw):
    q, kc, vc, ks, vs, table, start = args
    got = _run(*args, priors, **kw).cpu().double()
    assert bool(torch.isfinite(got).all())
    okw = dict(sm_scale=kw["sm_scale"], k_scale=ks, v_scale=vs, sinks=kw.get("sinks"), window=kw.get("window", 0),
               q_off=2.0 ** -16 if fmt == "int8" else 0.0)
    at = [(r, i) for r in range(len(priors)) for i in range(start[r + 1] - start[r])]
    pick = range(len(at)) if rows is None else rows
    want, off = ob.decode(q[list(pick)], kc, vc, table, [priors[at[t][0]] + at[t][1] + 1 for t in pick],
                          rows=[at[t][0] for t in pick], **okw)
    over = (got[list(pick)] - want).abs() - off
    assert float(over.max()) <= 1e-30, f"{float((got[list(pick)] - want).abs().max()):.3e} off, {float(over.max()):.3e} over"
    return got


SHAPES = [(4, 2, 128, 16, 16), (3, 3, 64, 32, 16), (16, 1, 64, 48, 48), (10, 2, 128, 64, 32), (5, 1, 128, 128, 128)]


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("H,G,d,P,bt", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, False), (37, True), (1, False)])
def test_ragged_chunks(fmt, H, G, d, P, bt, window, sinks):
    """Chunks of 0 to 150 tokens after 0 to 200, at the tiles', groups' and pages' edges."""
    announce(f"chunks {fmt} H={H} G={G} d={d} P={P} bt={bt} window={window} sinks={sinks}")
    priors, counts = [0, 0, 7, 64, 200, 33, 15], [1, 64, 150, 0, 3, 65, 17]
    args = _case(H + P, priors, counts, H, G, d, P, bt, fmt, extra=2)
    _check(args, priors, fmt, sm_scale=d ** -0.5, window=window, sinks=torch.randn(H, generator=gen(1)) if sinks else None)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("n", [1, 16, 17, 31, 32, 33, 47, 48, 64])
def test_one_tile(fmt, n):
    """Prompts whose tables name at most one tile, or half of one."""
    announce(f"one tile {fmt} {n}")
    for P in (16, 32, 64):
        args = _case(n + P, [0, 0], [n, max(1, n - 5)], 8, 2, 128, P, 16, fmt)
        _check(args, [0, 0], fmt, sm_scale=0.1)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("d,bt", [(128, 16), (64, 64)])
def test_splits(fmt, d, bt):
    """Few queries after long priors: the keys are split and merged; a tail that is one key."""
    announce(f"splits {fmt} d={d}")
    priors, counts = [4095, 2700, 10], [5, 33, 2]
    args = _case(d, priors, counts, 8, 1, d, 64, bt, fmt)
    assert _lib.load().sna_prefill_workspace_bytes(3, 33, 8, 1, d, 64, args[5].shape[1], 0) > 0
    _check(args, priors, fmt, sm_scale=d ** -0.5)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_one_long_chunk_among_many_tokens(fmt):
    """The query blocks there are, counted out among 150 requests (some without tokens) instead of given to each."""
    announce(f"mixed {fmt}")
    R = 150
    priors = [(7 * r) % 50 for r in range(R)]
    counts = [0 if r % 13 == 5 else 1 for r in range(R)]
    counts[70], counts[149] = 700, 33
    args = _case(17, priors, counts, 8, 8, 64, 16, 16, fmt)
    at = sum(counts[:70])
    _check(args, priors, fmt, rows=[0, 1, 40, at, at + 127, at + 128, at + 400, at + 699, at + 700, sum(counts) - 40,
                                    sum(counts) - 1], sm_scale=0.125)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_restaged_scales(fmt):
    """More tiles than scales are staged at a time (256), whole and with a window that starts behind them."""
    announce(f"restaged {fmt}")
    n, H, G, d = 64 * 256 * 2 + 77, 8, 8, 64
    args = _case(3, [n - 300], [300], H, G, d, 16, 16, fmt, hide=False)
    q, kc, vc, ks, vs, table, start = args
    for window in (0, n - 200):
        q_start, prior = _i32(start).to(DEV), _i32([n - 300]).to(DEV)
        dev = to(DEV, q, kc, vc, table, ks, vs)
        lib = _lib.load()
        out = torch.empty(300, H, d, dtype=torch.bfloat16, device=DEV)
        # without a workspace the launch never splits
        rc = lib.sna_prefill_attention_blocks(
            dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), dev[4].data_ptr(), dev[5].data_ptr(), ks.stride(0),
            ks.stride(1), 16, dev[3].data_ptr(), table.shape[1], table.shape[1], q_start.data_ptr(), prior.data_ptr(), 300, 1,
            300, None, 0.125, window, out.data_ptr(), H, G, d, 16, kc.shape[0], 3 if fmt == "int8" else 1, None, 0,
            torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, "prefill_attention_blocks")
        some = [0, 150, 299]
        want, off = ob.decode(q[some], kc, vc, table, [n - 300 + t + 1 for t in some], rows=[0] * 3, sm_scale=0.125, k_scale=ks,
                              v_scale=vs, window=window,
                              q_off=2.0 ** -16 if fmt == "int8" else 0.0)
        assert float(((out[some].cpu().double() - want).abs() - off).max()) <= 0


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_queries_of_one_large_element(fmt):
    """An outlier channel in q and a small one in K: the rest of the row still counts within its bound."""
    announce(f"outlier {fmt}")
    priors, counts = [40], [70]
    q, kc, vc, ks, vs, table, start = _case(5, priors, counts, 8, 2, 64, 16, 16, fmt)
    q = q.clone()
    q[..., 3] = 60.0
    _check((q, kc, vc, ks, vs, table, start), priors, fmt, sm_scale=0.125)
    zero = q.clone()
    zero[5:9] = 0
    _check((zero, kc, vc, ks, vs, table, start), priors, fmt, sm_scale=0.125)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_missing_pages_and_nan(fmt):
    """Pages that are none, queries that see nothing, NaN scales and queries, long tables: nobody else is touched."""
    announce(f"missing, nan {fmt}")
    priors, counts = [40, 0], [70, 40]
    H = 4
    q, kc, vc, ks, vs, table, start = _case(6, priors, counts, H, 2, 64, 16, 16, fmt, extra=5)
    table[0, 2], table[0, 3], table[1, :] = -1, kc.shape[0] + 9, -1
    got = _check((q, kc, vc, ks, vs, table, start), priors, fmt, sm_scale=0.125)
    assert bool((got[70:] == 0).all())
    # the scale of a block that only later queries see; a query that is no number
    want, off = ob.prefill(q, kc, vc, table, start, priors, sm_scale=0.125, k_scale=ks, v_scale=vs,
                           q_off=2.0 ** -16 if fmt == "int8" else 0.0)
    first = 80  # the first position of column 5, in chunk row 40
    for name in ("k", "v"):
        bad = {"k": ks.clone(), "v": vs.clone()}
        bad[name][int(table[0, 5]), 0, 0] = math.nan
        out = _run(q, kc, vc, bad["k"], bad["v"], table, start, priors, sm_scale=0.125).cpu().double()
        assert bool(out[first - 40:70, :2].isnan().all())
        clean = torch.ones(110, H, dtype=torch.bool)
        clean[first - 40:70, :2] = False
        assert float(((out - want).abs() - off)[clean].max()) <= 1e-30
    for x in (math.nan, math.inf):
        qq = q.clone()
        qq[7, 1, 9] = x
        out = _run(qq, kc, vc, ks, vs, table, start, priors, sm_scale=0.125).cpu().double()
        assert bool(out[7, 1].isnan().all())
        clean = torch.ones(110, H, dtype=torch.bool)
        clean[7, 1] = False
        assert float(((out - want).abs() - off)[clean].max()) <= 1e-30


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_stores_behind_a_nan_token(d, fmt):
    """A NaN token makes its block NaN; tokens that later calls store in that block reach nobody who does not see it: queries
    whose window has left it, and earlier queries of a chunk that two calls stored."""
    announce(f"prefill behind a NaN token {fmt} d={d}")
    G, H, P, n = 2, 4, 16, 240
    g = gen(d)
    table = (torch.randperm(n // P, generator=g) + 1).to(torch.int32).view(1, -1)
    tab = table.to(DEV)
    for window, nan_at, calls in ((20, 36, (36, 37, n)), (0, 50, (52, n))):
        caches = [torch.zeros(n // P + 1, G, P, d, dtype=FMTS[fmt], device=DEV) for _ in range(2)]
        scales = [torch.zeros(n // P + 1, G, 1, device=DEV) for _ in range(2)]
        k, v = (tokens(g, n, G, d).to(torch.bfloat16) for _ in range(2))
        k[nan_at, 0, 3] = v[nan_at, 0, 7] = math.nan
        at = 0
        for end in calls:
            ops.kv_store_blocks(k[at:end].to(DEV), v[at:end].to(DEV), *caches, tab, _i32([at]).to(DEV),
                                q_start=_i32([0, end - at]).to(DEV), max_q_len=end - at, k_scale=scales[0], v_scale=scales[1])
            at = end
        prior = calls[-2] if window else 0
        q = torch.randn(n - prior, H, d, generator=g).to(torch.bfloat16)
        args = (q, *(c.cpu() for c in caches), *(s.cpu() for s in scales), table, [0, n - prior])
        got = _run(*args, [prior], sm_scale=0.125, window=window).cpu().double()
        want, off = ob.prefill(q, *args[1:3], table, [0, n - prior], [prior], sm_scale=0.125, k_scale=args[3], v_scale=args[4],
                               window=window, q_off=ob.INT8_QUERY_OFF if fmt == "int8" else 0.0)
        first = nan_at - nan_at % P  # the block that is NaN, for KV head 0
        sees = torch.tensor([prior + i >= first and (window == 0 or prior + i - window + 1 < first + P) for i in range(n - prior)])
        assert bool(got[sees, :H // G].isnan().all())
        clean = torch.ones(n - prior, H, dtype=torch.bool)
        clean[sees, :H // G] = False
        assert bool(torch.isfinite(got[clean]).all()), int(got[clean].isnan().any(-1).sum())
        assert float(((got - want).abs() - off)[clean].max()) <= 1e-30


@pytest.mark.parametrize("d,lens", [(64, (9, 40)), (128, (60, 3)), (64, (700, 300))])
def test_bf16_rows_without_pages(d, lens):
    """bf16 caches: requests whose table names no page give zeros, whatever the output held, the others their attention."""
    announce(f"bf16 without pages {d} {lens}")
    q, kc, vc, ks, vs, table, start = _case(9, [0, 5], list(lens), 4, 2, d, 16, 16, "bf16", extra=1)
    table[0, :] = -1
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    got = _check((q, kc, vc, ks, vs, table, start), [0, 5], "bf16", sm_scale=0.125, out=out)
    assert bool((got[:lens[0]] == 0).all())


def test_sinks_without_end():
    announce("prefill sinks")
    priors, counts = [0], [20]
    args = _case(8, priors, counts, 4, 2, 64, 16, 16, "int8")
    got = _run(*args, priors, sm_scale=0.125, sinks=torch.tensor([math.inf, -math.inf, 0.0, 50.0])).cpu()
    plain = _run(*args, priors, sm_scale=0.125).cpu()
    assert bool((got[:, 0] == 0).all()) and torch.equal(got[:, 1], plain[:, 1])


@pytest.mark.parametrize("fmt", list(FMTS))
def test_a_chunk_is_its_tokens(fmt):
    """Chunks stored, attended, and the last queries attended again one by one by the token form: within both bounds."""
    announce(f"chunk and tokens {fmt}")
    H, G, d, P, bt = 8, 2, 128, 64, 32
    g = gen(31)
    priors, counts = [100, 0], [90, 130]
    table, nb = table_of(g, [p + n for p, n in zip(priors, counts)], P)
    caches = [torch.zeros(nb, G, P, d, dtype=FMTS[fmt], device=DEV) for _ in range(2)]
    scales = [None if fmt == "bf16" else torch.zeros(nb, G, P // bt, device=DEV) for _ in range(2)]
    tab = table.to(DEV)
    for at, n in (([0, 0], [100, 0]), (priors, counts)):
        start = [0, n[0], n[0] + n[1]]
        k, v = (tokens(g, start[-1], G, d).to(torch.bfloat16).to(DEV) for _ in range(2))
        ops.kv_store_blocks(k, v, *caches, tab, _i32(at).to(DEV), q_start=_i32(start).to(DEV), max_q_len=max(n),
                            k_scale=scales[0], v_scale=scales[1])
    q = torch.randn(220, H, d, generator=g).to(torch.bfloat16)
    cpu = [None if t is None else t.cpu() for t in (*caches, *scales)]
    args = (q, cpu[0], cpu[1], cpu[2], cpu[3], table, [0, 90, 220])
    got = _check(args, priors, fmt, sm_scale=d ** -0.5)
    rows, lens = [0] * 90 + [1] * 130, [101 + i for i in range(90)] + [1 + i for i in range(130)]
    one = ops.paged_decode_blocks(q.to(DEV), *caches, tab, _i32(lens).to(DEV), sm_scale=d ** -0.5, k_scale=scales[0],
                                  v_scale=scales[1], rows=_i32(rows).to(DEV)).cpu().double()
    want, off = ob.decode(q, cpu[0], cpu[1], table, lens, rows=rows, sm_scale=d ** -0.5, k_scale=cpu[2], v_scale=cpu[3])
    assert float(((one - want).abs() - off).max()) <= 1e-30
    assert float((got - one).abs().max()) < 0.1


def test_captured_and_replayed():
    announce("prefill graph")
    for priors, counts in (([200, 50], [70, 40]), ([4000], [5])):
        q, kc, vc, ks, vs, table, start = _case(9, priors, counts, 8, 2, 128, 64, 32, "int8", hide=False)
        dev = to(DEV, q, kc, vc, table, _i32(start), _i32(priors))
        kw = dict(max_q_len=max(counts), sm_scale=0.1, k_scale=ks.to(DEV), v_scale=vs.to(DEV))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.prefill_attention_blocks(*dev, **kw)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.prefill_attention_blocks(*dev, **kw)
        for _ in range(4):
            graph.replay()
            want = ops.prefill_attention_blocks(*dev, **kw)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            dev[0].mul_(-0.7)
