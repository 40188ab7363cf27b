"""ops.paged_decode_blocks, ops.paged_decode_selected, ops.block_scores and ops.select_blocks against their definitions in 64
bits, on pools that hold garbage wherever nothing was stored. The bounds are oracle.blocks.attend's."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import blocks as ob
from oracle import weights as ow
from sglang_neuron_amd import _lib, ops
from tests._block_cases import FMTS, gen, hide_unstored, pool, same_bits, table_of, to, tokens
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _within(got, want, off, what=""):
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), what
    over = (got - want).abs() - off
    assert float(over.max()) <= 1e-30, f"{what}: {float((got - want).abs().max()):.3e} off, {float(over.max()):.3e} over"


def _case(seed, lens, H, G, d, P, bt, fmt, extra=1, rows=None, hide=True):
    g = gen(seed)
    table, nb = table_of(g, lens, P, extra)
    kc, ks = pool(g, nb + 1, G, P, d, bt, fmt)
    vc, vs = pool(g, nb + 1, G, P, d, bt, fmt)
    if hide:
        for c, s in ((kc, ks), (vc, vs)):
            hide_unstored(c, s, table, lens, P)
    T = len(lens) if rows is None else len(rows)
    return torch.randn(T, H, d, generator=g).to(torch.bfloat16), kc, vc, ks, vs, table


def _run(q, kc, vc, ks, vs, table, lens, **kw):
    kc, vc, ks, vs, table, q = to(DEV, kc, vc, ks, vs, table, q)
    kw = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    lens = lens.to(DEV) if isinstance(lens, torch.Tensor) else _i32(lens).to(DEV)
    if "blocks" in kw:
        return ops.paged_decode_selected(q, kc, vc, table, lens, kw.pop("blocks"), k_scale=ks, v_scale=vs, **kw)
    return ops.paged_decode_blocks(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, **kw)


SHAPES = [(4, 2, 128, 16, 16), (3, 3, 64, 32, 16), (16, 1, 64, 48, 48), (10, 2, 128, 64, 32), (5, 1, 128, 128, 128),
          (8, 8, 64, 256, 64)]


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("H,G,d,P,bt", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, False), (37, True), (1, False)])
def test_rows_of_all_lengths(fmt, H, G, d, P, bt, window, sinks):
    """From no key to several pages: the tile's, half-tile's and page's edges, with a window and sinks."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]
    announce(f"decode {fmt} H={H} G={G} d={d} P={P} bt={bt} window={window} sinks={sinks}")
    q, kc, vc, ks, vs, table = _case(H + P, lens, H, G, d, P, bt, fmt)
    sk = torch.randn(H, generator=gen(1)) if sinks else None
    kw = dict(sm_scale=d ** -0.5, sinks=sk, window=window)
    want, off = ob.decode(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, **kw)
    got = _run(q, kc, vc, ks, vs, table, lens, **kw)
    _within(got, want, off, "decode")
    assert bool((got[0] == 0).all())


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("T,lo,hi,H,G,d,P,bt", [(1, 5000, 5000, 8, 1, 128, 16, 16), (2, 3000, 9000, 8, 2, 64, 32, 32),
                                                (70, 1, 700, 32, 8, 128, 16, 16), (520, 1, 90, 2, 1, 64, 16, 16)])
def test_few_and_many_rows(fmt, T, lo, hi, H, G, d, P, bt):
    """Rows cut into many splits, into few, and whole; more than 256 table columns a split."""
    g = gen(T)
    lens = torch.randint(lo, hi + 1, (T,), generator=g).tolist()
    announce(f"decode rows {fmt} T={T} {lo}..{hi}")
    q, kc, vc, ks, vs, table = _case(T, lens, H, G, d, P, bt, fmt, hide=hi < 1000)
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.1, k_scale=ks, v_scale=vs)
    _within(_run(q, kc, vc, ks, vs, table, lens, sm_scale=0.1), want, off)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_whole_rows_past_256_columns(fmt):
    """512 workgroups of whole rows: a row's pages are staged 256 at a time."""
    H, G, d, P = 2, 1, 64, 16
    T, n = 512, 16 * 300 + 5
    announce(f"decode whole rows {fmt}")
    g = gen(2)
    table, nb = table_of(g, [n] * 3, P)
    kc, ks = pool(g, nb, G, P, d, 16, fmt)
    vc, vs = pool(g, nb, G, P, d, 16, fmt)
    rows = [i % 3 for i in range(T)]
    lens = [n - i // 3 for i in range(T)]
    q = torch.randn(T, H, d, generator=g).to(torch.bfloat16)
    some = [0, 1, 200, 511]
    want, off = ob.decode(q[some], kc, vc, table, [lens[i] for i in some], sm_scale=0.2, k_scale=ks, v_scale=vs,
                          rows=[rows[i] for i in some])
    got = _run(q, kc, vc, ks, vs, table, lens, sm_scale=0.2, rows=_i32(rows))
    _within(got[some], want, off)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("H,G,d,P,bt", SHAPES)
def test_selected_pages(fmt, H, G, d, P, bt):
    """Lists of each query and head: padded, unordered, out of the table, empty, past the row's length."""
    lens = [0, 1, 40, 3 * P, 5 * P + 3, 9 * P - 1, 700]
    announce(f"selected {fmt} H={H} G={G} d={d} P={P} bt={bt}")
    q, kc, vc, ks, vs, table = _case(H + P, lens, H, G, d, P, bt, fmt)
    W, n = table.shape[1], 5
    g = gen(7)
    lists = [torch.stack([torch.randperm(max(W, n), generator=g)[:n] for _ in range(G)]) for _ in lens]
    lists = torch.stack(lists).to(torch.int32)
    lists[3, :, 1:3] = -1
    lists[4, 0] = -1
    lists[5, :, 0], lists[5, :, 4] = 0, 2 ** 31 - 1
    kw = dict(sm_scale=d ** -0.5, sinks=torch.randn(H, generator=g))
    want, off = ob.decode(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, blocks=lists, **kw)
    _within(_run(q, kc, vc, ks, vs, table, lens, blocks=lists, **kw), want, off)
    # every page, in order, is the whole row
    whole = torch.arange(W, dtype=torch.int32).expand(len(lens), G, W).contiguous()
    want, off = ob.decode(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, **kw)
    _within(_run(q, kc, vc, ks, vs, table, lens, blocks=whole, **kw), want, off)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_long_lists(fmt):
    """More than 256 pages of a list, cut into splits and (many queries) whole."""
    H, G, d, P = 4, 1, 64, 16
    announce(f"selected long lists {fmt}")
    lens = [16 * 900, 16 * 700 + 3]
    q, kc, vc, ks, vs, table = _case(11, lens, H, G, d, P, 16, fmt, hide=False)
    g = gen(8)
    lists = torch.stack([torch.randperm(700, generator=g)[:301].sort().values for _ in lens]).to(torch.int32)[:, None]
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.125, k_scale=ks, v_scale=vs, blocks=lists)
    _within(_run(q, kc, vc, ks, vs, table, lens, blocks=lists, sm_scale=0.125), want, off)
    T = 512
    rows = [i % 2 for i in range(T)]
    got = _run(q[rows], kc, vc, ks, vs, table, [lens[r] for r in rows], blocks=lists[rows], sm_scale=0.125, rows=_i32(rows))
    _within(got[[0, 511]], want, off)


def _by_page(T, R, W, n, H, G, d, P, fmt):
    """Whether a call goes page by page: its workspace is a partial for each listed page's 64 keys."""
    need = _lib.load().sna_block_decode_workspace_bytes(T, H, G, d, P, W, R, 0, n, ops._BLOCK_CODES[FMTS[fmt]])
    return need == T * n * -(-P // 64) * H * (d + 2) * 4


@pytest.mark.parametrize("H,G,d,P,bt,fmt,T,n,cols", [
    (16, 8, 128, 64, 64, "bf16", 840, 5, 8), (4, 2, 128, 64, 16, "fp8", 800, 41, 8), (3, 3, 64, 64, 32, "int8", 700, 32, 9),
    (6, 2, 64, 80, 16, "bf16", 700, 47, 8), (2, 2, 64, 96, 32, "fp8", 840, 40, 7), (1, 1, 128, 128, 128, "bf16", 840, 40, 8),
    (24, 8, 64, 128, 64, "int8", 330, 50, 8), (2, 1, 64, 64, 64, "bf16", 4100, 8, 3), (1, 1, 64, 64, 16, "fp8", 2000, 33, 3)])
def test_selected_pages_of_many_queries(H, G, d, P, bt, fmt, T, n, cols):
    """Prompts' queries: few rows, many queries a page (more than a workgroup lists at a time), lengths that end inside pages,
    rows outside the table, pages listed twice, unordered, invalid."""
    announce(f"selected by page {fmt} H={H} G={G} d={d} P={P} bt={bt} T={T} n={n}")
    R = 3
    lens = [cols * P, (cols - 1) * P + 3, 1]
    q, kc, vc, ks, vs, table = _case(P + T, lens, H, G, d, P, bt, fmt, rows=[0] * T)
    W = table.shape[1]
    assert _by_page(T, R, W, n, H, G, d, P, fmt)
    if cols > 3:
        table[0, 2], table[1, 1] = -1, kc.shape[0] + 5
    g = gen(T)
    rows = (torch.rand(T, generator=g) < 0.3).long()
    at = torch.where(rows == 0, torch.randint((cols - 1) * P - 5, cols * P + 1, (T,), generator=g),
                     (cols - 1) * P + torch.randint(0, 4, (T,), generator=g))
    some = torch.randperm(T, generator=g)[:12].tolist()  # (of nobody else's lengths)
    for t, (r, n_t) in zip(some, [(2, 1), (2, 0), (-1, 9), (3, 9), (2 ** 31 - 1, 9), (0, 1), (0, -4), (0, P), (1, 16), (0, 0),
                                  (1, 2 * P + 1), (0, 3 * P - 1)]):
        rows[t], at[t] = r, n_t
    lists = torch.randint(0, cols, (T, G, n), generator=g).to(torch.int32)
    lists[::2, :, 0] = cols - 1
    lists[1::7, :, 3] = lists[1::7, :, 1]
    lists[2::9, 0] = -1
    lists[4::9, :, 2], lists[5::9, :, 3] = 2 ** 31 - 1, W
    kw = dict(sm_scale=d ** -0.5, sinks=torch.randn(H, generator=g))
    want, off = ob.decode(q, kc, vc, table, at.tolist(), k_scale=ks, v_scale=vs, blocks=lists, rows=rows.tolist(), **kw)
    got = _run(q, kc, vc, ks, vs, table, at.to(torch.int32), blocks=lists, rows=rows.to(torch.int32), **kw)
    _within(got, want, off)
    again = _run(q, kc, vc, ks, vs, table, at.to(torch.int32), blocks=lists, rows=rows.to(torch.int32), **kw)
    assert same_bits(got, again)


def test_selected_pages_of_many_queries_specials():
    """Page by page, captured and replayed with other lists; NaN reaches the queries that see it and no others."""
    announce("selected by page, graph")
    H, G, d, P, T, R, n, cols = 4, 2, 128, 64, 2080, 2, 8, 24
    q, kc, vc, ks, vs, table = _case(5, [cols * P] * R, H, G, d, P, 64, "bf16", rows=[0] * T, hide=False)
    assert _by_page(T, R, table.shape[1], n, H, G, d, P, "bf16")
    g = gen(6)
    rows = _i32([i % 2 for i in range(T)])
    at = torch.randint(1, cols * P + 1, (T,), generator=g).to(torch.int32)
    pick = lambda: torch.stack([torch.stack([torch.randperm(cols, generator=g)[:n] for _ in range(G)])
                                for _ in range(T)]).to(torch.int32)
    vc[int(table[0, 3]), 1, 7, 2] = float("nan")
    state = to(DEV, q, kc, vc, table, at, pick(), rows)

    def call():
        s = state
        return ops.paged_decode_selected(s[0], s[1], s[2], s[3], s[4], s[5], sm_scale=0.1, rows=s[6])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        lists = pick()
        state[5].copy_(lists)
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert same_bits(got.isnan(), eager.isnan()) and same_bits(got.nan_to_num(), eager.nan_to_num())
        want, off = ob.decode(q, kc, vc, table, at.tolist(), sm_scale=0.1, blocks=lists, rows=rows.tolist())
        nan = got.isnan().cpu()
        sees = (lists[:, 1] == 3).any(-1) & (rows == 0) & (at > 3 * P + 7)
        assert bool(sees.any()) and torch.equal(nan[:, 2:, 2], sees[:, None].expand(T, 2))
        nan[:, 2:, 2] = False
        assert not bool(nan.any())
        ok = ~got.isnan().cpu()
        _within(torch.where(ok, got.cpu().float(), 0.0), torch.where(ok, want, 0.0), torch.where(ok, off, 0.0))


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_selected_pages_of_many_queries_scales(fmt):
    """Page by page: a scale that is NaN reaches the queries that see its block and no others, whatever they share."""
    announce(f"selected by page, NaN scales {fmt}")
    H, G, d, P, T, R, n, cols = 8, 4, 64, 64, 2100, 2, 8, 6
    q, kc, vc, ks, vs, table = _case(8, [cols * P] * R, H, G, d, P, 16, fmt, rows=[0] * T, hide=False)
    assert _by_page(T, R, table.shape[1], n, H, G, d, P, fmt)
    g = gen(9)
    rows = torch.arange(T) % 2
    at = torch.randint(5 * P - 20, cols * P + 1, (T,), generator=g)
    lists = torch.randint(0, cols, (T, G, n), generator=g).to(torch.int32)
    want, off = ob.decode(q, kc, vc, table, at.tolist(), k_scale=ks, v_scale=vs, sm_scale=0.1, blocks=lists, rows=rows.tolist())
    ks[int(table[0, 5]), 0, 2] = float("nan")
    vs[int(table[1, 5]), 0, 1] = float("nan")
    got = _run(q, kc, vc, ks, vs, table, at.to(torch.int32), sm_scale=0.1, blocks=lists, rows=rows.to(torch.int32)).cpu()
    sees = (lists[:, 0] == 5).any(-1) & (at > 5 * P + torch.where(rows == 0, 32, 16))
    assert bool(sees.any()) and bool((~sees & (lists[:, 0] == 5).any(-1) & (at > 5 * P)).any())
    assert bool(got[sees, :2].isnan().all())
    _within(got[:, 2:], want[:, 2:], off[:, 2:])
    _within(got[~sees, :2], want[~sees, :2], off[~sees, :2])


def test_rows_and_strided_tables():
    """Several queries of a row at lengths of their own; rows outside the table see nothing; tables that are views."""
    announce("decode rows, strides")
    lens = [100, 37]
    H, G, d, P = 4, 2, 64, 16
    rows = [1, 0, 0, 0, 1, 5, -3]
    at = [37, 100, 99, 98, 5, 20, 20]
    q, kc, vc, ks, vs, table = _case(4, lens, H, G, d, P, 16, "fp8", rows=rows)
    want, off = ob.decode(q, kc, vc, table, at, sm_scale=0.125, k_scale=ks, v_scale=vs, rows=rows)
    wide = torch.full((2, 40), 7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for tab in (table, wide.to(DEV)[:, :table.shape[1]], table.t().contiguous().t().to(DEV), table.long()):
        got = _run(q, kc, vc, ks, vs, tab, at, sm_scale=0.125, rows=torch.tensor(rows))
        _within(got, want, off)
        assert bool((got[5:] == 0).all())
    # one row for all queries, expanded; an output of the caller's; queries that are a view
    one = table[:1].to(DEV).expand(7, -1)
    want, off = ob.decode(q, kc, vc, table, at, sm_scale=0.125, k_scale=ks, v_scale=vs, rows=[0] * 7)
    out = torch.full((7, H, d), 9.0, dtype=torch.bfloat16, device=DEV)
    wide_q = torch.cat([q, q], 1).to(DEV)[:, :H]
    args = to(DEV, kc, vc)
    got = ops.paged_decode_blocks(wide_q, *args, one, _i32(at).to(DEV), sm_scale=0.125, k_scale=ks.to(DEV),
                                  v_scale=vs.to(DEV), out=out)
    assert got.data_ptr() == out.data_ptr()
    _within(got, want, off)


def test_scales_of_other_strides():
    """One scale for all pages (expanded), scales that are views, K's and V's of different strides."""
    announce("decode scale strides")
    lens, H, G, d, P = [70, 33], 4, 2, 64, 32
    q, kc, vc, ks, vs, table = _case(6, lens, H, G, d, P, 16, "int8", hide=False)
    one = torch.tensor([0.02, 0.03]).view(1, G, 1).expand(kc.shape[0], G, 1)
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.125, k_scale=one.contiguous(), v_scale=one.contiguous())
    dev = torch.tensor([0.02, 0.03], device=DEV).view(1, G, 1).expand(kc.shape[0], G, 1)
    args = to(DEV, q, kc, vc, table, _i32(lens))
    _within(ops.paged_decode_blocks(*args, sm_scale=0.125, k_scale=dev, v_scale=dev), want, off)
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.125, k_scale=ks, v_scale=vs)
    both = torch.stack([ks, vs], 1).to(DEV)  # [blocks, 2, G, n]
    _within(ops.paged_decode_blocks(*args, sm_scale=0.125, k_scale=both[:, 0], v_scale=both[:, 1]), want, off)
    odd = vs.permute(2, 0, 1).contiguous().permute(1, 2, 0).to(DEV)
    _within(ops.paged_decode_blocks(*args, sm_scale=0.125, k_scale=ks.to(DEV), v_scale=odd), want, off)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_scales_far_apart(fmt):
    """Blocks whose values differ by 2^60, and blocks of zeros at the least scale, weigh what they should."""
    announce(f"decode far scales {fmt}")
    lens, H, G, d, P = [150, 16 * 9], 4, 2, 64, 16
    q, kc, vc, ks, vs, table = _case(12, lens, H, G, d, P, 16, fmt, hide=False)
    g = gen(3)
    vs = vs * torch.exp2(torch.randint(-40, 20, vs.shape, generator=g).float())
    vs[::3] = 2.0 ** -100
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.125, k_scale=ks, v_scale=vs)
    _within(_run(q, kc, vc, ks, vs, table, lens, sm_scale=0.125), want, off)


def test_special_values():
    """NaN reaches the rows that see it and no others; sinks of +-inf; scores far beyond the exponential's range."""
    announce("decode specials")
    lens, H, G, d, P = [40, 40, 40], 4, 2, 64, 16
    q, kc, vc, ks, vs, table = _case(13, lens, H, G, d, P, 16, "int8")
    want, off = ob.decode(q, kc, vc, table, lens, sm_scale=0.125, k_scale=ks, v_scale=vs)
    bad = ks.clone()
    bad[int(table[1, 2]), 0, 0] = math.nan
    got = _run(q, kc, vc, bad, vs, table, lens, sm_scale=0.125)
    assert bool(got[1, :2].isnan().all())
    keep = torch.ones(3, H, dtype=torch.bool)
    keep[1, :2] = False
    _within(got.cpu()[keep], want[keep], off[keep])
    # a window that does not reach the block
    w2, o2 = ob.decode(q, kc, vc, table, [32, 32, 32], sm_scale=0.125, k_scale=ks, v_scale=vs)
    _within(_run(q, kc, vc, bad, vs, table, [32, 32, 32], sm_scale=0.125), w2, o2)
    sinks = torch.tensor([math.inf, -math.inf, 0.5, 300.0])
    got = _run(q, kc, vc, ks, vs, table, lens, sm_scale=0.125, sinks=sinks).cpu()
    assert bool((got[:, 0] == 0).all())
    _within(got[:, 1], want[:, 1], off[:, 1])
    assert float(got[:, 3].abs().max()) < 1e-30
    want, off = ob.decode(q * 2000, kc, vc, table, lens, sm_scale=0.125, k_scale=ks, v_scale=vs)
    _within(_run(q * 2000, kc, vc, ks, vs, table, lens, sm_scale=0.125), want, off)


@pytest.mark.parametrize("H,G,d,P", [(4, 2, 128, 16), (3, 3, 64, 48), (16, 1, 64, 64), (10, 2, 128, 128)])
def test_scores(H, G, d, P):
    """Every page's bound, up to 200 columns, invalid pages, rows, counts. fp32 sums of 2 d exact products: 2 d 2^-24 off."""
    announce(f"scores H={H} G={G} d={d} P={P}")
    lens = [0, 1, P, P + 1, 17 * P - 1, 64 * P, 65 * P + 3, 200 * P]
    g = gen(P)
    table, nb = table_of(g, lens, P, 3)
    table[6, 5], table[6, 6] = -1, nb + 7
    b = tokens(g, nb, G, 3, d)
    bounds = torch.stack([b.amin(2), b.amax(2)], 2).to(torch.bfloat16)
    bounds[0] = math.nan
    rows = [3, 0, 7, 6, 9, 4, 5, 1, 2, 6]
    at = [lens[r] if r < 8 else 30 for r in rows]
    q = torch.randn(len(rows), H, d, generator=g).to(torch.bfloat16)
    q[2, 0, :5] = 0.0
    q[2, 1, :5] = -0.0
    for rr, ll in ((rows, at), (None, lens)):
        qq = q[:len(ll)]
        want, size, counts = ob.scores(qq, bounds, table, ll, P, rr)
        got, n = ops.block_scores(*to(DEV, qq, bounds, table, _i32(ll)), page_size=P,
                                  rows=None if rr is None else _i32(rr).to(DEV))
        assert n.tolist() == counts
        got = got.cpu().double()
        assert torch.equal(got == -math.inf, want == -math.inf)
        ok = want > -math.inf
        assert bool(((got - want).abs()[ok] <= 2 * d * 2.0 ** -24 * size[ok]).all())


@pytest.mark.parametrize("H,G,d,P", [(4, 2, 128, 16), (3, 3, 64, 48), (16, 1, 64, 64), (10, 2, 128, 128)])
def test_scores_of_infinite_bounds(H, G, d, P):
    """Pages with infinite keys and with dimensions that are NaN in every key, as the writer leaves their bounds, among ordinary
    ones; query elements of 0, infinite and NaN. Infinite and NaN scores are the definition's, the others as near as ever."""
    announce(f"scores, infinite bounds H={H} G={G} d={d} P={P}")
    lens, inf = [64 * P, 3 * P, 20 * P], math.inf
    g = gen(P + 1)
    table, nb = table_of(g, lens, P)
    b = tokens(g, nb, G, 3, d)
    bounds = torch.stack([b.amin(2), b.amax(2)], 2).to(torch.bfloat16)
    kinds = [(-inf, None), (None, inf), (-inf, inf), (inf, -inf), (inf, inf), (-inf, -inf)]
    for c in range(64):  # (every third page of row 0, one to three dimensions of each KV head; all pages of row 1)
        for r in range(2):
            if (r == 0 and c % 3) or (r == 1 and c > 2):
                continue
            for gg in range(G):
                for at in torch.randperm(d, generator=g)[:1 + c % 3].tolist():
                    lo, hi = kinds[int(torch.randint(len(kinds), (1,), generator=g))]
                    page = int(table[r, c])
                    if lo is not None:
                        bounds[page, gg, 0, at] = lo
                    if hi is not None:
                        bounds[page, gg, 1, at] = hi
    rows = [0, 0, 0, 1, 1, 2, 2]
    q = torch.randn(len(rows), H, d, generator=g).to(torch.bfloat16)
    q[1, :, ::2] = 0.0
    q[1, :, 1::4] = -0.0
    q[2, 0, 5], q[2, H - 1, 7], q[4, 0, 1], q[6, H - 1, 2] = math.nan, inf, math.nan, -inf
    at = [lens[r] for r in rows]
    want, size, counts = ob.scores(q, bounds, table, at, P, rows)
    got, n = ops.block_scores(*to(DEV, q, bounds, table, _i32(at)), page_size=P, rows=_i32(rows).to(DEV))
    assert n.tolist() == counts
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    assert int((want == inf).sum()) > 20 and int(fin.sum()) > 20
    # (a finite score among heads whose own sums are infinite: its magnitudes are at most those of all finite bounds)
    fb = torch.where(bounds.double().isinf(), 0.0, bounds.double())
    for t, r in enumerate(rows):
        for gg in range(G):
            for c in range(counts[t]):
                if fin[t, gg, c]:
                    x = torch.nan_to_num(q[t, gg * (H // G):(gg + 1) * (H // G)].double(), posinf=0.0, neginf=0.0)
                    most = float((x.abs() @ fb[int(table[r, c]), gg].abs().amax(0)).max())
                    assert abs(float(got[t, gg, c] - want[t, gg, c])) <= 2 * d * 2.0 ** -24 * most


def test_a_page_of_infinite_keys_is_selected():
    """Stored with bounds: an infinite key's page scores what its other heads and elements give, or is the first of all."""
    announce("selection, infinite keys")
    G, d, P, keep = 1, 64, 16, 3
    g = gen(8)
    k = torch.randint(-4, 5, (10 * P, G, d), generator=g).to(torch.bfloat16)
    k[5 * P + 3, 0, 7] = math.inf    # q's element 7 is positive: page 5 is the first of all
    k[7 * P, 0, 9] = -math.inf       # q's element 9 is positive: page 7 by its other elements
    caches = [torch.zeros(11, G, P, d, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(11, G, 1, device=DEV) for _ in range(2)]
    bounds = torch.zeros(11, G, 2, d, dtype=torch.bfloat16, device=DEV)
    table = (torch.randperm(10, generator=g) + 1).to(torch.int32).view(1, 10)
    ops.kv_store_blocks(k.to(DEV), k.to(DEV).nan_to_num(posinf=0.0, neginf=0.0), *caches, table.to(DEV), _i32([0]).to(DEV),
                        q_start=_i32([0, 10 * P]).to(DEV), max_q_len=10 * P, k_scale=scales[0], v_scale=scales[1],
                        k_bounds=bounds)
    q = torch.randint(1, 5, (1, 2, d), generator=g).to(torch.bfloat16)
    want, _, pages = ob.scores(q, bounds.cpu(), table, [10 * P], P)
    assert want[0, 0, 5] == math.inf and bool(torch.isfinite(want[0, 0, 7]))
    got, _ = ops.block_scores(q.to(DEV), bounds, table.to(DEV), _i32([10 * P]).to(DEV), page_size=P)
    assert torch.equal(got.cpu().double(), want)  # (small whole numbers: exact)
    chosen, _ = ow.select_tokens(want.float(), pages, keep, 0, 0)
    sel = ops.select_blocks(q.to(DEV), bounds, table.to(DEV), _i32([10 * P]).to(DEV), keep=keep, page_size=P, first=0, recent=0)
    assert torch.equal(sel.cpu(), chosen) and 5 in chosen[0, 0].tolist()


def test_writer_to_selection_to_attention():
    """The operators as they are used: chunks, then tokens, appended with bounds; each query's pages selected; attention over
    them. Scores of small whole numbers are exact, so the selection has to be the definition's."""
    announce("writer, selection, attention")
    H, G, d, P, bt, keep = 6, 2, 64, 32, 16, 5
    g = gen(21)
    priors, counts = [0, 0, 0], [400, 90, 33]
    table, nb = table_of(g, [p + n + 3 for p, n in zip(priors, counts)], P)
    for fmt in FMTS:
        caches = [torch.zeros(nb, G, P, d, dtype=FMTS[fmt]) for _ in range(2)]
        scales = [None if fmt == "bf16" else torch.zeros(nb, G, P // bt) for _ in range(2)]
        bounds = torch.zeros(nb, G, 2, d, dtype=torch.bfloat16)
        dc, ds, db = to(DEV, *caches), to(DEV, *scales), bounds.to(DEV)
        lens = priors
        for step, n in enumerate((counts, [1, 1, 1], [1, 1, 1])):
            start = [sum(n[:r]) for r in range(4)]
            k = torch.randint(-8, 9, (start[-1], G, d), generator=g).to(torch.bfloat16)
            v = tokens(g, start[-1], G, d).to(torch.bfloat16)
            ops.kv_store_blocks(k.to(DEV), v.to(DEV), *dc, table.to(DEV), _i32(lens).to(DEV),
                                q_start=_i32(start).to(DEV) if step == 0 else None, max_q_len=max(n), k_scale=ds[0],
                                v_scale=ds[1], k_bounds=db)
            ob.append(caches[0], scales[0], k, table, start, lens, bounds)
            ob.append(caches[1], scales[1], v, table, start, lens)
            lens = [a + b for a, b in zip(lens, n)]
            q = torch.randint(-8, 9, (3, H, d), generator=g).to(torch.bfloat16)
            want, _, pages = ob.scores(q, bounds, table, lens, P)
            chosen, _ = ow.select_tokens(want.float(), pages, keep, 1, 1)
            got = ops.select_blocks(q.to(DEV), db, table.to(DEV), _i32(lens).to(DEV), keep=keep, page_size=P)
            assert torch.equal(got.cpu(), chosen)
            o, off = ob.decode(q, caches[0], caches[1], table, lens, sm_scale=0.02, k_scale=scales[0], v_scale=scales[1],
                               blocks=chosen)
            _within(ops.paged_decode_selected(q.to(DEV), *dc, table.to(DEV), _i32(lens).to(DEV), got, sm_scale=0.02,
                                              k_scale=ds[0], v_scale=ds[1]), o, off, fmt)


def test_captured_and_replayed():
    """A step (append, scores, selection, attention dense and selected) captured once and replayed with other contents, eager
    work between the replays; split and whole rows. Every replay equals the eager call on the same state."""
    announce("graph")
    H, G, d, P, bt = 8, 2, 128, 16, 16
    for T, n in ((2, 700), (300, 60)):
        g = gen(T)
        table, nb = table_of(g, [n + 8] * T, P)
        kc, ks = pool(g, nb, G, P, d, bt, "fp8")
        vc, vs = pool(g, nb, G, P, d, bt, "fp8")
        b = tokens(g, nb, G, 3, d)
        state = to(DEV, kc, vc, ks, vs, torch.stack([b.amin(2), b.amax(2)], 2).to(torch.bfloat16))
        tab, lens = table.to(DEV), torch.full((T,), n, dtype=torch.int32, device=DEV)
        prior = lens - 1
        q, k, v = (torch.randn(T, h, d, generator=g).to(torch.bfloat16).to(DEV) for h in (H, G, G))

        def step(s):
            ops.kv_store_blocks(k, v, s[0], s[1], tab, prior, k_scale=s[2], v_scale=s[3], k_bounds=s[4])
            pages = ops.select_blocks(q, s[4], tab, lens, keep=3, page_size=P)
            return (pages, ops.paged_decode_blocks(q, s[0], s[1], tab, lens, sm_scale=0.1, k_scale=s[2], v_scale=s[3]),
                    ops.paged_decode_selected(q, s[0], s[1], tab, lens, pages, sm_scale=0.1, k_scale=s[2], v_scale=s[3]))

        eager = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step([t.clone() for t in state])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(state)
        for i in range(4):
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            for a, c in zip((*got, *state), (*want, *eager)):
                assert same_bits(a, c)
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
            lens += 1
            prior += 1


def test_two_streams_at_once():
    announce("two streams")
    lens, H, G, d, P = [900, 777], 8, 2, 64, 16
    cases = [_case(s, lens, H, G, d, P, 16, "int8", hide=False) for s in (1, 2)]
    args = [to(DEV, q, kc, vc, table, _i32(lens), ks, vs) for q, kc, vc, ks, vs, table in cases]
    want = [ops.paged_decode_blocks(*a[:5], sm_scale=0.1, k_scale=a[5], v_scale=a[6]) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[] for _ in args]
    for _ in range(20):
        for i, (s, a) in enumerate(zip(streams, args)):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_decode_blocks(*a[:5], sm_scale=0.1, k_scale=a[5], v_scale=a[6]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_empty_calls():
    announce("empty")
    kc = torch.zeros(2, 1, 16, 64, dtype=torch.int8, device=DEV)
    s = torch.ones(2, 1, 1, device=DEV)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.paged_decode_blocks(none, kc, kc.clone(), table, lens, sm_scale=1.0, k_scale=s, v_scale=s).shape == (0, 2, 64)
    ops.kv_store_blocks(none[:, :1], none[:, :1], kc, kc.clone(), table, lens, k_scale=s, v_scale=s.clone())
    bounds = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    scores, counts = ops.block_scores(none, bounds, table, lens, page_size=16)
    assert scores.shape == (0, 1, 3) and counts.shape == (0,)
