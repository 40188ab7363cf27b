"""The operators over caches whose blocks of tokens carry scales where sizes are extreme: offsets past 32 bits, wide tables,
pages of the largest size, and the refusals that need device tensors."""

from __future__ import annotations

import pytest
import torch

from oracle import blocks as ob
from sglang_neuron_amd import ops
from tests._block_cases import gen, tokens
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _gather(t, pages):
    return None if t is None else t[torch.tensor(pages, device=DEV)].cpu()


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Pages behind the first 4 GiB of a cache: stored, attended as a token, as a chunk and by a list."""
    announce(f"far pages {dtype}")
    G, d, P, H = 1, 128, 128, 4
    nb = (1 << 32) // (G * d * P) // (2 if dtype == torch.bfloat16 else 1) + 100
    caches = [torch.empty(nb, G, P, d, dtype=dtype, device=DEV) for _ in range(2)]
    scales = [None, None] if dtype == torch.bfloat16 else [torch.empty(nb, G, 4, device=DEV) for _ in range(2)]
    bounds = torch.empty(nb, G, 2, d, dtype=torch.bfloat16, device=DEV)
    pages, n = [nb - 1, 5, nb - 3], 300
    assert (nb - 3) * G * P * d * caches[0].element_size() > 1 << 32
    table = _i32([pages]).to(DEV)
    g = gen(1)
    k, v = (tokens(g, n, G, d).to(torch.bfloat16) for _ in range(2))
    for lo, hi in ((0, 130), (130, 300)):
        ops.kv_store_blocks(k[lo:hi].to(DEV), v[lo:hi].to(DEV), *caches, table, _i32([lo]).to(DEV),
                            q_start=_i32([0, hi - lo]).to(DEV), max_q_len=hi - lo, k_scale=scales[0], v_scale=scales[1],
                            k_bounds=bounds)
    small = [torch.zeros(3, G, P, d, dtype=dtype) for _ in range(2)]
    s_small = [None, None] if dtype == torch.bfloat16 else [torch.zeros(3, G, 4) for _ in range(2)]
    b_small = torch.zeros(3, G, 2, d, dtype=torch.bfloat16)
    near = _i32([[0, 1, 2]])
    for lo, hi in ((0, 130), (130, 300)):
        ob.append(small[0], s_small[0], k[lo:hi], near, [0, hi - lo], [lo], b_small)
        ob.append(small[1], s_small[1], v[lo:hi], near, [0, hi - lo], [lo])
    for c, s in zip(caches, small):
        assert torch.equal(_gather(c, pages).reshape(-1, d)[:n], s.reshape(-1, d)[:n])  # (one head)
    assert torch.equal(_gather(bounds, pages), b_small)
    q = torch.randn(20, H, d, generator=g).to(torch.bfloat16)
    kw = dict(sm_scale=0.1, k_scale=s_small[0], v_scale=s_small[1])
    dev = dict(sm_scale=0.1, k_scale=scales[0], v_scale=scales[1])
    want, off = ob.prefill(q, *small, near, [0, 20], [n - 20], q_off=2.0 ** -16 if dtype == torch.int8 else 0.0, **kw)
    got = ops.prefill_attention_blocks(q.to(DEV), *caches, table, _i32([0, 20]).to(DEV), _i32([n - 20]).to(DEV), max_q_len=20,
                                       **dev)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0
    want, off = ob.decode(q[:1], *small, near, [n], **kw)
    got = ops.paged_decode_blocks(q[:1].to(DEV), *caches, table, _i32([n]).to(DEV), **dev)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0
    lists = _i32([[[2, 0]]])
    want, off = ob.decode(q[:1], *small, near, [n], blocks=lists, **kw)
    got = ops.paged_decode_selected(q[:1].to(DEV), *caches, table, _i32([n]).to(DEV), lists.to(DEV), **dev)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0


def test_bounds_past_32_bits():
    announce("far bounds")
    G, d, H = 1, 128, 2
    nb = (1 << 32) // (2 * d * 2) + 50
    bounds = torch.empty(nb, G, 2, d, dtype=torch.bfloat16, device=DEV)
    pages = [nb - 1, 3, nb - 7]
    x = tokens(gen(2), 3, G, 4, d)
    near = torch.stack([x.amin(2), x.amax(2)], 2).to(torch.bfloat16)
    bounds[torch.tensor(pages, device=DEV)] = near.to(DEV)
    q = torch.randn(1, H, d, generator=gen(3)).to(torch.bfloat16)
    want, size, _ = ob.scores(q, near, _i32([[0, 1, 2]]), [90], 32)
    got, counts = ops.block_scores(q.to(DEV), bounds, _i32([pages]).to(DEV), _i32([90]).to(DEV), page_size=32)
    assert counts.tolist() == [3]
    assert bool(((got.cpu().double() - want).abs() <= 2 * d * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("P,bt", [(4096, 16), (4096, 4096), (4080, 48), (1008, 1008)])
def test_largest_pages(P, bt):
    """Pages of 4096 tokens, in blocks of 16 and in one; odd multiples of 16."""
    announce(f"large pages {P} {bt}")
    G, d, H = 1, 64, 2
    g = gen(P + bt)
    caches = [torch.zeros(4, G, P, d, dtype=torch.int8) for _ in range(2)]
    scales = [torch.zeros(4, G, P // bt) for _ in range(2)]
    dev = [t.to(DEV) for t in (*caches, *scales)]
    table, n = _i32([[2, 3]]), P + 77
    at = 0
    for m in (P - 20, 60, 37):
        k, v = (tokens(g, m, G, d).to(torch.bfloat16) for _ in range(2))
        ops.kv_store_blocks(k.to(DEV), v.to(DEV), dev[0], dev[1], table.to(DEV), _i32([at]).to(DEV),
                            q_start=_i32([0, m]).to(DEV), max_q_len=m, k_scale=dev[2], v_scale=dev[3])
        ob.append(caches[0], scales[0], k, table, [0, m], [at])
        ob.append(caches[1], scales[1], v, table, [0, m], [at])
        at += m
    assert at == n
    for a, b in zip(dev, (*caches, *scales)):
        assert torch.equal(a.cpu(), b)
    q = torch.randn(2, H, d, generator=g).to(torch.bfloat16)
    kw = dict(sm_scale=0.125, k_scale=scales[0], v_scale=scales[1])
    dkw = dict(sm_scale=0.125, k_scale=dev[2], v_scale=dev[3])
    want, off = ob.decode(q, *caches, table, [n, P + 1], rows=[0, 0], **kw)
    got = ops.paged_decode_blocks(q.to(DEV), dev[0], dev[1], table.to(DEV), _i32([n, P + 1]).to(DEV), rows=_i32([0, 0]).to(DEV),
                                  **dkw)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0
    lists = _i32([[[1]], [[0]]])
    want, off = ob.decode(q, *caches, table, [n, P + 1], rows=[0, 0], blocks=lists, **kw)
    got = ops.paged_decode_selected(q.to(DEV), dev[0], dev[1], table.to(DEV), _i32([n, P + 1]).to(DEV), lists.to(DEV),
                                    rows=_i32([0, 0]).to(DEV), **dkw)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0
    want, off = ob.prefill(q, *caches, table, [0, 2], [n - 2], q_off=2.0 ** -16, **kw)
    got = ops.prefill_attention_blocks(q.to(DEV), dev[0], dev[1], table.to(DEV), _i32([0, 2]).to(DEV), _i32([n - 2]).to(DEV),
                                       max_q_len=2, **dkw)
    assert float(((got.cpu().double() - want).abs() - off).max()) <= 0


def test_wide_tables_and_lengths_past_them():
    """A table as wide as a graph would be captured for; lengths past the table, and below 0."""
    announce("wide table")
    G, d, P, H, nb = 2, 64, 16, 4, 12
    g = gen(9)
    x = tokens(g, nb, G, P, d)
    s = x.reshape(nb, G, 1, -1).abs().amax(-1) / 127
    kc = ob.round_codes(x / s[..., None], torch.int8)
    vc, vs = kc.flip(0).contiguous(), s.flip(0).contiguous()
    q = torch.randn(3, H, d, generator=g).to(torch.bfloat16)
    table = torch.full((3, 9000), -1, dtype=torch.int32)
    table[:, :3] = _i32([[1, 2, 3], [4, 5, 6], [7, 8, 9]])
    dev = [t.to(DEV) for t in (q, kc, vc)]
    for tab, lens in ((table, [40, 1, 48]), (table[:, :2].contiguous(), [40, 2 ** 31 - 1, 33]), (table, [-5, -2 ** 31, 7])):
        want, off = ob.decode(q, kc, vc, tab, lens, sm_scale=0.125, k_scale=s, v_scale=vs)
        got = ops.paged_decode_blocks(*dev, tab.to(DEV), _i32(lens).to(DEV), sm_scale=0.125, k_scale=s.to(DEV),
                                      v_scale=vs.to(DEV))
        assert float(((got.cpu().double() - want).abs() - off).max()) <= 1e-30
    bounds = torch.zeros(nb, G, 2, d, dtype=torch.bfloat16)
    scores, counts = ops.block_scores(dev[0], bounds.to(DEV), table[:, :2].contiguous().to(DEV),
                                      _i32([40, 2 ** 31 - 1, -7]).to(DEV), page_size=P)
    assert counts.tolist() == [3, 2 ** 27, 0] and scores.shape == (3, G, 2) and bool((scores[2] == -torch.inf).all())
    picked = ops.select_blocks(dev[0], bounds.to(DEV), table[:, :2].contiguous().to(DEV), _i32([40, 2 ** 31 - 1, -7]).to(DEV),
                               keep=3, page_size=P)
    assert picked[0, 0].tolist() == [0, 1, -1] and picked[1, 1].tolist() == [0, 1, -1] and picked[2, 0].tolist() == [-1] * 3


def test_refusals_of_device_tensors():
    G, d, P, H, nb = 2, 64, 32, 4, 6
    z = lambda *shape, dt=torch.bfloat16: torch.zeros(*shape, dtype=dt, device=DEV)  # noqa: E731
    kc, vc = z(nb, G, P, d, dt=torch.int8), z(nb, G, P, d, dt=torch.int8)
    ks, vs = z(nb, G, 2, dt=torch.float32), z(nb, G, 2, dt=torch.float32)
    table, one = z(2, 3, dt=torch.int32), z(2, dt=torch.int32)
    x, q, bounds = z(2, G, d), z(2, H, d), z(nb, G, 2, d)
    store = dict(k=x, v=x, k_cache=kc, v_cache=vc, block_table=table, prior_lens=one, k_scale=ks, v_scale=vs)
    start = _i32([0, 1, 2]).to(DEV)
    for change in (dict(v=z(2, G, d, dt=torch.float32)), dict(k=z(2, 1, d)), dict(k=z(3, G, d), v=z(3, G, d)), dict(v_cache=kc),
                   dict(v_scale=ks), dict(k_scale=z(nb, 2 * G, 2, dt=torch.float32)[:, ::2]), dict(k_bounds=z(nb, G, d)),
                   dict(k_bounds=z(nb, G, 2, 2 * d)[..., ::2]), dict(block_table=z(1, 3, dt=torch.int32)), dict(max_q_len=2),
                   dict(q_start=start[:2]), dict(q_start=start, max_q_len=0), dict(q_start=start, host_q_start=[0, 2, 2]),
                   dict(q_start=start, max_q_len=2, host_q_start=[0, 2, 1]),
                   dict(q_start=start, max_q_len=2, host_q_start=[0, 1, 1])):
        with pytest.raises(ValueError):
            ops.kv_store_blocks(**{**store, **change})
    dec = dict(q=q, k_cache=kc, v_cache=vc, block_table=table, seq_lens=one, sm_scale=1.0, k_scale=ks, v_scale=vs)
    for change in (dict(q=z(2, H, 128)), dict(q=z(2, 5, d)), dict(q=z(3, H, d)), dict(block_table=z(1, 3, dt=torch.int32)),
                   dict(rows=z(3, dt=torch.int32)), dict(sinks=z(3, dt=torch.float32)), dict(out=z(2, H, d, dt=torch.float32)),
                   dict(out=z(2, H, 2 * d)[..., ::2]), dict(sm_scale=0.0), dict(window=-1), dict(k_scale=None)):
        with pytest.raises(ValueError):
            ops.paged_decode_blocks(**{**dec, **change})
    for blocks in (z(2, G, 0, dt=torch.int32), z(2, H, 3, dt=torch.int32), z(2, 3, dt=torch.int32)):
        with pytest.raises(ValueError):
            ops.paged_decode_selected(blocks=blocks, **dec)
    pre = dict(q=q, k_cache=kc, v_cache=vc, block_table=table, q_start=start, prior_lens=one, max_q_len=1, sm_scale=1.0,
               k_scale=ks, v_scale=vs)
    for change in (dict(q=z(2, 5, d)), dict(q_start=start[:2]), dict(max_q_len=0), dict(host_q_start=[0, 2, 2]),
                   dict(sinks=z(3, dt=torch.float32)), dict(out=z(3, H, d)), dict(window=-1)):
        with pytest.raises(ValueError):
            ops.prefill_attention_blocks(**{**pre, **change})
    for change in (dict(k_bounds=z(nb, G, 2, 32)), dict(k_bounds=z(nb, 3, 2, d)),
                   dict(k_bounds=z(nb, G, 2, d, dt=torch.float32)),
                   dict(page_size=0), dict(seq_lens=z(3, dt=torch.int32))):
        with pytest.raises(ValueError):
            ops.block_scores(**{**dict(q=q, k_bounds=bounds, block_table=table, seq_lens=one, page_size=P), **change})
    with pytest.raises(ValueError):
        ops.select_blocks(q, bounds, table, one, keep=1, page_size=P, first=1, recent=1)
