"""ops.select_tokens, ops.compact_tokens and ops.evict_tokens against the oracle (oracle/weights.py): positions, lengths,
weights and cache bytes are equal, and a prompt weighed, thinned and decoded on as a serving loop does it."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


def _weights(seed, R, G, N, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2.5 * torch.randn(R, G, N, generator=g) - 4)
    if kind == "ties":
        w = torch.randint(0, 3, (R, G, N), generator=g).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(R, G, N, generator=g) < 0.9, 0.0, w)
    elif kind == "strange":
        w = torch.randn(R, G, N, generator=g)
        w[torch.rand(R, G, N, generator=g) < 0.1] = float("nan")
        w[torch.rand(R, G, N, generator=g) < 0.1] = math.inf
        w[torch.rand(R, G, N, generator=g) < 0.1] = -math.inf
        w[torch.rand(R, G, N, generator=g) < 0.2] = -0.0
        w[torch.rand(R, G, N, generator=g) < 0.2] = 0.0
    elif kind == "close":  # neighbours in the last bits
        w = (torch.randint(0, 1 << 12, (R, G, N), generator=g) + 0x3F800000).to(torch.int32).view(torch.float32)
    return w


@pytest.mark.parametrize("G,N,lens,keep,first,recent,kind", [
    (1, 8, [0, 1, 2, 7, 8], 2, 0, 0, "plain"),
    (2, 100, [100, 33, 50], 33, 4, 8, "plain"),
    (2, 100, [100, 34, 99], 33, 16, 17, "ties"),
    (3, 2050, [2050, 2049, 64, 63], 64, 0, 1, "ties"),
    (2, 3000, [3000, 2999], 1000, 4, 0, "zeros"),
    (2, 3000, [3000, 1500], 1, 0, 0, "strange"),
    (2, 3000, [3000, 1500], 900, 3, 7, "strange"),
    (1, 5000, [5000, 4097, 4096], 4095, 1, 1, "close"),
    (2, 33333, [33333, 20000], 5000, 4, 64, "plain"),
    (1, 131072, [131072, 90001], 8192, 16, 512, "close"),
    (1, 300, [500, -3], 300, 0, 0, "plain"),  # lengths outside the weights are held to them
    (1, 70000, [70000], 69999, 0, 0, "ties"),
])
def test_select(G, N, lens, keep, first, recent, kind):
    announce(f"select N={N} keep={keep} {kind}")
    R = len(lens)
    w = _weights(N + keep, R, G, N, kind)
    want, new = ow.select_tokens(w, lens, keep, first, recent)
    dl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.full((R, G, keep + 5), -7.0, device=DEV)
    kept, got_new = ops.select_tokens(w.to(DEV), dl, keep=keep, first=first, recent=recent, weights_out=out)
    assert torch.equal(kept.cpu(), want) and got_new.tolist() == new
    live = want >= 0
    carried = torch.where(live, torch.gather(w, 2, want.clamp(min=0).long()), 0.0)
    assert torch.equal(out[..., :keep].cpu().nan_to_num(99.0), carried.nan_to_num(99.0)) and bool((out[..., keep:] == 0).all())
    # in place
    buf = w.to(DEV)
    kept2, _ = ops.select_tokens(buf, dl, keep=keep, first=first, recent=recent, weights_out=buf)
    assert torch.equal(kept2, kept)
    assert torch.equal(buf[..., :keep].cpu().nan_to_num(99.0), carried.nan_to_num(99.0)) and bool((buf[..., keep:] == 0).all())


def test_select_strided_weights():
    w = _weights(3, 4, 2, 300, "plain")
    wide = torch.full((2, 4, 400), 99.0, device=DEV)
    wide[..., 50:350] = w.transpose(0, 1).to(DEV)
    view = wide[..., 50:350].transpose(0, 1)
    lens = [300, 200, 61, 59]
    want, _ = ow.select_tokens(w, lens, 60, 2, 3)
    kept, _ = ops.select_tokens(view, torch.tensor(lens, device=DEV), keep=60, first=2, recent=3, weights_out=view)
    assert torch.equal(kept.cpu(), want)
    assert bool((wide[..., :50] == 99).all()) and bool((wide[..., 350:] == 99).all())
    assert bool((view[..., 60:] == 0).all())


def _cache(seed, nb, G, P, d, fp8):
    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(0, 256, (nb, G, P, d * (1 if fp8 else 2)), generator=g, dtype=torch.uint8)
    return bits.view(FP8) if fp8 else bits.view(torch.bfloat16)


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


def _table(seed, pages, nb, width, first=1):
    g = torch.Generator().manual_seed(seed)
    perm = (torch.randperm(nb - first, generator=g) + first).tolist()
    t = torch.full((len(pages), width), -1, dtype=torch.int32)
    for r, n in enumerate(pages):
        for c in range(n):
            t[r, c] = perm.pop()
    return t


@pytest.mark.parametrize("G,P,d,fp8,lens,keep", [
    (1, 16, 64, True, [5], 2), (2, 16, 128, True, [300, 40, 1], 37), (2, 16, 128, False, [300, 40, 0], 37),
    (3, 7, 64, False, [100, 99], 64), (1, 128, 128, False, [3000, 2500], 2000), (8, 16, 64, True, [900] * 5, 512),
    (2, 64, 128, True, [9000], 4500), (1, 16, 128, False, [1200], 1199),
    # in place by columns of 64 and of 128 bytes, more than a tile of each
    (2, 16, 128, False, [1400, 5, 1101] * 7, 1100), (8, 16, 128, True, [520 + 10 * i for i in range(32)], 515),
    (2, 48, 128, False, [600] * 64, 513)])
@pytest.mark.parametrize("where", ["in-place", "other-pages"])
def test_compact(G, P, d, fp8, lens, keep, where):
    announce(f"compact {where} {lens} -> {keep}")
    R = len(lens)
    pages = [-(-n // P) for n in lens]
    other = [-(-min(n, keep) // P) for n in lens]
    nb = 2 + sum(pages) + (sum(other) if where == "other-pages" else 0)
    table = _table(1, pages, nb, max(pages) + 1)
    dst = None
    if where == "other-pages":
        free = sorted(set(range(1, nb)) - set(table.flatten().tolist()))
        dst = torch.full((R, -(-keep // P)), -1, dtype=torch.int32)
        for r in range(R):
            for c in range(other[r]):
                dst[r, c] = free.pop()
    k, v = _cache(2, nb, G, P, d, fp8), _cache(3, nb, G, P, d, fp8)
    w = _weights(4, R, G, max(lens), "plain")
    kept, _ = ow.select_tokens(w, lens, keep, 1 if keep > 1 else 0, 1)
    dk, dv = k.to(DEV), v.to(DEV)
    for _ in range(1 if dst is None else 2):
        ops.compact_tokens(dk, dv, table.to(DEV), kept.to(DEV), dst_table=None if dst is None else dst.to(DEV))
    raw = lambda t: t.view(torch.uint8) if fp8 else t.view(torch.int16)  # noqa: E731
    assert torch.equal(_bytes(dk), _bytes(ow.compact_tokens(raw(k), table, kept, dst)))
    assert torch.equal(_bytes(dv), _bytes(ow.compact_tokens(raw(v), table, kept, dst)))


def test_compact_table_given_twice_is_in_place_and_holes_move_nothing():
    table = _table(1, [10, 8], 30, 10)
    k, v = _cache(5, 30, 2, 16, 64, True), _cache(6, 30, 2, 16, 64, True)
    kept, _ = ow.select_tokens(_weights(7, 2, 2, 160, "plain"), [160, 128], 60, 0, 0)
    table[0, 3], table[1, 1], table[1, 2] = -1, 10 ** 6, -5
    kept[1, 0, 5:9] = -1
    kept[0, 1, 59] = 10 ** 6  # past the table
    dk, dv, dt = k.to(DEV), v.to(DEV), table.to(DEV)
    ops.compact_tokens(dk, dv, dt, kept.to(DEV), dst_table=dt)
    assert torch.equal(_bytes(dk), _bytes(ow.compact_tokens(k.view(torch.uint8), table, kept)))
    assert torch.equal(_bytes(dv), _bytes(ow.compact_tokens(v.view(torch.uint8), table, kept)))


def test_shared_pages_evict_to_pages_of_their_own():
    """Two rows on one cached prefix: each keeps its own tokens of it, in its own pages, and the prefix stays whole."""
    P, G, d = 16, 2, 128
    table = torch.tensor([[1, 2, 3, 4], [1, 2, 5, -1]], dtype=torch.int32)
    dst = torch.tensor([[6, 7], [8, 9]], dtype=torch.int32)
    k, v = _cache(8, 10, G, P, d, False), _cache(9, 10, G, P, d, False)
    w = _weights(10, 2, G, 64, "plain")
    lens = torch.tensor([64, 40], dtype=torch.int32, device=DEV)
    dk, dv = k.to(DEV), v.to(DEV)
    kept, new = ops.evict_tokens(dk, dv, table.to(DEV), lens, w.to(DEV), keep=30, first=2, recent=4, dst_table=dst.to(DEV))
    want, _ = ow.select_tokens(w, [64, 40], 30, 2, 4)
    assert torch.equal(kept.cpu(), want) and new.tolist() == [30, 30]
    assert torch.equal(_bytes(dk), _bytes(ow.compact_tokens(k.view(torch.int16), table, want, dst)))
    assert torch.equal(_bytes(dv), _bytes(ow.compact_tokens(v.view(torch.int16), table, want, dst)))


@pytest.mark.parametrize("fp8", [True, False])
def test_a_prompt_weighed_thinned_and_decoded(fp8):
    """A prompt's cache weighed by its last 16 queries, thinned in place, and decoded on: the decode over the thinned pages
    equals, bit for bit, one over a fresh cache that holds only the kept tokens, per KV head; the steps' weights go on."""
    G, H, d, P = 2, 8, 128, 16
    lens, keep = [500, 333, 20], 96
    R = len(lens)
    g = torch.Generator().manual_seed(12)
    pages = [-(-(n + 2) // P) for n in lens]
    nb = 1 + sum(pages)
    table = _table(13, pages, nb, max(pages)).to(DEV)
    tok = [[torch.randn(n, G, d, generator=g).to(torch.bfloat16).to(DEV) for n in lens] for _ in range(2)]
    ks = vs = None
    if fp8:
        ks, vs = (ops.kv_absmax_scale(torch.cat(t)) for t in tok)
    kc = torch.zeros(nb, G, P, d, dtype=FP8 if fp8 else torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    slot = lambda r, i: table[r, i // P].long() * P + i % P  # noqa: E731
    slots = torch.cat([slot(r, torch.arange(n, device=DEV)) for r, n in enumerate(lens)])
    ops.kv_store_mha(torch.cat(tok[0]), torch.cat(tok[1]), slots, kc, vc, ks, vs)
    q = torch.randn(16 * R, H, d, generator=g).to(torch.bfloat16).to(DEV)
    start = torch.arange(R + 1, dtype=torch.int32, device=DEV) * 16
    w = ops.prefill_attention_weights(q, kc, table, start, torch.tensor([n - 16 for n in lens], device=DEV), max_q_len=16,
                                      sm_scale=d ** -0.5, k_scale=ks)
    before = w.clone()
    dl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept, new = ops.evict_tokens(kc, vc, table, dl, w, keep=keep, first=4, recent=16, weights_out=w)
    want, _ = ow.select_tokens(before.cpu(), lens, keep, 4, 16)
    assert torch.equal(kept.cpu(), want) and new.tolist() == [96, 96, 20]
    # a fresh cache of the kept tokens
    fk, fv = torch.zeros_like(kc), torch.zeros_like(vc)
    for r in range(R):
        n = int(new[r])
        at = torch.arange(n, device=DEV)
        rows = [torch.stack([t[r][kept[r, h, :n].long(), h] for h in range(G)], 1) for t in tok]
        ops.kv_store_mha(rows[0].contiguous(), rows[1].contiguous(), slot(r, at), fk, fv, ks, vs)
    step = [torch.randn(R, n, d, generator=g).to(torch.bfloat16).to(DEV) for n in (H, G, G)]
    ns = torch.stack([slot(r, new[r]) for r in range(R)])
    kw = dict(sm_scale=d ** -0.5, k_scale=ks, v_scale=vs, new_slots=ns)
    a = ops.paged_decode_gqa(step[0], kc, vc, table, new + 1, step[1], step[2], **kw)
    b = ops.paged_decode_gqa(step[0], fk, fv, table, new + 1, step[1], step[2], **kw)
    assert torch.equal(a, b)
    carried = w.clone()
    ops.decode_attention_weights(step[0], kc, table, new + 1, sm_scale=d ** -0.5, k_scale=ks, weights=w)
    alone = ops.decode_attention_weights(step[0], fk, table, new + 1, sm_scale=d ** -0.5, k_scale=ks)
    assert torch.equal(w, carried + alone)
    for r in range(R):
        n = int(new[r])
        assert bool((w[r, :, n] > 0).all()) and bool((w[r, :, n + 1:] == 0).all())
    # and thinned again, with the new token among the recent ones
    kept, new = ops.evict_tokens(kc, vc, table, new + 1, w, keep=64, first=4, recent=8, weights_out=w)
    assert new.tolist() == [64, 64, 21] and bool((kept[0, :, -1] == 96).all())


def test_refusals():
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)  # noqa: E731
    i32 = torch.int32
    w, lens = z(2, 2, 64), z(2, dtype=i32)
    for kw in (dict(keep=0), dict(keep=4, first=3, recent=2), dict(keep=4, first=-1),
               dict(keep=8, weights_out=z(2, 2, 7)), dict(keep=8, weights_out=w[:, :, 8:])):
        with pytest.raises(ValueError):
            ops.select_tokens(w, lens, **kw)
    with pytest.raises(ValueError, match="overlap"):
        ops.select_tokens(z(1, 1, 64).expand(2, 2, 64), lens, keep=4)
    k = z(5, 2, 16, 64, dtype=torch.bfloat16)
    t, kept = z(2, 4, dtype=i32), z(2, 2, 8, dtype=i32)
    with pytest.raises(ValueError, match="one tensor"):
        ops.compact_tokens(k, k, t, kept)
    with pytest.raises(ValueError, match="kept"):
        ops.compact_tokens(k, k.clone(), t, z(2, 3, 8, dtype=i32))
    with pytest.raises(ValueError, match="dst_table"):
        ops.compact_tokens(k, k.clone(), t, z(2, 2, 40, dtype=i32), dst_table=z(2, 2, dtype=i32))
    with pytest.raises(ValueError, match="weights"):
        ops.evict_tokens(k, k.clone(), t, lens, z(2, 3, 64), keep=4)
    with pytest.raises(ValueError, match="head_dim"):
        ops.compact_tokens(z(5, 2, 16, 32, dtype=torch.bfloat16), z(5, 2, 16, 32, dtype=torch.bfloat16), t, kept)


def test_a_refused_eviction_leaves_the_weights():
    """Nothing of an eviction runs unless all of its arguments are good: weights_out is the weights themselves here."""
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    t, lens = torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.full((2,), 64, dtype=torch.int32, device=DEV)
    w = _weights(1, 2, 2, 64, "plain").to(DEV)
    was = w.clone()
    for k, v, dst in ((z(5, 2, 16, 32), z(5, 2, 16, 32), None), (z(5, 2, 16, 64), z(5, 2, 8, 64), None),
                      (z(5, 2, 16, 64), z(5, 2, 16, 64), t[:, :1])):
        with pytest.raises(ValueError):
            ops.evict_tokens(k, v, t, lens, w, keep=20, weights_out=w, dst_table=dst)
    both = z(6, 2, 16, 64)
    with pytest.raises(ValueError, match="overlap"):
        ops.evict_tokens(both[:5], both[1:], t, lens, w, keep=20, weights_out=w)
    with pytest.raises(ValueError, match="another stride"):
        ops.evict_tokens(z(5, 2, 16, 64), z(5, 2, 16, 64), t, lens, w, keep=20, weights_out=w,
                         dst_table=t.view(-1)[:6].view(2, 3))
    torch.cuda.synchronize()
    assert torch.equal(w, was)


def test_the_first_pages_of_the_table_as_target_are_in_place():
    table = _table(1, [6, 5], 20, 6)
    k, v = _cache(5, 20, 2, 16, 64, False), _cache(6, 20, 2, 16, 64, False)
    w = _weights(7, 2, 2, 96, "plain")
    lens = torch.tensor([96, 77], dtype=torch.int32, device=DEV)
    dk, dv, dt = k.to(DEV), v.to(DEV), table.to(DEV)
    kept, new = ops.evict_tokens(dk, dv, dt, lens, w.to(DEV), keep=40, dst_table=dt[:, :3])
    want, _ = ow.select_tokens(w, [96, 77], 40, 0, 0)
    assert torch.equal(kept.cpu(), want) and new.tolist() == [40, 40]
    assert torch.equal(_bytes(dk), _bytes(ow.compact_tokens(k.view(torch.int16), table, want)))
    assert torch.equal(_bytes(dv), _bytes(ow.compact_tokens(v.view(torch.int16), table, want)))


@pytest.mark.parametrize("where", ["in-place", "other-pages"])
def test_cache_offsets_past_32_bits(where):
    """Tokens move between pages far behind 4 GiB of a pool as between the first ones."""
    P, G, d, lens, keep = 64, 8, 128, [900, 333], 100
    pages = [15, 6]
    near = _table(1, pages, 22 + 4, 15)
    dst = _table(2, [2, 2], 4, 2, first=0) + 22 if where == "other-pages" else None
    near = torch.where(near >= 22, -1, near)  # (the last four are the targets': holes)
    k, v = _cache(3, 26, G, P, d, False), _cache(4, 26, G, P, d, False)
    kept, _ = ow.select_tokens(_weights(5, 2, G, 900, "plain"), lens, keep, 2, 10)
    far = (2 ** 32 + 2 ** 30) // (G * P * d * 2)
    big = [torch.zeros(far + 26, G, P, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for b, t in zip(big, (k, v)):
        b[far:] = t.to(DEV)
    up = lambda t: None if t is None else torch.where(t >= 0, t + far, t).to(DEV)  # noqa: E731
    ops.compact_tokens(*big, up(near), kept.to(DEV), dst_table=up(dst))
    assert torch.equal(_bytes(big[0][far:]), _bytes(ow.compact_tokens(k.view(torch.int16), near, kept, dst)))
    assert torch.equal(_bytes(big[1][far:]), _bytes(ow.compact_tokens(v.view(torch.int16), near, kept, dst)))
    assert not bool(big[0][:far].any())


def test_graph_and_side_stream():
    P, G, d, R = 16, 2, 128, 3
    lens, keep = [400, 100, 50], 64
    pages = [-(-n // P) for n in lens]
    other = [4, 4, 4]
    nb = 1 + sum(pages) + 12
    both = _table(1, [p + o for p, o in zip(pages, other)], nb, max(pages) + 4)
    table = torch.stack([torch.cat([both[r, 4:]]) for r in range(R)])
    dst = both[:, :4].contiguous()
    k, v = _cache(2, nb, G, P, d, True).to(DEV), _cache(3, nb, G, P, d, True).to(DEV)
    w = _weights(4, R, G, 400, "ties").to(DEV)
    dt, dd, dl = table.to(DEV), dst.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.empty(R, G, keep, device=DEV)
    run = lambda: ops.evict_tokens(k, v, dt, dl, w, keep=keep, first=1, recent=2, dst_table=dd, weights_out=out)  # noqa: E731
    eager = [t.clone() for t in (*run(), out, k.view(torch.uint8), v.view(torch.uint8))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(4):
        for t in (*outs, out):
            t.fill_(7)
        k.view(torch.uint8)[dd[:2].long().flatten()] = 1  # (the third row is short: its pages' last slots get nothing)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*outs, out, k.view(torch.uint8), v.view(torch.uint8)), eager):
            assert torch.equal(a, b)
