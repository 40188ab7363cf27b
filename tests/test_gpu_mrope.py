"""ops.qkv_norm_mrope_store against the 64-bit oracle (oracle/weights.mrope_rows).

Tolerance. Before its one rounding an output is off by fp32 steps: the norm (d / 8 additions in sequence and 4 folds under
a square root, so half of at most 24 steps, then three products: under 16 steps of 2^-24), and the rotation: a sine or
cosine off by at most 2^-21 (the fraction of a turn, half a step of 1/2, times 2 pi, under 2^-22.6; the function's own
error and rounding under 4 steps of 2^-24; the 64-bit angle's below both for these positions) and two products and a sum.
So off <= (|x c| + |y s|) * E with |c|, |s| <= 1 taken as 1, E = 2^-21 + 20 * 2^-24, and the rounding adds half a step of
the result: 2^-8 (bf16) or 2^-4 relative (e4m3fn; 2^-10 absolute below 2^-6). FP8 bytes are compared as values * scale."""

from __future__ import annotations

import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
E = 2.0 ** -21 + 20 * 2.0 ** -24


def _make(seed, T, Hq, Hkv, d, P, fp8, norm, rot, A, base, extra=2):
    g = torch.Generator().manual_seed(seed)
    nb = -(-max(T, 1) // P) + 1 + extra
    qkv = torch.randn(T, (Hq + 2 * Hkv) * d, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 4096, (A, T), generator=g) + base
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float32) / (rot // 2))
    gam = [(1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16) for _ in range(2)] if norm else [None, None]
    slots = (torch.randperm((nb - 1) * P, generator=g)[:T] + P)
    dt = FP8 if fp8 else torch.bfloat16
    k = torch.randn(nb, Hkv, P, d, generator=g).to(dt)
    v = torch.randn(nb, Hkv, P, d, generator=g).to(dt)
    sc = [torch.rand(Hkv, generator=g) * 0.02 + 0.003 for _ in range(2)] if fp8 else [None, None]
    return qkv, pos, inv, gam, slots, k, v, sc


def _near(got, want, size, fp8, scale, what):
    got, half_step = got.double(), 2.0 ** -4 if fp8 else 2.0 ** -8
    if fp8:
        s = scale.double().view(1, -1, 1)
        got = got * s
        want = want.clamp(-448 * s, 448 * s)
        # (the quotient's fp32 rounding is one more step of 2^-24)
        tol = want.abs() * (half_step + 2.0 ** -23) + size * E * (1 + half_step) + 2.0 ** -10 * s
    else:
        tol = want.abs() * half_step + size * E * (1 + half_step) + 2.0 ** -134
    off = (got - want).abs()
    assert bool((off <= tol).all()), f"{what}: off by {float((off - tol).max()):.3e} past the tolerance"


def _run(qkv, pos, inv, axes, Hq, Hkv, d, k, v, slots, gam, sc, **kw):
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    dk, dv = k.to(DEV), v.to(DEV)
    q = ops.qkv_norm_mrope_store(dev(qkv), positions=dev(pos), inv_freq=dev(inv), axes=axes, num_q_heads=Hq,
                                 num_kv_heads=Hkv, d_head=d, k_cache=dk, v_cache=dv, slot_mapping=dev(slots),
                                 q_norm=dev(gam[0]), k_norm=dev(gam[1]), k_scale=dev(sc[0]), v_scale=dev(sc[1]), **kw)
    return q.cpu(), dk.cpu(), dv.cpu()


CASES = [
    # T, Hq, Hkv, d, P, fp8, norm, sections, interleaved, base
    (1, 4, 1, 128, 16, False, True, (16, 24, 24), False, 0),
    (1, 16, 8, 128, 16, True, False, (24, 20, 20), True, 0),
    (7, 8, 2, 64, 16, False, True, (32,), False, 1000),
    (9, 24, 4, 64, 32, False, False, (8, 8), False, 10 ** 6),
    (33, 5, 1, 128, 7, True, True, (1, 30, 1), False, 0),
    (130, 32, 8, 128, 16, True, True, (16, 24, 24), False, 2 ** 24),
    (65, 3, 3, 64, 16, True, False, (8, 4, 2, 2), False, -2000),
    (40, 6, 2, 128, 64, False, True, (2, 3, 3), False, 2 ** 31),
]


@pytest.mark.parametrize("T,Hq,Hkv,d,P,fp8,norm,sections,interleaved,base", CASES)
def test_writer(T, Hq, Hkv, d, P, fp8, norm, sections, interleaved, base):
    announce(f"mrope T={T} {Hq}/{Hkv} d={d} {sections}")
    rot = 2 * sum(sections)
    axes = ops.mrope_axes(sections, interleaved)
    qkv, pos, inv, gam, slots, k, v, sc = _make(T + Hq, T, Hq, Hkv, d, P, fp8, norm, rot, len(sections), base)
    q, kc, vc = _run(qkv, pos, inv, axes, Hq, Hkv, d, k, v, slots, gam, sc)
    wq, wk, wv, size = ow.mrope_rows(qkv, pos, inv, axes, Hq, Hkv, d, gam[0], gam[1], 1e-6)
    _near(q, wq, size[:, :Hq], False, None, "q")
    page, off = slots // P, slots % P
    _near(kc.float()[page, :, off], wk, size[:, Hq:], fp8, sc[0], "k")
    if fp8:
        want = (wv.float() / sc[1].view(1, -1, 1)).clamp(-448, 448).to(FP8)  # one correctly rounded division
        assert torch.equal(vc.view(torch.uint8)[page, :, off], want.view(torch.uint8))
    else:
        assert torch.equal(vc[page, :, off], wv.to(torch.bfloat16))
    raw = (lambda t: t.view(torch.uint8)) if fp8 else (lambda t: t.view(torch.int16))
    untouched = torch.ones(k.shape[0], P, dtype=torch.bool)
    untouched[page, off] = False
    for a, b in ((kc, k), (vc, v)):
        assert torch.equal(raw(a).transpose(1, 2)[untouched], raw(b).transpose(1, 2)[untouched])


def test_one_axis_in_every_section_is_plain_rope():
    """Equal axes give the same bits whatever the sections, and the rotation of the one-axis writer within its roundings."""
    T, Hq, Hkv, d, P = 50, 4, 2, 128, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(3, T, Hq, Hkv, d, P, False, True, 128, 1, 500)
    p3 = pos.expand(3, T)
    a = _run(qkv, p3, inv, ops.mrope_axes([16, 24, 24]), Hq, Hkv, d, k, v, slots, gam, sc)
    b = _run(qkv, pos, inv, [0] * 64, Hq, Hkv, d, k, v, slots, gam, sc)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    angle = pos[0].double()[:, None] * inv.double()
    cos, sin = (f(torch.cat([angle, angle], 1)).to(torch.bfloat16).to(DEV) for f in (torch.cos, torch.sin))
    dk, dv = k.to(DEV), v.to(DEV)
    q = ops.qkv_norm_rope_store(qkv.to(DEV), cos=cos, sin=sin, num_q_heads=Hq, num_kv_heads=Hkv, d_head=d, k_cache=dk,
                                v_cache=dv, slot_mapping=slots.to(DEV), q_norm=gam[0].to(DEV), k_norm=gam[1].to(DEV))
    _, _, _, size = ow.mrope_rows(qkv, pos, inv, [0] * 64, Hq, Hkv, d, gam[0], gam[1], 1e-6)
    # that writer's bf16 roundings: two of the norm, one of cos / sin, two of the products and their sum, and this one's
    assert bool(((q.cpu().double() - a[0].double()).abs() <= size[:, :Hq] * 7 * 2.0 ** -8).all())
    assert torch.equal(dv.cpu(), a[2])


def test_strides_slots_and_nan():
    T, Hq, Hkv, d, P = 20, 4, 2, 64, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(5, T, Hq, Hkv, d, P, True, False, 64, 2, 0)
    axes = ops.mrope_axes([16, 16])
    slots[3], slots[4] = -1, 10 ** 9  # both to slot 0, the reserved page's
    k.view(torch.uint8)[0], v.view(torch.uint8)[0] = 0, 0
    qkv[7, Hq * d + 5] = float("nan")          # K head 0, a rotated pair
    qkv[8, (Hq + Hkv) * d + 1] = float("nan")  # V head 0
    wide = torch.zeros(T, qkv.shape[1] + 24, dtype=torch.bfloat16, device=DEV)
    wide[:, :qkv.shape[1]] = qkv.to(DEV)
    wpos = torch.zeros(2, T + 9, dtype=torch.int64, device=DEV)
    wpos[:, :T] = pos.to(DEV)
    q, kc, vc = _run(wide[:, :qkv.shape[1]], wpos[:, :T], inv, axes, Hq, Hkv, d, k, v, slots, gam, sc)
    q2, kc2, vc2 = _run(qkv, pos.to(torch.int32), inv, axes, Hq, Hkv, d, k, v, slots, gam, sc)
    keep = torch.tensor([t for t in range(T) if t not in (3, 4)])
    assert torch.equal(q, q2)
    assert torch.equal(kc.view(torch.uint8)[1:], kc2.view(torch.uint8)[1:])
    assert torch.equal(vc.view(torch.uint8)[1:], vc2.view(torch.uint8)[1:])
    page, off = slots[keep] // P, slots[keep] % P
    nan = kc.float()[page, :, off].isnan()
    want = torch.zeros_like(nan)
    want[keep.tolist().index(7), 0, 5] = want[keep.tolist().index(7), 0, 37] = True
    assert torch.equal(nan, want)
    assert int(vc.float()[page, :, off].isnan().sum()) == 1
    assert bool((kc.view(torch.uint8)[0, :, 1:] == 0).all())  # only slot 0 of the reserved page is written


@pytest.mark.parametrize("fp8", [False, True])
def test_cache_offsets_past_32_bits(fp8):
    """Slots far behind 4 GiB of a pool receive what the first ones do."""
    T, Hq, Hkv, d, P = 40, 8, 4, 128, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(11, T, Hq, Hkv, d, P, fp8, True, 128, 3, 77)
    axes = ops.mrope_axes([16, 24, 24])
    q, kc, vc = _run(qkv, pos, inv, axes, Hq, Hkv, d, k, v, slots, gam, sc)
    far = (2 ** 32 + 2 ** 30) // (k[0].numel() * k.element_size())
    big = [torch.zeros(far + len(k), Hkv, P, d, dtype=torch.uint8 if fp8 else torch.int16, device=DEV).view(k.dtype)
           for _ in range(2)]
    raw = lambda t: t.view(torch.uint8 if fp8 else torch.int16)  # noqa: E731
    for b, t in zip(big, (k, v)):
        raw(b)[far:] = raw(t).to(DEV)
    got = ops.qkv_norm_mrope_store(
        qkv.to(DEV), positions=pos.to(DEV), inv_freq=inv.to(DEV), axes=axes, num_q_heads=Hq, num_kv_heads=Hkv, d_head=d,
        k_cache=big[0], v_cache=big[1], slot_mapping=(slots + far * P).to(DEV), q_norm=gam[0].to(DEV),
        k_norm=gam[1].to(DEV), k_scale=sc[0].to(DEV) if fp8 else None, v_scale=sc[1].to(DEV) if fp8 else None)
    assert torch.equal(got.cpu(), q)
    assert torch.equal(raw(big[0])[far:].cpu(), raw(kc)) and torch.equal(raw(big[1])[far:].cpu(), raw(vc))
    assert not bool(raw(big[0])[:far].any())


@pytest.mark.parametrize("fp8", [False, True])
def test_an_image_prompt_written_weighed_thinned_and_read(fp8):
    """A prompt of text, an image's patches and text goes in by the writer, its keys are weighed by its last queries, the
    cache is thinned in place, and the next token is written behind it at the position that follows the prompt's: its
    attention and weights equal, bit for bit, those over a fresh cache that holds the kept rows alone."""
    Hq, G, d, P, keep, scale = 8, 2, 128, 16, 70, 128 ** -0.5
    lens = [300, 41]
    R, T = len(lens), sum(lens)
    g = torch.Generator().manual_seed(21)
    rows = torch.randn(T + R, (Hq + 2 * G) * d, generator=g).to(torch.bfloat16).to(DEV)
    inv = (10000.0 ** (-torch.arange(64) / 64)).float().to(DEV)
    axes = ops.mrope_axes([16, 24, 24])
    gam = [torch.rand(d, generator=g).add(0.5).to(torch.bfloat16).to(DEV) for _ in range(2)]
    pos, after = [], []
    for n in lens:
        text, side = n // 4, 5
        patches = n // 2
        p = torch.stack([torch.arange(n)] * 3)
        at = torch.arange(patches)
        p[:, text:text + patches] = text + torch.stack([at * 0, at // side, at % side])
        p[:, text + patches:] = int(p[:, :text + patches].max()) + 1 + torch.arange(n - text - patches)
        pos.append(p)
        after.append(p[:, -1:] + 1)
    pos, after = torch.cat(pos, 1).to(DEV), torch.cat(after, 1).to(DEV)
    pages = [-(-(n + 1) // P) for n in lens]
    nb = 1 + sum(pages)
    perm = (torch.randperm(nb - 1, generator=g) + 1).tolist()
    table = torch.full((R, max(pages)), -1, dtype=torch.int32)
    for r, n in enumerate(pages):
        table[r, :n] = torch.tensor([perm.pop() for _ in range(n)])
    table = table.to(DEV)
    slot = lambda r, i: table[r, i // P].long() * P + i % P  # noqa: E731
    slots = torch.cat([slot(r, torch.arange(n, device=DEV)) for r, n in enumerate(lens)])
    cache = [torch.zeros(nb, G, P, d, dtype=FP8 if fp8 else torch.bfloat16, device=DEV) for _ in range(2)]
    sc = [torch.full((G,), 0.02, device=DEV) if fp8 else None for _ in range(2)]

    def write(x, at, where, kc, vc):
        return ops.qkv_norm_mrope_store(x, positions=at, inv_freq=inv, axes=axes, num_q_heads=Hq, num_kv_heads=G, d_head=d,
                                        k_cache=kc, v_cache=vc, slot_mapping=where, q_norm=gam[0], k_norm=gam[1],
                                        k_scale=sc[0], v_scale=sc[1])

    q = write(rows[:T], pos, slots, *cache)
    whole = [c.clone() for c in cache]
    last = torch.cat([torch.arange(n - 16, n) + sum(lens[:r]) for r, n in enumerate(lens)]).to(DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    w = ops.prefill_attention_weights(q[last], cache[0], table, i32([0, 16, 32]), i32([n - 16 for n in lens]), max_q_len=16,
                                      sm_scale=scale, k_scale=sc[0])
    # without sinks every query's probabilities sum to 1: fp32 sums of at most 300 keys and 64 rows of scores whose products
    # add up to at most scale * (1.5 * sqrt(d))^2 < 26 (normed rows times gammas under 1.5)
    total = w.double().sum(-1)
    assert bool(((total - 16 * Hq // G).abs() <= 16 * Hq // G * (2 * (d + 8) * 26 + 400) * 2.0 ** -24).all())
    kept, new = ops.evict_tokens(*cache, table, i32(lens), w, keep=keep, first=4, recent=16, weights_out=w)
    assert new.tolist() == [70, 41]
    fresh = [torch.zeros_like(c) for c in cache]
    raw = lambda t: t.view(torch.uint8 if fp8 else torch.int16)  # noqa: E731
    for r in range(R):
        n = int(new[r])
        to = slot(r, torch.arange(n, device=DEV))
        for h in range(G):
            src = slot(r, kept[r, h, :n].long())
            for a, b in zip(fresh, whole):
                raw(a)[to // P, h, to % P] = raw(b)[src // P, h, src % P]
    step = torch.stack([slot(r, new[r]) for r in range(R)])
    outs = []
    for kc, vc in (cache, fresh):
        sq = write(rows[T:], after, step, kc, vc)
        k, v = (raw(c)[step // P, :, step % P].view(c.dtype) for c in (kc, vc))
        at = ops.decode_attention_weights(sq, kc, table, new + 1, sm_scale=scale, k_scale=sc[0])
        out = ops.prefill_attention(sq, kc, vc, table, i32([0, 1, 2]), new, max_q_len=1, sm_scale=scale, k_scale=sc[0],
                                    v_scale=sc[1])
        outs.append((sq, raw(k), raw(v), at, out))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert bool((outs[0][3][0, :, :71] > 0).all()) and bool((outs[0][3][0, :, 71:] == 0).all())


def test_refusals_and_empty():
    T, Hq, Hkv, d, P = 4, 2, 1, 64, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(7, T, Hq, Hkv, d, P, True, False, 64, 2, 0)
    axes = ops.mrope_axes([16, 16])
    bad = [dict(axes=axes[:-1]), dict(axes=[2] * 32), dict(pos=pos[:, :3]), dict(sc=[None, sc[1]]),
           dict(slots=slots[:2]), dict(inv=inv[:4], axes=[0] * 4), dict(gam=[torch.ones(64).bfloat16(), None])]
    for kw in bad:
        a = dict(qkv=qkv, pos=pos, inv=inv, axes=axes, Hq=Hq, Hkv=Hkv, d=d, k=k, v=v, slots=slots, gam=gam, sc=sc) | kw
        with pytest.raises(ValueError):
            _run(**a)
    q, kc, vc = _run(qkv[:0], pos[:, :0], inv, axes, Hq, Hkv, d, k, v, slots[:0], gam, sc)
    assert q.shape == (0, Hq, d) and torch.equal(kc.view(torch.uint8), k.view(torch.uint8))


def test_graph_and_side_stream():
    T, Hq, Hkv, d, P = 37, 8, 2, 128, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(9, T, Hq, Hkv, d, P, True, True, 128, 3, 0)
    t = [x.to(DEV) for x in (qkv, pos, inv, gam[0], gam[1], slots, k, v, sc[0], sc[1])]
    axes = ops.mrope_axes([24, 20, 20], True)

    def run():
        return ops.qkv_norm_mrope_store(t[0], positions=t[1], inv_freq=t[2], axes=axes, num_q_heads=Hq, num_kv_heads=Hkv,
                                        d_head=d, k_cache=t[6], v_cache=t[7], slot_mapping=t[5], q_norm=t[3], k_norm=t[4],
                                        k_scale=t[8], v_scale=t[9])

    eager = [x.clone() for x in (run(), t[6].view(torch.uint8), t[7].view(torch.uint8))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(other, eager[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):
        out.zero_()
        t[6].view(torch.uint8)[slots.to(DEV) // P] = 0
        run()
        torch.cuda.synchronize()
        t[6].view(torch.uint8).copy_(eager[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, t[6].view(torch.uint8), t[7].view(torch.uint8)), eager))
