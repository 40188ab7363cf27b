"""The definitions of oracle.blocks by hand and by closed forms. CPU only."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import blocks as ob
from tests._block_cases import gen, pool, table_of


def _one(values, d=4):
    """[n, 1, d] bf16 tokens whose elements are 0 but for the first."""
    x = torch.zeros(len(values), 1, d)
    x[:, 0, 0] = torch.tensor(values)
    return x.to(torch.bfloat16)


def test_a_block_starts_grows_and_starts_anew():
    cache, scale = torch.full((3, 1, 32, 4), 99, dtype=torch.int8), torch.full((3, 1, 2), math.nan)
    table = torch.tensor([[2, 1]])
    ob.append(cache, scale, _one([127.0, -63.0]), table, [0, 2], [0])
    assert scale[2, 0, 0] == 1 and cache[2, 0, :3, 0].tolist() == [127, -63, 99] and bool(scale[2, 0, 1].isnan())
    ob.append(cache, scale, _one([10.0]), table, [0, 1], [2])  # smaller: the scale stays
    assert scale[2, 0, 0] == 1 and cache[2, 0, :3, 0].tolist() == [127, -63, 10]
    ob.append(cache, scale, _one([254.0]), table, [0, 1], [3])  # twice: earlier tokens at half their codes, ties to even
    assert scale[2, 0, 0] == 2 and cache[2, 0, :5, 0].tolist() == [64, -32, 5, 127, 99]
    ob.append(cache, scale, _one([1.0]), table, [0, 1], [0])  # its first token again: anew
    assert float(scale[2, 0, 0]) == pytest.approx(1 / 127) and cache[2, 0, 0, 0] == 127
    ob.append(cache, scale, torch.zeros(20, 1, 4, dtype=torch.bfloat16), table, [0, 20], [16])  # zeros, over a page's end
    assert scale[2, 0, 1] == 2.0 ** -100 == scale[1, 0, 0] and bool((cache[2, 0, 16:] == 0).all())
    assert bool((cache[0] == 99).all()) and bool((cache[1, 0, 4:] == 99).all())


def test_special_elements_of_a_block():
    for dtype, top in ((torch.int8, 127.0), (ob.FP8, 448.0)):
        cache, scale = torch.zeros(2, 1, 16, 4).to(dtype), torch.zeros(2, 1, 1)
        ob.append(cache, scale, _one([math.inf, -2.0, -math.inf]), torch.tensor([[1]]), [0, 3], [0])
        assert float(scale[1, 0, 0]) == pytest.approx(2 / top)
        assert cache[1, 0, :3, 0].float().tolist() == [top, -top, -top]
        ob.append(cache, scale, _one([math.nan]), torch.tensor([[1]]), [0, 1], [3])
        assert bool(scale[1].isnan().all())
        ob.append(cache, scale, _one([1.0]), torch.tensor([[1]]), [0, 1], [4])
        assert bool(scale[1].isnan().all())


def test_bounds_hold_every_key():
    g = gen(1)
    bounds = torch.full((4, 2, 2, 8), math.nan, dtype=torch.bfloat16)
    cache = torch.zeros(4, 2, 16, 8, dtype=torch.bfloat16)
    table, at = torch.tensor([[3, 1]]), 0
    keys = torch.randn(30, 2, 8, generator=g).to(torch.bfloat16)
    for n in (1, 4, 13, 12):
        ob.append(cache, None, keys[at:at + n], table, [0, n], [at], bounds)
        at += n
    assert torch.equal(cache[3], keys[:16].transpose(0, 1)) and torch.equal(cache[1, :, :14], keys[16:].transpose(0, 1))
    for page, part in ((3, keys[:16]), (1, keys[16:])):
        assert torch.equal(bounds[page, :, 0], part.amin(0)) and torch.equal(bounds[page, :, 1], part.amax(0))
    # no key scores more than its page
    q = torch.randn(1, 4, 8, generator=g).to(torch.bfloat16)
    s, size, counts = ob.scores(q, bounds, table, [30], 16)
    assert counts == [2] and bool((s.abs() <= size).all())
    for c, part in enumerate((keys[:16], keys[16:])):
        for h in range(4):
            assert bool(((part[:, h // 2].double() @ q[0, h].double()) <= s[0, h // 2, c]).all())
    s, _, counts = ob.scores(q, bounds, table, [16], 16)
    assert counts == [1] and s[0, 0, 1] == -math.inf
    assert ob.scores(q, bounds, table, [0], 16)[2] == [0]


@pytest.mark.parametrize("dtype", [ob.FP8, torch.int8])
def test_cached_keys_pass_their_bounds_by_their_roundings(dtype):
    """Scores bound the keys as given. A cached key passes its page's by no more than its codes' roundings, one for each scale
    that its block has had (their halves of a step: 2^-4 of the element or 2^-10 of the scale, half a scale), and some do."""
    g = gen(4)
    for seed in range(20):
        cache, scale = torch.zeros(2, 1, 16, 8).to(dtype), torch.zeros(2, 1, 1)
        bounds, table = torch.zeros(2, 1, 2, 8, dtype=torch.bfloat16), torch.tensor([[1]])
        keys = (torch.randn(16, 1, 8, generator=g) * torch.linspace(1, 1 + seed / 4, 16).view(16, 1, 1)).to(torch.bfloat16)
        slack = torch.zeros(16, 8, dtype=torch.float64)
        for at in range(16):
            had = float(scale[1])
            ob.append(cache, scale, keys[at:at + 1], table, [0, 1], [at], bounds)
            s = float(scale[1])
            x = keys[:at + 1, 0].double().abs() + slack[:at + 1]
            half = torch.maximum(x * 2.0 ** -4, torch.tensor(s * 2.0 ** -10)) if dtype == ob.FP8 else torch.full_like(x, s / 2)
            slack[:at] += half[:at] if s > had else 0.0
            slack[at] = half[at]
        q = torch.randn(1, 1, 8, generator=g).to(torch.bfloat16)
        score = ob.scores(q, bounds, table, [16], 16)[0][0, 0, 0]
        got = (cache[1, 0].double() * float(scale[1])) @ q[0, 0].double()
        assert bool(((keys[:, 0].double() @ q[0, 0].double()) <= score).all())
        assert bool((got <= score + (1 + 2.0 ** -20) * (slack @ q[0, 0].double().abs())).all())
    # the one key of a page passes its score by the rounding of its second element, for a query of that or the other sign
    cache, scale = torch.zeros(2, 1, 16, 8).to(dtype), torch.zeros(2, 1, 1)
    bounds = torch.zeros(2, 1, 2, 8, dtype=torch.bfloat16)
    key = torch.zeros(1, 1, 8, dtype=torch.bfloat16)
    key[0, 0, 0], key[0, 0, 1] = 100.0, 1.2
    ob.append(cache, scale, key, torch.tensor([[1]]), [0, 1], [0], bounds)
    q = torch.zeros(2, 1, 8, dtype=torch.bfloat16)
    q[0, 0, 1], q[1, 0, 1] = 1.0, -1.0
    score = ob.scores(q, bounds, torch.tensor([[1], [1]]), [1, 1], 16)[0][:, 0, 0]
    got = q[:, 0].double() @ (cache[1, 0, 0].double() * float(scale[1]))
    assert int((got > score).sum()) == 1


def test_scores_of_infinite_bounds():
    """A bound that a query element does not take, or takes times 0, does not count; one that counts makes the score infinite."""
    inf = math.inf
    # of two dimensions: (lo, hi) of each page
    pages = [([-inf, -1.0], [2.0, 3.0]), ([-1.0, -1.0], [inf, 3.0]), ([inf, -1.0], [-inf, 3.0]), ([-inf, -1.0], [-inf, 3.0])]
    bounds = torch.tensor([[lo, hi] for lo, hi in pages]).to(torch.bfloat16).view(4, 1, 2, 2)
    table = torch.arange(4).view(1, 4)
    for q, want in (([1.0, 1.0], [5.0, inf, inf, -inf]), ([-1.0, 1.0], [inf, 4.0, inf, inf]), ([0.0, -2.0], [2.0] * 4)):
        s, _, _ = ob.scores(torch.tensor(q, dtype=torch.bfloat16).view(1, 1, 2), bounds, table, [64], 16)
        assert s.reshape(-1).tolist() == want
    # infinities of both signs are no number: the head counts only where it is alone
    bounds = torch.tensor([[-inf, 1.0], [-inf, inf]]).to(torch.bfloat16).view(1, 1, 2, 2)
    q = torch.tensor([[1.0, 1.0], [0.0, -2.0]], dtype=torch.bfloat16).view(1, 2, 2)
    assert ob.scores(q, bounds, table[:, :1], [16], 16)[0].item() == -2.0
    assert ob.scores(q[:, :1], bounds, table[:, :1], [16], 16)[0].isnan().all()


def test_int8_query_rounding():
    """The whole numbers that a prompt's queries become over int8 codes, step by step in fp32: every bf16 element up to 4 octaves
    below every largest one of an octave. The stated bound holds, and 2^-16 would not."""
    top = (1 + torch.arange(128) / 128.0).to(torch.float32)
    x = torch.cat([top * 2.0 ** -e for e in range(5)])
    worst = 0.0
    for amp in top:
        v = x[x <= amp]
        n = torch.round(v * (torch.tensor(32600.0) / amp))
        assert float(n.max()) == 32600
        value = n.double() * (amp / torch.tensor(32600.0)).double()
        worst = max(worst, float(((value - v.double()).abs() / amp.double()).max()))
    assert 2.0 ** -16 < worst <= ob.INT8_QUERY_OFF < 1.56e-5


def test_attention_of_equal_keys():
    G, d, P = 1, 8, 16
    table = torch.tensor([[2, 1]])
    v = torch.randn(3, G, P, d, generator=gen(2)).to(torch.bfloat16)
    k = torch.ones(3, G, P, d).to(torch.bfloat16)
    q = torch.randn(1, 2, d, generator=gen(3)).to(torch.bfloat16)
    rows = torch.cat([v[2, 0], v[1, 0]]).double()
    out, off = ob.decode(q, k, v, table, [20], sm_scale=0.5)
    assert torch.allclose(out[0], rows[:20].mean(0).expand(2, d)) and bool((off > 0).all())
    assert torch.allclose(ob.decode(q, k, v, table, [20], sm_scale=0.5, window=7)[0][0], rows[13:20].mean(0).expand(2, d))
    # a sink as heavy as one key; one without end; none
    z = float(q[0, 0].double().sum()) * 0.5
    out, _ = ob.decode(q, k, v, table, [20], sm_scale=0.5, sinks=torch.tensor([z, -math.inf]))
    assert torch.allclose(out[0, 0], rows[:20].sum(0) / 21, rtol=1e-6) and torch.allclose(out[0, 1], rows[:20].mean(0))
    # lists: one page, none, out of the table; a row out of the table; scales
    lists = torch.tensor([[[1, -1, 7]]])
    assert torch.allclose(ob.decode(q, k, v, table, [20], sm_scale=0.5, blocks=lists)[0][0], rows[16:20].mean(0).expand(2, d))
    assert bool((ob.decode(q, k, v, table, [20], sm_scale=0.5, blocks=torch.full((1, 1, 2), -1))[0] == 0).all())
    assert bool((ob.decode(q, k, v, table, [20], sm_scale=0.5, rows=[1])[0] == 0).all())
    vs = torch.tensor([1.0, 2.0, 4.0]).view(3, 1, 1)
    out, _ = ob.decode(q, k, v, table, [32], sm_scale=0.5, k_scale=torch.ones(3, 1, 1), v_scale=vs)
    assert torch.allclose(out[0, 0], (4 * rows[:16].sum(0) + 2 * rows[16:].sum(0)) / 32)


def test_a_chunk_is_its_tokens():
    g = gen(4)
    table, nb = table_of(g, [40, 9], 16)
    k, ks = pool(g, nb, 2, 16, 8, 16, "int8")
    v, vs = pool(g, nb, 2, 16, 8, 16, "int8")
    q = torch.randn(12, 4, 8, generator=g).to(torch.bfloat16)
    kw = dict(sm_scale=0.3, k_scale=ks, v_scale=vs, window=11)
    out, _ = ob.prefill(q, k, v, table, [0, 10, 12], [30, 7], **kw)
    one, _ = ob.decode(q[[3]], k, v, table, [34], rows=[0], **kw)
    assert torch.equal(out[3], one[0])
    one, _ = ob.decode(q[[11]], k, v, table, [9], rows=[1], **kw)
    assert torch.equal(out[11], one[0])
