"""ops.kv_store_blocks against the definition: scales and bounds equal, codes equal bit for bit (quotients are correctly
rounded), nothing written elsewhere."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import blocks as ob
from sglang_neuron_amd import ops
from tests._block_cases import FMTS, garbage, gen, pool, same_bits, table_of, to, tokens
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(k, v, caches, scales, table, start, prior, bounds=None, max_q=None, slices=False):
    """One call on the GPU and the definition on the CPU, compared whole."""
    max_q = max([start[r + 1] - start[r] for r in range(len(prior))] + [1]) if max_q is None else max_q
    got = to(DEV, *caches, *scales, bounds)
    kd, vd = k.to(DEV), v.to(DEV)
    if slices:  # views of one projection's rows
        T, G, d = k.shape
        wide = torch.zeros(T, 3 * G * d + 8, dtype=torch.bfloat16, device=DEV)
        wide[:, 8:8 + G * d], wide[:, 8 + G * d:8 + 2 * G * d] = kd.reshape(T, -1), vd.reshape(T, -1)
        kd, vd = wide[:, 8:8 + G * d].view(T, G, d), wide[:, 8 + G * d:8 + 2 * G * d].view(T, G, d)
    single = all(start[r + 1] - start[r] == 1 for r in range(len(prior)))
    ops.kv_store_blocks(kd, vd, got[0], got[1], table.to(DEV), torch.tensor(prior, dtype=torch.int32, device=DEV),
                        q_start=None if single else torch.tensor(start, dtype=torch.int32, device=DEV), max_q_len=max_q,
                        k_scale=got[2], v_scale=got[3], k_bounds=got[4])
    for x, cache, scale, b in ((k, caches[0], scales[0], bounds), (v, caches[1], scales[1], None)):
        ob.append(cache, scale, x, table, start, prior, b, max_q)
    for name, a, b in zip(("k", "v", "k_scale", "v_scale", "bounds"), got, (*caches, *scales, bounds)):
        if b is None:
            continue
        if b.dtype == torch.float32:
            assert torch.equal(torch.nan_to_num(a.cpu(), nan=-1.0), torch.nan_to_num(b, nan=-1.0)), name
        else:
            a, b = a.cpu(), b
            if a.dtype == torch.bfloat16:
                a, b = a.view(torch.int16), b.view(torch.int16)
            assert same_bits(a, b), (name, int((a.view(torch.uint8) != b.view(torch.uint8)).sum()))
    return got


def _setup(seed, R, G, d, P, bt, fmt, priors, counts, extra=0, dirty=False):
    g = gen(seed)
    lens = [p + n for p, n in zip(priors, counts)]
    table, nb = table_of(g, lens, P, extra)
    kc, ks = pool(g, nb + 2, G, P, d, bt, fmt)
    vc, vs = pool(g, nb + 2, G, P, d, bt, fmt)
    start = [sum(counts[:r]) for r in range(R + 1)]
    k, v = (tokens(g, start[-1], G, d).to(torch.bfloat16) for _ in range(2))
    b = tokens(g, nb + 2, G, 3, d)
    bounds = torch.stack([b.amin(2), b.amax(2)], 2).to(torch.bfloat16)
    return k, v, (kc, vc), (ks, vs), table, start, bounds


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("G,d,P,bt", [(2, 128, 16, 16), (1, 64, 32, 16), (3, 64, 48, 48), (2, 128, 64, 32), (1, 128, 128, 128),
                                      (2, 64, 256, 64)])
def test_one_token_a_row(fmt, G, d, P, bt):
    """A decode step at every kind of place: a block's first token, a page's, a block's last, the first of all."""
    priors = [0, 1, 15, 16, P - 1, P, P + 5, 2 * P - 1, 3 * P]
    announce(f"store step {fmt} G={G} d={d} P={P} bt={bt}")
    k, v, caches, scales, table, start, bounds = _setup(P + d, len(priors), G, d, P, bt, fmt, priors, [1] * len(priors))
    _check(k, v, caches, scales, table, start, priors, bounds)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("G,d,P,bt", [(2, 128, 16, 16), (1, 64, 48, 16), (2, 128, 64, 64), (1, 64, 128, 32), (1, 128, 160, 80),
                                      (1, 128, 512, 256)])
@pytest.mark.parametrize("slices", [False, True])
def test_chunks(fmt, G, d, P, bt, slices):
    """Ragged chunks, an empty one among them, that start and end anywhere in a block."""
    priors, counts = [0, 5, 2 * P + 17, 31, P], [3 * P + 7, 1, 200, 0, P]
    announce(f"store chunks {fmt} G={G} d={d} P={P} bt={bt} slices={slices}")
    k, v, caches, scales, table, start, bounds = _setup(P + bt, 5, G, d, P, bt, fmt, priors, counts, extra=2)
    _check(k, v, caches, scales, table, start, priors, bounds if slices else None, slices=slices)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_one_long_chunk_among_many_tokens(fmt):
    """The pages there are, counted out among 150 requests (some without tokens) instead of given to each."""
    announce(f"store mixed {fmt}")
    R, P = 150, 16
    priors = [(7 * r) % 50 for r in range(R)]
    counts = [0 if r % 13 == 5 else 1 for r in range(R)]
    counts[70], counts[149] = 700, 33
    k, v, caches, scales, table, start, bounds = _setup(41, R, 2, 64, P, 16, fmt, priors, counts)
    _check(k, v, caches, scales, table, start, priors, bounds)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_token_by_token_is_the_block_grown(fmt):
    """40 tokens one at a time, on a pool that held garbage: the scale only grows and every step's codes are as defined."""
    announce(f"store token by token {fmt}")
    G, d, P, bt = 2, 64, 32, 16
    g = gen(5)
    caches = [torch.empty(4, G, P, d, dtype=FMTS[fmt]) for _ in range(2)]
    scales = [torch.empty(4, G, P // bt) for _ in range(2)]
    for c, s in zip(caches, scales):
        garbage(c, s)
    bounds = torch.full((4, G, 2, d), float("nan"), dtype=torch.bfloat16)
    table = torch.tensor([[2, 1]], dtype=torch.int32)
    for i in range(40):
        k, v = (tokens(g, 1, G, d).to(torch.bfloat16) for _ in range(2))
        _check(k, v, caches, scales, table, [0, 1], [i], bounds)
    assert bool(torch.isfinite(scales[0][2]).all()) and bool(torch.isnan(scales[0][3]).all())


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_special_elements(fmt):
    """Zeros, subnormals, the largest bf16 values, infinities and NaN."""
    announce(f"store specials {fmt}")
    G, d, P, bt = 1, 64, 32, 16
    kinds = [0.0, -0.0, 1e-40, 2.0 ** -126, -2.0 ** -110, 1.0, -3.3895e38, 3.3895e38, math.inf, -math.inf, math.nan]
    for seed, pick in enumerate([kinds[:2], kinds[:3], kinds[:5], kinds[:8], kinds[:10], kinds]):
        g = gen(seed)
        caches, scales = [], []
        for _ in range(2):
            c, s = pool(g, 5, G, P, d, bt, fmt)
            caches.append(c)
            scales.append(s)
        x = torch.tensor(pick)[torch.randint(len(pick), (40, G, d), generator=g)].to(torch.bfloat16)
        finite = torch.where(x.isnan(), torch.zeros_like(x), x)
        bounds = torch.zeros(5, G, 2, d, dtype=torch.bfloat16)
        got = to(DEV, *caches, *scales, bounds)
        table = torch.tensor([[3, 1, 4]], dtype=torch.int32)
        ops.kv_store_blocks(x.to(DEV), finite.to(DEV), got[0], got[1], table.to(DEV),
                            torch.tensor([7], dtype=torch.int32, device=DEV),
                            q_start=torch.tensor([0, 40], dtype=torch.int32, device=DEV), max_q_len=40, k_scale=got[2],
                            v_scale=got[3], k_bounds=got[4])
        ob.append(caches[0], scales[0], x, table, [0, 40], [7], bounds)
        ob.append(caches[1], scales[1], finite, table, [0, 40], [7])
        for i in range(2):
            assert torch.equal(torch.nan_to_num(got[2 + i].cpu(), nan=-1.0), torch.nan_to_num(scales[i], nan=-1.0))
            # (the codes of a block whose scale is NaN may be anything)
            ok = ~scales[i].isnan().repeat_interleave(bt, 2)
            a, b = got[i].cpu().float()[ok], caches[i].float()[ok]
            assert torch.equal(a, b), int((a != b).sum())
        assert torch.equal(got[4].cpu().float() + 0.0, bounds.float() + 0.0)


@pytest.mark.parametrize("bt", [16, 64, 128])  # a wave, two and four waves a block
@pytest.mark.parametrize("had", [math.nan, math.inf])
def test_no_code_is_nan_behind_a_scale_that_is_no_number(bt, had):
    """Finite tokens behind a block whose scale is NaN (a NaN token before them) or infinite: the scale stays, and their e4m3fn
    codes are numbers, so that a product with a probability of 0 is 0."""
    announce(f"store behind a scale of {had} bt={bt}")
    G, d, P = 2, 128, 128
    g = gen(bt)
    caches = [torch.zeros(3, G, P, d, dtype=FMTS["fp8"], device=DEV) for _ in range(2)]
    scales = [torch.full((3, G, P // bt), had, device=DEV) for _ in range(2)]
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=DEV)
    at = 5
    for n in (1, 9, 120):
        k, v = (tokens(g, n, G, d).to(torch.bfloat16).to(DEV) for _ in range(2))
        ops.kv_store_blocks(k, v, *caches, table, torch.tensor([at], dtype=torch.int32, device=DEV),
                            q_start=torch.tensor([0, n], dtype=torch.int32, device=DEV), max_q_len=n, k_scale=scales[0],
                            v_scale=scales[1])
        at += n
        for c, s in zip(caches, scales):
            assert bool(((c.view(torch.uint8) & 0x7F) != 0x7F).all()), n
            assert bool((s[1, :, 0].isnan() if math.isnan(had) else s[1, :, 0].isinf()).all())


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_tokens_without_a_page_are_not_stored(fmt):
    """Entries outside the pool, columns past the table, chunks longer than max_q_len, a negative position."""
    announce(f"store no page {fmt}")
    G, d, P, bt = 1, 64, 16, 16
    k, v, caches, scales, table, start, bounds = _setup(3, 4, G, d, P, bt, fmt, [3, 20, 0, 0], [50, 10, 40, 9])
    table[0, 1], table[1, 1], table[2, 0] = -1, 10 ** 6, -7
    table = table[:, :3].contiguous()
    got = _check(k, v, caches, scales, table, start, [3, 20, 0, 0], bounds, max_q=30)
    before = [None if t is None else t.clone() for t in got]
    ops.kv_store_blocks(k[:1].to(DEV), v[:1].to(DEV), got[0], got[1], table[:1].to(DEV),
                        torch.tensor([-1], dtype=torch.int32, device=DEV), k_scale=got[2], v_scale=got[3], k_bounds=got[4])
    for a, b in zip(got, before):
        assert a is None or same_bits(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_the_same_call_again_changes_nothing():
    announce("store twice")
    k, v, caches, scales, table, start, bounds = _setup(9, 2, 2, 128, 64, 16, "int8", [37, 5], [100, 70])
    once = _check(k, v, caches, scales, table, start, [37, 5], bounds)
    for _ in range(2):
        again = _check(k, v, caches, scales, table, start, [37, 5], bounds)
        for a, b in zip(once, again):
            assert torch.equal(a, b)
