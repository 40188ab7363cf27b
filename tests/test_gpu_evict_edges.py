"""ops.select_tokens and ops.evict_tokens in place on buffers wider or narrower than the weights, and into views that share
a buffer with them without sharing an element."""

from __future__ import annotations

import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(seed, *shape):
    return torch.exp(2.5 * torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) - 4)


def _want(w, lens, keep, first, recent):
    kept, new = ow.select_tokens(w, lens, keep, first, recent)
    return kept, new, torch.where(kept >= 0, torch.gather(w, 2, kept.clamp(min=0).long()), 0.0)


@pytest.mark.parametrize("R,G", [(1, 1), (1, 3), (3, 1), (2, 2)])
@pytest.mark.parametrize("N,M,keep", [(200, 300, 60), (200, 80, 60), (17000, 18000, 700), (17000, 900, 700)])
def test_in_place_on_another_width(R, G, N, M, keep):
    """The weights of the present length are the front of a wider buffer, which is thinned in place, or only its front is."""
    announce(f"in place R={R} G={G} {N} of {M}")
    buf = torch.full((R, G, max(N, M)), 5.0, device=DEV)
    w = _weights(N + G, R, G, N)
    buf[..., :N] = w.to(DEV)
    lens = [N, N // 2, keep - 1][:R]
    want, new, carried = _want(w, lens, keep, 4, 8)
    kept, got = ops.select_tokens(buf[..., :N], torch.tensor(lens, device=DEV), keep=keep, first=4, recent=8,
                                  weights_out=buf[..., :M])
    assert torch.equal(kept.cpu(), want) and got.tolist() == new
    assert torch.equal(buf[..., :keep].cpu(), carried) and bool((buf[..., keep:M] == 0).all())
    assert torch.equal(buf[..., M:N].cpu(), w[..., M:])


def test_a_batch_that_shrinks_to_one_row_is_thinned_in_place():
    P, G, d, n, keep = 16, 2, 64, 100, 40
    table = torch.arange(1, 8, dtype=torch.int32, device=DEV)[None]
    cache = [torch.randn(8, G, P, d, device=DEV).to(torch.bfloat16) for _ in range(2)]
    was = [c.clone() for c in cache]
    buf = torch.zeros(1, G, 7 * P, device=DEV)
    w = _weights(5, 1, G, n)
    buf[..., :n] = w.to(DEV)
    want, _, carried = _want(w, [n], keep, 2, 5)
    kept, new = ops.evict_tokens(*cache, table, torch.tensor([n], device=DEV), buf[..., :n], keep=keep, first=2, recent=5,
                                 weights_out=buf)
    assert torch.equal(kept.cpu(), want) and new.tolist() == [keep]
    assert torch.equal(buf[..., :keep].cpu(), carried) and bool((buf[..., keep:] == 0).all())
    for c, b in zip(cache, was):
        for g in range(G):
            rows = b[1:, g].reshape(-1, d)
            assert torch.equal(c[1:, g].reshape(-1, d)[:keep], rows[kept[0, g].long()])


@pytest.mark.parametrize("N,keep", [(150, 40), (16500, 300)])
def test_views_of_one_buffer_that_share_no_element(N, keep):
    announce(f"disjoint views {N}")
    R, G = 3, 2
    w = _weights(N, R, G, N)
    lens = [N, N - 7, keep - 1]
    want, _, carried = _want(w, lens, keep, 1, 2)
    dl = torch.tensor(lens, device=DEV)
    for shape, src, dst in (((R, G, 2 * N), lambda b: b[..., :N], lambda b: b[..., N:]),
                            ((R, G, 2 * N), lambda b: b[..., N:], lambda b: b[..., :N]),
                            ((2 * R, G, N), lambda b: b[::2], lambda b: b[1::2]),
                            ((R, 2 * G, N), lambda b: b[:, :G], lambda b: b[:, G:]),
                            ((G, R, 2 * N), lambda b: b[..., :N].transpose(0, 1), lambda b: b[..., N:].transpose(0, 1))):
        buf = torch.full(shape, 9.0, device=DEV)
        src(buf).copy_(w)
        kept, _ = ops.select_tokens(src(buf), dl, keep=keep, first=1, recent=2, weights_out=dst(buf))
        assert torch.equal(kept.cpu(), want) and torch.equal(src(buf).cpu(), w)
        assert torch.equal(dst(buf)[..., :keep].cpu(), carried) and bool((dst(buf)[..., keep:] == 0).all())
    buf = torch.zeros(R, G, 2 * N, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.select_tokens(buf[..., :N], dl, keep=keep, weights_out=buf[..., N - 1:2 * N - 1])
