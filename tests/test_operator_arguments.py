"""How the tensor-level entry points read their arguments, before any launch. CPU only."""

from __future__ import annotations

import array
import random

import numpy as np
import pytest
import torch

from sglang_neuron_amd import _lib, ops


@pytest.mark.parametrize("R,N", [(1, 1), (1, 5), (3, 1), (3, 5), (2, 0), (0, 4)])
def test_strided_rows_stay_inside_their_tensor(R, N):
    wide = torch.arange(R * (N + 4) + 64, dtype=torch.int32)
    views = [wide[:R * N].view(R, N), wide.as_strided((R, N), (N + 4, 1), 2), wide.as_strided((R, N), (0, 1), 7),
             wide.as_strided((R, N), (1, 1), 3), wide.as_strided((R, N), (1, max(R, 1))),
             wide[:max(N, 1)][None, :N].expand(R, N), wide[:1, None].expand(R, N), wide.as_strided((R, N), (2 * N, 2))]
    for v in views:
        t, stride = ops._strided_rows(v)
        assert t.shape == v.shape and stride >= N and torch.equal(t, v)
        if R * N == 0:
            continue
        flat = t.as_strided((R, N), (stride, 1))  # what a kernel reads
        assert torch.equal(flat, v)
        assert t.storage_offset() + (R - 1) * stride + N <= t.untyped_storage().nbytes() // 4
    # rows apart are taken where they lie
    t, stride = ops._strided_rows(views[1])
    assert t.data_ptr() == views[1].data_ptr() or R * N == 0


def test_axes_are_read_element_by_element():
    axes = ops.mrope_axes([16, 24, 24])
    for same in (axes, list(axes), bytes(axes), bytearray(axes), np.array(axes), np.array(axes, dtype=np.int8),
                 np.repeat(np.arange(3), [16, 24, 24]), array.array("i", axes), memoryview(array.array("q", axes)),
                 torch.tensor(axes), torch.tensor(axes, dtype=torch.uint8)):
        assert ops._axis_bytes(same) == bytes(axes), type(same)
    for bad in ([300], [-1], np.array([256]), np.array([-1])):
        with pytest.raises(ValueError):
            ops._axis_bytes(bad)
    for bad in ([0.0, 1.0], np.array([0.0, 1.0])):
        with pytest.raises(TypeError):
            ops._axis_bytes(bad)


def test_overlap_of_views_of_one_buffer():
    rng = random.Random(1)
    buf = torch.zeros(600)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        R, G, N, M = rng.randint(1, 4), rng.randint(1, 4), rng.randint(0, 6), rng.randint(0, 6)
        wide = max(N, M, 1)
        inner = wide + rng.randint(0, 8)
        outer = inner * G + rng.randint(0, 9)
        strides = (outer, inner, 1) if rng.random() < 0.5 else (inner, inner * R + rng.randint(0, 9), 1)
        at = [rng.randint(0, 90) for _ in range(2)]
        a, b = (buf.as_strided((R, G, n), strides, o) for n, o in zip((N, M), at))
        elements = [set(torch.arange(600).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist())
                    for t in (a, b)]
        want = bool(elements[0] & elements[1])
        assert ops._overlap(a, b) == ops._overlap(b, a) == want, (R, G, N, M, strides, at)
        seen[want] += 1
    assert min(seen.values()) > 500
    # strides that differ: never told to be apart where they meet
    for _ in range(2000):
        R, G, N = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 5)
        views = []
        for _ in range(2):
            inner = N + rng.randint(0, 5)
            views.append(buf.as_strided((R, G, N), (inner * G + rng.randint(0, 5), inner, 1), rng.randint(0, 80)))
        elements = [set(torch.arange(600).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist())
                    for t in views]
        assert ops._overlap(*views) or not elements[0] & elements[1]


# The C ABI refuses on the host, before any launch: no pointer below is followed.
A = 1 << 20
MOST = 2 ** 30 - 2 ** 15


@pytest.mark.parametrize("width,keep,out", [(MOST + 1, 5, 0), (2 ** 31 - 1 - 16384, 2 ** 30, 0), (8, MOST + 1, 0),
                                            (8, 2 ** 31 - 1, 0), (8, 5, MOST + 1), (8, 5, 2 ** 31 - 1 - 2 ** 20)])
def test_selections_that_32_bits_cannot_number_are_refused(width, keep, out):
    """A place past 2^31 would wrap to a negative one: rows, kept tokens and columns stop before."""
    lib = _lib.load()
    args = (A, width, width, width, A, 1, 1, keep, 1, 1, A, A, A + 4096 if out else None, out, out, out, A, 1 << 60)
    assert lib.sna_select_tokens(*args, None) == -4 and "at most" in _lib.last_error()
    w, row, head, n, lens, R, _, *rest = args
    caches = (A, A, 4, 1, 16, 64, 0, A, 2, 2, None, 2, 2)
    assert lib.sna_evict_tokens(*caches, w, row, head, n, lens, R, *rest, None) == -4 and "at most" in _lib.last_error()


@pytest.mark.parametrize("keep", [MOST + 1, 2 ** 31 - 1])
@pytest.mark.parametrize("dst", [None, 2 * A])
def test_compactions_that_32_bits_cannot_number_are_refused(keep, dst):
    assert _lib.load().sna_compact_tokens(A, A, 4, 1, 16, 64, 0, A, 2, 2, dst, 2, 2, A, 1, keep, None) == -4
    assert "at most" in _lib.last_error()


@pytest.mark.parametrize("N,M,keep", [(2 ** 32 + 100, 0, 5), (2 ** 32 + 100, 2 ** 32 + 100, 5), (100, 2 ** 32 + 5, 5),
                                      (100, 0, 2 ** 32 + 5)])
def test_selections_whose_sizes_would_wrap_at_the_c_boundary(N, M, keep):
    w = torch.empty(1, 1, N, device="meta")
    out = torch.empty(1, 1, M, device="meta") if M else None
    lens = torch.empty(1, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="under 2"):
        ops._select_args(w.device, w, lens, keep, 1, 1, out)
