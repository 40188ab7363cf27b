"""How the tensor-level entry points read their arguments, before any launch. CPU only."""

from __future__ import annotations

import pytest
import torch

from sglang_neuron_amd import ops


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
