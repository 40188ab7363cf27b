"""ops.qkv_norm_mrope_store at the edges of its arguments: axes in other containers, positions past every float's whole
numbers, infinite elements that no rotation touches. Tolerance as in test_gpu_mrope.py."""

from __future__ import annotations

import array

import numpy as np
import pytest
import torch

from sglang_neuron_amd import ops
from tests.test_gpu_mrope import _make, _run

pytestmark = pytest.mark.gpu


def test_axes_in_any_container():
    T, Hq, Hkv, d, P = 20, 4, 2, 128, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(31, T, Hq, Hkv, d, P, False, True, 128, 3, 100)
    axes = ops.mrope_axes([16, 24, 24])
    want = _run(qkv, pos, inv, axes, Hq, Hkv, d, k, v, slots, gam, sc)
    for same in (list(axes), bytes(axes), bytearray(axes), np.array(axes), np.array(axes, dtype=np.int32),
                 np.repeat(np.arange(3), [16, 24, 24]), array.array("i", axes), memoryview(array.array("q", axes)),
                 torch.tensor(axes)):
        got = _run(qkv, pos, inv, same, Hq, Hkv, d, k, v, slots, gam, sc)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), type(same)
    for bad in (np.full(64, 300), np.full(64, -1), np.full(64, 3)):
        with pytest.raises(ValueError):
            _run(qkv, pos, inv, bad, Hq, Hkv, d, k, v, slots, gam, sc)
