"""ops.qkv_norm_mrope_store at the edges of its arguments: axes in other containers, positions past every float's whole
numbers, infinite elements that no rotation touches. Tolerance as in test_gpu_mrope.py."""

from __future__ import annotations

import array
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import ops
from tests.conftest import announce
from tests.test_gpu_mrope import E, _make, _run

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


def _pi(bits=400):
    """pi * 2^bits, by Machin's formula in whole numbers."""
    def atan(n):
        term = s = (1 << bits + 32) // n
        i = 1
        while term:
            term //= n * n
            i += 2
            s += (-1 if i // 2 % 2 else 1) * (term // i)
        return s
    return 4 * (4 * atan(5) - atan(239)) >> 32


@pytest.mark.parametrize("rot", [128, 32])
@pytest.mark.parametrize("base", [0, -5, 2 ** 24 + 1, 2 ** 31 + 3, -2 ** 33 - 7, 2 ** 40 + 9, 2 ** 52 + 1, 2 ** 53 + 1,
                                  2 ** 62 + 12345, 2 ** 63 - 8, -2 ** 63])
def test_positions_of_any_size(base, rot):
    """Each angle's fraction of a turn from whole numbers; the same tolerance at every position."""
    announce(f"positions from {base} rot {rot}")
    T, Hq, Hkv, d, P, n = 8, 2, 1, 128, 16, rot // 2
    qkv, _, inv, gam, slots, k, v, sc = _make(33, T, Hq, Hkv, d, P, False, False, rot, 1, 0)
    pos = torch.tensor([[base + t for t in range(T)]], dtype=torch.int64)
    q, kc, _ = _run(qkv, pos, inv, [0] * n, Hq, Hkv, d, k, v, slots, gam, sc)
    two_pi = Fraction(2 * _pi(), 1 << 400)
    x = qkv.double().view(T, Hq + 2 * Hkv, d)[:, :Hq + Hkv]
    want, size = x.clone(), x.abs().clone()
    for t in range(T):
        for i in range(n):
            turns = int(pos[0, t]) * Fraction(float(inv[i])) / two_pi
            angle = 2 * math.pi * float(turns - round(turns))
            c, s = math.cos(angle), math.sin(angle)
            a, b = x[t, :, i], x[t, :, i + n]
            want[t, :, i], want[t, :, i + n] = a * c - b * s, b * c + a * s
            size[t, :, i] = size[t, :, i + n] = a.abs() + b.abs()
    got = torch.cat([q.double(), kc.double()[slots // P, :, slots % P]], 1)
    tol = want.abs() * 2.0 ** -8 + size * E * (1 + 2.0 ** -8) + 2.0 ** -134
    assert bool(((got - want).abs() <= tol).all()), f"off by {float(((got - want).abs() - tol).max()):.3e} past the tolerance"


@pytest.mark.parametrize("d,rot", [(128, 64), (64, 16)])
def test_infinite_elements_that_are_not_rotated_stay(d, rot):
    T, Hq, Hkv, P = 9, 3, 1, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(35, T, Hq, Hkv, d, P, False, False, rot, 2, 10)
    x = qkv.view(T, Hq + 2 * Hkv, d)
    x[2, 0, rot], x[3, 1, d - 1], x[4, Hq, rot + 3], x[5, Hq + Hkv, 0] = math.inf, -math.inf, -math.inf, math.inf
    x[6, 2, rot + 1], x[6, Hq, rot + 1] = -0.0, -0.0
    q, kc, vc = _run(qkv, pos, inv, ops.mrope_axes([rot // 4, rot // 4]), Hq, Hkv, d, k, v, slots, gam, sc)
    at = (slots // P, slice(None), slots % P)
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(q[..., rot:]), bits(x[:, :Hq, rot:]))
    assert torch.equal(bits(kc[at][..., rot:]), bits(x[:, Hq:Hq + Hkv, rot:]))
    assert torch.equal(bits(vc[at]), bits(x[:, Hq + Hkv:]))
    assert bool(torch.isfinite(q[..., :rot]).all())


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("power", [-50, -62, -63, -64, -65])
def test_norm_of_tiny_rows_without_an_eps(power, d):
    """Down to mean squares that fp32 holds in fewer bits. (2^-130 in steps of 2^-149 is off by 2^-20 at most, and so is each of
    its d squares, all of one sign: the norm by half of both, 2^-20.)"""
    T, Hq, Hkv, P = 6, 2, 1, 16
    qkv, pos, inv, gam, slots, k, v, sc = _make(37, T, Hq, Hkv, d, P, False, True, d, 1, 10)
    qkv = (qkv.double() * 2.0 ** power).to(torch.bfloat16)
    q, kc, _ = _run(qkv, pos, inv, [0] * (d // 2), Hq, Hkv, d, k, v, slots, gam, sc, norm_eps=0.0)
    wq, wk, _, size = ow.mrope_rows(qkv, pos, inv, [0] * (d // 2), Hq, Hkv, d, gam[0], gam[1], 0.0)
    got, want = torch.cat([q.double(), kc.double()[slots // P, :, slots % P]], 1), torch.cat([wq, wk], 1)
    tol = want.abs() * 2.0 ** -8 + size * (E + 2.0 ** -20) * (1 + 2.0 ** -8)
    assert bool(((got - want).abs() <= tol).all())
    # a row of zeros has no direction: 0 / 0
    qkv[2] = 0
    q, _, _ = _run(qkv, pos, inv, [0] * (d // 2), Hq, Hkv, d, k, v, slots, gam, sc, norm_eps=0.0)
    assert bool(q[2].isnan().all()) and bool(torch.isfinite(q[[0, 1, 3, 4, 5]]).all())
