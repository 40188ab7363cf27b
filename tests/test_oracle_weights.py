"""The 64-bit oracle of the attention weights, the eviction and the multi-axis writer (oracle/weights.py) against closed
forms and invariants, and the host refusals of their entry points. CPU only."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import _lib, ops


def test_weights_of_equal_keys_and_their_sum():
    k = torch.zeros(3, 1, 4, 2)
    q = torch.ones(3, 2, 2)
    table = torch.tensor([[1, 2]])
    w, _ = ow.attention_weights(q, k, table, [0, 3], [2], 8, sm_scale=1.0)
    # positions 2, 3, 4 see 3, 4 and 5 equal keys, two heads each
    want = torch.tensor([1 / 3 + 1 / 4 + 1 / 5] * 3 + [1 / 4 + 1 / 5, 1 / 5, 0, 0, 0], dtype=torch.float64) * 2
    assert torch.allclose(w[0, 0], want, rtol=1e-14)
    w, _ = ow.attention_weights(q, k, table, [0, 3], [2], 8, sm_scale=1.0, window=1)
    assert w[0, 0].tolist() == [0, 0, 2, 2, 2, 0, 0, 0]
    w, _ = ow.attention_weights(q, k, table, [0, 3], [2], 8, sm_scale=1.0, sinks=torch.full((2,), math.log(5.0), dtype=torch.float64))
    assert abs(float(w.sum()) - 2 * (3 / 8 + 4 / 9 + 5 / 10)) < 1e-12


def test_selection_against_a_hand_made_row():
    w = torch.tensor([[[9.0, 1.0, 3.0, float("nan"), 3.0, -0.0, 0.0, 3.0, 7.0]]])
    kept, new = ow.select_tokens(w, [9], 5, 1, 1)
    assert kept[0, 0].tolist() == [0, 2, 3, 4, 8] and new == [5]
    kept, _ = ow.select_tokens(w, [8], 7, 0, 0)
    assert kept[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 7]
    kept, new = ow.select_tokens(w, [3], 5, 1, 1)
    assert kept[0, 0].tolist() == [0, 1, 2, -1, -1] and new == [3]


def test_compaction_of_a_hand_made_table():
    cache = torch.arange(4 * 2 * 2).view(4, 1, 2, 2)  # token o of page p: [4 p + 2 o, 4 p + 2 o + 1]
    out = ow.compact_tokens(cache, torch.tensor([[2, 1, 3]]), torch.tensor([[[0, 3, 4, -1]]]))
    assert out[2, 0].tolist() == [[8, 9], [6, 7]] and out[1, 0].tolist() == [[12, 13], [6, 7]]
    assert torch.equal(out[3], cache[3]) and torch.equal(out[0], cache[0])
    out = ow.compact_tokens(cache, torch.tensor([[2, 1, -1]]), torch.tensor([[[1, 2, 4]]]), torch.tensor([[3, 9]]))
    assert out[3, 0].tolist() == [[10, 11], [4, 5]] and torch.equal(out[:3], cache[:3])


def test_mrope_rotation_is_complex_multiplication():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 3 * 4, generator=g).double()
    pos = torch.tensor([[5, 100000, -7], [2, 9, 11]])
    inv = torch.tensor([1.0, 0.25])
    q, k, v, _ = ow.mrope_rows(x, pos, inv, [0, 1], 1, 1, 4, None, None, 1e-6)
    for i, axis in enumerate([0, 1]):
        turn = torch.polar(torch.ones(3, dtype=torch.float64), pos[axis].double() * inv[i].double())
        want = torch.complex(x[:, i], x[:, i + 2]) * turn
        assert torch.allclose(q[:, 0, i], want.real) and torch.allclose(q[:, 0, i + 2], want.imag)
    assert torch.equal(v[:, 0], x[:, 8:])


def test_mrope_axes():
    assert ops.mrope_axes([2, 1, 1]) == (0, 0, 1, 2)
    assert ops.mrope_axes([4, 2, 2], interleaved=True) == (0, 1, 2, 0, 1, 2, 0, 0)
    assert ops.mrope_axes([24, 20, 20], interleaved=True).count(0) == 24
    for bad in ([], [1, 1, 1, 1, 1], [0, 0], [-1, 3]):
        with pytest.raises(ValueError):
            ops.mrope_axes(bad)
    with pytest.raises(ValueError, match="axis 0"):
        ops.mrope_axes([1, 5, 2], interleaved=True)


def test_cpu_tensors_are_refused():
    z = torch.zeros
    cache = z(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensors"):
        ops.decode_attention_weights(z(1, 1, 64, dtype=torch.bfloat16), cache, z(1, 1, dtype=torch.int32),
                                     z(1, dtype=torch.int32), sm_scale=1.0)
    with pytest.raises(ValueError, match="device tensors"):
        ops.select_tokens(z(1, 1, 8), z(1, dtype=torch.int32), keep=2)
    with pytest.raises(ValueError, match="device tensors"):
        ops.compact_tokens(cache, cache.clone(), z(1, 1, dtype=torch.int32), z(1, 1, 2, dtype=torch.int32))


# The C ABI refuses on the host, before any launch: no pointer below is followed.
P = 1 << 20


def _weights_call(fn="sna_prefill_attention_weights", **kw):
    a = dict(q=P, k=P, ks=P, table=P, ts=4, tw=4, q_start=P, lens=P, T=8, R=2, max_q=8, sinks=None, scale=1.0, window=0,
             w=P, row=128, head=64, width=64, add=0, H=8, G=2, d=128, page=16, nb=9, dtype=_lib.DTYPE_BF16, ws=P,
             bytes=1 << 40) | kw
    lib = _lib.load()
    if fn == "sna_decode_attention_weights":
        return lib.sna_decode_attention_weights(
            a["q"], a["k"], a["ks"], a["table"], a["ts"], a["tw"], a["lens"], a["R"], a["sinks"], a["scale"], a["window"],
            a["w"], a["row"], a["head"], a["width"], a["add"], a["H"], a["G"], a["d"], a["page"], a["nb"], a["dtype"],
            a["ws"], a["bytes"], None)
    return lib.sna_prefill_attention_weights(
        a["q"], a["k"], a["ks"], a["table"], a["ts"], a["tw"], a["q_start"], a["lens"], a["T"], a["R"], a["max_q"],
        a["sinks"], a["scale"], a["window"], a["w"], a["row"], a["head"], a["width"], a["add"], a["H"], a["G"], a["d"],
        a["page"], a["nb"], a["dtype"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("fn", ["sna_prefill_attention_weights", "sna_decode_attention_weights"])
@pytest.mark.parametrize("bad,code", [
    (dict(H=7), -1), (dict(R=-1), -1), (dict(window=-1), -1), (dict(nb=0), -1), (dict(ts=3), -1), (dict(page=0), -1),
    (dict(d=96), -4), (dict(H=258, G=2), -4), (dict(dtype=7), -4), (dict(tw=1 << 28, ts=1 << 28), -4),
    (dict(q=None), -1), (dict(k=None), -1), (dict(lens=None), -1), (dict(w=None), -1), (dict(table=None), -1),
    (dict(dtype=_lib.DTYPE_FP8_E4M3FN, ks=None), -1), (dict(q=P + 8), -1), (dict(k=P + 8), -1), (dict(R=65536), -1),
    (dict(head=63), -1), (dict(row=63), -1), (dict(bytes=16), -2), (dict(ws=None), -2), (dict(ws=P + 8), -1),
    (dict(T=1 << 30, R=1 << 15, H=256), -4)])
def test_weights_refusals(fn, bad, code):
    if fn.endswith("decode_attention_weights") and "T" in bad:
        pytest.skip("a decode step has one token a row")
    if code == -2:  # (a table that is too wide for the launch that needs no workspace)
        bad = bad | dict(tw=4096, ts=4096)
    assert _weights_call(fn, **bad) == code, _lib.last_error()


def test_weights_refuse_a_grid_past_its_numbers():
    assert _weights_call(R=65535, G=64, H=64, tw=1 << 20, ts=1 << 20, T=65535, bytes=1 << 62) == -4


@pytest.mark.parametrize("bad", [dict(R=-1), dict(G=0), dict(N=0), dict(keep=0), dict(first=-1), dict(recent=-1),
                                 dict(first=3, recent=3), dict(row=7), dict(head=7), dict(w=None), dict(lens=None),
                                 dict(kept=None), dict(new=None), dict(out=P, M=4), dict(out=P, orow=7),
                                 dict(R=65536)])
def test_select_refusals(bad):
    a = dict(w=P, row=16, head=8, N=8, lens=P, R=2, G=2, keep=5, first=1, recent=1, kept=P, new=P, out=None, orow=16,
             ohead=8, M=8) | bad
    rc = _lib.load().sna_select_tokens(a["w"], a["row"], a["head"], a["N"], a["lens"], a["R"], a["G"], a["keep"], a["first"],
                                       a["recent"], a["kept"], a["new"], a["out"], a["orow"], a["ohead"], a["M"], None, 0,
                                       None)
    assert rc == -1, _lib.last_error()


def test_select_workspace_refusals():
    lib = _lib.load()
    assert lib.sna_select_workspace_bytes(2, 2, 16384, 5, 1) == 0
    need, more = (lib.sna_select_workspace_bytes(2, 2, 40000, 5, p) for p in (0, 1))
    assert 0 < need < more
    for ws, size in ((None, need), (P, need - 1), (P + 4, need)):
        rc = lib.sna_select_tokens(P, 80000, 40000, 40000, P, 2, 2, 5, 1, 1, P, P, None, 0, 0, 0, ws, size, None)
        assert rc in (-1, -2) and "workspace" in _lib.last_error()


@pytest.mark.parametrize("bad,code", [(dict(R=-1), -1), (dict(G=0), -1), (dict(nb=0), -1), (dict(page=0), -1),
                                      (dict(keep=0), -1), (dict(ts=1), -1), (dict(dst=2 * P, dw=0), -1),
                                      (dict(dst=2 * P, dw=2, dstride=1), -1), (dict(d=80), -4), (dict(dtype=9), -4),
                                      (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1),
                                      (dict(kept=None), -1), (dict(k=P + 8), -1), (dict(R=65536), -1),
                                      (dict(G=40000), -1)])
def test_compact_refusals(bad, code):
    a = dict(k=P, v=P, nb=4, G=2, page=16, d=64, dtype=0, table=P, ts=2, tw=2, dst=None, dstride=2, dw=2, kept=P, R=1,
             keep=8) | bad
    rc = _lib.load().sna_compact_tokens(a["k"], a["v"], a["nb"], a["G"], a["page"], a["d"], a["dtype"], a["table"], a["ts"],
                                        a["tw"], a["dst"], a["dstride"], a["dw"], a["kept"], a["R"], a["keep"], None)
    assert rc == code, _lib.last_error()


@pytest.mark.parametrize("bad,code,what", [(dict(d=80), -4, "head_dim"), (dict(k=P + 8), -1, "aligned"),
                                           (dict(tw=0), -1, "bad sizes"), (dict(keep=0), -1, "bad sizes"),
                                           (dict(lens=None), -1, "null"), (dict(table=None), -1, "null"),
                                           (dict(out=P, M=4), -1, "weights_out"), (dict(N=20000, row=40000, head=20000), -2,
                                                                                  "workspace"),
                                           (dict(dst=P, dstride=3, table=P, R=2), -1, "another stride")])
def test_evict_refuses_before_either_launch(bad, code, what):
    a = dict(k=P, v=P, nb=4, G=2, page=16, d=64, dtype=0, table=P, ts=2, tw=2, dst=None, dstride=2, dw=2, w=P, row=16, head=8,
             N=8, lens=P, R=1, keep=5, first=1, recent=1, kept=P, new=P, out=None, M=8) | bad
    rc = _lib.load().sna_evict_tokens(a["k"], a["v"], a["nb"], a["G"], a["page"], a["d"], a["dtype"], a["table"], a["ts"],
                                      a["tw"], a["dst"], a["dstride"], a["dw"], a["w"], a["row"], a["head"], a["N"],
                                      a["lens"], a["R"], a["keep"], a["first"], a["recent"], a["kept"], a["new"], a["out"],
                                      16, 8, a["M"], None, 0, None)
    assert rc == code and what in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("bad,code", [(dict(T=-1), -1), (dict(Hq=0), -1), (dict(d=96), -4), (dict(A=0), -4),
                                      (dict(A=5), -4), (dict(n=4), -4), (dict(n=72), -4), (dict(stride=8), -1),
                                      (dict(pstride=3), -1), (dict(kn=None), -1), (dict(dtype=2), -4),
                                      (dict(dtype=5), -1), (dict(axes=bytes([3] * 64)), -1), (dict(axes=None), -1),
                                      (dict(qkv=None), -1), (dict(pos=None), -1), (dict(inv=None), -1),
                                      (dict(slots=None), -1), (dict(dtype=1, ks=None), -1), (dict(qkv=P + 2), -1),
                                      (dict(stride=(8 + 4) * 128 + 4), -1), (dict(eps=-1.0), -1),
                                      (dict(T=1 << 32, pstride=1 << 32), -1)])
def test_mrope_refusals(bad, code):
    a = dict(qkv=P, stride=(8 + 4) * 128, T=4, Hq=8, Hkv=2, d=128, qn=P, kn=P, eps=1e-6, pos=P, pstride=4, A=3, inv=P, n=64,
             axes=bytes([0] * 64), slots=P, qo=P, k=P, v=P, ks=P, vs=P, nb=2, page=16, dtype=0) | bad
    rc = _lib.load().sna_qkv_norm_mrope_store(a["qkv"], a["stride"], a["T"], a["Hq"], a["Hkv"], a["d"], a["qn"], a["kn"],
                                              a["eps"], a["pos"], a["pstride"], a["A"], a["inv"], a["n"], a["axes"],
                                              a["slots"], a["qo"], a["k"], a["v"], a["ks"], a["vs"], a["nb"], a["page"],
                                              a["dtype"], None)
    assert rc == code, _lib.last_error()
