"""What the operators over caches whose blocks of tokens carry scales refuse, before any launch. CPU only: no pointer below is
followed, and tensors lie on the meta device where a device is asked for."""

from __future__ import annotations

import ctypes

import pytest
import torch

from sglang_neuron_amd import _lib, ops

A = 1 << 20  # an address that nothing reads
BF16, FP8, MUL, INT8 = 0, 1, 2, 3


def _refused(fn, args, change, code, text):
    lib = _lib.load()
    names = [n for n, _ in args]
    for n in change:
        assert n in names, n
    rc = getattr(lib, fn)(*[change.get(n, v) for n, v in args], None)
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


STORE = [("k", A), ("v", A), ("k_row", 256), ("v_row", 256), ("T", 10), ("table", A), ("stride", 4), ("W", 4), ("q_start", A),
         ("prior", A), ("R", 3), ("max_q", 5), ("k_cache", A), ("v_cache", 2 * A), ("ks", A), ("vs", A), ("tokens", 16),
         ("bounds", None), ("nb", 8), ("G", 2), ("P", 32), ("d", 128), ("dtype", INT8)]


@pytest.mark.parametrize("change,code,text", [
    (dict(k=None), -1, "null"), (dict(v=None), -1, "null"), (dict(table=None), -1, "null"), (dict(prior=None), -1, "null"),
    (dict(k_cache=None), -1, "null"), (dict(ks=None), -1, "null"), (dict(vs=None), -1, "null"),
    (dict(k=A + 8), -1, "aligned"), (dict(v_cache=A + 4), -1, "aligned"),
    (dict(T=-1), -1, "bad sizes"), (dict(R=-1), -1, "bad sizes"), (dict(G=0), -1, "bad sizes"), (dict(nb=0), -1, "bad sizes"),
    (dict(W=0), -1, "bad sizes"), (dict(stride=3), -1, "bad sizes"), (dict(max_q=-1), -1, "bad sizes"),
    (dict(k_row=248), -1, "apart"), (dict(v_row=260), -1, "apart"), (dict(k_row=2 ** 31), -1, "apart"),
    (dict(d=96), -4, "head_dim"), (dict(P=24), -4, "page_size"), (dict(P=0), -4, "page_size"), (dict(P=8192), -4, "page_size"),
    (dict(tokens=8), -1, "a scale for"), (dict(tokens=24), -1, "a scale for"), (dict(tokens=64), -1, "a scale for"),
    (dict(dtype=MUL), -4, "dtype"), (dict(dtype=7), -4, "dtype"), (dict(q_start=None), -1, "without q_start"),
    (dict(q_start=None, max_q=1), -1, "without q_start"),
    (dict(R=2 ** 20, max_q=2 ** 20, T=2 ** 30), -1, "exceed the grid"),
])
def test_store_refusals(change, code, text):
    _refused("sna_kv_store_blocks", STORE, change, code, text)


@pytest.mark.parametrize("change", [dict(T=0), dict(R=0), dict(max_q=0)])
def test_stores_of_nothing(change):
    assert _lib.load().sna_kv_store_blocks(*[change.get(n, v) for n, v in STORE], None) == 0


DECODE = [("q", A), ("k_cache", A), ("v_cache", A), ("ks", A), ("vs", A), ("s_page", 4), ("s_head", 2), ("tokens", 16),
          ("table", A), ("stride", 4), ("W", 4), ("rows_n", 600), ("rows", None), ("lens", A), ("blocks", None), ("n", 0),
          ("sinks", None), ("window", 0), ("scale", 1.0), ("out", A), ("T", 600), ("H", 4), ("G", 2), ("d", 128), ("P", 32),
          ("nb", 8), ("dtype", FP8), ("ws", None), ("ws_n", 0)]


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(out=None), -1, "null"), (dict(table=None), -1, "null"),
    (dict(ks=None), -1, "null"), (dict(q=A + 8), -1, "aligned"), (dict(k_cache=A + 8), -1, "aligned"),
    (dict(out=A + 2), -1, "aligned"), (dict(T=-1), -1, "bad sizes"), (dict(H=5), -1, "bad sizes"), (dict(H=0), -1, "bad sizes"),
    (dict(window=-1), -1, "bad sizes"), (dict(nb=0), -1, "bad sizes"), (dict(W=0), -1, "bad sizes"),
    (dict(stride=2), -1, "bad sizes"), (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"),
    (dict(rows_n=599), -1, "over a table"), (dict(rows_n=0, rows=A), -1, "no rows"), (dict(H=34), -4, "group"),
    (dict(d=80), -4, "head_dim"), (dict(P=40), -4, "page_size"), (dict(P=4112), -4, "page_size"), (dict(dtype=MUL), -4, "dtype"),
    (dict(tokens=0), -1, "a scale for"), (dict(tokens=48), -1, "a scale for"), (dict(s_page=-1), -1, "a scale for"),
    (dict(blocks=A, n=0), -1, "a list"), (dict(blocks=A, n=3, window=5), -1, "a list"),
    (dict(W=2 ** 27, stride=2 ** 27), -4, "32 bits"), (dict(blocks=A, n=2 ** 27), -4, "32 bits"),
    (dict(T=2 ** 23, rows_n=2 ** 23), -1, "exceed the grid"), (dict(T=1, rows_n=1, W=100, stride=100), -2, "workspace"),
    (dict(T=1, rows_n=1, W=100, stride=100, ws=A + 4, ws_n=1 << 30), -1, "workspace"),
])
def test_decode_refusals(change, code, text):
    _refused("sna_paged_decode_blocks", DECODE, change, code, text)


def test_decode_workspace_sizes():
    fn = _lib.load().sna_block_decode_workspace_bytes
    bf16, fp8 = _lib.DTYPE_BF16, _lib.DTYPE_FP8_E4M3FN
    good = (600, 4, 2, 128, 32, 4, 0, 0, 0, fp8)
    assert fn(*good) == 0
    few = fn(1, 32, 8, 128, 16, 8192, 0, 0, 0, fp8)
    assert few > 0 and few % (32 * 130 * 4) == 0
    assert fn(1, 32, 8, 128, 16, 8192, 0, 128, 0, fp8) < few and 0 < fn(1, 32, 8, 128, 16, 8192, 0, 0, 64, fp8) <= few
    for at, bad in ((0, 0), (1, 0), (4, 0), (5, 0), (6, -1), (7, -1), (8, -1)):
        assert fn(*good[:at], bad, *good[at + 1:]) == 0
    # the most that any size asks for: 256 splits a query
    assert fn(512, 4, 1, 64, 4096, 2 ** 19, 0, 0, 0, fp8) <= 512 * 256 * 4 * 66 * 4
    # page by page, of 2 rows: a partial for each listed page's 64 keys, of at most 1 GiB
    assert fn(512, 16, 8, 128, 64, 256, 2, 0, 16, bf16) == 512 * 16 * 16 * 130 * 4
    assert fn(512, 16, 8, 128, 160, 100, 2, 0, 16, fp8) == 512 * 16 * 3 * 16 * 130 * 4
    assert fn(512, 24, 8, 128, 64, 256, 2, 0, 16, bf16) == 512 * 16 * 24 * 130 * 4
    for other in ((512, 16, 8, 128, 64, 256, 0, 0, 16, bf16), (512, 16, 4, 128, 64, 256, 2, 0, 16, bf16),
                  (512, 24, 8, 128, 64, 256, 2, 0, 16, fp8), (512, 16, 8, 128, 48, 256, 2, 0, 16, bf16),
                  (512, 16, 8, 128, 64, 1025, 2, 0, 16, bf16), (255, 16, 8, 128, 64, 256, 2, 0, 16, bf16),
                  (511, 16, 8, 128, 64, 256, 2, 0, 16, fp8), (2 ** 14, 16, 8, 128, 64, 256, 2, 0, 16, bf16)):
        assert fn(*other) < other[0] * other[8] * 16 * 130 * 4


SCORES = [("q", A), ("bounds", A), ("table", A), ("stride", 4), ("W", 4), ("rows_n", 5), ("rows", None), ("lens", A),
          ("scores", A), ("counts", A), ("T", 5), ("H", 4), ("G", 2), ("d", 64), ("P", 32), ("nb", 8)]


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), -1, "null"), (dict(bounds=None), -1, "null"), (dict(counts=None), -1, "null"), (dict(scores=None), -1, "null"),
    (dict(q=A + 2), -1, "aligned"), (dict(bounds=A + 8), -1, "aligned"), (dict(T=-2), -1, "bad sizes"),
    (dict(G=3), -1, "bad sizes"), (dict(P=0), -1, "bad sizes"), (dict(nb=0), -1, "bad sizes"), (dict(stride=1), -1, "bad sizes"),
    (dict(H=64), -4, "group"), (dict(d=256), -4, "head_dim"), (dict(rows_n=4), -1, "over a table"),
    (dict(rows_n=0, rows=A), -1, "no rows"), (dict(W=2 ** 30, stride=2 ** 30), -1, "exceed the grid"),
])
def test_score_refusals(change, code, text):
    _refused("sna_block_scores", SCORES, change, code, text)


PREFILL = [("q", A), ("k_cache", A), ("v_cache", A), ("ks", A), ("vs", A), ("s_page", 4), ("s_head", 2), ("tokens", 16),
           ("table", A), ("stride", 4), ("W", 4), ("q_start", A), ("prior", A), ("T", 20), ("R", 3), ("max_q", 9),
           ("sinks", None), ("scale", 1.0), ("window", 0), ("out", A), ("H", 4), ("G", 2), ("d", 128), ("P", 32), ("nb", 8),
           ("dtype", INT8), ("ws", None), ("ws_n", 0)]


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), -1, "null"), (dict(ks=None), -1, "null"), (dict(prior=None), -1, "null"), (dict(q=A + 8), -1, "aligned"),
    (dict(out=A + 8), -1, "aligned"), (dict(R=-1), -1, "bad sizes"), (dict(H=5), -1, "bad sizes"), (dict(T=-1), -1, "queries"),
    (dict(window=-1), -1, "bad sizes"), (dict(d=72), -4, "head_dim"), (dict(P=20), -4, "page_size"),
    (dict(P=8192), -1, "a scale for"), (dict(tokens=12), -1, "a scale for"), (dict(s_head=-1), -1, "a scale for"),
    (dict(dtype=MUL), -4, "dtype"), (dict(dtype=9), -4, "dtype"), (dict(H=258), -4, "query heads"),
    (dict(R=70000), -1, "exceed the grid"), (dict(W=400, stride=400, ws=A, ws_n=16), -2, "workspace"),
])
def test_prefill_refusals(change, code, text):
    _refused("sna_prefill_attention_blocks", PREFILL, change, code, text)


@pytest.mark.parametrize("src,dst,item", [(A, 2 * A, 6), (A, 2 * A, 2), (A + 2, 2 * A, 4), (A, 2 * A + 1, 4), (A, 2 * A, 0)])
def test_page_copies_of_broken_words(src, dst, item):
    """Pages' scales are copied as items of whole words (on whole words)."""
    lens, items = (ctypes.c_int64 * 1)(64), (ctypes.c_int64 * 1)(item)
    rc = _lib.load().sna_page_items_copy((ctypes.c_uint64 * 1)(src), lens, (ctypes.c_uint64 * 1)(dst), lens, items, 1, A, A, 3,
                                         None)
    assert rc == -1 and "multiples of 4" in _lib.last_error()


@pytest.mark.parametrize("item", [4, 24])
def test_wire_buffers_hold_whole_vectors(item):
    lens, items, ptrs = (ctypes.c_int64 * 1)(96), (ctypes.c_int64 * 1)(item), (ctypes.c_uint64 * 1)(A)
    lib = _lib.load()
    for rc in (lib.sna_page_items_pack(ptrs, lens, items, 1, A, 2, A, 4096, None),
               lib.sna_page_items_unpack(A, 4096, ptrs, lens, items, 1, A, 2, None)):
        assert rc == -1 and "multiples of 16" in _lib.last_error()


def test_int8_is_for_blocks_only():
    assert _lib.DTYPE_INT8 == INT8
    with pytest.raises(ValueError):
        ops.cache_dtype_code(torch.int8)
    lib = _lib.load()
    assert lib.sna_prefill_attention(A, A, A, A, A, A, 4, 4, A, A, 3, 9, None, 1.0, 0, A, 4, 2, 128, 32, 8, INT8, None) == -4
    assert lib.sna_kv_store_mha(A, A, A, 4, A, A, A, A, 8, 2, 32, 128, INT8, None) < 0


def _cache(nb=6, G=2, P=32, d=64, dtype=torch.int8):
    return torch.zeros(nb, G, P, d, dtype=dtype)


def _scale(nb=6, G=2, n=2):
    return torch.ones(nb, G, n)


@pytest.mark.parametrize("k,v,ks,vs,text", [
    (_cache(dtype=torch.float16), _cache(dtype=torch.float16), None, None, "unsupported cache dtype"),
    (_cache(dtype=torch.uint8), _cache(dtype=torch.uint8), _scale(), _scale(), "unsupported cache dtype"),
    (_cache(), _cache(dtype=torch.bfloat16), _scale(), _scale(), "of one type"),
    (_cache(), _cache(P=16), _scale(), _scale(), "of one type"),
    (_cache()[:, :, :, :32], _cache()[:, :, :, :32], _scale(), _scale(), "contiguous"),
    (_cache(), _cache(), None, _scale(), "needs"),
    (_cache(), _cache(), _scale(n=3), _scale(n=3), "scales must be"),
    (_cache(), _cache(), _scale(n=4), _scale(n=4), "scales must be"),
    (_cache(), _cache(), _scale(nb=5), _scale(nb=5), "scales must be"),
    (_cache(), _cache(), _scale(), _scale(n=1), "scales must be"),
    (_cache(), _cache(), _scale().double(), _scale().double(), "scales must be"),
    (_cache(), _cache(), torch.ones(2), torch.ones(2), "scales must be"),
])
def test_caches_that_are_refused(k, v, ks, vs, text):
    with pytest.raises(ValueError, match=text):
        ops._block_cache(k, v, ks, vs)


def test_scale_strides():
    k, v = _cache(), _cache()
    code, shape, a, b, page, head, tokens = ops._block_cache(k, v, _scale(), _scale())
    assert (code, tuple(shape), page, head, tokens) == (INT8, (6, 2, 32, 64), 4, 2, 16)
    one = torch.ones(2).view(1, 2, 1).expand(6, 2, 1)
    _, _, a, _, page, head, tokens = ops._block_cache(k, v, one, one)
    assert (page, head, tokens) == (0, 1, 32) and a.data_ptr() == one.data_ptr()
    both = torch.rand(6, 2, 2, 2)
    _, _, a, b, page, head, _ = ops._block_cache(k, v, both[:, 0], both[:, 1])
    assert (page, head) == (8, 2) and a.data_ptr() == both.data_ptr()
    other = torch.rand(2, 6, 2).transpose(0, 1)  # V's heads apart, K's not
    _, _, a, b, page, head, _ = ops._block_cache(k, v, _scale(), other)
    assert a.is_contiguous() and torch.equal(b, other) and b.is_contiguous() and (page, head) == (4, 2)
    odd = torch.rand(6, 2, 4)[..., ::2]  # columns apart
    _, _, a, b, page, head, _ = ops._block_cache(k, v, odd, odd)
    assert a.is_contiguous() and torch.equal(a, odd) and (page, head) == (4, 2)
    assert ops._block_cache(_cache(dtype=torch.bfloat16), _cache(dtype=torch.bfloat16), None, None)[2:] == (None, None, 0, 0, 32)


def test_rows_of_heads_stay_inside_their_tensor():
    for x in (torch.randn(5, 2, 64), torch.randn(5, 3, 2, 64)[:, 1], torch.randn(5, 200)[:, 8:136].view(5, 2, 64),
              torch.randn(5, 201)[:, 8:136].unflatten(1, (2, 64)), torch.randn(2, 5, 64).transpose(0, 1),
              torch.randn(1, 2, 64).expand(5, 2, 64), torch.randn(5, 2, 128)[..., ::2]):
        y = ops._head_rows(x)
        assert torch.equal(x, y) and y.stride(0) % 8 == 0 and y.stride(0) >= 128
        assert torch.equal(y.as_strided((5, 128), (y.stride(0), 1)), x.reshape(5, 128))


def test_cpu_tensors_are_refused():
    k, s = _cache(), _scale()
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    bounds = torch.zeros(6, 2, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.kv_store_blocks(q, q, k, k.clone(), table, lens, k_scale=s, v_scale=s.clone()),
                 lambda: ops.paged_decode_blocks(q, k, k, table, lens, sm_scale=1.0, k_scale=s, v_scale=s),
                 lambda: ops.paged_decode_selected(q, k, k, table, lens, torch.zeros(1, 2, 1), sm_scale=1.0, k_scale=s,
                                                   v_scale=s),
                 lambda: ops.prefill_attention_blocks(q, k, k, table, torch.tensor([0, 1]), lens, max_q_len=1, sm_scale=1.0,
                                                      k_scale=s, v_scale=s),
                 lambda: ops.block_scores(q, bounds, table, lens, page_size=32),
                 lambda: ops.select_blocks(q, bounds, table, lens, keep=2, page_size=32)):
        with pytest.raises(ValueError, match="CPU"):
            call()
