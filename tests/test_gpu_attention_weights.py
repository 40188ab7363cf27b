"""ops.prefill_attention_weights and ops.decode_attention_weights against the 64-bit oracle (oracle/weights.py) on the
same pool bytes.

Tolerance. A score is an fp32 sum of d exact products (bf16 times bf16 or e4m3fn values): it is off by at most
d * 2^-24 * A, A the largest sm_scale * sum |q k|; its scale constant, product and difference to the row's maximum add at
most 4 roundings of a value of at most 2 A (log2 e < 1.45 times A, the maximum taken away). A probability is the quotient
of two exponentials that are off by so much each, plus the exponential's own step and the roundings of its row's sum (at
most one a block of keys and 64 inside a block) and of the reciprocal, and a key's weight adds its rows' in fp32. So
  |W - W64| <= W64 * (2 * (d + 8) * 2^-24 * A + (128 + blocks + rows) * 2^-24)   (plus 1e-30, what flushes to zero)."""

from __future__ import annotations

import types

import pytest
import torch

from oracle import weights as ow
from sglang_neuron_amd import _lib, ops
from sglang_neuron_amd.attention import NeuronAttnBackend
from sglang_neuron_amd.mem_cache import NeuronMHATokenToKVPool
from tests.conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


def make(seed, H, G, d, P, lens, counts, fp8, spare=2, junk=True, holes=0):
    """A pool of random pages with a table of random pages, the queries and their offsets. Slots of the pool that hold no
    token are NaN (``junk``): nothing may read them into a result. ``holes``: table entries inside rows set to -1."""
    g = torch.Generator().manual_seed(seed)
    R = len(lens)
    pages = [-(-n // P) for n in lens]
    nb = 1 + sum(pages) + spare
    width = max(pages + [1]) + 1
    perm = (torch.randperm(nb - 1, generator=g) + 1).tolist()
    table = torch.full((R, width), -1, dtype=torch.int32)
    k = torch.randn(nb, G, P, d, generator=g)
    ks = None
    if fp8:
        ks = k.abs().amax((0, 2, 3)) / 448
        k = k / ks.view(1, G, 1, 1)
    live = torch.zeros(nb, P, dtype=torch.bool)
    for r, n in enumerate(lens):
        for c in range(pages[r]):
            page = perm.pop()
            table[r, c] = page
            live[page, :min(P, n - c * P)] = True
    if junk:
        k = torch.where(live[:, None, :, None], k, float("nan"))
    for _ in range(holes):
        r = int(torch.randint(0, R, (1,), generator=g))
        if pages[r] > 1:
            table[r, int(torch.randint(0, pages[r], (1,), generator=g))] = -1
    k = k.to(FP8) if fp8 else k.to(torch.bfloat16)
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    q = torch.randn(start[-1], H, d, generator=g).to(torch.bfloat16)
    return types.SimpleNamespace(q=q, k=k, ks=ks, table=table, start=start, prior=[n - c for n, c in zip(lens, counts)],
                                 lens=lens, counts=counts, P=P, G=G, H=H, d=d, scale=d ** -0.5)


def oracle(c, width, **kw):
    return ow.attention_weights(c.q, c.k, c.table, c.start, c.prior, width, sm_scale=c.scale, k_scale=c.ks, **kw)


def prefill(c, **kw):
    host = kw.pop("host", True)
    return ops.prefill_attention_weights(
        c.q.to(DEV), c.k.to(DEV), c.table.to(DEV), torch.tensor(c.start, dtype=torch.int32, device=DEV),
        torch.tensor(c.prior, dtype=torch.int32, device=DEV), max_q_len=max(c.counts + [1]), sm_scale=c.scale,
        k_scale=None if c.ks is None else c.ks.to(DEV), host_q_start=c.start if host else None, **kw)


def check(c, got, want, reach, what):
    rows = max(c.counts + [1]) * (c.H // c.G)
    blocks = -(-max(c.lens + [1]) // 256)
    rel = 2 * (c.d + 8) * 2.0 ** -24 * reach + (128 + blocks + rows) * 2.0 ** -24
    off = (got.double().cpu() - want).abs()
    worst = float((off - rel * want).max()) if want.numel() else 0.0
    assert worst <= 1e-30, f"{what}: off by {float(off.max()):.3e} at {float(want.flatten()[off.argmax()]):.3e} (rel {rel:.1e})"


CASES = [
    # name, H, G, d, P, lens, queries, fp8, window, sinks, holes
    ("one-token", 1, 1, 64, 16, [1], [1], False, 0, False, 0),
    ("one-key-each", 8, 2, 128, 16, [1, 1, 1], [1, 1, 1], True, 0, True, 0),
    ("odd-mix", 6, 2, 128, 16, [37, 300, 5, 517], [37, 3, 5, 129], False, 0, False, 0),
    ("odd-mix-fp8", 6, 2, 128, 32, [37, 300, 5, 517], [37, 3, 5, 129], True, 0, True, 0),
    ("no-queries", 4, 4, 64, 16, [100, 20, 257], [2, 0, 1], True, 0, False, 0),
    ("group-5-d64", 10, 2, 64, 48, [255, 256, 257], [1, 2, 70], False, 0, True, 0),
    ("group-40", 40, 1, 64, 16, [130, 33], [9, 33], True, 0, False, 0),
    ("group-128", 128, 1, 128, 16, [70], [5], False, 0, False, 0),
    ("window", 8, 2, 128, 16, [600, 90, 1000], [600, 90, 10], False, 100, False, 0),
    ("window-1", 4, 2, 64, 16, [300], [300], True, 1, True, 0),
    ("window-wide", 4, 2, 64, 16, [300, 700], [20, 400], True, 5000, True, 0),
    ("holes", 8, 2, 128, 16, [300, 400, 64], [40, 1, 64], False, 0, False, 9),
    ("holes-window", 8, 2, 64, 16, [300, 400, 64], [300, 7, 64], True, 20, False, 40),
    ("page-7", 4, 2, 64, 7, [100, 30], [33, 30], False, 0, False, 0),
    ("long-window-of-queries", 4, 1, 128, 64, [3000], [32], True, 0, False, 0),
    ("runs-of-queries", 64, 1, 64, 16, [100, 300], [100, 70], True, 0, True, 2),
    ("runs-window", 96, 2, 128, 16, [150, 40], [150, 40], False, 33, False, 0),
    ("runs-far-window", 8, 1, 64, 16, [5000, 300, 90], [600, 300, 45], False, 128, True, 4),
    ("runs-wide-window", 8, 1, 64, 16, [1500, 900], [700, 31], True, 300, False, 0),
    ("runs-group-3", 12, 4, 128, 16, [2000, 700, 1], [333, 700, 1], True, 0, True, 3),
    ("runs-odd-prior", 8, 1, 64, 16, [777, 1333], [500, 65], False, 0, False, 0),
    ("many-tiles", 16, 1, 128, 16, [700], [530], True, 0, False, 0),
    ("many-rows-merged", 16, 2, 64, 16, [700, 650], [700, 300], True, 0, True, 2),
    ("many-rows", 2, 1, 64, 16, [5 + 13 * i for i in range(40)], [1 + i % 4 for i in range(40)], True, 0, False, 0),
]


@pytest.mark.parametrize("name,H,G,d,P,lens,counts,fp8,window,sinks,holes", CASES, ids=[c[0] for c in CASES])
def test_prefill_weights(name, H, G, d, P, lens, counts, fp8, window, sinks, holes):
    announce(f"weights {name}")
    c = make(len(name) * 7 + H, H, G, d, P, lens, counts, fp8, holes=holes)
    sk = torch.randn(H, generator=torch.Generator().manual_seed(3)) if sinks else None
    kw = dict(window=window)
    width = c.table.shape[1] * P
    want, reach = oracle(c, width, sinks=sk, **kw)
    got = prefill(c, sinks=None if sk is None else sk.to(DEV), **kw)
    assert got.shape == (len(lens), G, width) and got.dtype == torch.float32
    check(c, got, want, reach, name)
    assert bool((got.cpu()[want == 0] == 0).all())
    again = prefill(c, sinks=None if sk is None else sk.to(DEV), host=False, **kw)
    assert torch.equal(got, again), "two runs of one call differ"


@pytest.mark.parametrize("H,G,d,P,lens,fp8,window,sinks", [
    (4, 4, 64, 16, [1], False, 0, False),
    (16, 8, 128, 16, [128, 900, 1, 33], False, 0, False),
    (32, 8, 128, 16, [255, 256, 257, 2000], True, 0, False),
    (8, 1, 64, 16, [700, 1300, 5], True, 0, True),
    (8, 1, 64, 32, [700, 1300, 5], True, 128, True),
    (40, 1, 128, 16, [300, 17], False, 0, False),
    (128, 1, 64, 16, [300, 17], True, 50, False),
])
def test_decode_weights(H, G, d, P, lens, fp8, window, sinks):
    announce(f"decode weights {H} {G} {d} {lens}")
    c = make(5 + H + d, H, G, d, P, lens, [1] * len(lens), fp8)
    sk = torch.randn(H, generator=torch.Generator().manual_seed(4)) if sinks else None
    width = c.table.shape[1] * P
    want, reach = oracle(c, width, window=window, sinks=sk)
    args = (c.q.to(DEV), c.k.to(DEV), c.table.to(DEV), torch.tensor(lens, device=DEV))  # int64 lengths
    kw = dict(sm_scale=c.scale, k_scale=None if c.ks is None else c.ks.to(DEV), window=window,
              sinks=None if sk is None else sk.to(DEV))
    got = ops.decode_attention_weights(*args, **kw)
    check(c, got, want, reach, "decode")
    assert torch.equal(got, ops.decode_attention_weights(*args, **kw))


def few_rows(R, H, G, d, P, most, queries, fp8, holes=0, seed=0, table_width=None):
    """R requests of 0 to ``most`` keys (the first has them all) and up to ``queries`` queries each."""
    g = torch.Generator().manual_seed(seed + R + d + P)
    counts = [min(queries, 1 + int(x)) for x in torch.randint(0, queries, (R,), generator=g)]
    lens = [most] + [max(c, int(x)) for c, x in zip(counts[1:], torch.randint(1, most // 4, (R - 1,), generator=g))]
    counts[-1] = 0
    c = make(seed + R + P, H, G, d, P, lens, counts, fp8, holes=holes)
    if table_width:
        wide = torch.full((R, table_width), -1, dtype=torch.int32)
        wide[:, :c.table.shape[1]] = c.table
        c.table = wide
    return c


# Few query rows a request, in the forms that their number, the tables' width and the batch choose between.
@pytest.mark.parametrize("R,H,G,d,P,most,queries,fp8,window,sinks,holes,table_width", [
    (130, 4, 2, 64, 16, 2100, 1, True, 0, False, 0, None),    # a row's scores in LDS: two workgroups a CU
    (64, 8, 4, 128, 7, 2060, 3, False, 0, True, 20, None),    # the same, odd pages
    (64, 16, 4, 64, 48, 2200, 3, False, 300, True, 20, None), # one workgroup a CU
    (128, 32, 2, 128, 32, 2050, 1, True, 70, False, 5, None),
    (40, 56, 8, 64, 1, 2080, 2, True, 0, True, 0, None),      # pages of one token
    (512, 4, 2, 64, 16, 2111, 2, False, 2000, False, 9, None),  # two turns of workgroups
    (160, 16, 8, 64, 16, 900, 2, False, 0, False, 9, None),   # several chunks a workgroup, scores through memory
    (160, 16, 8, 128, 16, 700, 1, True, 200, True, 9, None),
    (3, 16, 2, 128, 16, 2500, 2, False, 0, True, 3, 4000),    # tables much wider than the keys
    (4, 64, 8, 64, 16, 700, 2, True, 0, False, 3, 17000),     # scores past the workspace's bound: computed twice
])
def test_few_rows(R, H, G, d, P, most, queries, fp8, window, sinks, holes, table_width):
    announce(f"few rows {R} {H} {G} {d} {P} {most} {queries} {fp8}")
    c = few_rows(R, H, G, d, P, most, queries, fp8, holes, table_width=table_width)
    sk = torch.randn(H, generator=torch.Generator().manual_seed(5)) if sinks else None
    sg = None if sk is None else sk.to(DEV)
    keys, full = max(c.lens), c.table.shape[1] * P
    want, reach = oracle(c, full, sinks=sk, window=window)
    got = prefill(c, sinks=sg, window=window)
    check(c, got, want, reach, "written")
    assert got.shape[2] == full and bool((got[want.to(DEV) == 0] == 0).all())
    assert torch.equal(got, prefill(c, sinks=sg, window=window, host=False))
    rel = 2 * (d + 8) * 2.0 ** -24 * reach + (128 + -(-keys // 256) + max(c.counts) * H // G) * 2.0 ** -24
    for width in (keys + 99, keys - 30):  # added to: wider than the keys, and narrower
        base = torch.full((R, G + 1, width + 5), -2.0, device=DEV)
        w = base[:, :G, 3:3 + width]
        w.fill_(3.0)
        prefill(c, sinks=sg, window=window, weights=w)
        part = torch.zeros(R, G, width, dtype=torch.float64)
        part[..., :min(width, full)] = want[..., :width]
        # (adding rounds once more: half a step of at most 3 + W)
        assert bool(((w.double().cpu() - (part + 3)).abs() <= part * rel + (part + 3) * 2.0 ** -24).all())
        rest = torch.arange(width, device=DEV) >= torch.tensor(c.lens, device=DEV)[:, None]
        assert bool((w[rest[:, None].expand(R, G, width)] == 3).all())
        assert bool((base[:, G] == -2).all() and (base[..., :3] == -2).all() and (base[..., 3 + width:] == -2).all())


@pytest.mark.parametrize("R,H,G,counts", [(64, 8, 4, 1), (3, 8, 4, 1), (3, 8, 4, 40)])
@pytest.mark.parametrize("width", [2500, 1900])
def test_written_widths_at_the_c_entry(R, H, G, counts, width):
    """The C entry writes any number of columns: fewer than the table's keys, or more."""
    c = few_rows(R, H, G, 64, 16, 2070, counts, False, seed=8)
    q, k, table = c.q.to(DEV), c.k.to(DEV), c.table.to(DEV)
    start, prior = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (c.start, c.prior))
    out = torch.full((R, G, width + 3), -2.0, device=DEV)
    lib = _lib.load()
    sizes = (len(q), R, max(c.counts))
    need = lib.sna_attention_weights_workspace_bytes(*sizes, H, G, 64, 16, table.shape[1], width, _lib.DTYPE_BF16, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    rc = lib.sna_prefill_attention_weights(
        q.data_ptr(), k.data_ptr(), None, table.data_ptr(), table.shape[1], table.shape[1], start.data_ptr(),
        prior.data_ptr(), *sizes, None, c.scale, 0, out.data_ptr(), G * (width + 3), width + 3, width, 0, H, G, 64, 16,
        k.shape[0], _lib.DTYPE_BF16, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    want, reach = oracle(c, width)
    check(c, out[..., :width], want, reach, "written")
    assert bool((out[..., width:] == -2).all())


def test_few_rows_bad_pages_and_nan():
    """The kernel that keeps a row's scores in LDS: pages past the pool, rows that see nothing, a NaN of a visible key."""
    c = few_rows(64, 8, 4, 64, 16, 2100, 1, False, seed=3)
    c.table[1, 0], c.table[2] = 10 ** 6, -1
    c.lens[3] = c.prior[3] = 0
    lens = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
    c.counts = [1] * 64
    c.start = list(range(65))
    g = torch.Generator().manual_seed(6)
    c.q = torch.randn(64, 8, 64, generator=g).to(torch.bfloat16)
    c.prior = [n - 1 for n in c.lens]
    want, reach = oracle(c, c.table.shape[1] * 16)
    want[3] = 0
    args = (c.q.to(DEV), c.k.to(DEV), c.table.to(DEV), lens)
    got = ops.decode_attention_weights(*args, sm_scale=c.scale)
    check(c, got, want, reach, "bad pages")
    assert bool((got[2:4] == 0).all())
    args[1][int(c.table[0, 5]), 1, 3] = float("nan")
    got = ops.decode_attention_weights(*args, sm_scale=c.scale).cpu()
    assert bool(got[0, 1, :2100].isnan().all()) and bool((got[0, 1, 2100:] == 0).all())
    got[0, 1] = 0
    want[0, 1] = 0
    check(c, got, want, reach, "beside a NaN")
    # most exponentials of a row underflow: a NaN of its sum reaches them all the same, in every form
    for n in (64, 4):
        few = ops.decode_attention_weights(args[0][:n], args[1], args[2][:n], lens[:n], sm_scale=40.0).cpu()
        assert bool(few[0, 1, :2100].isnan().all()) and bool((few[0, :, 2100:] == 0).all())
        assert bool(torch.isfinite(few[0, [0, 2, 3]]).all()) and bool(torch.isfinite(few[1:]).all())


def test_a_longest_query_count_past_the_tokens():
    """max_q_len is an upper bound: any that holds gives the same weights."""
    c = make(29, 8, 2, 64, 16, [300, 40], [40, 3], False)
    dev = [t.to(DEV) for t in (c.q, c.k, c.table)]
    start, prior = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (c.start, c.prior))
    want, reach = oracle(c, c.table.shape[1] * 16)
    for most in (40, 43, 10 ** 6, 2 ** 31 - 1):
        check(c, ops.prefill_attention_weights(*dev, start, prior, max_q_len=most, sm_scale=c.scale), want, reach, str(most))


def test_decode_rows_without_keys():
    c = make(9, 8, 2, 64, 16, [40, 40, 40], [1, 1, 1], False)
    c.table[1] = -1  # no valid page: a row that sees nothing
    lens = torch.tensor([40, 40, 0], dtype=torch.int32, device=DEV)
    got = ops.decode_attention_weights(c.q.to(DEV), c.k.to(DEV), c.table.to(DEV), lens, sm_scale=c.scale)
    want, reach = oracle(c, c.table.shape[1] * 16)
    want[2] = 0
    check(c, got, want, reach, "empty rows")
    assert bool((got[1:] == 0).all()) and bool((got[0] > 0).any())


def test_accumulates_into_strided_weights_and_leaves_the_rest():
    c = make(11, 8, 2, 128, 16, [300, 77], [5, 77], True)
    width = 280  # narrower than the first row: its last keys get nothing
    base = torch.full((2, 3, 512), -3.0, device=DEV)
    w = base[:, 1:, 100:100 + width]
    w.fill_(2.0)
    out = prefill(c, weights=w)
    assert out is w
    want, reach = oracle(c, width)
    # (adding to 2 rounds once more: half a step of at most 2 + W)
    off = (w.double().cpu() - (want + 2)).abs()
    rel = 2 * (128 + 8) * 2.0 ** -24 * reach + (128 + 2 + 5 * 77) * 2.0 ** -24
    assert bool((off <= want * rel + (2 + want) * 2.0 ** -24).all())
    assert bool((w[1, :, 77:] == 2.0).all())
    assert bool((base[:, 0] == -3).all()) and bool((base[:, :, :100] == -3).all()) and bool((base[:, :, 380:] == -3).all())
    # heads outermost: the row stride is the smaller one
    t = torch.zeros(2, 2, 320, device=DEV).transpose(0, 1)
    prefill(c, weights=t)
    want, reach = oracle(c, 320)
    check(c, t, want, reach, "transposed")


def test_accumulates_runs_of_queries():
    c = make(12, 64, 1, 64, 16, [100, 80], [90, 80], False)
    w = torch.full((2, 1, 128), 3.0, device=DEV)
    prefill(c, weights=w)
    want, reach = oracle(c, 128)
    off = (w.double().cpu() - (want + 3)).abs()
    rel = 2 * (64 + 8) * 2.0 ** -24 * reach + (128 + 1 + 64 * 90) * 2.0 ** -24
    assert bool((off <= want * rel + (3 + want) * 2.0 ** -24).all()) and bool((w[0, :, 100:] == 3).all())


def test_multipliers_and_strided_queries():
    c = make(13, 8, 2, 128, 16, [200, 60], [30, 60], True)
    m = (1.0 / c.ks.to(torch.bfloat16)).float()
    c.ks = m
    want, reach = oracle(c, c.table.shape[1] * 16, multiply=True)
    wide = torch.randn(90, 8, 256, device=DEV).to(torch.bfloat16)
    wide[..., :128] = c.q.to(DEV)
    c.q = wide[..., :128]
    got = prefill(c, scales_multiply=True)
    check(c, got, want, reach, "multipliers")


def test_a_chunk_of_its_own_sums_to_its_rows():
    """Without sinks every query's probabilities sum to 1: W sums to queries * heads of the group."""
    c = make(15, 32, 8, 128, 16, [2048, 1500], [700, 64], True)
    got = prefill(c).double().sum(-1).cpu()
    want = torch.tensor([[700.0 * 4] * 8, [64.0 * 4] * 8], dtype=torch.float64)
    assert bool(((got - want).abs() <= want * (128 + 8 + 2800) * 2.0 ** -24).all())


@pytest.mark.parametrize("R,counts", [(4, 1), (64, 1), (2, 40)])
def test_cache_offsets_past_32_bits(R, counts):
    """The same pages far behind 4 GiB of a pool give the same bits, in every form."""
    c = few_rows(R, 8, 4, 128, 16, 2060, counts, False, seed=31)
    nb, page = len(c.k), c.k[0].numel() * 2
    far = (2 ** 32 + 2 ** 30) // page
    k = torch.zeros(far + nb, *c.k.shape[1:], dtype=torch.bfloat16, device=DEV)
    k[far:] = c.k.to(DEV)
    start, prior = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (c.start, c.prior))
    table = c.table.to(DEV)
    got = ops.prefill_attention_weights(c.q.to(DEV), k, torch.where(table >= 0, table + far, table), start, prior,
                                        max_q_len=max(c.counts), sm_scale=c.scale)
    near = prefill(c)
    assert torch.equal(got, near) and bool((near[0] > 0).any())


def test_bad_offsets_and_lengths_stay_inside():
    """Device offsets outside q, chunks past max_q_len and lengths past the table are cut, never followed."""
    c = make(17, 8, 2, 64, 16, [64, 64], [8, 8], False, junk=False)
    args = (c.q.to(DEV), c.k.to(DEV), c.table.to(DEV))
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for start, prior in (((0, 8, 4000), (56, 56)), ((-5, 8, 2), (56, 2 ** 31 - 1)), ((9, 3, 16), (-100, 56)),
                         ((0, 16, 16), (-2 ** 31, 10 ** 6))):
        got = ops.prefill_attention_weights(*args, t(*start), t(*prior), max_q_len=8, sm_scale=c.scale)
        assert bool(torch.isfinite(got).all())
    got = ops.decode_attention_weights(c.q[:2].to(DEV), *args[1:], t(2 ** 31 - 1, -7), sm_scale=c.scale)
    assert bool(torch.isfinite(got).all()) and bool((got[1] == 0).all())
    # a table entry past the pool is no page
    c.table[0, 1] = 10 ** 6
    want, reach = oracle(c, c.table.shape[1] * 16)
    check(c, prefill(c), want, reach, "page past the pool")


def test_nan_of_a_visible_key_and_infinite_query():
    c = make(19, 4, 2, 64, 16, [50, 50], [50, 1], False)
    page = int(c.table[0, 1])
    c.k[page, 0, 4] = float("nan")  # key 20 of request 0, head 0
    got = prefill(c).cpu()
    assert bool(got[0, 0, :50].isnan().all()) and bool(torch.isfinite(got[0, 1]).all()) and bool(torch.isfinite(got[1]).all())
    assert bool((got[0, :, 50:] == 0).all())


def test_empty_batches():
    c = make(21, 4, 2, 64, 16, [50], [1], False)
    k = c.k.to(DEV)
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.decode_attention_weights(none, k, torch.zeros(0, 3, dtype=torch.int32, device=DEV), z,
                                        sm_scale=1.0).shape == (0, 2, 48)
    got = ops.prefill_attention_weights(none, k, c.table.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
                                        torch.full((1,), 50, dtype=torch.int32, device=DEV), max_q_len=0, sm_scale=1.0)
    assert got.shape == (1, 2, c.table.shape[1] * 16) and bool((got == 0).all())


def test_refusals():
    c = make(23, 8, 2, 64, 16, [50], [4], True)
    with pytest.raises(ValueError, match="k_scale"):
        prefill(types.SimpleNamespace(**{**vars(c), "ks": None}))
    with pytest.raises(ValueError, match="q_start"):
        prefill(types.SimpleNamespace(**{**vars(c), "start": [0, 5]}))
    with pytest.raises(ValueError, match="fp32"):
        prefill(c, weights=torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        prefill(c, weights=torch.zeros(1, 1, 64, device=DEV).expand(1, 2, 64))
    with pytest.raises(ValueError, match="bad sizes"):
        prefill(c, window=-1)


def test_graph_and_side_stream():
    c = make(25, 16, 8, 128, 16, [900, 130, 555], [1, 1, 1], True)
    p = make(27, 16, 8, 128, 16, [900, 130], [64, 20], False)
    dev = [t.to(DEV) for t in (c.q, c.k, c.table, torch.tensor(c.lens, dtype=torch.int32), c.ks)]
    pq = [t.to(DEV) for t in (p.q, p.k, p.table, torch.tensor(p.start, dtype=torch.int32),
                              torch.tensor(p.prior, dtype=torch.int32))]

    def both():
        return (ops.decode_attention_weights(*dev[:4], sm_scale=c.scale, k_scale=dev[4]),
                ops.prefill_attention_weights(*pq, max_q_len=64, sm_scale=p.scale))

    eager = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for _ in range(4):
        for t in outs:
            t.fill_(7.0)
        both()  # eager work of the same kind between the replays
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
