"""ops.prefill_attention_weights and ops.decode_attention_weights where their forms could part from each other: requests on
one table row, values that are not finite, and sinks past every score. The tolerance is that of
test_gpu_attention_weights.py."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_neuron_amd import ops
from tests.conftest import announce
from tests.test_gpu_attention_weights import DEV, check, few_rows, make, oracle, prefill

pytestmark = pytest.mark.gpu

# heads, requests and queries that take each form: scores in memory, scores in LDS, many rows (whole and in runs)
FORMS = [("scores", 8, 2, 3, 2, 600), ("lds", 8, 4, 64, 2, 2100), ("many", 8, 2, 3, 40, 600), ("runs", 64, 1, 2, 90, 300)]


def _table_call(c, table, q, starts, lens, queries):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    got = [ops.prefill_attention_weights(q, c.k.to(DEV), table, i32(starts), i32([n - queries for n in lens]),
                                         max_q_len=queries, sm_scale=c.scale)]
    got.append(ops.decode_attention_weights(q[:len(lens)], c.k.to(DEV), table, i32(lens), sm_scale=c.scale))
    return got


@pytest.mark.parametrize("form,H,G,R,queries,keys", FORMS, ids=[f[0] for f in FORMS])
def test_requests_on_one_table_row(form, H, G, R, queries, keys):
    """A table of one row for all requests (stride 0), and rows that overlap, give what their copies give."""
    announce(f"shared table row {form}")
    c = make(41, H, G, 64, 16, [keys], [queries], False)
    q = torch.randn(R * queries, H, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    lens = [keys - r % 5 for r in range(R)]
    starts = [r * queries for r in range(R + 1)]
    one = c.table.to(DEV)
    W = one.shape[1]
    long = torch.cat([one[0], one[0, :R]])
    for table in (one.expand(R, W), long.as_strided((R, W), (1, 1)), one[:, :1].expand(R, W)):
        assert table.stride(0) < W
        a = _table_call(c, table, q, starts, lens, queries)
        b = _table_call(c, table.contiguous(), q, starts, lens, queries)
        # (bits: the shifted rows bring the last page's empty slots, NaN, into view)
        assert all(torch.equal(x.view(torch.int32), y.view(torch.int32)) for x, y in zip(a, b))
    alone = _table_call(c, one.as_strided((1, W), (0, 1)), q[:queries], [0, queries], lens[:1], queries)
    whole = _table_call(c, one.contiguous(), q[:queries], [0, queries], lens[:1], queries)
    assert all(torch.equal(x, y) for x, y in zip(alone, whole)) and bool((whole[0] > 0).any())


def _compare(c, clean, sinks=None, window=0):
    """The oracle's NaN pattern, and its values elsewhere (``clean``: the same case without what is not finite, whose scores
    bound the rounding)."""
    width = c.table.shape[1] * c.P
    _, reach = oracle(clean, width, sinks=sinks, window=window)
    want, _ = oracle(c, width, sinks=sinks, window=window)
    got = prefill(c, sinks=None if sinks is None else sinks.to(DEV), window=window)
    assert torch.equal(got.isnan().cpu(), want.isnan())
    check(c, torch.where(got.isnan(), 0.0, got), want.nan_to_num(0.0), reach, "finite keys")
    return want


def _pair(build):
    return build(), build()


@pytest.mark.parametrize("name,build", [
    ("scores", lambda: make(43, 4, 2, 64, 16, [700, 60], [3, 1], False)),
    ("lds", lambda: few_rows(64, 8, 4, 64, 16, 2100, 3, False, seed=4)),
    ("many", lambda: make(43, 8, 2, 64, 16, [700, 60], [40, 3], False)),
    ("many-fp8", lambda: make(43, 6, 2, 128, 16, [900, 60], [70, 3], True)),
    ("runs", lambda: make(43, 64, 1, 64, 16, [300, 100], [90, 70], False)),
])
def test_a_query_that_is_nan_reaches_no_later_key(name, build):
    announce(f"NaN query {name}")
    c, clean = _pair(build)
    assert c.counts[0] > 1
    c.q[c.start[0], 1, 3] = float("nan")
    want = _compare(c, clean)
    first = c.lens[0] - c.counts[0]  # the NaN query's position
    assert bool(want[0, 0, :first + 1].isnan().any()) and bool(torch.isfinite(want[0, :, first + 1:]).all())


@pytest.mark.parametrize("name,build,window,key", [
    ("scores", lambda: make(47, 4, 2, 64, 16, [300, 60], [3, 1], False), 50, 249),
    ("lds", lambda: few_rows(64, 8, 4, 64, 16, 2100, 3, False, seed=4), 100, 1999),
    ("many", lambda: make(47, 8, 2, 64, 16, [600, 90], [600, 40], False), 100, 20),
    ("many-fp8", lambda: make(47, 8, 2, 128, 16, [600, 90], [600, 40], True), 30, 300),
    ("runs", lambda: make(47, 96, 2, 128, 16, [300, 40], [300, 40], False), 33, 60),
])
def test_a_key_that_is_nan_reaches_no_key_outside_its_windows(name, build, window, key):
    announce(f"NaN key {name}")
    c, clean = _pair(build)
    c.k[int(c.table[0, key // 16]), 0, key % 16, 5] = float("nan")
    want = _compare(c, clean, window=window)
    bad = want[0, 0].isnan().nonzero()[:, 0]
    # the queries that see it are at key .. key + window - 1 (the chunk's own ones), and so are the keys that they see
    lo, hi = max(key, c.lens[0] - c.counts[0]), min(key + window - 1, c.lens[0] - 1)
    assert bad.tolist() == list(range(max(lo - window + 1, 0), hi + 1))
    assert bool(torch.isfinite(want[0, 1]).all())


@pytest.mark.parametrize("name,build", [
    ("scores", lambda: make(53, 4, 2, 64, 16, [700, 60], [3, 1], False)),
    ("lds", lambda: few_rows(64, 8, 4, 64, 16, 2100, 1, False, seed=4)),
    ("many", lambda: make(53, 8, 2, 64, 16, [700, 400], [40, 300], False)),
    ("runs", lambda: make(53, 64, 1, 128, 16, [300, 200], [90, 70], False)),
])
def test_keys_whose_scores_are_minus_infinity(name, build):
    """They get nothing, and nothing from their rows is lost, where they fill a block of keys and where they do not."""
    announce(f"infinite keys {name}")
    c, clean = _pair(build)
    c.q[..., 0] = clean.q[..., 0] = -1.0
    keys = [*range(64, 192), 200, 203]
    for j in keys:
        c.k[int(c.table[0, j // 16]), :, j % 16, 0] = math.inf
    width = c.table.shape[1] * c.P
    _, reach = oracle(clean, width)
    want, _ = oracle(c, width)
    got = prefill(c)
    assert bool(torch.isfinite(got).all()) and bool((got[0, :, keys] == 0).all())
    check(c, got, want, reach, "beside them")


@pytest.mark.parametrize("form,H,G,R,queries,keys", FORMS, ids=[f[0] for f in FORMS])
def test_sinks_past_every_score(form, H, G, R, queries, keys):
    """A sink that is infinite, or finite and infinite in the log2 domain, leaves its head's keys nothing; one of the lowest
    value takes nothing."""
    announce(f"sinks {form}")
    c = few_rows(R, H, G, 64, 16, keys, queries, False, seed=6) if form in ("scores", "lds") else \
        make(59, H, G, 64, 16, [keys, 50, 70][:R], [queries, 3, 70][:R], False)
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(2))
    sinks[::4], sinks[1::8], sinks[2::8], sinks[3::8] = math.inf, 3.0e38, -math.inf, torch.finfo(torch.float32).min
    _compare(c, c, sinks=sinks)
    all_of = torch.full((H,), math.inf)
    got = prefill(c, sinks=all_of.to(DEV))
    assert bool((got == 0).all())


def test_bounds_past_32_bits():
    """A window, or a longest query count, that 32 bits do not hold bounds nothing."""
    c = make(61, 8, 2, 64, 16, [300, 40], [40, 3], False)
    dev = [t.to(DEV) for t in (c.q, c.k, c.table)]
    start, prior = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (c.start, c.prior))
    want = ops.prefill_attention_weights(*dev, start, prior, max_q_len=40, sm_scale=c.scale)
    check(c, want, *oracle(c, c.table.shape[1] * 16), "plain")
    for most in (2 ** 31, 2 ** 32 + 3, 2 ** 63):
        assert torch.equal(ops.prefill_attention_weights(*dev, start, prior, max_q_len=most, sm_scale=c.scale), want)
    windowed = ops.prefill_attention_weights(*dev, start, prior, max_q_len=40, sm_scale=c.scale, window=2 ** 31 - 1)
    for window in (2 ** 31, 2 ** 32 + 2, 2 ** 63):
        got = ops.prefill_attention_weights(*dev, start, prior, max_q_len=40, sm_scale=c.scale, window=window)
        assert torch.equal(got, windowed)
        check(c, got, *oracle(c, c.table.shape[1] * 16), "no key is outside")
