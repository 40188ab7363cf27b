"""ops.prefill_attention_weights and ops.decode_attention_weights where their forms could part from each other: requests on
one table row, values that are not finite, and sinks past every score. The tolerance is that of
test_gpu_attention_weights.py."""

from __future__ import annotations

import pytest
import torch

from sglang_neuron_amd import ops
from tests.conftest import announce
from tests.test_gpu_attention_weights import DEV, make

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
