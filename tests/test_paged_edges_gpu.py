"""Edges of the paged cache operators (rich_triplet_b200.paged): views that
overlap or repeat rows, infinities and NaN, weights far below the largest,
threads, streams and graphs, tables wider than the lengths.

Tolerances are those derived in test_paged_gpu.py, whose caches and 64-bit
definition are used here, except where a test says otherwise.
"""

import pytest
import torch

from test_paged_gpu import BF16, DEV, F16, F32, Cache, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,nq,nkv,d", [(BF16, 8, 4, 256), (F16, 8, 1, 64), (F32, 4, 2, 128)])
def test_decode_does_not_depend_on_where_pages_lie(dtype, nq, nkv, d):
    """Every row address is handed from one lane to the others: under another
    placement of the same pages the bits are the same, call after call."""
    from rich_triplet_b200 import paged

    lens = [1500, 1, 333, 8, 2049, 77]
    c = Cache(lens, nkv, d, 8, dtype)
    q = queries(len(lens), nq, d, dtype, 0, False)
    want = paged.attend_decode(q, *c.args(), scale=d ** -0.5)
    g = torch.Generator().manual_seed(5)
    for _ in range(40):
        to = torch.randperm(c.kp.shape[0], generator=g).to(DEV)
        kp, vp = torch.empty_like(c.kp), torch.empty_like(c.vp)
        kp[to], vp[to] = c.kp, c.vp
        table = torch.where(c.table >= 0, to[c.table.clamp(min=0).long()].int(), c.table)
        got = paged.attend_decode(q, kp, vp, table, c.lens_t, scale=d ** -0.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
