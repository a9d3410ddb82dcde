"""The paged operators' checks that need no GPU: null arguments across the C
ABI, tensors that are not on a GPU, page bookkeeping."""

import pytest
import torch


def test_null_arguments_are_rejected(rtlib):
    assert rtlib.rt_paged_append(None, None, None, None) == -1
    assert rtlib.rt_paged_decode(None, None, None, None) == -1
    assert rtlib.rt_paged_prompt(None, None, None, None) == -1
    assert rtlib.rt_paged_evict(None, None, None, None) == -1
    assert rtlib.rt_paged_scratch(None, None, 0, None) == -1


def test_host_tensors_and_wrong_kinds_are_refused():
    from rich_triplet_b200 import paged

    pools = [torch.zeros(4, 2, 16, 64) for _ in range(2)]
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 2, 64), torch.zeros(1, 2, 64)
    for call in (lambda: paged.attend_decode(q, *pools, table, lens, scale=1.0),
                 lambda: paged.attend_prompt(q, table[0], 1, *pools, table, lens, scale=1.0),
                 lambda: paged.kv_append(*pools, k, k, table, lens),
                 lambda: paged.kv_evict(*pools, table, lens, torch.zeros(1, 2, 32), table, budget=8)):
        with pytest.raises(ValueError, match="one GPU"):
            call()
    with pytest.raises(ValueError, match="must be a tensor"):
        paged.kv_append(1, 2, k, k, table, lens)
    with pytest.raises(ValueError, match="num_pages, kv_heads"):
        paged.attend_decode(q, pools[0][0], pools[1][0], table, lens, scale=1.0)
    with pytest.raises(ValueError, match="f32, f16 or bf16"):
        paged.attend_decode(q, pools[0].int(), pools[1].int(), table, lens, scale=1.0)
    with pytest.raises(TypeError):
        paged.attend_decode(q, *pools, table, lens)  # no scale


def test_page_pool():
    from rich_triplet_b200.paged import PagePool

    p = PagePool(5)
    a, b = p.take(2), p.take(3)
    assert sorted(a + b) == [0, 1, 2, 3, 4] and p.free_pages == 0
    with pytest.raises(ValueError, match="1 pages wanted, 0 of 5 free"):
        p.take(1)
    p.give(b)
    assert p.free_pages == 3 and sorted(p.take(3)) == sorted(b)


def test_cache_bookkeeping_on_the_host():
    """Pages and lengths of PagedKvCache need no kernel."""
    from rich_triplet_b200.paged import PagedKvCache

    c = PagedKvCache(2, 3, 12, 8, 1, 64, 64, device="cpu")
    c.extend([9, 1, 0])
    assert c.lens == [9, 1, 0] and c.pool.free_pages == 9
    assert [[int(x) >= 0 for x in row[:3]] for row in c.page_table] == [[True, True, False], [True, False, False], [False] * 3]
    c.extend([30, 7, 1])
    assert c.lens == [39, 8, 1] and c.lens_device.tolist() == [39, 8, 1] and c.pool.free_pages == 12 - 7
    c.drop(window=10, sinks=3)  # the next token of sequence 0 sees from position 30 on, and 0 .. 2
    assert [p for p in range(5) if int(c.page_table[0, p]) >= 0] == [0, 3, 4]
    assert c.pool.free_pages == 12 - 5
    with pytest.raises(ValueError, match="extend"):
        c.extend([26, 0, 0])
    with pytest.raises(ValueError, match="pages wanted"):
        c.extend([0, 56, 56])
    assert c.lens == [39, 8, 1]
