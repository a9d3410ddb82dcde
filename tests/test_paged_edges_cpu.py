"""Edges of the paged cache's host side: contexts, size limits of the C entry
points, bookkeeping of pages.  No GPU."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch


def test_forget_and_sync_without_a_context():
    """A device that no call has used has no context to wait for."""
    from rich_triplet_b200 import paged

    paged._ext.forget(5)
    assert paged._ext.sync(5) is None
    with pytest.raises(TypeError):
        paged._ext.sync()


class Kv(ctypes.Structure):
    """rt_paged_kv"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("slot_stride", ctypes.c_int64), ("num_pages", ctypes.c_int64),
                ("fmt", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
                ("table_width", ctypes.c_int32), ("num_seqs", ctypes.c_int32), ("lens", ctypes.c_void_p)]


class Attn(ctypes.Structure):
    """rt_paged_attn"""
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("q_row_stride", ctypes.c_int64),
                ("q_head_stride", ctypes.c_int64), ("out_row_stride", ctypes.c_int64),
                ("out_head_stride", ctypes.c_int64), ("lse", ctypes.c_void_p), ("lse_row_stride", ctypes.c_int64),
                ("rows", ctypes.c_int64), ("num_heads", ctypes.c_int32), ("window", ctypes.c_int32),
                ("sinks", ctypes.c_int32), ("max_new", ctypes.c_int32), ("scale", ctypes.c_float),
                ("mass_cap", ctypes.c_int32), ("q_start", ctypes.c_void_p), ("mass", ctypes.c_void_p),
                ("mass_seq_stride", ctypes.c_int64), ("mass_head_stride", ctypes.c_int64),
                ("scratch", ctypes.c_void_p), ("scratch_bytes", ctypes.c_uint64)]


SCRATCH = """
import ctypes, sys
sys.path[:0] = {path!r}
import test_paged_edges_cpu as t
from rich_triplet_b200._lib import lib
for kv, attn in {calls!r}:
    kv, a, n = t.Kv(**kv), t.Attn(**attn), ctypes.c_uint64(7)
    print(lib().rt_paged_scratch(ctypes.byref(kv), ctypes.byref(a), 0, ctypes.byref(n)), n.value)
"""


def test_scratch_of_any_sizes_answers():
    """In a process of its own: sizes that no call takes get an answer, not a hang."""

    def call(page, width, rows, heads):
        return (dict(fmt=0, kv_heads=2, head_dim=64, page_size=page, table_width=width, num_seqs=3),
                dict(rows=rows, num_heads=heads, mass=16, mass_cap=9))

    bad = [call(page, 5, 3, 4) for page in (2 ** 30 + 1, 2 ** 31 - 1, 512, 24, 0, -8)]
    bad += [call(256, 2 ** 31 - 1, 3, 4), call(256, -1, 3, 4), call(16, 5, -1, 4), call(16, 5, 3, 0)]
    bad += [call(256, 2 ** 23 - 1, 2 ** 27, 2 ** 20)]  # the product passes 64 bits
    here = os.path.dirname(os.path.abspath(__file__))
    code = SCRATCH.format(path=[here, os.path.dirname(here)], calls=[call(16, 5, 3, 4)] + bad)
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0, got.stderr
    got = [tuple(int(x) for x in line.split()) for line in got.stdout.splitlines()]
    # 3 x 4 rows of 5 pages of 16 positions, and their maxima and sums
    assert got[0] == (0, 256 + 3840)
    assert [status for status, _ in got[1:]] == [-4] * len(bad)


def cache(layers=2, sequences=3, pages=12, page=8, heads=1, d=64, max_len=64, **kw):
    from rich_triplet_b200.paged import PagedKvCache

    return PagedKvCache(layers, sequences, pages, page, heads, d, max_len, device="cpu", **kw)


def accounted(c):
    """Every page is in the table once or free once."""
    used = [int(p) for p in c.page_table.flatten() if p >= 0]
    assert torch.equal(c.page_table, c._table) and c.lens_device.tolist() == c.lens
    return sorted(used + c.pool._free) == list(range(c.pool.num_pages))


def test_extend_refuses_negative_counts():
    c = cache()
    c.extend([9, 1, 16])
    with pytest.raises(ValueError, match="negative counts"):
        c.extend([-9, 0, 0])
    assert c.lens == [9, 1, 16] and accounted(c)
    c.extend([7, 7, 1])
    assert c.lens == [16, 8, 17] and accounted(c)


def plain_evict(k, v, table, lens, mass, dst, *, budget, sinks=0, recent=0):
    """kv_evict in plain torch."""
    page = k.shape[2]
    kept = torch.full((len(lens), k.shape[1], budget), -1, dtype=torch.int32)
    out = torch.zeros_like(mass)
    for b, n in enumerate(lens.tolist()):
        for h in range(k.shape[1]):
            ends = [j for j in range(n) if j < sinks or j >= n - recent] if n > budget else range(n)
            rest = sorted(set(range(n)) - set(ends), key=lambda j: (-float(mass[b, h, j]), j))
            keep = sorted((list(ends) + rest)[:budget])
            for i, j in enumerate(keep):
                kept[b, h, i], out[b, h, i] = j, mass[b, h, j]
                for pool in (k, v):
                    pool[dst[b, i // page], h, i % page] = pool[table[b, j // page], h, j % page]
    return kept, lens.clamp(max=budget), out


def filled(monkeypatch, lens, **kw):
    from rich_triplet_b200 import paged

    monkeypatch.setattr(paged, "kv_evict", plain_evict)
    c = cache(sequences=len(lens), totals=True, **kw)
    c.extend(lens)
    g = torch.Generator().manual_seed(2)
    for b, n in enumerate(lens):
        c.mass[:, b, :, :n] = torch.rand(c.mass.shape[0], c.mass.shape[2], n, generator=g)
        for j in range(n):
            at = int(c.page_table[b, j // c.page_size]), slice(None), j % c.page_size
            for layer in range(c.k.shape[0]):
                c.k[layer][at] = 1000.0 * layer + 100 * b + j
                c.v[layer][at] = -(1000.0 * layer + 100 * b + j)
    return c


def check_trimmed(c, lens, before, kept, budget, sinks, recent):
    """The cache holds what a trim of `lens` positions with totals `before` leaves."""
    assert c.lens == [min(n, budget) for n in lens] and accounted(c)
    for layer in range(c.k.shape[0]):
        for b, n in enumerate(lens):
            m = min(n, budget)
            for h in range(c.k.shape[2]):
                ends = [j for j in range(n) if j < sinks or j >= n - recent] if n > budget else range(n)
                rest = sorted(set(range(n)) - set(ends), key=lambda j: (-float(before[layer, b, h, j]), j))
                keep = sorted((list(ends) + rest)[:budget])
                assert kept[layer][b, h].tolist() == keep + [-1] * (budget - m)
                assert c.mass[layer, b, h, :m].tolist() == [float(before[layer, b, h, j]) for j in keep]
                assert (c.mass[layer, b, h, m:] == 0).all()
                for i, j in enumerate(keep):
                    at = int(c.page_table[b, i // c.page_size]), h, i % c.page_size
                    assert (c.k[layer][at] == 1000.0 * layer + 100 * b + j).all()
                    assert (c.v[layer][at] == -(1000.0 * layer + 100 * b + j)).all()


def test_evict(monkeypatch):
    lens = [40, 7, 0, 16, 33]
    c = filled(monkeypatch, lens, pages=32, heads=2, dtype=torch.float32)
    before = c.mass.clone()
    check_trimmed(c, lens, before, c.evict(16, sinks=2, recent=5), 16, 2, 5)


def test_evict_that_is_refused_changes_nothing(monkeypatch):
    from rich_triplet_b200 import paged

    lens = [40, 7]
    c = filled(monkeypatch, lens, pages=20, dtype=torch.float32)
    mass, table = c.mass.clone(), c.page_table.clone()
    for kw in (dict(budget=16, sinks=10, recent=7), dict(budget=0), dict(budget=16, sinks=-1), dict(budget=16, recent=-1)):
        with pytest.raises(ValueError, match="must lie in"):
            c.evict(**kw)
    calls = []

    def fails_late(*a, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("a launch failed")
        return plain_evict(*a, **kw)

    monkeypatch.setattr(paged, "kv_evict", fails_late)
    with pytest.raises(RuntimeError, match="a launch failed"):
        c.evict(16)
    assert c.lens == lens and accounted(c) and torch.equal(c.mass, mass) and torch.equal(c.page_table, table)


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 30])
def test_evict_in_a_pool_with_few_free_pages(monkeypatch, spare):
    """Sequences take turns on the free pages; with none, one at a time goes
    through a copy outside the pool.  Those within the budget keep their pages."""
    lens = [40, 7, 0, 17, 33, 64]
    used = sum(-(-n // 8) for n in lens)
    c = filled(monkeypatch, lens, pages=used + spare, heads=2, dtype=torch.float32)
    before, short = c.mass.clone(), c.page_table[1].clone()
    assert c.pool.free_pages == spare
    check_trimmed(c, lens, before, c.evict(16, sinks=2, recent=5), 16, 2, 5)
    assert torch.equal(c.page_table[1], short)
    # 16 positions in 2 pages each now, but for 7 in one and none
    assert c.pool.num_pages - c.pool.free_pages == 9


def test_evict_after_dropped_pages(monkeypatch):
    """Dropped positions have no rows to keep: their slots read as zeros, and the
    page counts still add up, in a full pool too."""
    c = filled(monkeypatch, [64, 40], pages=13, dtype=torch.float32)
    c.drop(window=20)
    assert accounted(c)
    c.pool.take(c.pool.free_pages)  # someone else has the rest
    monkeypatch.setattr("rich_triplet_b200.paged.kv_evict", lambda k, v, table, lens, mass, dst, *, budget, **kw: (
        torch.zeros(len(lens), 1, budget, dtype=torch.int32), lens.clamp(max=budget), torch.zeros_like(mass)))
    c.evict(16)
    assert c.lens == [16, 16]
    used = [int(p) for p in c.page_table.flatten() if p >= 0]
    assert len(set(used)) == 4 and torch.equal(c.page_table, c._table)


def test_drop_takes_back_what_no_later_token_sees():
    """Any order of growth, windows and first tokens: the pages that one pass over
    every table entry would give back, once each."""
    import random

    rng = random.Random(3)
    for _ in range(60):
        c = cache(layers=1, sequences=3, pages=30, max_len=80)
        table = [[-1] * 10 for _ in range(3)]  # which entries hold a page
        for _ in range(25):
            if rng.random() < 0.6:
                counts = [rng.randint(0, min(9, 80 - n)) for n in c.lens]
                for b, (n, m) in enumerate(zip(c.lens, counts)):
                    for p in range(-(-n // 8), -(-(n + m) // 8)):
                        table[b][p] = 1
                c.extend(counts)
            else:
                window, sinks = rng.choice([0, 1, 5, 8, 20, 33, 70]), rng.choice([0, 0, 1, 8, 9, 30])
                if window:
                    for b, n in enumerate(c.lens):
                        for p in range(-(-sinks // 8), max(0, n + 1 - window) // 8):
                            table[b][p] = -1
                c.drop(window, sinks)
            assert [[min(1, max(-1, int(x))) if x < 0 else 1 for x in row] for row in c.page_table] == table
            assert accounted(c)
    for bad in ((-1, 0), (4, -1)):
        with pytest.raises(ValueError, match="negative"):
            c.drop(*bad)


def test_drop_every_step_costs_the_same_late_in_a_long_sequence():
    """A step's drop looks at the entries that it gives back, not at all of them."""
    seen = []

    class Watched(torch.Tensor):
        def __getitem__(self, at):
            seen.append(at)
            return super().__getitem__(at)

    c = cache(layers=1, sequences=8, pages=8 * 4200, max_len=32768)
    c.extend([32000] * 8)
    c.drop(1024, 4)
    c._table = c._table.as_subclass(Watched)
    for _ in range(32):
        c.extend([1] * 8)
        c.drop(1024, 4)
    assert len(seen) <= 2 * 8 * 32 // 8 + 8 and accounted(c)


def test_prompt_without_row_starts_is_refused():
    """Not taken for a decode step, which has none."""
    from rich_triplet_b200 import paged

    pools = [torch.zeros(4, 2, 16, 64) for _ in range(2)]
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="q_start must be a tensor"):
        paged.attend_prompt(torch.zeros(1, 2, 64), None, 1, *pools, table, lens, scale=1.0)


def test_model_refuses_budgets_that_no_trim_takes():
    """Before anything is made, not in the middle of the step that trims first."""
    from rich_triplet_b200.model import Config4
    from rich_triplet_b200.paged_model import PagedGemma3

    class Weights:
        cfg = Config4.tiny()

    for kw in (dict(budget=32), dict(budget=70, sinks=7), dict(budget=-1), dict(budget=64, recent=-1)):
        with pytest.raises(ValueError, match="must lie in 0..budget"):
            PagedGemma3(Weights, 1, 64, **kw)
