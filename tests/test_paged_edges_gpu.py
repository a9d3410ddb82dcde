"""Edges of the paged cache operators (rich_triplet_b200.paged): views that
overlap or repeat rows, infinities and NaN, weights far below the largest,
threads, streams and graphs, tables wider than the lengths.

Tolerances are those derived in test_paged_gpu.py, whose caches and 64-bit
definition are used here, except where a test says otherwise.
"""

import math
import threading

import pytest
import torch

from rich_triplet_b200._lib import RtError
from test_paged_gpu import BF16, DEV, F16, F32, U, Cache, close, e32, is_visible, queries, reference

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


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_table_row_for_all_sequences(dtype):
    """Samples that share one prompt's pages: an expanded table (row stride 0),
    and a view whose rows overlap, give what a copy of the rows gives."""
    from rich_triplet_b200 import paged

    c = Cache([500], 2, 64, 16, dtype, spare=12)
    lens = torch.tensor([500, 17, 0, 333], dtype=torch.int32, device=DEV)
    shared = c.table.expand(4, -1)
    sliding = torch.as_strided(c.table, (4, 20), (3, 1))  # sequence b starts three pages after b - 1
    assert shared.stride(0) == 0 and sliding.stride(0) < sliding.size(1)
    for table, n in ((shared, lens), (sliding, lens.clamp(max=320))):
        copied = table.clone(memory_format=torch.contiguous_format)
        q = queries(4, 4, 64, dtype, 1, False)
        mass = [torch.zeros(4, 2, 512, device=DEV) for _ in range(4)]
        got = paged.attend_decode(q, c.kp, c.vp, table, n, scale=0.125, mass=mass[0])
        want = paged.attend_decode(q, c.kp, c.vp, copied, n, scale=0.125, mass=mass[1])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(mass[0], mass[1])
        start = torch.tensor([0, 5, 9, 9, 20], dtype=torch.int32, device=DEV)
        q = queries(20, 4, 64, dtype, 2, False)
        got = paged.attend_prompt(q, start, 11, c.kp, c.vp, table, n, scale=0.125, mass=mass[2])
        want = paged.attend_prompt(q, start, 11, c.kp, c.vp, copied, n, scale=0.125, mass=mass[3])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(mass[2], mass[3])
        dst = c.free[:12].view(4, 3).to(DEV)
        total = torch.rand(4, 2, 512, device=DEV)
        kept = paged.kv_evict(c.kp, c.vp, table, n, total, dst, budget=40)
        again = paged.kv_evict(c.kp, c.vp, copied, n, total, dst, budget=40)
        assert all(torch.equal(x, y) for x, y in zip(kept, again))


def refused(error, match, fn, *args, **kw):
    with pytest.raises(error, match=match):
        fn(*args, **kw)


def test_outputs_whose_rows_overlap_are_refused():
    """Expanded totals and outputs would be written by several CTAs at once."""
    from rich_triplet_b200 import paged

    c = Cache([40, 9], 2, 64, 16, BF16)
    q = queries(2, 4, 64, BF16, 0, False)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    one = torch.zeros(1, 1, 50, device=DEV)
    wide = torch.zeros(400, device=DEV)
    for mass in (one.expand(2, 2, -1), one.expand(2, 1, -1).repeat(1, 2, 1)[:1].expand(2, -1, -1),
                 torch.as_strided(wide, (2, 2, 50), (49, 100, 1)), torch.as_strided(wide, (2, 2, 50), (60, 49, 1))):
        refused(RtError, "rows of mass overlap", paged.attend_decode, q, *c.args(), scale=0.1, mass=mass)
        refused(RtError, "rows of mass overlap", paged.attend_prompt, q, start, 1, *c.args(), scale=0.1, mass=mass)
    for out in (torch.zeros(1, 4, 64, dtype=BF16, device=DEV).expand(2, -1, -1),
                torch.zeros(2, 1, 64, dtype=BF16, device=DEV).expand(-1, 4, -1)):
        refused(RtError, "rows of out overlap", paged.attend_decode, q, *c.args(), scale=0.1, out=out)
        refused(RtError, "rows of out overlap", paged.attend_prompt, q, start, 1, *c.args(), scale=0.1, out=out)
    # rows that lie apart in any order are taken
    want = torch.zeros(2, 2, 50, device=DEV)
    o, z = paged.attend_decode(q, *c.args(), scale=0.1, mass=want)
    for mass in (torch.zeros(2, 2, 50, device=DEV).transpose(0, 1), torch.as_strided(wide, (2, 2, 50), (51, 150, 1)),
                 torch.zeros(5, 3, 70, device=DEV)[1:4:2, 1:, 8:58]):
        paged.attend_decode(q, *c.args(), scale=0.1, mass=mass)
        assert torch.equal(mass, want)
    out = torch.zeros(4, 2, 64, dtype=BF16, device=DEV).transpose(0, 1)
    assert torch.equal(paged.attend_decode(q, *c.args(), scale=0.1, out=out)[0], o) and torch.equal(out, o)
    # one sequence: its stride says nothing
    c = Cache([40], 1, 64, 16, BF16)
    mass = torch.as_strided(wide, (1, 1, 50), (0, 0, 1)).zero_()
    paged.attend_decode(q[:1], *c.args(), scale=0.1, mass=mass)
    assert abs(float(mass.sum()) - 4) < 1e-3


def test_a_closed_context_is_not_used_again():
    from rich_triplet_b200 import paged

    c = Cache([300, 41], 2, 128, 16, BF16)
    q = queries(2, 4, 128, BF16, 0, False)
    want = paged.attend_decode(q, *c.args(), scale=0.1)
    ctx = paged.context(DEV)
    assert paged.context("cuda:0") is ctx
    ctx.close()
    ctx.close()
    got = paged.attend_decode(q, *c.args(), scale=0.1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert paged.context(DEV) is not ctx
    paged.context(DEV).sync()


def test_threads_and_streams_at_once():
    """Four threads, each with its own stream, and two that share one: splits and
    joins of one stream do not touch another's."""
    from rich_triplet_b200 import paged

    c = Cache([3000, 700, 64, 1], 2, 128, 32, BF16)
    start = torch.tensor([0, 8, 16, 24, 25], dtype=torch.int32, device=DEV)
    shared = torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in range(4)] + [shared, shared]
    qd = [queries(4, 8, 128, BF16, i, False) for i in range(6)]
    qp = [queries(25, 8, 128, BF16, 50 + i, False) for i in range(6)]
    torch.cuda.synchronize()

    def once(i):
        mass = torch.zeros(4, 2, 3000, device=DEV)
        a = paged.attend_decode(qd[i], *c.args(), scale=0.1, mass=mass)
        b = paged.attend_prompt(qp[i], start, 8, *c.args(), scale=0.1, mass=mass)
        return (*a, *b, mass)

    want = [once(i) for i in range(6)]
    torch.cuda.synchronize()
    wrong, contexts = [], set()

    def work(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(30):
                    got = once(i)
                    if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                        wrong.append(i)
            contexts.add(id(paged.context(DEV)))
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(contexts) == 1
    paged.context(DEV).sync()


def test_a_graph_outlives_the_thread_that_captured_it():
    """Its kernels use the workspace of the stream, which is still there."""
    from rich_triplet_b200 import paged

    c = Cache([4000, 33], 2, 128, 16, F16)
    q = queries(2, 4, 128, F16, 0, False)
    want, _ = paged.attend_decode(q, *c.args(), scale=0.1)
    torch.cuda.synchronize()
    made = {}

    def capture():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            paged.attend_decode(q, *c.args(), scale=0.1)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out, _ = paged.attend_decode(q, *c.args(), scale=0.1)
        made.update(graph=g, out=out, stream=s)

    t = threading.Thread(target=capture)
    t.start()
    t.join()
    for _ in range(3):
        made["out"].zero_()
        made["graph"].replay()
        torch.cuda.synchronize()
        assert torch.equal(made["out"], want)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_row_starts_outside_the_rows(dtype):
    """q_start is read on the device: sequences that begin before row 0 or end
    past the last row read and write no row that is not there."""
    from rich_triplet_b200 import paged

    c = Cache([40, 50, 60], 2, 64, 16, dtype)
    room = torch.full((30, 4, 64), 5.0, dtype=dtype, device=DEV)
    q = queries(30, 4, 64, dtype, 0, False)[10:20]
    out = room[10:20]
    mass = torch.zeros(3, 2, 60, device=DEV)
    for starts in ([-7, -2, 3, 10], [-9, 4, 4, 1000], [12, 15, 20, 25]):
        room.fill_(5.0)
        mass.zero_()
        start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        _, lse = paged.attend_prompt(q, start, 10, *c.args(), scale=0.1, mass=mass, out=out)
        assert (room[:10] == 5).all() and (room[20:] == 5).all()
        for b in range(3):
            first, end = starts[b], min(starts[b + 1], 10)
            # token i of the starts[b + 1] - first ones is at position c.lens[b] - (starts[b + 1] - first) + i
            rows = [r for r in range(max(0, first), end) if c.lens[b] - starts[b + 1] + r >= 0] if first >= 0 else []
            assert abs(float(mass[b].sum()) - 4 * len(rows)) < 1e-2
            assert torch.isfinite(lse[rows]).all()
        k = torch.randn(10, 2, 64, device=DEV)
        before = c.kp.clone()
        paged.kv_append(c.kp, c.vp, k, k, c.table, c.lens_t, q_start=start)
        c.kp.copy_(before)
        c.vp.copy_(before)


def test_evict_budget_at_the_limit():
    """Loops over a row of nearly 2^31 entries end at its end (the kept positions
    take 8.6 GB)."""
    from rich_triplet_b200 import paged

    most = 2 ** 31 - 257
    c = Cache([50, 0], 1, 64, 256, F16, spare=3)
    dst = torch.full((1, 2 ** 23 - 1), int(c.free[0]), dtype=torch.int32, device=DEV)
    mass = torch.rand(1, 1, 50, device=DEV)
    one = (c.kp, c.vp, c.table[:1], c.lens_t[:1])
    kept, lens, out = paged.kv_evict(*one, mass, dst, budget=most)
    assert lens.tolist() == [50] and torch.equal(out, mass)
    assert kept[0, 0, :50].tolist() == list(range(50))
    assert int(kept[0, 0, 50:].max()) == -1 and int(kept[0, 0, 50:].min()) == -1
    del kept
    torch.cuda.empty_cache()
    dst = torch.zeros(1, 2 ** 23, dtype=torch.int32, device=DEV)
    refused(RtError, "at most 2147483391 positions", paged.kv_evict, *one, mass, dst, budget=most + 1)
    torch.cuda.empty_cache()


def test_prompt_totals_read_the_queries_after_the_outputs():
    """An output over the queries is refused where the totals need them again; one
    beside them in the same rows is taken."""
    from rich_triplet_b200 import paged

    c = Cache([40, 9], 2, 64, 16, BF16)
    start = torch.tensor([0, 20, 26], dtype=torch.int32, device=DEV)
    wide = torch.randn(26, 10, 64, device=DEV).to(BF16)
    q = wide[:, 1:5]
    mass = torch.zeros(2, 2, 40, device=DEV)
    o, z = paged.attend_prompt(q.clone(), start, 20, *c.args(), scale=0.1, mass=mass)
    for out in (q, wide[:, 2:6], wide[:, :8:2]):
        refused(RtError, "out overlaps q", paged.attend_prompt, q, start, 20, *c.args(), scale=0.1, mass=mass.clone(),
                out=out)
    for q2, out in ((q, wide[:, 5:9]), (wide[:, :8:2], wide[:, 1:9:2]), (wide.view(260, 64)[:104].view(26, 4, 64),
                                                                       wide.view(260, 64)[104:208].view(26, 4, 64))):
        q2.copy_(torch.randn(26, 4, 64, device=DEV))
        got = [torch.zeros_like(mass) for _ in range(2)]
        want, _ = paged.attend_prompt(q2.clone(), start, 20, *c.args(), scale=0.1, mass=got[0])
        paged.attend_prompt(q2, start, 20, *c.args(), scale=0.1, mass=got[1], out=out)
        assert torch.equal(out, want) and torch.equal(got[0], got[1])
    # without totals, and for single tokens, every query is read before an output is written
    x = wide[:, 1:5].clone()
    assert torch.equal(paged.attend_prompt(x, start, 20, *c.args(), scale=0.1, out=x)[0],
                       paged.attend_prompt(wide[:, 1:5], start, 20, *c.args(), scale=0.1)[0])


def check_beside_nan(dtype, nq, nkv, d, lens, new, bad, window=0, sinks=0):
    """Prompt rows of which those in `bad` (row, head) have a NaN query: NaN there,
    the definition elsewhere, totals NaN where such a token sees a position."""
    from rich_triplet_b200 import paged

    c = Cache(lens, nkv, d, 32, dtype)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = queries(starts[-1], nq, d, dtype, 3, False)
    for r, h in bad:
        q[r, h, (r * 7 + h) % d] = float("nan")
    mass = torch.zeros(len(lens), nkv, max(lens), device=DEV)
    start = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out, lse = paged.attend_prompt(q, start, max(new), *c.args(), scale=d ** -0.5, window=window, sinks=sinks, mass=mass)
    for b, (n, m) in enumerate(zip(lens, new)):
        t = torch.arange(n - m, n, device=DEV)
        rows = slice(starts[b], starts[b + 1])
        o, ob, z, zb, _, _ = reference(c, b, q[rows], t, d ** -0.5, window, sinks)
        nan = torch.isnan(z)
        assert nan.any() == any(starts[b] <= r < starts[b + 1] for r, _ in bad)
        assert torch.equal(torch.isnan(lse[rows]), nan)
        assert torch.equal(torch.isnan(out[rows]), nan[..., None].expand(-1, -1, d))
        close(lse[rows][~nan], z[~nan], zb[~nan], f"lse of sequence {b}")
        close(out[rows][~nan], o[~nan], ob[~nan], f"out of sequence {b}")
        # the totals: of each token's weights where it sees a position
        j = torch.arange(n, device=DEV)
        seen = is_visible(t, j, window, sinks)
        touched = (seen[:, None, :] & nan.view(m, nkv, -1).any(-1)[..., None]).any(0)
        assert torch.equal(torch.isnan(mass[b, :, :n]), touched)
        # positions that no NaN token sees: the other tokens' weights
        clean = q[rows].clone()
        clean[nan] = 0
        _, _, _, _, w, wb = reference(c, b, clean, t, d ** -0.5, window, sinks)
        close(mass[b, :, :n][~touched], w[~touched], wb[~touched], f"mass of sequence {b}")


@pytest.mark.parametrize("dtype,nq,nkv,d", [(BF16, 8, 4, 256), (F16, 4, 2, 128), (BF16, 8, 1, 64), (F32, 4, 2, 64),
                                            (F16, 3, 1, 128)])
def test_prompt_queries_with_nan(dtype, nq, nkv, d):
    # a long prompt, a short one on a filled cache (its walk is split), one without NaN
    check_beside_nan(dtype, nq, nkv, d, [300, 2000, 70], [300, 5, 9], [(0, 0), (100, 1), (131, 2), (301, 0)])
    check_beside_nan(dtype, nq, nkv, d, [300, 700], [300, 8], [(40, 0), (305, 1)], window=50, sinks=3)


@pytest.mark.parametrize("dtype,d", [(BF16, 256), (F16, 128), (F32, 64)])
def test_prompt_keys_with_nan_or_infinity(dtype, d):
    """Tokens that see such a key get NaN, the earlier ones of the same tile do not."""
    from rich_triplet_b200 import paged

    for value in (float("nan"), float("inf")):
        c = Cache([200], 2, d, 16, dtype)
        c.kp[c.table[0, 150 // 16].long(), 1, 150 % 16, 5] = value
        q = queries(200, 4, d, dtype, 0, False)
        q[:, :, 5] = q[:, :, 5].abs() + 0.5  # infinity times zero or a negative number is another case
        start = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
        mass = torch.zeros(1, 2, 200, device=DEV)
        out, lse = paged.attend_prompt(q, start, 200, *c.args(), scale=0.1, mass=mass)
        assert torch.isnan(out[150:, 2:]).all() and torch.isfinite(out[:150]).all() and torch.isfinite(out[:, :2]).all()
        assert torch.isfinite(lse[:150]).all() and torch.isfinite(lse[:, :2]).all() and not torch.isfinite(lse[150:, 2:]).any()
        assert torch.isfinite(mass[:, 0]).all() and torch.isnan(mass[:, 1, :151]).all()


@pytest.mark.parametrize("dtype,nq,nkv,d", [(BF16, 8, 4, 256), (F16, 16, 1, 128), (F32, 4, 2, 64), (F16, 8, 1, 64)])
def test_decode_queries_with_nan(dtype, nq, nkv, d):
    from rich_triplet_b200 import paged

    lens = [1, 5, 300, 20000]
    c = Cache(lens, nkv, d, 32, dtype)
    q = queries(4, nq, d, dtype, 3, False)
    q[0, 0], q[2, nq - 1, 3], q[3, 1, 9] = float("nan"), float("nan"), float("nan")
    mass = torch.zeros(4, nkv, 20000, device=DEV)
    out, lse = paged.attend_decode(q, *c.args(), scale=d ** -0.5, mass=mass)
    for b, n in enumerate(lens):
        o, ob, z, zb, w, wb = reference(c, b, q[b:b + 1], torch.tensor([n - 1], device=DEV), d ** -0.5, 0, 0)
        nan = torch.isnan(z)
        assert torch.equal(torch.isnan(lse[b:b + 1]), nan)
        assert torch.equal(torch.isnan(out[b:b + 1]), nan[..., None].expand(-1, -1, d))
        close(lse[b:b + 1][~nan], z[~nan], zb[~nan], f"lse of sequence {b}")
        close(out[b:b + 1][~nan], o[~nan], ob[~nan], f"out of sequence {b}")
        touched = torch.isnan(w)
        assert torch.equal(torch.isnan(mass[b, :, :n]), touched) and (mass[b, :, n:] == 0).all()
        close(mass[b, :, :n][~touched], w[~touched], wb[~touched], f"mass of sequence {b}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scores_of_minus_infinity(dtype):
    """Every visible score -inf: nothing carries weight, as with nothing visible."""
    from rich_triplet_b200 import paged

    c = Cache([30, 40], 1, 64, 16, dtype)
    q = queries(2, 2, 64, dtype, 0, False)
    # over an f32 cache a product that overflows: an infinite element would have parts that are NaN
    c.kp[c.table[0, :2].long(), 0, :, 0] = -2.0 ** 120 if dtype == F32 else -float("inf")
    q[:1, :, 0] = 2.0 ** 120 if dtype == F32 else 1.0
    mass = torch.zeros(2, 1, 40, device=DEV)
    out, lse = paged.attend_decode(q, *c.args(), scale=0.1, mass=mass)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and (mass[0] == 0).all()
    assert torch.isfinite(lse[1]).all() and abs(float(mass[1].sum()) - 2) < 1e-3
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    mass.zero_()
    out, lse = paged.attend_prompt(q, start, 1, *c.args(), scale=0.1, mass=mass)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and (mass[0] == 0).all()
    assert torch.isfinite(lse[1]).all() and abs(float(mass[1].sum()) - 2) < 1e-3


@pytest.mark.parametrize("nq,nkv,d", [(4, 1, 64), (8, 1, 128), (12, 1, 256), (2, 1, 256)])
@pytest.mark.parametrize("below", [20.0, 24.6, 25.3])
@pytest.mark.parametrize("at", [0, -1])
def test_f16_weights_far_below_the_largest(nq, nkv, d, below, at):
    """One position 2^below heavier than each of 131070 others, which hold the
    only values that are not 0: their share of the output must not be lost.

    Weights are taken 2^7 above the largest one, so f16's smallest step rounds
    each by at most 2^-25 2^-7, and all of them by n 2^-32 of the sum, which is at
    least the largest weight; the rest of the bound is that of every output."""
    from rich_triplet_b200 import paged

    n, page = 131071, 256
    scale = d ** -0.5
    c = Cache.__new__(Cache)
    c.lens, c.page, c.dtype, c.nkv, c.d = [n], page, F16, nkv, d
    k = torch.zeros(nkv, n, d, dtype=F16, device=DEV)
    v = torch.ones(nkv, n, d, dtype=F16, device=DEV)
    k[:, at, 0], v[:, at] = 8.0, 0.0
    c.k, c.v = [k.double()], [v.double()]
    pages = -(-n // page)
    kp, vp = (torch.nn.functional.pad(x, (0, 0, 0, pages * page - n)).view(nkv, pages, page, d).transpose(0, 1).contiguous()
              for x in (k, v))
    table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.zeros(3, nq, d, dtype=F16, device=DEV)
    q[:, :, 0] = below * math.log(2.0) / 8.0 / scale
    u, e = 2.0 ** -11, e32(n)

    def check(out, lse, t, what):
        o, _, z, zb, _, _ = reference(c, 0, q[:len(t)], t, scale, 0, 0)
        delta = 2 * e32(d) * below  # the one product's size
        A = o.abs()
        bound = u * (o.abs() + A) + (2 * delta + 2 * e) * A + n * 2.0 ** -32 + 2.0 ** -25
        close(out, o.expand_as(out), bound.expand_as(out), what)
        close(lse, z.expand_as(lse), zb.expand_as(lse), what + " lse")
        assert float((o - bound).min()) > 0  # nothing would not do

    out, lse = paged.attend_decode(q[:1], kp, vp, table, lens, scale=scale)
    check(out, lse, torch.tensor([n - 1], device=DEV), "decode")
    # sequences on the same pages, so many that hardly one is split over CTAs
    many = 300
    shared = (kp, vp, table.expand(many, -1), lens.repeat(many))
    qs = q[:1].expand(many, -1, -1)
    out, lse = paged.attend_decode(qs, *shared, scale=scale)
    check(out, lse, torch.tensor([n - 1], device=DEV), "decode of many")
    start = torch.arange(many + 1, dtype=torch.int32, device=DEV)
    out, lse = paged.attend_prompt(qs, start, 1, *shared, scale=scale)
    check(out, lse, torch.tensor([n - 1], device=DEV), "prompt of many")
    if at == 0:  # every token sees the heavy position
        start = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
        out, lse = paged.attend_prompt(q, start, 3, kp, vp, table, lens, scale=scale)
        check(out, lse, torch.arange(n - 3, n, device=DEV), "prompt")


@pytest.mark.parametrize("window,sinks", [(0, 0), (1000, 200)])
def test_totals_of_more_positions_than_32_bits_hold_rows(window, sinks):
    """2^27 and some positions times 16 heads pass 2^31 (all on one page of 256
    rows, so the weights of a slot are equal everywhere)."""
    from rich_triplet_b200 import paged

    n, page, d, G = 2 ** 27 + 2 ** 12, 256, 64, 16
    g = torch.Generator().manual_seed(1)
    kp, vp = (torch.randn(1, 1, page, d, generator=g).to(DEV).to(BF16) for _ in range(2))
    table = torch.zeros(1, n // page, dtype=torch.int32, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = queries(2, G, d, BF16, 0, False)
    start = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    mass = torch.zeros(1, 1, n, device=DEV)
    paged.attend_prompt(q, start, 2, kp, vp, table, lens, scale=0.125, window=window, sinks=sinks, mass=mass)
    s = torch.exp(torch.einsum("tgd,pd->tgp", q.double(), kp[0, 0].double()) * 0.125)  # of a slot
    want = torch.zeros(n, dtype=torch.float64, device=DEV)
    for i in range(2):
        t = n - 2 + i
        count = torch.zeros(n, dtype=torch.bool, device=DEV)
        if window:
            count[:sinks] = True
            count[t + 1 - window:t + 1] = True
        else:
            count[:t + 1] = True
        seen = count.view(-1, page)
        total = (seen.sum(0).double()[None] * s[i]).sum(1, keepdim=True)
        want += (seen * (s[i] / total).sum(0)).flatten()
    got = mass[0, 0].double()
    same = bool(((got > 0) == (want > 0)).all())
    assert same
    # relative: a score's error, 2 e32(d) of at most 64 x 5 x 5 x 0.125, and 2^16 additions to a row's sum
    worst = float(((got - want).abs() - want * 1e-2).max())
    assert worst <= 0
    assert abs(float(got.sum()) - 2 * G) < 0.1
    del mass, got, want
    torch.cuda.empty_cache()


@pytest.mark.parametrize("spare", [0, 3, 60])
def test_cache_trims_in_full_pools(spare):
    """PagedKvCache.evict with none, a few and enough free pages: the rows and
    totals of kv_evict."""
    from rich_triplet_b200 import paged

    lens, page, d = [700, 90, 0, 301, 1000], 16, 64
    used = sum(-(-n // page) for n in lens)
    c = paged.PagedKvCache(2, 5, used + spare, page, 2, d, 1024, BF16, totals=True)
    c.extend(lens)
    k = torch.randn(2, c.pool.num_pages, 2, page, d, device=DEV).to(BF16)
    c.k.copy_(k)
    c.v.copy_(-k)
    live = torch.arange(1024, device=DEV) < c.lens_device[:, None, None]
    c.mass.copy_(torch.rand(2, 5, 2, 1024, device=DEV) * live)
    want = []
    for i in range(2):  # all five, into pages behind the pool's
        room = [torch.cat([x[i], torch.zeros(5 * 8, 2, page, d, dtype=BF16, device=DEV)]) for x in (c.k, c.v)]
        dst = torch.arange(c.pool.num_pages, c.pool.num_pages + 40, dtype=torch.int32, device=DEV).view(5, 8)
        want.append((*paged.kv_evict(*room, c.page_table, c.lens_device, c.mass[i], dst, budget=120, sinks=4, recent=30),
                     room, dst))
    kept = c.evict(120, sinks=4, recent=30)
    assert c.lens == [120, 90, 0, 120, 120]
    for i, (positions, lens_t, mass, room, dst) in enumerate(want):
        assert torch.equal(kept[i], positions) and torch.equal(c.lens_device, lens_t) and torch.equal(c.mass[i], mass)
        for b, n in enumerate(c.lens):
            j = torch.arange(n, device=DEV)
            for x, y in zip((c.k[i], c.v[i]), room):
                assert torch.equal(x[c.page_table[b, j // page].long(), :, j % page], y[dst[b, j // page].long(), :, j % page])
    used = [int(p) for p in c.page_table.flatten() if p >= 0]
    assert sorted(used + c.pool._free) == list(range(c.pool.num_pages))


def test_gradients_are_refused_not_dropped():
    from rich_triplet_b200 import paged

    c = Cache([40, 9], 2, 64, 16, F32, spare=2)
    kp, vp, table, lens = c.args()
    q, k = queries(2, 4, 64, F32, 0, False), torch.randn(2, 2, 64, device=DEV)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    mass = torch.zeros(2, 2, 50, device=DEV)
    dst = c.free[:2].view(2, 1).to(DEV)

    def grad(x):
        return x.detach().clone().requires_grad_()

    calls = [lambda: paged.attend_decode(grad(q), kp, vp, table, lens, scale=0.1),
             lambda: paged.attend_decode(grad(q) * 2, kp, vp, table, lens, scale=0.1),
             lambda: paged.attend_decode(q, grad(kp), vp, table, lens, scale=0.1),
             lambda: paged.attend_decode(q, kp, vp, table, lens, scale=0.1, mass=grad(mass)),
             lambda: paged.attend_prompt(q, start, 1, kp, grad(vp), table, lens, scale=0.1),
             lambda: paged.attend_prompt(grad(q), start, 1, kp, vp, table, lens, scale=0.1),
             lambda: paged.kv_append(kp, vp, grad(k), k, table, lens),
             lambda: paged.kv_append(kp, vp, k, grad(k), table, lens),
             lambda: paged.kv_evict(kp, vp, table, lens, grad(mass), dst, budget=8)]
    for call in calls:
        refused(ValueError, "not differentiable", call)
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_of_extents_of_one_say_nothing(dtype):
    """One row, head or page: torch gives its stride any value."""
    from rich_triplet_b200 import paged

    c = Cache([40], 1, 64, 64, dtype, spare=1)
    kp, vp = c.kp[c.table[0, :1].long()], c.vp[c.table[0, :1].long()]  # one page
    table = torch.zeros_like(c.table)
    q = queries(1, 4, 64, dtype, 0, False)
    start = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    mass = torch.zeros(2, 1, 1, 40, device=DEV)
    want = paged.attend_decode(q, kp, vp, table, c.lens_t, scale=0.1, mass=mass[0])

    def odd(x, *strides):
        return torch.as_strided(x, x.shape, strides)

    kp, vp = odd(kp, 3, 5, 64, 1), odd(vp, 7, 9, 64, 1)
    for q1, out in ((odd(q, 259, 64, 1), None), (q, odd(torch.zeros_like(q), 1, 64, 1))):
        got = paged.attend_decode(q1, kp, vp, table, c.lens_t, scale=0.1, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = paged.attend_prompt(q1, start, 1, kp, vp, table, c.lens_t, scale=0.1, mass=mass[1].zero_(), out=out)
        assert torch.allclose(got[0], want[0], rtol=0.02, atol=0.02) and torch.allclose(mass[1], mass[0], rtol=1e-3)
    one = odd(q[:, :1], 3, 5, 1)
    got = paged.attend_decode(one, kp, vp, table, c.lens_t, scale=0.1)
    assert torch.allclose(got[0], want[0][:, :1], rtol=0.02, atol=0.02)
    k = torch.randn(1, 1, 64, device=DEV)
    paged.kv_append(kp, vp, odd(k, 3, 5, 1), odd(k, 2, 1, 1), table, c.lens_t)
    assert torch.equal(kp[0, 0, 39], k[0, 0].to(dtype)) and torch.equal(vp[0, 0, 39], k[0, 0].to(dtype))
    # larger extents count
    c = Cache([40, 9], 2, 64, 16, dtype)
    q = torch.zeros(2, 259, dtype=dtype, device=DEV)[:, :256].view(2, 4, 64)
    refused(RtError, "multiples of 16 bytes", paged.attend_decode, q, *c.args(), scale=0.1)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_graphs_of_every_operator(dtype):
    """Append, decode and prompt with totals and eviction in one captured graph,
    replayed with other lengths and rows: the bits of plain calls."""
    from rich_triplet_b200 import paged

    nkv, d, page = 2, 64, 16
    c = Cache([300, 64, 200], nkv, d, page, dtype, spare=24)
    dst = c.free[:24].view(3, 8).to(DEV)
    q, k = queries(3, 4, d, dtype, 0, False), torch.randn(3, nkv, d, device=DEV)
    qp = queries(12, 4, d, dtype, 1, False)
    start = torch.tensor([0, 5, 6, 12], dtype=torch.int32, device=DEV)
    kp, vp, lens = torch.empty_like(c.kp), torch.empty_like(c.vp), c.lens_t.clone()

    def calls():
        mass = torch.zeros(3, nkv, 320, device=DEV)
        paged.kv_append(kp, vp, k, k, c.table, lens)
        a = paged.attend_decode(q, kp, vp, c.table, lens, scale=0.1, window=150, sinks=3, mass=mass)
        b = paged.attend_prompt(qp, start, 6, kp, vp, c.table, lens, scale=0.1, mass=mass)
        e = paged.kv_evict(kp, vp, c.table, lens, mass, dst, budget=120, sinks=3, recent=9)
        return (*a, *b, mass, *e)

    def fill(n, seed):
        kp.copy_(c.kp)
        vp.copy_(c.vp)
        lens.copy_(torch.tensor(n))
        g = torch.Generator().manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=g))
        qp.copy_(torch.randn(qp.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fill([300, 64, 200], 0)
        calls()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = calls()
    for n, seed in (([300, 64, 200], 1), ([121, 7, 199], 2), ([290, 60, 6], 3)):
        fill(n, seed)
        want = [x.clone() for x in calls()]
        pools = kp.clone(), vp.clone()
        fill(n, seed)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip((*got, kp, vp), (*want, *pools)):
            assert torch.equal(x.nan_to_num(7.0) if x.is_floating_point() else x, y.nan_to_num(7.0) if y.is_floating_point() else y)
    paged.context(DEV).sync()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_tables_and_totals_wider_than_the_lengths(dtype, window, sinks):
    """Room for 70000 positions a sequence, as a cache that may grow has: outputs,
    totals and kept positions are those of tables that just fit."""
    from rich_triplet_b200 import paged

    lens, new, nkv, d, page, wide = [700, 33, 0, 260], [200, 33, 0, 1], 2, 64, 16, 70000
    c = Cache(lens, nkv, d, page, dtype, spare=4 * 8)
    table = torch.full((4, wide // page), -1, dtype=torch.int32, device=DEV)
    table[:, :c.table.shape[1]] = c.table
    q, qp = queries(4, 4, d, dtype, 0, False), queries(234, 4, d, dtype, 1, False)
    start = torch.tensor([0, 200, 233, 233, 234], dtype=torch.int32, device=DEV)
    seen = dict(scale=0.125, window=window, sinks=sinks)
    dst = c.free[:32].view(4, 8).to(DEV)
    got = []
    for t, cap in ((c.table, 700), (table, wide)):
        mass = torch.zeros(4, nkv, cap, device=DEV)
        a = paged.attend_decode(q, c.kp, c.vp, t, c.lens_t, mass=mass, **seen)
        b = paged.attend_prompt(qp, start, 200, c.kp, c.vp, t, c.lens_t, mass=mass, **seen)
        kept, n, out = paged.kv_evict(c.kp, c.vp, t, c.lens_t, mass, dst, budget=120, sinks=4, recent=30)
        assert (mass[..., 700:] == 0).all() and (out[..., 120:] == 0).all()
        got.append((*a, *b, mass[..., :700], kept, n, out[..., :700]))
    u = U[dtype]
    for i, (x, y) in enumerate(zip(*got)):
        if x.dtype == torch.int32:
            continue
        # prompts and their totals may be split differently over CTAs: each is within
        # about u (1 + |value|) of the definition
        assert torch.equal(torch.isinf(x), torch.isinf(y))
        fin = torch.isfinite(y)
        off = (x[fin].double() - y[fin].double()).abs()
        assert float((off - 4 * u * (1 + y[fin].double().abs())).max() if off.numel() else 0) <= 0, i
    # the totals decide; equal ones, equal positions
    mass = got[0][4].contiguous()
    full = torch.zeros(4, nkv, wide, device=DEV)
    full[..., :700] = mass
    a = paged.kv_evict(c.kp, c.vp, c.table, c.lens_t, mass, dst, budget=120, sinks=4, recent=30)
    b = paged.kv_evict(c.kp, c.vp, table, c.lens_t, full, dst, budget=120, sinks=4, recent=30)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2][..., :700])


@pytest.mark.parametrize("dtype,fmt", [(BF16, 30), (F16, 1), (F32, 0)])
def test_c_calls_without_lse(dtype, fmt):
    """rt_paged_prompt and rt_paged_decode with totals and lse NULL: the scratch of
    rt_paged_scratch stands in, its end untouched; too little of it is refused."""
    import ctypes

    from rich_triplet_b200 import paged
    from rich_triplet_b200._lib import lib
    from test_paged_edges_cpu import Attn, Kv

    nkv, nq, d, page = 2, 4, 64, 16
    c = Cache([130, 9, 0], nkv, d, page, dtype)
    start = torch.tensor([0, 40, 49, 49], dtype=torch.int32, device=DEV)
    scale = 0.125
    ctx = paged.context(DEV)
    ctx.sync()
    kv = Kv(k=c.kp.data_ptr(), v=c.vp.data_ptr(), page_stride=c.kp.stride(0), head_stride=c.kp.stride(1),
            slot_stride=c.kp.stride(2), num_pages=c.kp.shape[0], fmt=fmt, kv_heads=nkv, head_dim=d, page_size=page,
            page_table=c.table.data_ptr(), table_stride=c.table.shape[1], table_width=c.table.shape[1], num_seqs=3,
            lens=c.lens_t.data_ptr())
    for prompt in (1, 0):
        rows = 49 if prompt else 3
        q = queries(rows, nq, d, dtype, prompt, False)
        want_mass = torch.zeros(3, nkv, 130, device=DEV)
        if prompt:
            want, _ = paged.attend_prompt(q, start, 40, *c.args(), scale=scale, mass=want_mass)
        else:
            want, _ = paged.attend_decode(q, *c.args(), scale=scale, mass=want_mass)
        out, mass = torch.empty_like(q), torch.zeros_like(want_mass)
        a = Attn(q=q.data_ptr(), out=out.data_ptr(), q_row_stride=nq * d, q_head_stride=d, out_row_stride=nq * d,
                 out_head_stride=d, rows=rows, num_heads=nq, max_new=40, scale=scale, mass_cap=130,
                 q_start=start.data_ptr() if prompt else None, mass=mass.data_ptr(), mass_seq_stride=nkv * 130,
                 mass_head_stride=130)
        need = ctypes.c_uint64()
        assert lib().rt_paged_scratch(ctypes.byref(kv), ctypes.byref(a), prompt, ctypes.byref(need)) == 0
        assert need.value >= rows * nq * 4
        room = torch.full((need.value + 512,), 77, dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()
        call = lib().rt_paged_prompt if prompt else lib().rt_paged_decode
        a.scratch, a.scratch_bytes = room.data_ptr(), need.value - 1
        assert call(ctx.h, ctypes.byref(kv), ctypes.byref(a), None) == -1 and "scratch" in ctx.last_error()
        a.scratch_bytes = need.value
        assert call(ctx.h, ctypes.byref(kv), ctypes.byref(a), None) == 0, ctx.last_error()
        ctx.sync()
        assert torch.equal(out, want) and torch.equal(mass, want_mass) and (room[need.value:] == 77).all()


def test_a_replay_beside_another_threads_calls_on_the_capture_stream():
    """Streams come from a pool, so two threads may hold the same one: a graph that
    the first captured there, replayed elsewhere, meets the second's calls."""
    from rich_triplet_b200 import paged

    c = Cache([9000, 33], 2, 128, 16, BF16)
    q = [queries(2, 4, 128, BF16, i, False) for i in range(2)]
    want = [paged.attend_decode(x, *c.args(), scale=0.1)[0] for x in q]
    s, elsewhere = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        paged.attend_decode(q[0], *c.args(), scale=0.1)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out, _ = paged.attend_decode(q[0], *c.args(), scale=0.1)
    wrong, stop = [], threading.Event()

    def other():
        with torch.cuda.stream(s):
            for _ in range(300):
                if not torch.equal(paged.attend_decode(q[1], *c.args(), scale=0.1)[0], want[1]):
                    wrong.append("other")
        stop.set()

    t = threading.Thread(target=other)
    t.start()
    with torch.cuda.stream(elsewhere):
        while not stop.is_set():
            g.replay()
            if not torch.equal(out, want[0]):
                wrong.append("replay")
    t.join()
    assert not wrong
    paged.context(DEV).sync()
