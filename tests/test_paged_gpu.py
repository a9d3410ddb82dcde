"""Paged cache operators (rich_triplet_b200.paged) against their definitions in
64 bits.

Every slot of the pools that holds no visible position is NaN, and page-table
entries without a visible position are out of range, so a kernel that reads
what it must not shows it.

Tolerances come from the arithmetic.  With u32 = 2^-24 and e(n) = (n + 16) u32:
a score, a sum of D products in 32 bits in any order, is off by at most
delta = 2 e(D) scale max_j sum |q k_j| (twice, for an accumulator that cuts off
instead of rounding); a weight then by the factor 1 + 2 delta + e(n) with its
normalisation; an output sum over n positions by (2 delta + 2 e(n)) A, with
A = sum_j p_j |v_j|.  A 16-bit cache adds the rounding of the output, u |o|, and
of the weights before they multiply V, u A, with u = 2^-8 (bf16) or 2^-11 (f16)
(plus f16's smallest step 2^-24 for weights and outputs below its normal
range).  32-bit caches may run on the tensor cores with each operand split in
two 11-bit parts: u = 2^-20 covers what the dropped product and the parts'
rounding leave.  The log of the sum is off by delta + e(n) + u32 |lse|, with
2^-20 sum |q k| scale for split operands.
"""

import math

import pytest
import torch

from rich_triplet_b200._lib import RtError

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}
U32 = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def e32(n):
    return (n + 16) * U32


def is_visible(t, j, window, sinks):
    """[len(t), len(j)]: whether a token at t sees position j."""
    t, j = t[:, None], j[None, :]
    ok = j <= t
    if window:
        ok = ok & ((j > t - window) | (j < sinks))
    return ok


class Cache:
    """Sequences of the given lengths in pages that are scattered over a pool
    and poisoned outside `seen(b)`, the positions that some token sees."""

    def __init__(self, lens, nkv, d, page, dtype, layout="head", seed=0, seen=None, width=None, spare=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.dtype, self.nkv, self.d = list(lens), page, dtype, nkv, d
        need = [-(-n // page) for n in lens]
        width = max(need + [width or 1])
        pages = sum(need) + 5 + spare
        shape = (pages, nkv, page, d) if layout == "head" else (pages, page, nkv, d)
        both = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
        self.kp, self.vp = both if layout == "head" else [x.transpose(1, 2) for x in both]
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32)
        self.k, self.v = [], []  # f64 values of the cached rows, [nkv, n, d]
        at = 0
        for b, n in enumerate(lens):
            k = torch.randn(nkv, n, d, generator=g).to(DEV).to(dtype)
            v = (torch.randn(nkv, n, d, generator=g) + torch.randn(nkv, 1, d, generator=g)).to(DEV).to(dtype)
            self.k.append(k.double())
            self.v.append(v.double())
            ids = order[at:at + need[b]]
            at += need[b]
            j = torch.arange(n) if seen is None else seen(b)
            self.table[b, torch.unique(j // page)] = ids[torch.unique(j // page)].int()
            pg, sl = ids[j // page].to(DEV), (j % page).to(DEV)
            self.kp[pg, :, sl] = k[:, j.to(DEV)].transpose(0, 1)
            self.vp[pg, :, sl] = v[:, j.to(DEV)].transpose(0, 1)
        self.free = order[at:].int()
        self.table = self.table.to(DEV)
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device=DEV)

    def args(self):
        return self.kp, self.vp, self.table, self.lens_t


def reference(cache, b, q, t, scale, window, sinks):
    """Sequence b's outputs for q [m, nq, D] at positions t [m] in 64 bits, with
    their bounds: out, its bound, lse, its bound, weight totals [nkv, n], theirs."""
    n, d, nkv = cache.lens[b], cache.d, cache.nkv
    u, tiny = U[cache.dtype], TINY[cache.dtype]
    m, nq = q.shape[:2]
    G = nq // nkv
    qd = q.double().view(m, nkv, G, d)
    k, v = cache.k[b], cache.v[b]
    s = torch.einsum("mhgd,hnd->mhgn", qd, k) * scale
    size = torch.einsum("mhgd,hnd->mhgn", qd.abs(), k.abs()) * scale
    ok = is_visible(t, torch.arange(n, device=DEV), window, sinks)[:, None, None, :]
    s = s.masked_fill(~ok, -math.inf)
    size = size.masked_fill(~ok, 0.0)
    some = ok.any(-1)
    lse = torch.logsumexp(s, -1) if n else torch.full((m, nkv, G), -math.inf, dtype=torch.float64, device=DEV)
    lse = torch.where(some, lse, -math.inf)
    p = torch.where(ok, torch.exp(s - torch.where(some, lse, 0.0)[..., None]), 0.0)
    big = size.amax(-1) if n else torch.zeros_like(lse)
    delta = (2 * e32(d) + (2.0 ** -20 if cache.dtype == F32 else 0.0)) * big
    out = torch.einsum("mhgn,hnd->mhgd", p, v)
    A = torch.einsum("mhgn,hnd->mhgd", p, v.abs())
    vmax = v.abs().amax(1)[None, :, None, :] if n else torch.zeros_like(A)
    bound = u * (out.abs() + A) + (2 * delta[..., None] + 2 * e32(n)) * A + tiny * (1 + n * vmax)
    lse_bound = delta + e32(n) + U32 * torch.where(some, lse, 0.0).abs()
    mass = p.sum((0, 2))
    mass_bound = ((2 * delta[..., None] + e32(n)) * p).sum((0, 2)) + e32(m * G) * mass
    return (out.reshape(m, nq, d), bound.reshape(m, nq, d), lse.reshape(m, nq), lse_bound.reshape(m, nq), mass,
            mass_bound)


def close(got, want, bound, what):
    got = got.double()
    same = got == want  # infinities
    bad = ~(same | ((got - want).abs() <= bound))
    if bad.any():
        off = (got - want).abs()
        i = int(torch.where(torch.isnan(off), torch.inf, off / bound.clamp(min=1e-300)).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds; worst got "
                             f"{got.flatten()[i]:.8g}, want {want.flatten()[i]:.8g}, bound {bound.flatten()[i]:.3g}")


def queries(rows, nq, d, dtype, seed, fused):
    """Random queries; `fused`: as slices of wider rows."""
    g = torch.Generator().manual_seed(seed + 99)
    wide = torch.randn(rows, (nq + 3) * d if fused else nq * d, generator=g).to(DEV).to(dtype)
    return wide[:, (2 if fused else 0) * d:][:, :nq * d].view(rows, nq, d)


def check_decode(lens, nq, nkv, d, page, dtype, window=0, sinks=0, layout="head", fused=False, mass=False, seed=0,
                 width=None, q_mul=1.0, cap=None):
    from rich_triplet_b200 import paged

    def seen(b):
        n = lens[b]
        j = torch.arange(n)
        return j[is_visible(torch.tensor([n - 1]), j, window, sinks)[0]] if n else j

    c = Cache(lens, nkv, d, page, dtype, layout, seed, seen, width)
    q = queries(len(lens), nq, d, dtype, seed, fused) * q_mul
    scale = 1.0 / math.sqrt(d)
    cap = cap or max(lens + [1]) + 3
    total = torch.rand(len(lens), nkv, cap, device=DEV) if mass else None
    before = total.clone() if mass else None
    out, lse = paged.attend_decode(q, *c.args(), scale=scale, window=window, sinks=sinks, mass=total)
    for b, n in enumerate(lens):
        t = torch.tensor([n - 1], device=DEV)
        o, ob, z, zb, m, mb = reference(c, b, q[b:b + 1], t, scale, window, sinks)
        close(out[b:b + 1], o, ob, f"out of sequence {b} (length {n})")
        close(lse[b:b + 1], z, zb, f"lse of sequence {b} (length {n})")
        if mass:
            x = min(n, cap)
            want = before[b].double()
            add = torch.zeros_like(want)
            add[:, :x] = m[:, :x]
            slack = torch.zeros_like(want)
            slack[:, :x] = mb[:, :x]
            close(total[b], want + add, slack + 2 * U32 * (want + add) * (add > 0), f"mass of sequence {b} (length {n})")
    again, lse2 = paged.attend_decode(q, *c.args(), scale=scale, window=window, sinks=sinks)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


EDGE_LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nq,nkv,d", [(8, 4, 256), (32, 16, 128), (4, 1, 256), (2, 1, 128), (8, 1, 64)])
def test_decode_lengths(dtype, nq, nkv, d):
    check_decode(EDGE_LENS, nq, nkv, d, 16, dtype, seed=d + nq)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 1), (5, 1), (12, 2), (9, 1), (16, 1)])
@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 128), (F16, 256)])
def test_decode_head_groups(nq, nkv, dtype, d):
    check_decode([70, 1, 333], nq, nkv, d, 32, dtype, seed=nq, mass=True)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["head", "slot"])
def test_decode_pages_and_layouts(page, layout):
    check_decode([513, 255, 256, 257], 8, 4, 256, page, BF16, layout=layout, fused=True, width=60, seed=page)
    check_decode([513, 7, 100], 4, 2, 64, page, F32, layout=layout, fused=True, seed=page)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 3), (64, 64), (128, 0), (1000, 4), (64, 1000)])
@pytest.mark.parametrize("dtype,d", [(BF16, 256), (F32, 128), (F16, 64)])
def test_decode_window_and_sinks(window, sinks, dtype, d):
    check_decode([0, 1, 5, 64, 101, 700, 65], 4, 2, d, 16, dtype, window=window, sinks=sinks, mass=True, seed=window)


@pytest.mark.parametrize("lens", [[5000], [20011, 3, 0, 9000], [1] * 97, [40] * 300])
def test_decode_split_and_many(lens):
    check_decode(lens, 4, 2, 128, 32, BF16, seed=len(lens), mass=True)


def test_decode_large_scores():
    """Scores in the hundreds: the running maximum has to move."""
    check_decode([400, 77], 8, 4, 256, 16, BF16, q_mul=40.0, mass=True)
    check_decode([400, 77], 8, 4, 256, 16, F32, q_mul=40.0, mass=True)


def test_decode_mass_shorter_than_the_sequences():
    check_decode([400, 77], 8, 4, 256, 16, BF16, mass=True, cap=100)


def check_prompt(lens, new, nq, nkv, d, page, dtype, window=0, sinks=0, layout="head", fused=False, mass=False, seed=0,
                 max_new=None, cap=None, q_mul=1.0):
    from rich_triplet_b200 import paged

    def seen(b):
        n, m = lens[b], new[b]
        j = torch.arange(n)
        t = torch.arange(max(0, n - m), n)
        return j[is_visible(t, j, window, sinks).any(0)] if n and len(t) else j[:0]

    c = Cache(lens, nkv, d, page, dtype, layout, seed, seen)
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    q = queries(starts[-1], nq, d, dtype, seed, fused) * q_mul
    start_t = torch.tensor(starts, dtype=torch.int32, device=DEV)
    scale = 1.0 / math.sqrt(d)
    cap = cap or max(lens + [1]) + 2
    total = torch.rand(len(lens), nkv, cap, device=DEV) if mass else None
    before = total.clone() if mass else None
    max_new = max_new if max_new is not None else max(new + [0])
    args = dict(scale=scale, window=window, sinks=sinks)
    out, lse = paged.attend_prompt(q, start_t, max_new, *c.args(), mass=total, **args)
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0:
            if mass:
                assert torch.equal(total[b], before[b])
            continue
        rows = slice(starts[b], starts[b + 1])
        t = torch.arange(n - m, n, device=DEV)
        o, ob, z, zb, w, wb = reference(c, b, q[rows], t, scale, window, sinks)
        close(out[rows], o, ob, f"out of sequence {b} ({m} of {n})")
        close(lse[rows], z, zb, f"lse of sequence {b} ({m} of {n})")
        if mass:
            x = min(n, cap)
            want = before[b].double()
            add, slack = torch.zeros_like(want), torch.zeros_like(want)
            add[:, :x], slack[:, :x] = w[:, :x], wb[:, :x]
            close(total[b], want + add, slack + 2 * U32 * (want + add) * (add > 0), f"mass of sequence {b} ({m} of {n})")
    again, lse2 = paged.attend_prompt(q, start_t, max_new, *c.args(), **args)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nq,nkv,d", [(8, 4, 256), (4, 2, 128), (4, 1, 256), (8, 1, 64)])
def test_prompt_lengths(dtype, nq, nkv, d):
    new = [1, 2, 31, 0, 64, 65, 127, 128, 129, 260]
    check_prompt(new, new, nq, nkv, d, 16, dtype, seed=d + nq)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 128), (F16, 256)])
def test_prompt_on_a_filled_cache(dtype, d):
    check_prompt([500, 129, 64, 200, 1000], [8, 1, 64, 130, 3], 8, 4, d, 32, dtype, mass=True, seed=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 3), (64, 64), (128, 130), (1000, 4), (64, 1000)])
@pytest.mark.parametrize("dtype,d", [(BF16, 256), (F32, 64), (F16, 128)])
def test_prompt_window_and_sinks(window, sinks, dtype, d):
    check_prompt([600, 333, 1], [200, 333, 1], 4, 2, d, 16, dtype, window=window, sinks=sinks, mass=True, seed=window)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 1), (6, 2), (9, 1), (16, 1)])
@pytest.mark.parametrize("dtype,d", [(BF16, 256), (F16, 64), (F32, 128)])
def test_prompt_head_groups(nq, nkv, dtype, d):
    check_prompt([150, 40], [141, 7], nq, nkv, d, 64, dtype, mass=True, seed=nq)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["head", "slot"])
def test_prompt_pages_and_layouts(page, layout):
    check_prompt([513, 255, 7], [300, 255, 7], 8, 4, 256, page, BF16, layout=layout, fused=True, mass=True, seed=page)
    check_prompt([513, 100], [120, 100], 4, 2, 64, page, F16, layout=layout, fused=True, seed=page, window=50, sinks=2)


def test_prompt_tokens_before_position_zero_see_nothing():
    """More new tokens than positions: the first ones get 0 and -inf."""
    from rich_triplet_b200 import paged

    c = Cache([5, 0], 2, 128, 16, BF16)
    q = queries(14, 4, 128, BF16, 0, False)
    start = torch.tensor([0, 8, 14], dtype=torch.int32, device=DEV)
    out, lse = paged.attend_prompt(q, start, 8, *c.args(), scale=0.1)
    hidden = [0, 1, 2, 8, 9, 10, 11, 12, 13]
    assert (out[hidden] == 0).all() and torch.isneginf(lse[hidden]).all()
    o, ob, z, zb, _, _ = reference(c, 0, q[3:8], torch.arange(5, device=DEV), 0.1, 0, 0)
    close(out[3:8], o, ob, "out")
    close(lse[3:8], z, zb, "lse")


def test_prompt_rows_beyond_max_new_stay():
    from rich_triplet_b200 import paged

    c = Cache([50], 2, 128, 16, F16)
    q = queries(20, 4, 128, F16, 0, False)
    start = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    paged.attend_prompt(q, start, 12, *c.args(), scale=0.1, out=out)
    assert (out[12:] == 7).all()
    o, ob, _, _, _, _ = reference(c, 0, q[:12], torch.arange(30, 42, device=DEV), 0.1, 0, 0)
    close(out[:12], o, ob, "out")


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 256)])
def test_prompt_large_scores_and_long(dtype, d):
    check_prompt([900], [900], 2, 1, d, 64, dtype, q_mul=30.0, mass=True)
    check_prompt([3001, 1500], [1500, 1500], 2, 1, d, 128, dtype, window=700, sinks=5, mass=True)


def test_prompt_mass_shorter_than_the_sequences():
    check_prompt([400, 77], [300, 77], 8, 4, 256, 16, BF16, mass=True, cap=130)


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["head", "slot"])
def test_append(src, dtype, layout):
    from rich_triplet_b200 import paged

    lens, new, nkv, d = [40, 7, 0, 16, 300], [40, 1, 0, 3, 33], 3, 64
    c = Cache(lens, nkv, d, 16, dtype, layout)
    rows = sum(new)
    kv = torch.randn(rows, 2 * nkv * d, device=DEV).to(src)
    k, v = kv[:, :nkv * d].view(rows, nkv, d), kv[:, nkv * d:].view(rows, nkv, d)
    start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    want_k, want_v = c.kp.clone(), c.vp.clone()
    r = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            j = n - m + i
            want_k[c.table[b, j // 16].long(), :, j % 16] = k[r].to(dtype)
            want_v[c.table[b, j // 16].long(), :, j % 16] = v[r].to(dtype)
            r += 1
    paged.kv_append(c.kp, c.vp, k, v, c.table, c.lens_t, q_start=start)
    bits = torch.int32 if dtype == F32 else torch.int16
    assert torch.equal(c.kp.contiguous().view(bits), want_k.contiguous().view(bits))
    assert torch.equal(c.vp.contiguous().view(bits), want_v.contiguous().view(bits))


def test_append_one_each_and_dropped_rows():
    from rich_triplet_b200 import paged

    c = Cache([5, 0, 17], 2, 128, 8, BF16)
    k = torch.randn(3, 2, 128, device=DEV)
    before = c.kp.clone()
    paged.kv_append(c.kp, c.vp, k, k, c.table, c.lens_t)
    want = before.clone()
    want[c.table[0, 0].long(), :, 4] = k[0].to(BF16)
    want[c.table[2, 2].long(), :, 0] = k[2].to(BF16)  # the empty sequence's row is dropped
    assert torch.equal(c.kp.view(torch.int16), want.view(torch.int16))
    # rows before position 0, and a page number outside the pool
    before = c.kp.clone()
    start = torch.tensor([0, 7, 7, 8], dtype=torch.int32, device=DEV)
    k = torch.randn(8, 2, 128, device=DEV)
    table = c.table.clone()
    table[2, 2] = 10 ** 6
    paged.kv_append(c.kp, c.vp, k, k, table, c.lens_t, q_start=start)
    want = before.clone()
    for j in range(5):
        want[c.table[0, 0].long(), :, j] = k[2 + j].to(BF16)
    assert torch.equal(c.kp.view(torch.int16), want.view(torch.int16))


def check_evict(lens, nkv, d, page, dtype, budget, sinks, recent, layout="head", seed=0, mass=None, cap=None):
    from rich_triplet_b200 import paged

    width = -(-budget // page)
    c = Cache(lens, nkv, d, page, dtype, layout, seed, spare=width * len(lens))
    cap = cap or max(lens + [1])
    if mass is None:
        g = torch.Generator().manual_seed(seed)
        mass = torch.rand(len(lens), nkv, cap, generator=g).pow(6).to(DEV)
    dst = c.free[:width * len(lens)].view(len(lens), width).to(DEV)
    before = mass.clone()
    kept, new_lens, out = paged.kv_evict(c.kp, c.vp, c.table, c.lens_t, mass, dst, budget=budget, sinks=sinks,
                                         recent=recent)
    assert torch.equal(torch.nan_to_num(mass, 7.0), torch.nan_to_num(before, 7.0))
    for b, n in enumerate(lens):
        m = min(n, budget)
        assert int(new_lens[b]) == m
        for h in range(nkv):
            rank = [(-math.inf if math.isnan(x) else x) for x in before[b, h].tolist()]
            first = [j for j in range(n) if j < sinks or j >= n - recent]
            rest = sorted((j for j in range(n) if not (j < sinks or j >= n - recent)),
                          key=lambda j: (-(rank[j] if j < cap else -math.inf), j))
            want = sorted((first + rest)[:m]) if n > budget else list(range(n))
            assert kept[b, h].tolist() == want + [-1] * (budget - m), (b, h)
            w = torch.tensor(want, dtype=torch.long, device=DEV)
            i = torch.arange(m, device=DEV)
            for pool, rows in ((c.kp, c.k), (c.vp, c.v)):
                got = pool[dst[b].long()[i // page], h, i % page].double()
                assert torch.equal(got, rows[b][h][w])
            z = before[b, h][w.clamp(max=cap - 1)]
            assert torch.equal(torch.nan_to_num(out[b, h, :m], 7.0), torch.nan_to_num(z, 7.0)[:cap])
            assert (out[b, h, m:] == 0).all()


@pytest.mark.parametrize("dtype,d", [(F32, 64), (F16, 128), (BF16, 256)])
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("layout", ["head", "slot"])
def test_evict(dtype, d, page, layout):
    check_evict([700, 100, 0, 101, 1, 99], 3, d, page, dtype, 100, 4, 30, layout, seed=page)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 0, 0), (64, 64, 0), (64, 0, 64),
                                                 (64, 10, 54), (1025, 4, 100)])
def test_evict_budgets(budget, sinks, recent):
    check_evict([1500, 64, 65, 5000], 2, 64, 32, BF16, budget, sinks, recent, seed=budget)


def test_evict_long():
    check_evict([70001, 33000], 1, 64, 256, BF16, 5000, 4, 1000, seed=1)


def test_evict_ties_and_special_values():
    lens = [500, 500, 500, 500]
    mass = torch.zeros(4, 1, 500, device=DEV)  # all equal
    mass[1] = torch.randint(0, 4, (500,), device=DEV).float()  # many ties
    mass[1, 0, ::5] = -0.0
    mass[2] = torch.randn(500, device=DEV)
    mass[2, 0, ::7] = float("nan")
    mass[2, 0, 3::7] = -math.inf
    mass[3] = torch.rand(500, device=DEV)
    mass[3, 0, ::50] = math.inf
    check_evict(lens, 1, 64, 16, BF16, 450, 0, 0, mass=mass)
    check_evict(lens, 1, 64, 16, BF16, 40, 2, 5, mass=mass)


def test_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^32 (keys and values 9 GB each)."""
    from rich_triplet_b200 import paged

    nkv, d, page = 4, 256, 64
    pages = (2 ** 32) // (nkv * page * d) + 64
    kp = torch.empty(pages, nkv, page, d, dtype=BF16, device=DEV)
    vp = torch.empty_like(kp)
    n = 200
    ids = torch.tensor([pages - 1 - i for i in range(4)], dtype=torch.int32, device=DEV)
    table, lens = ids.view(1, 4), torch.tensor([n], dtype=torch.int32, device=DEV)
    k, v = torch.randn(n, nkv, d, device=DEV).to(BF16), torch.randn(n, nkv, d, device=DEV).to(BF16)
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    paged.kv_append(kp, vp, k, v, table, lens, q_start=start)
    c = Cache.__new__(Cache)
    c.lens, c.d, c.nkv, c.dtype = [n], d, nkv, BF16
    c.k, c.v = [k.double().transpose(0, 1)], [v.double().transpose(0, 1)]
    q = queries(n, 8, d, BF16, 0, False)
    out, lse = paged.attend_prompt(q, start, n, kp, vp, table, lens, scale=1 / 16)
    o, ob, z, zb, _, _ = reference(c, 0, q, torch.arange(n, device=DEV), 1 / 16, 0, 0)
    close(out, o, ob, "prompt out")
    close(lse, z, zb, "prompt lse")
    one, z1 = paged.attend_decode(q[-1:], kp, vp, table, lens, scale=1 / 16)
    close(one, o[-1:], ob[-1:], "decode out")
    mass = torch.rand(1, nkv, n, device=DEV)
    dst = torch.tensor([[pages - 9, 3]], dtype=torch.int32, device=DEV)
    kept, _, _ = paged.kv_evict(kp, vp, table, lens, mass, dst, budget=100)
    i = torch.arange(100, device=DEV)
    for h in range(nkv):
        assert torch.equal(kp[dst[0].long()[i // page], h, i % page], k[kept[0, h].long(), h])
    del kp, vp
    torch.cuda.empty_cache()


def test_runs_on_the_current_stream():
    """Inputs made on a side stream, the operators called there, without any
    synchronisation in between; then again on the default stream."""
    from rich_triplet_b200 import paged

    c = Cache([900, 30], 4, 256, 32, BF16)
    want, _ = paged.attend_decode(queries(2, 8, 256, BF16, 1, False), *c.args(), scale=1 / 16)
    q0 = queries(2, 8, 256, BF16, 1, False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            big = big @ big * 1e-4
        q = q0 + (big.sum() * 0).nan_to_num().to(BF16)
        got, _ = paged.attend_decode(q, *c.args(), scale=1 / 16)
        got = got * 1
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(paged.attend_decode(q0, *c.args(), scale=1 / 16)[0], want)


def test_in_a_graph():
    """Captured once, replayed with other lengths and pages in the same buffers."""
    from rich_triplet_b200 import paged

    a, b = Cache([300, 64], 2, 128, 16, F16, seed=1), Cache([17, 290], 2, 128, 16, F16, seed=2)
    q = queries(2, 4, 128, F16, 0, False)
    want = [paged.attend_decode(q, *x.args(), scale=0.1)[0] for x in (a, b)]
    table, lens = a.table.clone(), a.lens_t.clone()
    kp, vp = a.kp.clone(), a.vp.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged.attend_decode(q, kp, vp, table, lens, scale=0.1)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out, _ = paged.attend_decode(q, kp, vp, table, lens, scale=0.1)
    for x, w in ((a, want[0]), (b, want[1]), (a, want[0])):
        n = min(kp.shape[0], x.kp.shape[0])
        kp[:n], vp[:n] = x.kp[:n], x.vp[:n]
        table.copy_(x.table)
        lens.copy_(x.lens_t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_no_sequences_and_no_rows():
    from rich_triplet_b200 import paged

    c = Cache([5], 2, 128, 16, F16)
    none = (c.kp, c.vp, c.table[:0], c.lens_t[:0])
    out, lse = paged.attend_decode(torch.empty(0, 4, 128, dtype=F16, device=DEV), *none, scale=0.1)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    paged.attend_prompt(torch.empty(0, 4, 128, dtype=F16, device=DEV), start, 0, *c.args(), scale=0.1)
    paged.kv_append(c.kp, c.vp, torch.empty(0, 2, 128, device=DEV), torch.empty(0, 2, 128, device=DEV), c.table, c.lens_t,
                    q_start=start)


def test_refusals():
    from rich_triplet_b200 import paged

    c = Cache([40, 9], 2, 128, 16, BF16)
    kp, vp, table, lens = c.args()
    q = queries(2, 4, 128, BF16, 0, False)
    ok = dict(scale=0.1)

    def refused(error, match, fn, *args, **kw):
        with pytest.raises(error, match=match):
            fn(*args, **kw)

    dec = paged.attend_decode
    refused(ValueError, "q must be", dec, q.half(), *c.args(), **ok)
    refused(ValueError, "q must be", dec, q[..., :64], *c.args(), **ok)
    refused(ValueError, "query rows", dec, q[:1], *c.args(), **ok)
    refused(ValueError, "same strides", dec, q, kp, vp[:, :1], table, lens, **ok)
    refused(ValueError, "f32, f16 or bf16", dec, q, kp.to(torch.float64), vp.to(torch.float64), table, lens, **ok)
    refused(ValueError, "page_table", dec, q, kp, vp, table.long(), lens, **ok)
    refused(ValueError, "lens", dec, q, kp, vp, table, lens[:1], **ok)
    refused(ValueError, "lens", dec, q, kp, vp, table, lens.cpu(), **ok)
    refused(ValueError, "one GPU", dec, q, kp.cpu(), vp.cpu(), table, lens, **ok)
    refused(ValueError, "mass", dec, q, *c.args(), mass=torch.zeros(2, 1, 50, device=DEV), **ok)
    refused(ValueError, "out must be", dec, q, *c.args(), out=torch.empty(2, 4, 64, dtype=BF16, device=DEV), **ok)
    refused(RtError, "scale", dec, q, *c.args(), scale=0.0)
    refused(RtError, "scale", dec, q, *c.args(), scale=float("nan"))
    refused(RtError, "negative window", dec, q, *c.args(), window=-1, **ok)
    refused(RtError, "query heads", dec, queries(2, 5, 128, BF16, 0, False), *c.args(), **ok)
    refused(RtError, "query heads", dec, queries(2, 34, 128, BF16, 0, False), *c.args(), **ok)
    odd = Cache([40], 1, 96, 16, BF16)
    refused(RtError, "head_dim 96", dec, queries(1, 2, 96, BF16, 0, False), *odd.args(), **ok)
    odd = Cache([40], 1, 64, 24, BF16)
    refused(RtError, "page_size 24", dec, queries(1, 2, 64, BF16, 0, False), *odd.args(), **ok)
    odd = torch.empty(40 * 128 + 1, dtype=BF16, device=DEV)[1:].view(10, 4, 128)
    refused(RtError, "16-byte aligned", dec, odd[:2], *c.args(), **ok)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    refused(ValueError, "q_start", paged.attend_prompt, q, start[:2], 1, *c.args(), **ok)
    refused(RtError, "max_new", paged.attend_prompt, q, start, -1, *c.args(), **ok)
    k = torch.zeros(2, 2, 128, device=DEV)
    refused(ValueError, "kv_append", paged.kv_append, kp, vp, k[..., :64], k[..., :64], table, lens)
    refused(ValueError, "f32, f16 or bf16", paged.kv_append, kp, vp, k.double(), k.double(), table, lens)
    refused(RtError, "rows for", paged.kv_append, kp, vp, k[:1], k[:1], table, lens)
    mass = torch.zeros(2, 2, 50, device=DEV)
    dst = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    refused(ValueError, "dst_table", paged.kv_evict, kp, vp, table, lens, mass, dst, budget=17)
    refused(ValueError, "mass", paged.kv_evict, kp, vp, table, lens, mass[:1], dst, budget=16)
    refused(RtError, "budget", paged.kv_evict, kp, vp, table, lens, mass, dst, budget=16, sinks=10, recent=7)
    refused(RtError, "budget", paged.kv_evict, kp, vp, table, lens, mass, dst, budget=0)
    # and after all that the operators still work
    dec(q, *c.args(), **ok)
    torch.cuda.synchronize()


def test_prompt_more_row_tiles_than_sms():
    """Several waves of CTAs over long windowed walks, and again: a wait that is
    only sometimes late shows here."""
    for _ in range(3):
        check_prompt([2600, 900], [2000, 900], 16, 4, 256, 64, F16, window=1024, sinks=4, seed=5)
        check_prompt([2600, 900], [2000, 900], 16, 4, 128, 64, BF16, seed=6)
    from rich_triplet_b200 import paged
    paged.context(DEV).sync()  # raises if a wait gave up


def test_evict_mass_shorter_than_the_sequences():
    """Positions at or beyond the mass tensor's end rank as -inf and have no mass."""
    from rich_triplet_b200 import paged

    c = Cache([300, 90], 2, 64, 16, F16, spare=2 * 8)
    mass = torch.rand(2, 2, 120, device=DEV)
    dst = c.free[:16].view(2, 8).to(DEV)
    kept, lens, out = paged.kv_evict(c.kp, c.vp, c.table, c.lens_t, mass, dst, budget=125, sinks=2, recent=3)
    assert lens.tolist() == [125, 90]
    # all 120 ranked positions, the last three, and two of the others: the lowest
    assert kept[0, 0].tolist() == list(range(122)) + [297, 298, 299]
    assert torch.equal(out[0], mass[0]) and torch.equal(out[1, :, :90], mass[1, :, :90]) and (out[1, :, 90:] == 0).all()


def test_first_call_on_a_stream_inside_a_capture_is_refused():
    """The stream's workspace cannot be made there; the capture stays usable."""
    from rich_triplet_b200 import paged

    c = Cache([40], 2, 128, 16, BF16)
    q = queries(1, 4, 128, BF16, 0, False)
    want, _ = paged.attend_decode(q, *c.args(), scale=0.1)
    s = torch.cuda.Stream(priority=-1)
    x = torch.zeros(4, device=DEV)
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(RtError, match="workspace does not exist"):
            paged.attend_decode(q, *c.args(), scale=0.1)
        x += 1
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1, 1, 1, 1]
    assert torch.equal(paged.attend_decode(q, *c.args(), scale=0.1)[0], want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences_and_strided_tables(dtype):
    """More sequences than threads of a CTA, lengths of zero among them, a page
    table that is a slice of a wider one, outputs into a given strided tensor."""
    from rich_triplet_b200 import paged

    lens = [(7 * i) % 45 for i in range(700)]
    c = Cache(lens, 1, 64, 8, dtype, seed=3)
    wide = torch.full((700, c.table.shape[1] + 9), 10 ** 8, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + c.table.shape[1]] = c.table
    table = wide[:, 4:4 + c.table.shape[1]]
    q = queries(700, 2, 64, dtype, 0, True)
    room = torch.full((700, 5, 64), 9.0, dtype=dtype, device=DEV)
    out, lse = paged.attend_decode(q, c.kp, c.vp, table, c.lens_t, scale=0.125, out=room[:, 1:3])
    assert out.data_ptr() == room[:, 1:3].data_ptr()
    assert (room[:, 0] == 9).all() and (room[:, 3:] == 9).all()
    for b in range(0, 700, 13):
        o, ob, z, zb, _, _ = reference(c, b, q[b:b + 1], torch.tensor([lens[b] - 1], device=DEV), 0.125, 0, 0)
        close(out[b:b + 1], o, ob, f"out of sequence {b}")
        close(lse[b:b + 1], z, zb, f"lse of sequence {b}")
    start = torch.arange(701, dtype=torch.int32, device=DEV)
    again, _ = paged.attend_prompt(q, start, 1, c.kp, c.vp, table, c.lens_t, scale=0.125)
    for b in range(0, 700, 13):
        o, ob, _, _, _, _ = reference(c, b, q[b:b + 1], torch.tensor([lens[b] - 1], device=DEV), 0.125, 0, 0)
        close(again[b:b + 1], o, ob, f"prompt out of sequence {b}")
