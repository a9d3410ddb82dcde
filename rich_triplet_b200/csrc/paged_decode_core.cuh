// paged_decode_core.cuh -- attention of one or a few new tokens per sequence over
// a paged cache: the kernel behind rt_paged_decode (paged_decode.cu) and, over
// f32 caches, rt_paged_prompt (paged_prompt32.cu).
//
// Bound by HBM: every visible key and value row is read once.
//
// Work.  The visible positions of a (sequence, KV head) item, counted without
// the gap between the first tokens and the window, are cut into units of 4
// tiles, and the units of all items, in order, are dealt evenly to the CTAs
// of one persistent grid, from the lengths on the device: a CTA's share is a
// contiguous range that may end inside an item, so one long sequence and many
// ragged ones both load every SM to within a unit.  An item whose range spans
// several CTAs is joined by whichever of them finishes last (an atomic
// counter per first CTA), in CTA order, so results do not depend on timing.
//
// A warp takes every fourth tile of its CTA's range and keeps its own running
// maximum m, sum l and output for the G query heads of the KV head.  Its
// tiles' K and V rows come through a private ring of shared-memory slots
// filled by 16-byte cp.async from page-table addresses (rows past the end are
// zero-filled, so masked rows add nothing whatever they hold): NS - 1 slots
// are in flight while one is read, and no barrier stands between the warps.
//
// Arithmetic: mma.sync with the cache rows as the 16-row operand and the query
// heads as its 8 columns (S^T = K Q^T, O^T = V^T P^T), so up to 8 heads read
// each row at no extra cost; the memory stream leaves the tensor cores mostly
// idle and tcgen05's 64-row operand would be mostly padding here.  The weights are split
// in two 16-bit parts (hi + lo) before they multiply V, so their rounding stays
// below the output's: 2^-16 of a bf16 weight, 2^-22 of an f16 one, and where that
// is less than f16's smallest step, 2^-32 of the largest weight (kLift).  With
// G <= 4 the low parts ride in columns 4..7 of the same product.  f32 rows: tf32 products of hi and lo parts of
// both operands, relative error about 2^-22; for the scores the queries are the
// 16-row operand, hi parts above lo parts, so two products give all four terms.
//
// Measured (B200): one sequence of 131071 positions, 8 heads on 4 of 256, bf16:
// 95 us, 5.6 TB/s (the SMs finish between 62 and 84 us, the join of 74 parts
// takes 8).  64 sequences, 1.05 GB of f32: 194 us, 5.4 TB/s (205 to 212 in a row of
// calls).  64 windows of 1028: 45 us, 5.8 TB/s.  301 positions: 9.0 us, six
// dependent trips to memory (length, page, rows, part, counter, parts).
//
// A state has seen no weight where its sum is 0, whatever its maximum: NaN scores
// do not move the maximum, but their NaN is in the sum and in the output.
//
// The maximum is only moved when a score exceeds it by more than 8 (powers of
// two), so weights stay below 2^8 (2^15 for f16 rows) and most tiles rescale nothing.
#pragma once

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"

namespace rt {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSlotBytes = 8192;  // K or V rows of a tile, head_dim 256
constexpr int kRingBytes = 3 * kSlotBytes;  // per warp
constexpr float kMaxSlack = 8.f;
// Weights of f16 rows are taken 2^7 above the largest one: f16's smallest step is
// 2^-24, and with the slack of 2^8 they stay below its 65504.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int kMinFew = 4;

template <typename T, int D, int NT>
struct DecCfg {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int kRows = kF32 ? 8 : 16;                 // positions of a tile
    static constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
    static constexpr int kSlot = kRows * kRowBytes;
    static constexpr int NS = kRingBytes / kSlot;               // 3, 6 or 12
    static constexpr int kUnit = kRows * kWarps;
    // An item's start (page lookups, an empty ring, a combine at its end) takes
    // about as long as kStart units; it is dealt out like units without rows.
    static constexpr int kStart = 256 / D;
    static constexpr int kWhole = 3 * 256 / D;                   // units that cost what a join does
    static constexpr int kQBytes = kF32 ? NT * (D / 8) * 32 * 16 : 0;  // f32: query fragments
    static constexpr int CS = D + 4;                            // floats of a combine row
    static constexpr int kCombBytes = kWarps * NT * 8 * CS * 4;
    static constexpr int kMain = kWarps * kRingBytes > kCombBytes ? kWarps * kRingBytes : kCombBytes;
    static constexpr int kOffQ = kMain;
    static constexpr int kOffMisc = kOffQ + kQBytes;            // m, l of every warp and column; block scan
    static constexpr int kOffRows = kOffMisc + kWarps * NT * 8 * 8 + 64;  // [warp][16] byte offsets of a tile's rows
    static constexpr int kSmem = kOffRows + kWarps * 16 * 8;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void cp16_all(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ int64_t lds64(uint32_t a) {
    int64_t v;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts64(uint32_t a, int64_t v) { asm volatile("st.shared.b64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float lds32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// x = hi + lo with hi's 11 leading bits; the product reads 11 bits of lo, which
// leaves out at most 2^-21 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float residual(float x) { return x - to_f32(from_f32<T>(x)); }

// Weight of a state with maximum m under the joint maximum M (powers of two).
__device__ __forceinline__ float rel2(float m, float M) { return m == -INFINITY ? 0.f : exp2f(m - M); }

__device__ __forceinline__ void store4(float* p, float4 v, float f) {
    *reinterpret_cast<float4*>(p) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v, float f) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x * f, v.y * f, T()), pack2(v.z * f, v.w * f, T()));
}

struct DecWork {
    float* part;        // [2 * grid][G][D + 4]: output, m, l
    uint32_t* cnt;      // [grid], zero between calls
    float* scores;      // null, or [nseq][nq][score_stride]: scores (powers of two) by visible position
    int64_t score_stride;
    float2* norm;       // with scores: [nseq][nq] maximum and 1 / sum
    float scale2;       // scale * log2(e)
};

// G <= 4: columns c and c + 4 are both head c (the second carries the low
// parts of the weights); else column c is head c.
template <bool DUP>
__device__ __forceinline__ int head_of(int col) { return DUP ? (col & 3) : col; }

// The new tokens of a sequence: `count` of them are computed, at positions pos0 on.
struct Tokens {
    int first, count, pos0;
};
__device__ __forceinline__ Tokens tokens_of(const PagedKv& kv, const PagedAttn& a, int b) {
    const int first = a.q_start[b], all = a.q_start[b + 1] - first;
    Tokens t = {first, 0, kv.len(b) - all};
    if (first >= 0 && all > 0) t.count = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(min(all, a.max_new)), a.rows - first)));
    return t;
}
// What the tokens at positions t_first .. t_last see together.
__device__ __forceinline__ Visible visible_to(int t_first, int t_last, int window, int sinks) {
    Visible v = {0, 0, 0};
    if (t_last < 0) return v;
    v.w0 = window > 0 && t_first >= window ? t_first - window + 1 : 0;
    v.sinks = min(sinks, v.w0);
    v.n = v.sinks + t_last + 1 - v.w0;
    return v;
}

// FEW = false: one token per sequence, an item is a (sequence, KV head) and its
// columns are the G heads.  FEW = true: several tokens per sequence; the (token,
// head) rows of a sequence and KV head are cut into tiles of 8 NT columns, an
// item is one such tile, and each column has its own mask.  All items of a
// sequence are dealt out as if they saw as much as its last token.
template <typename T, int D, int NT, bool DUP, bool FEW>
__global__ void __launch_bounds__(kThreads, 2) paged_decode_kernel(const PagedKv kv, const PagedAttn a, const DecWork wk) {
    using C = DecCfg<T, D, NT>;
    constexpr bool F32 = C::kF32;
    constexpr int ROWS = C::kRows, NS = C::NS, CS = C::CS, UNIT = C::kUnit;
    constexpr int CPR = C::kRowBytes / 16;          // 16-byte chunks of a row
    constexpr int COPIES = ROWS * CPR / 32;         // cp.async of a lane per slot
    constexpr int KQ = F32 ? 1 : D / 16;
    constexpr int MT = D / 16;                      // 16-row tiles of O^T
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kRingBytes;
    const uint32_t rows_at = smem_u32(smem) + C::kOffRows + warp * 16 * 8;
    float* comb = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(smem + C::kOffMisc);  // [warp][NT * 8]
    int* red = reinterpret_cast<int*>(smem + C::kOffMisc + kWarps * NT * 8 * 8);
    constexpr int COLS = NT * 8;
    const int G = a.G;

    // ---- this CTA's share of the units ----
    // Prefix sums over the sequences of (units of an item, items) in one word each half.
    const int chunk = (kv.nseq + kThreads - 1) / kThreads;
    const int sb0 = min(kv.nseq, static_cast<int>(threadIdx.x) * chunk), sb1 = min(kv.nseq, sb0 + chunk);
    auto units_of = [](int seen) { return seen > 0 ? C::kStart + (seen + UNIT - 1) / UNIT : 0; };
    auto item_tiles = [&](int b) -> int { return FEW ? (tokens_of(kv, a, b).count * G + COLS - 1) / COLS : 1; };
    auto item_units = [&](int b) -> int {
        if (!FEW) return units_of(visible(kv.len(b), a.window, a.sinks).n);
        const Tokens t = tokens_of(kv, a, b);
        if (t.count == 0) return 0;
        const int all = t.pos0 + t.count;  // the last token sees at most this
        const int64_t span = static_cast<int64_t>(a.window) + a.sinks + COLS / G + 1;
        return units_of(max(1, a.window > 0 && span < all ? static_cast<int>(span) : all));
    };
    int64_t mine = 0;
    int longest = 0;
    for (int b = sb0; b < sb1; ++b) {
        const int n = item_units(b);
        if (n > 0) mine += ((static_cast<int64_t>(1) << 40) + n) * item_tiles(b);
        longest = max(longest, n);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    int64_t* red64 = reinterpret_cast<int64_t*>(red);
    if (lane == 31) red64[warp] = x;
    if (lane == 0) red[12 + warp] = longest;
    __syncthreads();
    int64_t before = x - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += red64[w];
        all += red64[w];
        longest = max(longest, red[12 + w]);
    }
    constexpr int64_t kUnits = (static_cast<int64_t>(1) << 40) - 1;
    // Every CTA below `grid` has a unit at least.  Items stay whole, one to a
    // CTA, where the longest of them is at most kWhole units more than an even
    // share: a split item is drained, joined and followed by another's start,
    // which takes about as long (64 windows of 1028 positions on 4 heads of 256:
    // 51 us dealt evenly, 46 us whole).
    const int64_t U = (all & kUnits) * kv.nkv, items = (all >> 40) * kv.nkv;
    const bool by_item = items > 0 && items <= gridDim.x && longest <= U / min(static_cast<int64_t>(gridDim.x), U) + C::kWhole;
    // (with several tokens a part is 8 or 16 rows to join, so it gets kMinFew units)
    const int64_t grid = by_item ? items : min(static_cast<int64_t>(gridDim.x), FEW ? max(min(items, U), U / kMinFew) : U);
    const bool idle = blockIdx.x >= grid;
    const int64_t u_begin = idle ? U : blockIdx.x * U / grid;
    int64_t u_end = idle ? U : (blockIdx.x + 1) * U / grid;
    {
        // the one thread whose sequences hold this CTA's first unit (or item) finds it
        const int64_t at = by_item ? static_cast<int64_t>(blockIdx.x) : u_begin;
        const int shift = by_item ? 40 : 0;
        const int64_t lo = ((before >> shift) & kUnits) * kv.nkv, hi = lo + ((mine >> shift) & kUnits) * kv.nkv;
        if (!idle && at >= lo && at < hi) {
            int64_t u = (before & kUnits) * kv.nkv, v = lo;
            for (int b = sb0; b < sb1; ++b) {
                const int64_t n = item_units(b), its = static_cast<int64_t>(n > 0 ? item_tiles(b) : 0) * kv.nkv;
                const int64_t step = by_item ? its : n * its;
                if (at < v + step) {
                    red[8] = b;
                    red[9] = static_cast<int>(by_item ? at - v : (at - v) / n);
                    red64[5] = u;
                    break;
                }
                u += n * its;
                v += step;
            }
        }
    }
    // Sequences that see nothing: output 0, lse -inf.
    if (!FEW && (all >> 40) < kv.nseq)
        for (int b = blockIdx.x; b < kv.nseq; b += gridDim.x) {
            if (visible(kv.len(b), a.window, a.sinks).n > 0) continue;
            for (int i = threadIdx.x; i < a.nq * D; i += kThreads)
                static_cast<T*>(a.out)[b * a.out_row + (i / D) * a.out_head + i % D] = from_f32<T>(0.f);
            for (int i = threadIdx.x; i < a.nq; i += kThreads)
                if (a.lse) a.lse[b * a.lse_row + i] = -INFINITY;
        }
    pdl_launch_dependents();
    if (idle) return;
    __syncthreads();
    // item `it` of sequence b: head it / ntile, column tile it % ntile
    int b = red[8], it = red[9], ntile = item_tiles(b);
    int nun = item_units(b);
    int64_t u_item = red64[5] + static_cast<int64_t>(it) * nun;  // its first unit
    const int64_t u_first = by_item ? u_item : u_begin;
    if (by_item) u_end = u_item + nun;

    for (int64_t u = u_first; u < u_end;) {
        // units [t0, t1) of the item, less the ones that stand for its start
        const int seg_end = static_cast<int>(min(u_end - u_item, static_cast<int64_t>(nun)));
        const int t0 = max(0, static_cast<int>(u - u_item) - C::kStart), t1 = seg_end - C::kStart;
        if (t1 <= t0) {  // nothing but (a part of) the start: the next CTA reads the rows
            u = u_item + seg_end;
            continue;
        }
        const int h = it / ntile, row0 = FEW ? (it % ntile) * COLS : 0;
        Tokens tk = {b, 1, 0};
        Visible vis;
        if constexpr (FEW) {
            tk = tokens_of(kv, a, b);
            vis = visible_to(tk.pos0 + row0 / G, tk.pos0 + (min(tk.count * G, row0 + COLS) - 1) / G, a.window, a.sinks);
        } else {
            vis = visible(kv.len(b), a.window, a.sinks);
        }
        const int ncol = FEW ? min(COLS, tk.count * G - row0) : G;
        // column col: its query row, and its head of the KV head's G
        auto row_at = [&](int col) { return FEW ? tk.first + (row0 + col) / G : b; };
        auto head_at = [&](int col) { return h * G + (FEW ? (row0 + col) % G : col); };
        const int c_end = min(vis.n, t1 * UNIT);
        const int c_first = t0 * UNIT + warp * ROWS;  // this warp's tiles: c_first, + UNIT, ...
        const int tiles = c_first < c_end ? (c_end - c_first + UNIT - 1) / UNIT : 0;
        const int64_t hoff = h * kv.head_stride;

        // ---- copies: half-tile s = 2 i + (0: K, 1: V) of tile i to slot s % NS ----
        int issued = 0, islot = 0;
        bool whole_tile = true;
        const char* const kl = static_cast<const char*>(kv.k) + hoff * sizeof(T) + (lane % CPR) * 16;
        const char* const vl = static_cast<const char*>(kv.v) + hoff * sizeof(T) + (lane % CPR) * 16;
        auto row_of = [&](int i) -> int64_t {
            const int c = c_first + i * UNIT + (lane % ROWS);
            return i < tiles && c < c_end ? kv.row(b, vis.pos(c)) : -1;
        };
        int64_t off_next = row_of(0);
        auto issue = [&]() {
            const int half = issued & 1;
            __syncwarp();  // every lane has read the last tile's offsets, and the slot that is filled here
            if (half == 0) {
                if (lane < ROWS) sts64(rows_at + lane * 8, off_next < 0 ? -1 : off_next * static_cast<int64_t>(sizeof(T)));
                whole_tile = __all_sync(0xffffffffu, off_next >= 0);
                off_next = row_of((issued >> 1) + 1);
                __syncwarp();  // the offsets are there for the other lanes (a vote orders no memory)
            }
            if (issued < 2 * tiles) {
                const char* base = half ? vl : kl;
                const uint32_t dst = ring + islot * C::kSlot;
#pragma unroll
                for (int i = 0; i < COPIES; ++i) {
                    // a warp-wide copy is 32 / CPR rows, or a part of one
                    const int r = CPR >= 32 ? i / (CPR / 32) : i * (32 / CPR) + lane / CPR, part = CPR >= 32 ? i % (CPR / 32) : 0;
                    const int sw = r & 7, ch = part * 32 + lane % CPR;
                    const uint32_t to = dst + r * C::kRowBytes + ((ch ^ sw) << 4);
                    const int64_t o = lds64(rows_at + r * 8);
                    if (whole_tile) cp16_all(to, base + o + part * 512);
                    else cp16(to, base + (o < 0 ? 0 : o) + part * 512, o >= 0);
                }
            }
            cp_commit();
            ++issued;
            islot = islot + 1 == NS ? 0 : islot + 1;
        };
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) issue();

        // ---- queries: column n = g8 of Q^T ----
        uint32_t qf[NT][KQ][2];
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = head_of<DUP>(n * 8 + g8);
                const bool has = col < ncol;
                const T* qr = static_cast<const T*>(a.q) + static_cast<int64_t>(row_at(has ? col : 0)) * a.q_row + head_at(has ? col : 0) * a.q_head;
#pragma unroll
                for (int k = 0; k < KQ; ++k) {
                    qf[n][k][0] = has ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 2 * t4) : 0u;
                    qf[n][k][1] = has ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 8 + 2 * t4) : 0u;
                }
            }
        } else {
            uint4* qs = reinterpret_cast<uint4*>(smem + C::kOffQ);
            for (int i = threadIdx.x; i < NT * (D / 8) * 32; i += kThreads) {
                const int l = i & 31, k = (i >> 5) % (D / 8), n = (i >> 5) / (D / 8);
                const int col = head_of<DUP>(n * 8 + (l >> 2));
                uint4 f = make_uint4(0, 0, 0, 0);
                if (col < ncol) {
                    const float* qr = static_cast<const float*>(a.q) + static_cast<int64_t>(row_at(col)) * a.q_row + head_at(col) * a.q_head +
                                      8 * k + (l & 3);
                    split_tf32(qr[0], f.x, f.y);
                    split_tf32(qr[4], f.z, f.w);
                }
                qs[i] = f;
            }
            __syncthreads();
        }

        float o[NT][MT][4];
        // of columns 2 t4 and 2 t4 + 1 (f32 rows: [0] of column g8); m: the weights are 2^(score - m),
        // the maximum so far less kLift; l: this lane's positions only
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
        int when[NT][2];  // FEW: positions of the tokens of those columns, -1 for no column
        if constexpr (FEW) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int col = n * 8 + (F32 ? g8 : 2 * t4 + q);
                    when[n][q] = col < ncol ? tk.pos0 + (row0 + col) / G : -1;
                }
        }
        int slot = 0;
        for (int i = 0; i < tiles; ++i) {
            const int c0 = c_first + i * UNIT;
            // ---- scores of the tile: rows g8 (and g8 + 8), columns 2 t4, 2 t4 + 1 ----
            issue();
            cp_wait<NS - 1>();
            __syncwarp();
            float s[NT][4];
            const uint32_t ks = ring + slot * C::kSlot;
            if constexpr (!F32) {
                const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
                // chunk (2 k + lane / 16) ^ (r % 8): the swizzle only turns bits 0..2
                uint32_t at[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) at[k] = ks + r * C::kRowBytes + (((2 * k + (lane >> 4)) ^ (r & 7)) << 4);
                float acc[2][NT][4];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[q][n][e] = 0.f;
#pragma unroll
                for (int k = 0; k < KQ; ++k) {
                    uint32_t kf[4];
                    ldsm4(at[k & 3] + (k >> 2) * 128, kf);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16<T>(acc[k & 1][n], kf, qf[n][k][0], qf[n][k][1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = (acc[0][n][e] + acc[1][n][e]) * wk.scale2;
            } else {
                const uint4* qs = reinterpret_cast<const uint4*>(smem + C::kOffQ) + lane;
                // Rows 0..7 of the left operand are the columns' high parts, 8..15 their
                // low parts, the eight positions its columns: S = [q_hi; q_lo] (k_hi + k_lo)^T.
                const int r = lane & 7;
                const uint32_t at[2] = {ks + r * C::kRowBytes + (((lane >> 3) ^ r) << 4),
                                        ks + r * C::kRowBytes + (((4 + (lane >> 3)) ^ r) << 4)};
                // The tensor cores' f32 sums cut off instead of rounding: four short
                // chains for the large products, added here.
                float hh[4][NT][4], lo[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) hh[0][n][e] = hh[1][n][e] = hh[2][n][e] = hh[3][n][e] = lo[n][e] = 0.f;
#pragma unroll 4
                for (int k2 = 0; k2 < D / 16; ++k2) {  // chain 2 (k2 % 2) + k of hh
                    uint32_t kf[4];
                    ldsm4(at[k2 & 1] + (k2 >> 1) * 128, kf);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t h0, h1, l0, l1;
                        split_tf32(__uint_as_float(kf[2 * k]), h0, l0);
                        split_tf32(__uint_as_float(kf[2 * k + 1]), h1, l1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 f = qs[(n * (D / 8) + 2 * k2 + k) * 32];
                            mma8(hh[2 * (k2 & 1) + k][n], f.x, f.y, f.z, f.w, h0, h1);
                            mma8(lo[n], f.x, f.y, f.z, f.w, l0, l1);
                        }
                    }
                }
                // column g8, positions 2 t4 and 2 t4 + 1
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        s[n][e] = ((hh[0][n][e] + hh[1][n][e]) + (hh[2][n][e] + hh[3][n][e]) +
                                   (((hh[0][n][e + 2] + hh[1][n][e + 2]) + (hh[2][n][e + 2] + hh[3][n][e + 2])) +
                                    (lo[n][e] + lo[n][e + 2]))) * wk.scale2;
                    s[n][2] = s[n][3] = -INFINITY;
                }
            }
            slot = slot + 1 == NS ? 0 : slot + 1;
            // ---- weights ----
            constexpr int EL = F32 ? 2 : 4;  // values of a lane: positions g8, g8 + 8 of two columns (f32: 2 t4, 2 t4 + 1 of one)
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < EL; ++e) {
                    const int c = F32 ? c0 + 2 * t4 + e : c0 + g8 + (e >> 1) * 8, q = F32 ? 0 : (e & 1);
                    if (!FEW && wk.scores && c < c_end) {
                        const int col = n * 8 + (F32 ? g8 : 2 * t4 + q), head = head_of<DUP>(col);
                        if (head < G && (!DUP || col < 4))
                            wk.scores[(static_cast<int64_t>(b) * a.nq + h * G + head) * wk.score_stride + c] = s[n][e];
                    }
                    bool seen = c < c_end;
                    if constexpr (FEW) {
                        const int p = vis.pos(c), t = when[n][q];
                        seen = seen && p <= t && (a.window == 0 || p > t - a.window || p < a.sinks);
                    }
                    s[n][e] = seen ? s[n][e] : -INFINITY;
                    over |= s[n][e] > m[n][q] + (kMaxSlack + kLift<T>);
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[2];
#pragma unroll
                    for (int q = 0; q < (F32 ? 1 : 2); ++q) {
                        float v = F32 ? fmaxf(s[n][0], s[n][1]) : fmaxf(s[n][q], s[n][q + 2]);
#pragma unroll
                        for (int d = F32 ? 1 : 4; d < (F32 ? 4 : 32); d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                        const float mn = fmaxf(m[n][q], v - kLift<T>);
                        f[q] = rel2(m[n][q], mn);
                        m[n][q] = mn;
                        l[n][q] *= f[q];
                    }
                    if (F32) {  // the output's columns are 2 t4 and 2 t4 + 1
                        const float own = f[0];
                        f[0] = __shfl_sync(0xffffffffu, own, 8 * t4);
                        f[1] = __shfl_sync(0xffffffffu, own, 8 * t4 + 4);
                    }
#pragma unroll
                    for (int j = 0; j < MT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][j][e] *= f[e & 1];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < EL; ++e) {
                    const int q = F32 ? 0 : (e & 1);
                    s[n][e] = rel2(s[n][e], m[n][q]);
                    l[n][q] += s[n][e];
                }
            // ---- O^T += V^T P^T ----
            issue();
            cp_wait<NS - 1>();
            __syncwarp();
            const uint32_t vs = ring + slot * C::kSlot;
            if constexpr (!F32) {
                uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float p0 = s[n][2 * q], p1 = s[n][2 * q + 1];
                        const float r0 = residual<T>(p0), r1 = residual<T>(p1);
                        if (DUP) {
                            hi[n][q] = transpose8x8(t4 >= 2 ? pack2(r0, r1, T()) : pack2(p0, p1, T()));
                        } else {
                            hi[n][q] = transpose8x8(pack2(p0, p1, T()));
                            lo[n][q] = transpose8x8(pack2(r0, r1, T()));
                        }
                    }
                const int mi = lane >> 3, r = (lane & 7) + (mi >> 1) * 8;
                uint32_t at[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) at[j] = vs + r * C::kRowBytes + (((2 * j + (mi & 1)) ^ (r & 7)) << 4);
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    uint32_t vf[4];
                    ldsm4t(at[j & 3] + (j >> 2) * 128, vf);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16<T>(o[n][j], vf, hi[n][0], hi[n][1]);
                        if (!DUP) mma16<T>(o[n][j], vf, lo[n][0], lo[n][1]);
                    }
                }
            } else {
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < 2; ++q) split_tf32(s[n][q], ph[n][q], pl[n][q]);  // positions 2 t4 + q, column g8
                // value q of 16-dim tile j: dims 16 j + g8 + 8 (q & 1), positions 2 t4 + (q >> 1)
                // (the product's steps t4 and t4 + 4 may be any two positions);
                // its chunk 4 j + 2 (q & 1) + g8 / 4 is turned in bits 0..2 by the swizzle
                uint32_t at[2][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = 2 * t4 + (q >> 1);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        at[j][q] = vs + r * C::kRowBytes + (((4 * j + 2 * (q & 1) + (g8 >> 2)) ^ r) << 4) + (g8 & 3) * 4;
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    uint32_t vh[4], vl[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) split_tf32(lds32(at[j & 1][q] + (j >> 1) * 128), vh[q], vl[q]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float z[4];  // one tile's sum, added with rounding
                        mma8_zero(z, vh[0], vh[1], vh[2], vh[3], pl[n][0], pl[n][1]);
                        mma8(z, vl[0], vl[1], vl[2], vl[3], ph[n][0], ph[n][1]);
                        mma8(z, vh[0], vh[1], vh[2], vh[3], ph[n][0], ph[n][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][j][e] += z[e];
                    }
                }
            }
            slot = slot + 1 == NS ? 0 : slot + 1;
            __syncwarp();
        }
        cp_wait<0>();

        // ---- the CTA's state of this item: warps joined in warp order ----
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int d = F32 ? 1 : 4; d < (F32 ? 4 : 32); d <<= 1) l[n][q] += __shfl_xor_sync(0xffffffffu, l[n][q], d);
        __syncthreads();  // every warp is done with its ring (and the query fragments)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float* row = comb + (warp * NT * 8 + n * 8 + 2 * t4 + q) * CS;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    row[16 * j + g8] = o[n][j][q];
                    row[16 * j + g8 + 8] = o[n][j][q + 2];
                }
                if (!F32 && g8 == 0) ml[warp * NT * 8 + n * 8 + 2 * t4 + q] = make_float2(m[n][q], l[n][q]);
                if (F32 && q == 0 && t4 == 0) ml[warp * NT * 8 + n * 8 + g8] = make_float2(m[n][0], l[n][0]);
            }
        }
        __syncthreads();
        const bool whole = t0 == 0 && seg_end == nun;
        const int rec = 2 * blockIdx.x + (u == u_first ? 0 : 1);
        float* pr = wk.part + static_cast<int64_t>(rec) * (FEW ? COLS : G) * CS;
        for (int i = threadIdx.x; i < ncol * (D / 4); i += kThreads) {
            const int g = i / (D / 4), d = (i % (D / 4)) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * NT * 8 + g].x);
            float L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 s = ml[w * NT * 8 + g];
                const float f = rel2(s.x, M);
                L += s.y * f;
                const float* row = comb + (w * NT * 8 + g) * CS + d;
                float4 v = *reinterpret_cast<const float4*>(row);
                if (DUP) {
                    const float4 z = *reinterpret_cast<const float4*>(row + 4 * CS);
                    v = make_float4(v.x + z.x, v.y + z.y, v.z + z.z, v.w + z.w);
                }
                A.x += v.x * f;
                A.y += v.y * f;
                A.z += v.z * f;
                A.w += v.w * f;
            }
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                const int64_t row = row_at(g);
                const int head = head_at(g);
                store4(static_cast<T*>(a.out) + row * a.out_row + head * a.out_head + d, A, inv);
                if (d == 0) {
                    if (a.lse) a.lse[row * a.lse_row + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
                    if (!FEW && wk.norm) wk.norm[row * a.nq + head] = make_float2(M, inv);
                }
            } else {
                *reinterpret_cast<float4*>(pr + g * CS + d) = A;
                if (d == 0) *reinterpret_cast<float2*>(pr + g * CS + D) = make_float2(M, L);
            }
        }
        if (!whole) {
            // ---- the CTAs c_a .. c_z hold parts of this item; the last to arrive joins them in order ----
            const int64_t u_last = u_item + nun - 1;
            const int c_a = static_cast<int>(((u_item + C::kStart + 1) * grid - 1) / U), c_z = static_cast<int>(((u_last + 1) * grid - 1) / U);
            const int n = c_z - c_a + 1;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t old = atomicAdd(&wk.cnt[c_a], 1u);
                red[0] = old == static_cast<uint32_t>(n - 1);
                if (red[0]) wk.cnt[c_a] = 0u;
            }
            __syncthreads();
            if (red[0]) {
                __threadfence();
                // CTA c_a's part is its last segment, unless its share begins in the item
                const int first = 2 * c_a + (c_a * U / grid >= u_item ? 0 : 1);
                auto record = [&](int k) { return wk.part + static_cast<int64_t>(k ? 2 * (c_a + k) : first) * (FEW ? COLS : G) * CS; };
                float2* st = reinterpret_cast<float2*>(smem);  // [n][ncol] maximum and sum, then weight and sum
                for (int i = threadIdx.x; i < n * ncol; i += kThreads)
                    st[i] = __ldcg(reinterpret_cast<const float2*>(record(i / ncol) + (i % ncol) * CS + D));
                __syncthreads();
                for (int g = warp; g < ncol; g += kWarps) {
                    float M = -INFINITY, L = 0.f;
                    for (int k = lane; k < n; k += 32) M = fmaxf(M, st[k * ncol + g].x);
                    M = warp_max(M);
                    for (int k = lane; k < n; k += 32) {
                        const float f = rel2(st[k * ncol + g].x, M);
                        L += f * st[k * ncol + g].y;
                        st[k * ncol + g].x = f;
                    }
                    L = warp_sum(L);
                    if (lane == 0) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        st[n * ncol + g].x = inv;
                        const int64_t row = row_at(g);
                        const int head = head_at(g);
                        if (a.lse) a.lse[row * a.lse_row + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
                        if (!FEW && wk.norm) wk.norm[row * a.nq + head] = make_float2(M, inv);
                    }
                }
                __syncthreads();
                // kQuads float4 of the output a thread at a time; the loads of kBatch parts of each overlap
                auto add_up = [&](auto quads, auto batch) {
                    constexpr int kQuads = decltype(quads)::value, kBatch = decltype(batch)::value;
                    const int all_quads = ncol * (D / 4);
                    for (int i0 = threadIdx.x; i0 < all_quads; i0 += kThreads * kQuads) {
                        float4 A[kQuads];
#pragma unroll
                        for (int q = 0; q < kQuads; ++q) A[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int k0 = 0; k0 < n; k0 += kBatch) {
                            float4 v[kQuads][kBatch];
#pragma unroll
                            for (int k = 0; k < kBatch; ++k) {
                                const float* p = record(min(k0 + k, n - 1));
#pragma unroll
                                for (int q = 0; q < kQuads; ++q) {
                                    const int i = min(i0 + q * kThreads, all_quads - 1);
                                    v[q][k] = __ldcg(reinterpret_cast<const float4*>(p + (i / (D / 4)) * CS + (i % (D / 4)) * 4));
                                }
                            }
#pragma unroll
                            for (int k = 0; k < kBatch; ++k)
#pragma unroll
                                for (int q = 0; q < kQuads; ++q) {
                                    const int g = min(i0 + q * kThreads, all_quads - 1) / (D / 4);
                                    const float f = k0 + k < n ? st[(k0 + k) * ncol + g].x : 0.f;
                                    A[q].x += v[q][k].x * f;
                                    A[q].y += v[q][k].y * f;
                                    A[q].z += v[q][k].z * f;
                                    A[q].w += v[q][k].w * f;
                                }
                        }
#pragma unroll
                        for (int q = 0; q < kQuads; ++q) {
                            const int i = i0 + q * kThreads, g = i / (D / 4);
                            if (i < all_quads)
                                store4(static_cast<T*>(a.out) + static_cast<int64_t>(row_at(g)) * a.out_row + head_at(g) * a.out_head +
                                           (i % (D / 4)) * 4,
                                       A[q], st[n * ncol + g].x);
                        }
                    }
                };
                using std::integral_constant;
                if (ncol * (D / 4) > 2 * kThreads) add_up(integral_constant<int, 4>(), integral_constant<int, 5>());
                else if (n <= 4) add_up(integral_constant<int, 1>(), integral_constant<int, 4>());
                else if (n <= 8) add_up(integral_constant<int, 1>(), integral_constant<int, 8>());
                else add_up(integral_constant<int, 1>(), integral_constant<int, 20>());
            }
        }
        __syncthreads();  // the combine area is free for the next segment's copies

        u = u_item + seg_end;
        if (seg_end == nun) {  // next item: of this sequence, or the first of the next one that has any
            u_item += nun;
            if (++it == kv.nkv * ntile && u < u_end) {
                it = 0;
                do {
                    nun = item_units(++b);
                } while (nun == 0);
                ntile = item_tiles(b);
            }
        }
    }
}

template <typename T, int D, int NT, bool DUP, bool FEW>
cudaError_t launch(const PagedKv& kv, const PagedAttn& a, const DecWork& wk, int grid, cudaStream_t s) {
    auto kernel = paged_decode_kernel<T, D, NT, DUP, FEW>;
    constexpr int bytes = DecCfg<T, D, NT>::kSmem;
    static_assert(bytes <= 227 * 1024, "shared memory");
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) done[dev] = true;
    }
    kernel<<<grid, kThreads, bytes, s>>>(kv, a, wk);
    return cudaGetLastError();
}

inline int decode_grid(int num_sms) { return 2 * (num_sms > 0 ? num_sms : 148); }

}  // namespace

}  // namespace rt
