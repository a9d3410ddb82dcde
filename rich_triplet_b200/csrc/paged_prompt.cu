// paged_prompt.cu -- attention of several new tokens per sequence over a paged
// 16-bit cache (rt_paged_prompt) on the tcgen05 tensor cores.
//
// Bound by the tensor cores for long prompts (4 D flops per visible pair of
// positions and query head), by the exponentials at head_dim 64.
//
// Work.  The G query heads of a KV head share its keys, so a CTA's rows are
// (token, head) pairs: row i G + g is token i, head g.  A CTA takes NQ tiles
// of 128 rows (NQ = 2, or 1 at head_dim 256, where one output tile fills half
// of tensor memory) and walks the 128-position key tiles that one of its rows
// sees: those of the first tokens, then those from the window's start to the
// last row's position.  The CTAs of the longest walks start first.  With few
// rows (speculative verify) a walk is split over several CTAs, whose states
// are joined by whichever finishes last, in order.
//
// Roles.  Producer warp: K and V tiles, as 128-byte-swizzled boxes of
// min(page, 128) rows x 64 columns, one lane per box, page numbers read from
// the table; positions past the length and bad page numbers become
// out-of-range coordinates, which read as zeros.  MMA thread: S = Q K^T
// (operands in shared memory) and O += P V (P in tensor memory, V as it lies:
// the N-contiguous operand).  One warpgroup per row tile: one thread per row
// takes its 128 scores from tensor memory, masks them, keeps the running
// maximum and sum in 32 bits and writes the weights back in 16 bits, the
// operand type of the second product; the sum is of the unrounded weights.
// The maximum moves only when a score passes it by 2^8, so the output, which
// stays in tensor memory, is rescaled rarely.
//
// Tensor memory (512 columns): D = 256: O 256, one S, two P of 64, so that S
// is free for the next tile once read.  D = 64: two O of 64, two S, two P.
// D = 128: two O of 128 and two S, whose first 64 columns P overwrites; a
// tile's next S then waits for its P V, while the other tile's products run.
//
// Rows of V that none of the CTA's rows sees (beyond the last position, or
// between the first tokens and the window) are set to zero in shared memory
// before they are multiplied by weights of zero: they may hold anything.
//
// Every wait on an mbarrier gives up after a second: the CTA records
// kErrMbarTimeout, waits (bounded) for its copies and products in flight,
// frees its tensor memory and returns.
//
// Measured (B200): 8192 tokens, 32 heads on 16 of 128, all visible: 640 to 660 us
// in a row of calls, 850 TFLOP/s (615 us where it runs a few times only).  There
// a pair of 128 x 128 tiles takes 3800 clocks where its
// products take 2050: the chain scores -> weights (2000) -> product with V ->
// next scores of a tile is only half hidden behind the other tile's.  6185
// tokens in windows of 1024, 16 heads on 4 of 256: 167 us; a 128 x 128 tile
// takes 3200 clocks (products 2050), and every 128 rows read their own 128 KB
// of K and V a tile from L2, 10 TB/s over the GPU.  5 x 8 tokens over 2050
// positions: 22 us, nearly all of it start (5 us), two or three tiles (2.3 us
// each) and the join (6 us).  Tried and slower: one lane polling for a warp
// (745 against 682 us), a third to an eighth of the exponentials as a
// polynomial on the FMA pipe (640 against 621), the ring's first copies before
// the CTA's first barrier (252 against 244).
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "gemv.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace rt {

namespace {

constexpr int kKeys = 128;   // positions of a key tile
constexpr int kRows = 128;   // rows of a query tile
// Weights are taken 2^kLift above the largest one, 7 for f16, whose smallest step
// is 2^-24: a long tail of small weights then keeps its share (each is rounded by
// at most 2^-32 of the largest).  kMaxSlack: how far they may exceed that before
// the maximum is moved (powers of two; kMaxWeight: their sum), below f16's 65504.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr float kMaxSlack = 8.f;
template <typename T>
constexpr float kMaxWeight = std::is_same<T, __half>::value ? 32768.f : 256.f;
constexpr int kSoftRegs = 208, kOtherRegs = 88;
constexpr int kMaxSplit = 16;  // CTAs that share a walk, at most

template <int D>
struct PCfg {
    static constexpr int NQ = D == 256 ? 1 : 2;       // query tiles of a CTA
    static constexpr bool kAlias = D == 128;          // P in S's columns
    static constexpr int NP = D == 256 ? 2 : 1;       // P buffers of a query tile
    static constexpr int SPT = D == 256 ? 2 : 1;      // ring stages of a K or V tile
    static constexpr int SD = D / SPT;                // columns of a stage
    static constexpr int kChunk = kKeys * 128;        // 64 columns of 128 positions
    static constexpr int kStage = (SD / 64) * kChunk;
    static constexpr int NST = D == 64 ? 10 : 5;
    static constexpr int kQTile = (D / 64) * kChunk;
    static constexpr int kOffRing = NQ * kQTile;
    static constexpr int kOffBar = kOffRing + NST * kStage;
    static constexpr int kBars = 2 * NST + (2 + 3 * NP) * NQ + 2;
    static constexpr int kOffMisc = kOffBar + kBars * 8;
    static constexpr int kSmem = kOffMisc + 16 + 1024;  // + alignment of the tiles
    static constexpr int kSoftWarps = 4 * NQ;
    // With two query tiles the warps are 3 warpgroups of 168 registers a
    // thread, of which the third (producer, MMA, two idle warps) gives up 80 so
    // that the softmax threads have 208 (2 x 208 + 88 = 3 x 168).
    static constexpr int kThreads = NQ == 2 ? 384 : (kSoftWarps + 2) * 32;
    static constexpr uint32_t kS = D == 64 ? 128 : 256;                // S of query tile 0; the next 128 columns on
    static constexpr uint32_t kP = D == 128 ? kS : 384;                // P buffers 64 columns apart
    __host__ __device__ static constexpr uint32_t o_col(int t) { return static_cast<uint32_t>(t * D); }
    __host__ __device__ static constexpr uint32_t s_col(int t) { return kS + 128u * t; }
    __host__ __device__ static constexpr uint32_t p_col(int t, int j) {
        return kAlias ? s_col(t) : kP + 64u * (NP == 2 ? (j & 1) : t);
    }
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct PromptWork {
    float* part;    // split walks: [item][split][NQ * 128 rows][D + 4]: output, maximum (powers of two), sum
    uint32_t* cnt;  // [item], zero between calls
    int nsplit;
    int tiles;      // row tiles (of NQ * 128) of a sequence and KV head, at most
    float scale2;   // scale * log2(e)
};

__device__ __forceinline__ uint32_t pack16(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The key tiles of rows whose tokens stand at t_min .. t_max.
struct Walk {
    int first_tiles, w_tile, count;  // tiles of the first tokens, then from w_tile on
    int w_min;                       // the first position that the window of some row holds
    __device__ __forceinline__ int tile(int i) const { return i < first_tiles ? i : w_tile + i - first_tiles; }
};

__device__ __forceinline__ Walk make_walk(int t_min, int t_max, int window, int sinks) {
    Walk w = {0, 0, 0, 0};
    if (t_max < 0) return w;
    w.w_min = window > 0 && t_min >= window ? t_min - window + 1 : 0;
    w.w_tile = w.w_min / kKeys;
    const int s = min(sinks, w.w_min);
    w.first_tiles = min(w.w_tile, (s + kKeys - 1) / kKeys);
    w.count = w.first_tiles + t_max / kKeys + 1 - w.w_tile;
    return w;
}

template <typename T, int D>
__global__ void __launch_bounds__(PCfg<D>::kThreads, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PagedKv kv,
                        const PagedAttn a, const PromptWork wk) {
    using C = PCfg<D>;
    constexpr int NQ = C::NQ, SPT = C::SPT, NST = C::NST;
    constexpr bool BF16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];

    // ---- this CTA's rows and key tiles ----
    const int G = a.G;
    int64_t bid = blockIdx.x;
    const int split = static_cast<int>(bid % wk.nsplit);
    bid /= wk.nsplit;
    const int64_t bhs = static_cast<int64_t>(kv.nseq) * kv.nkv;
    const int ytile = wk.tiles - 1 - static_cast<int>(bid / bhs);
    const int b = static_cast<int>(bid % bhs) / kv.nkv, h = static_cast<int>(bid % bhs) % kv.nkv;
    const int64_t q_first = a.q_start[b];
    const int all = a.q_start[b + 1] - static_cast<int>(q_first), len = kv.len(b);
    // (rows * G fits 32 bits: checked by the caller)
    const int R = static_cast<int>(min(static_cast<int64_t>(min(all, a.max_new)), a.rows - q_first)) * G;
    const int row0 = ytile * NQ * kRows;
    if (all <= 0 || q_first < 0 || row0 >= R) return;
    const int nrows = min(R - row0, NQ * kRows);
    const int pos0 = len - all;  // position of the sequence's first new token (may be negative)
    const int t_min = pos0 + row0 / G, t_max = pos0 + (row0 + nrows - 1) / G;
    const Walk walk = make_walk(t_min, t_max, a.window, a.sinks);
    const int ns = max(1, min(wk.nsplit, (walk.count + 1) / 2));
    if (split >= ns) return;
    const int i0 = static_cast<int>(static_cast<int64_t>(walk.count) * split / ns);
    const int n = static_cast<int>(static_cast<int64_t>(walk.count) * (split + 1) / ns) - i0;
    // key tiles of each query tile: those up to its last row's position
    auto tiles_of = [&](int t) -> int {
        if (t * kRows >= nrows) return 0;
        const int last = pos0 + (row0 + min(nrows, (t + 1) * kRows) - 1) / G;
        if (last < 0) return 0;
        return max(0, min(n, walk.first_tiles + last / kKeys + 1 - walk.w_tile - i0));
    };

    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    uint8_t* ring = sm + C::kOffRing;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::kOffBar);
    uint64_t* empty = full + NST;
    uint64_t* s_full = empty + NST;   // [NQ] scores are in tensor memory
    uint64_t* s_free = s_full + NQ;   // [NQ] they have been read
    // One barrier per P buffer, so that no waiter is ever two phases behind (a parity could not tell):
    uint64_t* half_bars = s_free + NQ;              // [NQ][NP] the weights of the first 64 positions are there, the output is rescaled
    uint64_t* full_bars = half_bars + NQ * C::NP;   // [NQ][NP] the other 64 too
    uint64_t* pv_bars = full_bars + NQ * C::NP;     // [NQ][NP] their product with V has been added
    uint64_t* q_full = pv_bars + NQ * C::NP;
    uint64_t* drain = q_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::kOffMisc);
    volatile int* abort = reinterpret_cast<volatile int*>(sm + C::kOffMisc + 4);
    int* joined = reinterpret_cast<int*>(sm + C::kOffMisc + 8);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int t = 0; t < NQ; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&s_free[t], 4);
            for (int i = t * C::NP; i < (t + 1) * C::NP; ++i) {
                mbar_init(&half_bars[i], 4);
                mbar_init(&full_bars[i], 4);
                mbar_init(&pv_bars[i], 1);
            }
        }
        mbar_init(q_full, C::kSoftWarps);
        mbar_init(drain, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 0) tc::alloc(tmem_slot, 512);
    if (warp == C::kSoftWarps && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;

    auto p_half = [&](int t, int j) { return &half_bars[t * C::NP + j % C::NP]; };
    auto p_full = [&](int t, int j) { return &full_bars[t * C::NP + j % C::NP]; };
    auto pv_done = [&](int t, int j) { return &pv_bars[t * C::NP + j % C::NP]; };
    auto p_parity = [](int j) { return static_cast<uint32_t>(j / C::NP) & 1u; };

    // Ring order of the tiles: K0, K1, V0, K2, V1, ... (scores run a tile
    // ahead), or K0, V0, K1, V1, ... where P shares S's columns.
    auto k_seq = [&](int j) { return SPT * (C::kAlias ? 2 * j : (j == 0 ? 0 : 2 * j - 1)); };
    auto v_seq = [&](int j) { return SPT * (C::kAlias ? 2 * j + 1 : (j + 1 < n ? 2 * j + 2 : 2 * j + 1)); };

    if (warp >= C::kSoftWarps) {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == C::kSoftWarps) {
            // ---- producer ----
            const int rows = min(1 << kv.page_log2, kKeys), boxes = kKeys / rows;
            const int chunk = lane / boxes, box = lane % boxes;
            int done = 0;
            const int total = 2 * SPT * n;
            bool ok = true;
            for (int e = 0; e < total && ok; ++e) {
                // entry e of the ring: tile j, K or V, columns [col0, + SD)
                const int tile_e = e / SPT;
                bool is_v;
                int j;
                if (C::kAlias) {
                    is_v = tile_e & 1;
                    j = tile_e >> 1;
                } else {
                    is_v = tile_e >= 2 && (!(tile_e & 1) || tile_e == 2 * n - 1);
                    if (n == 1) is_v = tile_e == 1;
                    j = is_v ? (tile_e == 2 * n - 1 ? n - 1 : tile_e / 2 - 1) : (tile_e + 1) / 2;
                }
                const int col0 = (e % SPT) * C::SD;
                const int s = e % NST;
                const int p = walk.tile(i0 + j) * kKeys + box * rows;
                int page = -1;
                if (chunk < C::SD / 64 && p < len) page = kv.table[b * kv.table_stride + (p >> kv.page_log2)];
                if (static_cast<uint32_t>(page) >= static_cast<uint64_t>(kv.num_pages)) page = static_cast<int>(kv.num_pages);
                if (lane == 0) {
                    ok = e < NST || tc::wait_phase(&empty[s], static_cast<uint32_t>(e / NST - 1) & 1u, abort);
                    if (ok) mbar_arrive_expect_tx(&full[s], C::kStage);
                    else tc::give_up(abort, a.err);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (ok && chunk < C::SD / 64)
                    tc::tma_4d(ring + s * C::kStage + chunk * C::kChunk + box * rows * 128, is_v ? &tm_v : &tm_k, col0 + 64 * chunk,
                           p & ((1 << kv.page_log2) - 1), h, page, &full[s]);
                if (ok) ++done;
            }
            // no copy may still be landing when the CTA exits
            if (lane == 0)
                for (int e = max(0, done - NST); e < done; ++e)
                    (void)mbar_wait_timed(&full[e % NST], static_cast<uint32_t>(e / NST) & 1u);
        } else if (warp == C::kSoftWarps + 1) {
            // ---- MMA issuer: the warp walks, one elected lane issues ----
            constexpr uint32_t kIdS = tc::idesc_f16(BF16, kKeys, false), kIdO = tc::idesc_f16(BF16, C::SD, true);
            int nt[NQ];
#pragma unroll
            for (int t = 0; t < NQ; ++t) nt[t] = tiles_of(t);
            auto last_t = [&](int j) { return NQ == 2 && j < nt[NQ - 1] ? 1 : 0; };
            bool ok = tc::warp_wait(q_full, 0u, abort);
            auto scores = [&](int t, int j) {  // S_t = Q_t K_j^T
#pragma unroll
                for (int sp = 0; sp < SPT; ++sp) {
                    const int e = k_seq(j) + sp, s = e % NST;
                    ok = ok && tc::warp_wait(&full[s], static_cast<uint32_t>(e / NST) & 1u, abort);
                    if (!ok) return;
                    tc::fence_after();
                    const uint32_t kb = tc::uniform(tc::desc_lo(smem_u32(ring + s * C::kStage), 16));
                    const uint32_t qb = tc::uniform(tc::desc_lo(smem_u32(sm + t * C::kQTile + sp * C::kStage), 16));
                    const uint32_t st = tc::uniform(tmem + C::s_col(t));
                    if (tc::elect()) {
#pragma unroll
                        for (int k = 0; k < C::SD / 16; ++k) {
                            const uint32_t at = (k >> 2) * C::kChunk + (k & 3) * 32;
                            tc::mma_ss(st, tc::desc_sw128(qb, at), tc::desc_sw128(kb, at), kIdS, sp > 0 || k > 0);
                        }
                        if (t == last_t(j)) tc::commit(&empty[s]);
                        if (sp == SPT - 1) tc::commit(&s_full[t]);
                    }
                    __syncwarp();
                }
            };
            auto outputs = [&](int t, int j) {  // O_t += P_t V_j, as the halves of P_t come
                ok = ok && tc::warp_wait(p_half(t, j), p_parity(j), abort);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half) ok = ok && tc::warp_wait(p_full(t, j), p_parity(j), abort);
                    if (!ok) return;
                    tc::fence_after();
#pragma unroll
                    for (int sp = 0; sp < SPT; ++sp) {
                        const int e = v_seq(j) + sp, s = e % NST;
                        if (!half) {
                            ok = ok && tc::warp_wait(&full[s], static_cast<uint32_t>(e / NST) & 1u, abort);
                            if (!ok) return;
                            tc::fence_after();
                        }
                        const uint32_t vb = tc::uniform(tc::desc_lo(smem_u32(ring + s * C::kStage), C::kChunk));
                        const uint32_t ot = tc::uniform(tmem + C::o_col(t) + sp * C::SD), pt = tc::uniform(tmem + C::p_col(t, j));
                        const uint32_t more = tc::uniform(j > 0);
                        if (tc::elect()) {
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; ++k)
                                tc::mma_ts(ot, pt + 8 * k, tc::desc_sw128(vb, k * 2048), kIdO, k > 0 ? 1u : more);
                            if (half && t == last_t(j)) tc::commit(&empty[s]);
                            if (half && sp == SPT - 1) tc::commit(pv_done(t, j));
                        }
                        __syncwarp();
                    }
                }
            };
            for (int t = 0; t < NQ; ++t)
                if (nt[t] > 0) scores(t, 0);
            for (int j = 0; j < n && ok; ++j) {
                if (C::kAlias) {
                    for (int t = 0; t < NQ; ++t) {
                        if (j >= nt[t]) continue;
                        outputs(t, j);
                        if (j + 1 < nt[t]) {
                            ok = ok && tc::warp_wait(pv_done(t, j), p_parity(j), abort);
                            if (ok) scores(t, j + 1);
                        }
                    }
                } else {
                    for (int t = 0; t < NQ; ++t) {
                        if (j + 1 >= nt[t]) continue;
                        ok = ok && tc::warp_wait(&s_free[t], static_cast<uint32_t>(j) & 1u, abort);
                        if (!ok) break;
                        tc::fence_after();
                        scores(t, j + 1);
                    }
                    for (int t = 0; t < NQ; ++t)
                        if (j < nt[t]) outputs(t, j);
                }
            }
            if (!ok) tc::give_up(abort, a.err);
            // every product has completed before tensor memory is freed
            if (tc::elect()) tc::commit(drain);
            __syncwarp();
            (void)mbar_wait_timed(drain, 0u);
        }
    } else {
        // ---- one warpgroup per query tile, one thread per row ----
        if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int t = warp >> 2, r = t * kRows + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // tensor-memory lane 32 (warp % 4), bits 16 on
        const int nj = tiles_of(t), n0 = tiles_of(0);
        {
            // Q tile t into shared memory, rows past the end zero: a warp its own 32 rows
            constexpr int CPR = D / 8, RPI = 32 / CPR;  // 16-byte chunks of a row; rows of a warp-wide load
            const int own = r < nrows ? (row0 + r) / G : -1;  // this lane's row: its token
            const int64_t off = own < 0 ? -1 : (q_first + own) * a.q_row + (h * G + row0 + r - own * G) * a.q_head;
            const int ch = lane % CPR;
            uint8_t* dst = sm + t * C::kQTile + (ch >> 3) * C::kChunk + (warp & 3) * 32 * 128;
#pragma unroll 1
            for (int i0q = 0; i0q < 32; i0q += 8 * RPI) {
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, i0q + i * RPI + lane / CPR);
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (o >= 0) v[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + o + ch * 8);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = i0q + i * RPI + lane / CPR;
                    *reinterpret_cast<uint4*>(dst + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = v[i];
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const int rho = row0 + r;
        const bool live = r < nrows;
        const int tok = live ? rho / G : 0, head = live ? h * G + rho - tok * G : 0;
        const int pos = live ? pos0 + tok : -1;
        const int tile_lo = pos0 + (row0 + t * kRows) / G, tile_hi = pos0 + (row0 + min(nrows, (t + 1) * kRows) - 1) / G;
        const bool warp_live = t * kRows + (warp & 3) * 32 < nrows;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nj; ++j) {
            const uint32_t par = static_cast<uint32_t>(j) & 1u;
            ok = tc::warp_wait(&s_full[t], par, abort);
            if (!ok) break;
            tc::fence_after();
            float x[kKeys];
            if (warp_live) {
#pragma unroll
                for (int c = 0; c < kKeys; c += 32) tc::ld32(tmem + lanes + C::s_col(t) + c, x + c);
                tc::wait_ld();
#pragma unroll
                for (int c = 0; c < kKeys; c += 32) tc::tie32(x + c);
            }
            if (!C::kAlias) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[t]);
            }
            // The product that last read this P buffer has been added (with one
            // buffer in S's columns, these scores came after it).
            if (!C::kAlias && j >= C::NP) {
                ok = tc::warp_wait(pv_done(t, j - C::NP), p_parity(j - C::NP), abort);
                if (!ok) break;
                tc::fence_after();
            }
            const int j0 = walk.tile(i0 + j) * kKeys;
            if (warp_live && (j0 + kKeys - 1 > tile_lo || nrows < (t + 1) * kRows || (a.window > 0 && j0 <= tile_hi - a.window))) {
                // visible: c <= hi, and c > lo or c < first
                const int hi = pos - j0, lo = a.window > 0 ? pos - a.window - j0 : -1, first = a.window > 0 ? a.sinks - j0 : 0;
#pragma unroll
                for (int c = 0; c < kKeys; ++c)
                    if (c > hi || (c <= lo && c >= first)) x[c] = -INFINITY;
            }
            // rows of V that no row of this CTA sees: zero (once, by the first query tile that uses them)
            if ((t == 0 || j >= n0) && (j0 + kKeys - 1 > t_max || (a.window > 0 && j0 < walk.w_min))) {
                // entries up to V of the tile before have landed: full's parity is unambiguous
                if (C::NP == 2 && j > 0) {
                    ok = tc::warp_wait(pv_done(t, j - 1), p_parity(j - 1), abort);
                    if (!ok) break;
                }
                // a warp's 32 rows, four at a time: eight lanes to the 128 bytes of a row
                const int at = (warp & 3) * 32 + (lane >> 3);
#pragma unroll
                for (int sp = 0; sp < SPT; ++sp) {
                    const int e = v_seq(j) + sp, s = e % NST;
                    ok = ok && tc::warp_wait(&full[s], static_cast<uint32_t>(e / NST) & 1u, abort);
                    if (!ok) break;
                    uint8_t* stage = ring + s * C::kStage + (lane & 7) * 16;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const int q = j0 + at + i;
                        if (q <= t_max && (a.window == 0 || q >= walk.w_min || q < a.sinks)) continue;
#pragma unroll
                        for (int ch = 0; ch < C::SD / 64; ++ch)
                            *reinterpret_cast<uint4*>(stage + ch * C::kChunk + (at + i) * 128) = make_uint4(0, 0, 0, 0);
                    }
                }
                if (!ok) break;
                fence_proxy_async_smem();
            }
            if (!warp_live) {  // nobody reads these rows' outputs: whatever P holds will do
                tc::fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(p_half(t, j));
                    mbar_arrive(p_full(t, j));
                }
                continue;
            }
            const float2 sc = make_float2(wk.scale2, wk.scale2);
            float2 sum[2];
            uint32_t p[kKeys / 4];
            float m2 = m == -INFINITY ? 0.f : m * wk.scale2 - kLift<T>;
            // The running maximum moves to the row's largest score so far.
            auto raise = [&]() {
                float top[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) top[q] = x[q];
#pragma unroll
                for (int c = 8; c < kKeys; ++c) top[c & 7] = fmaxf(top[c & 7], x[c]);
#pragma unroll
                for (int q = 4; q > 0; q >>= 1)
#pragma unroll
                    for (int i = 0; i < q; ++i) top[i] = fmaxf(top[i], top[i + q]);
                const float mn = fmaxf(m, top[0]), f = m == -INFINITY ? 0.f : tc::ex2((m - mn) * wk.scale2);
                m = mn;
                m2 = m == -INFINITY ? 0.f : m * wk.scale2 - kLift<T>;
                l *= f;
                if (j == 0) return;
                ok = tc::warp_wait(pv_done(t, j - 1), p_parity(j - 1), abort);
                if (!ok) return;
                tc::fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    uint32_t u[32];
                    tc::ld32(tmem + lanes + C::o_col(t) + c, o);
                    tc::wait_ld();
                    tc::tie32(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(o[i] * f);
                    tc::st32(tmem + lanes + C::o_col(t) + c, u);
                }
                tc::wait_st();
            };
            auto weights = [&](int q) {  // of columns 32 q .. 32 q + 31
                const float2 nm = make_float2(-m2, -m2);
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float2 w = ffma2(make_float2(x[32 * q + c], x[32 * q + c + 1]), sc, nm);
                    w = make_float2(tc::ex2(w.x), tc::ex2(w.y));
                    sum[(c >> 1) & 1] = tc::add2(sum[(c >> 1) & 1], w);
                    p[16 * (q & 1) + c / 2] = pack16(w.x, w.y, T());
                }
            };
            // The first half's weights are taken under the old maximum, and the
            // maximum is raised (and they are taken again) only where their sum
            // or a score of the second half asks for it: looking for the largest
            // of 128 scores first costs 250 clocks a tile, the second half's
            // search hides behind the exponentials.
            const bool fresh = __any_sync(0xffffffffu, live && m == -INFINITY);
            if (fresh) raise();
            if (!ok) break;
            auto first_half = [&]() -> bool {
                sum[0] = sum[1] = make_float2(0.f, 0.f);
                float top[4] = {x[64], x[65], x[66], x[67]};
                weights(0);
#pragma unroll
                for (int c = 68; c < kKeys; ++c) top[c & 3] = fmaxf(top[c & 3], x[c]);
                weights(1);
                const float s = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                const float t2 = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                return s > kMaxWeight<T> || fmaf(t2, wk.scale2, -m2) > kMaxSlack + kLift<T>;
            };
            const bool over = first_half();
            if (!fresh && __any_sync(0xffffffffu, over)) {
                raise();
                if (!ok) break;
                (void)first_half();
            }
            tc::st32(tmem + lanes + C::p_col(t, j), p);
            weights(2);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_half(t, j));
            weights(3);
            tc::st32(tmem + lanes + C::p_col(t, j) + 32, p);
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(t, j));
        }
        if (ok && nj > 0) ok = tc::warp_wait(pv_done(t, nj - 1), p_parity(nj - 1), abort);
        if (!ok) tc::give_up(abort, a.err);
        tc::fence_after();
        constexpr int CS = D + 4;
        const int64_t item = bid;
        float* rec = wk.part + ((item * wk.nsplit + split) * NQ * kRows + r) * CS;
        T* out = static_cast<T*>(a.out) + (q_first + tok) * a.out_row + head * a.out_head;
        // no weight seen (NaN scores leave the maximum where it is, but not the sum)
        const bool none = l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
        if (ok && warp_live) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                if (nj > 0) {
                    tc::ld32(tmem + lanes + C::o_col(t) + c, o);
                    tc::wait_ld();
                    tc::tie32(o);
                }
                if (!live) continue;
                if (nj == 0 || none)
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                if (ns == 1) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4*>(out + c + i) =
                            make_uint4(pack16(o[i] * inv, o[i + 1] * inv, T()), pack16(o[i + 2] * inv, o[i + 3] * inv, T()),
                                       pack16(o[i + 4] * inv, o[i + 5] * inv, T()), pack16(o[i + 6] * inv, o[i + 7] * inv, T()));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(rec + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
            }
            if (live && ns == 1 && a.lse)
                a.lse[(q_first + tok) * a.lse_row + head] =
                    none ? -INFINITY : fmaf(m, wk.scale2, log2f(l) - kLift<T>) * 0.693147180559945309f;
            if (live && ns > 1) *reinterpret_cast<float2*>(rec + D) = make_float2(none ? -INFINITY : m * wk.scale2 - kLift<T>, l);
        }
        if (ns > 1) {
            // ---- the last of the walk's CTAs to get here joins their states in order ----
            constexpr int kSoft = C::kSoftWarps * 32;
            __threadfence();
            asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
            if (threadIdx.x == 0) {
                const uint32_t old = atomicAdd(&wk.cnt[item], 1u);
                *joined = old == static_cast<uint32_t>(ns - 1);
                if (*joined) wk.cnt[item] = 0u;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
            if (*joined) {
                __threadfence();
                const float* recs = wk.part + item * wk.nsplit * NQ * kRows * CS;
                constexpr int64_t kNext = static_cast<int64_t>(NQ) * kRows * CS;
                // [row][split] weights, 1 / sum with the last one (in the ring, which is free)
                float* wgt = reinterpret_cast<float*>(ring);
                for (int row = threadIdx.x; row < nrows; row += kSoft) {
                    const float* p = recs + static_cast<int64_t>(row) * CS + D;
                    float M = -INFINITY, L = 0.f;
                    float2 ml[kMaxSplit];
#pragma unroll
                    for (int s = 0; s < kMaxSplit; ++s)
                        if (s < ns) {
                            ml[s] = __ldcg(reinterpret_cast<const float2*>(p + s * kNext));
                            M = fmaxf(M, ml[s].x);
                        }
#pragma unroll
                    for (int s = 0; s < kMaxSplit; ++s)
                        if (s < ns) {
                            const float f = ml[s].x == -INFINITY ? 0.f : exp2f(ml[s].x - M);
                            L += ml[s].y * f;
                            wgt[row * (kMaxSplit + 1) + s] = f;
                        }
                    wgt[row * (kMaxSplit + 1) + kMaxSplit] = L == 0.f ? 0.f : 1.f / L;
                    const int rr = row0 + row, tk = rr / G;
                    if (a.lse)
                        a.lse[(q_first + tk) * a.lse_row + h * G + rr - tk * G] =
                            L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
                // eight float4 of the output a thread at a time, so that their loads overlap
                constexpr int kBatch = 8;
                const int quads = nrows * (D / 4);
#pragma unroll 1
                for (int i0q = threadIdx.x; i0q < quads; i0q += kSoft * kBatch) {
                    float4 A[kBatch];
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) A[q] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                    for (int s = 0; s < ns; ++s) {
#pragma unroll
                        for (int q = 0; q < kBatch; ++q) {
                            const int i = min(i0q + q * kSoft, quads - 1), row = i / (D / 4);
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(recs + s * kNext + row * CS + (i % (D / 4)) * 4));
                            const float f = wgt[row * (kMaxSplit + 1) + s];
                            A[q].x += v.x * f;
                            A[q].y += v.y * f;
                            A[q].z += v.z * f;
                            A[q].w += v.w * f;
                        }
                    }
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) {
                        const int i = i0q + q * kSoft, row = i / (D / 4);
                        if (i >= quads) continue;
                        const int rr = row0 + row, tk = rr / G;
                        const float iv = wgt[row * (kMaxSplit + 1) + kMaxSplit];
                        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (q_first + tk) * a.out_row + (h * G + rr - tk * G) * a.out_head +
                                                  (i % (D / 4)) * 4) =
                            make_uint2(pack16(A[q].x * iv, A[q].y * iv, T()), pack16(A[q].z * iv, A[q].w * iv, T()));
                    }
                }
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, 512);
    }
}

}  // namespace

// A pool as a 4-D tensor (column, slot, head, page); boxes of min(page, 128)
// slots x 64 columns in the 128-byte swizzle.
bool paged_pool_map(const PagedKv& kv, void* pool, CUtensorMap* out) {
    const TmapEncodeFn encode = tmap_encoder();
    if (!encode) return false;
    const cuuint64_t page = cuuint64_t{1} << kv.page_log2;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.D), page, static_cast<cuuint64_t>(kv.nkv),
                                static_cast<cuuint64_t>(kv.num_pages)};
    // the stride of an extent of one is never used
    const cuuint64_t row = static_cast<cuuint64_t>(kv.D) * 2;
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(kv.slot_stride) * 2,
                                   kv.nkv > 1 ? static_cast<cuuint64_t>(kv.head_stride) * 2 : row,
                                   kv.num_pages > 1 ? static_cast<cuuint64_t>(kv.page_stride) * 2 : row};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(std::min<cuuint64_t>(page, kKeys)), 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return encode(out, kv.type == kPagedF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, pool,
                  dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

template <typename T, int D>
cudaError_t launch(const PagedKv& kv, const PagedAttn& a, PromptWork wk, int num_sms, cudaStream_t s) {
    using C = PCfg<D>;
    auto kernel = paged_prompt_kernel<T, D>;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < 64) done[dev] = true;
    }
    CUtensorMap tk, tv;
    if (!paged_pool_map(kv, kv.k, &tk) || !paged_pool_map(kv, kv.v, &tv)) return cudaErrorInvalidValue;
    const int64_t rows = std::min<int64_t>(a.max_new, a.rows) * a.G;
    wk.tiles = static_cast<int>((rows + C::NQ * kRows - 1) / (C::NQ * kRows));
    const int64_t items = static_cast<int64_t>(wk.tiles) * kv.nseq * kv.nkv;
    const int64_t key_tiles = ((static_cast<int64_t>(kv.width) << kv.page_log2) + kKeys - 1) / kKeys;
    // few rows: each walk over as many CTAs as fill the SMs, two key tiles each at least
    wk.nsplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({num_sms / items, (key_tiles + 1) / 2, kMaxSplit})));
    if (items * wk.nsplit > INT32_MAX) return cudaErrorInvalidValue;
    kernel<<<static_cast<unsigned>(items * wk.nsplit), C::kThreads, C::kSmem, s>>>(tk, tv, kv, a, wk);
    return cudaGetLastError();
}

template <typename T>
cudaError_t by_dim(const PagedKv& kv, const PagedAttn& a, const PromptWork& wk, int num_sms, cudaStream_t s) {
    if (kv.D == 64) return launch<T, 64>(kv, a, wk, num_sms, s);
    if (kv.D == 128) return launch<T, 128>(kv, a, wk, num_sms, s);
    return launch<T, 256>(kv, a, wk, num_sms, s);
}

}  // namespace

// One record of every CTA of a split grid (one CTA per SM at most).
size_t paged_prompt_part_bytes(int num_sms) {
    const size_t d128 = 2 * kRows * (128 + 4), d256 = kRows * (256 + 4);
    return num_sms * std::max(d128, d256) * sizeof(float);
}

cudaError_t paged_prompt16_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s) {
    PromptWork wk = {};
    wk.cnt = static_cast<uint32_t*>(workspace);
    wk.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + paged_counter_bytes(num_sms));
    wk.scale2 = a.scale * 1.44269504088896341f;
    return kv.type == kPagedF16 ? by_dim<__half>(kv, a, wk, num_sms, s) : by_dim<__nv_bfloat16>(kv, a, wk, num_sms, s);
}

}  // namespace rt
