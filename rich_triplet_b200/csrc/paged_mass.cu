// paged_mass.cu -- attention weights of a prompt summed per cached position
// (the `mass` of rt_paged_prompt) for 16-bit caches, on the tcgen05 tensor
// cores.
//
// The weight exp(s - lse) needs the row's final log-sum, so this is a second
// pass over the scores, after the attention: 2 D flops per visible pair and
// head, one exponential.  It is transposed, S^T = K Q^T, so that a thread owns
// one position (a tensor-memory lane) and adds the weights of the rows, its
// columns, in registers, in a fixed order, with no exchange between threads.
//
// A CTA takes one tile of 128 positions of a (sequence, KV head), keeps its
// keys in shared memory and walks the (token, head) rows that see it, 128 at a
// time: the query rows come into a 128-byte-swizzled ring, the MMA thread forms
// the scores in one of four tensor-memory buffers, and two warpgroups take
// alternate tiles.  Where 128 is a multiple of G a tile's rows are one box of a
// (column, head, token) tensor per 64 columns, which TMA fetches; for other G a
// warpgroup gathers them with cp.async (its address arithmetic doubles a
// tile's time at head_dim 256).  Tiles of
// early positions, which most rows see, start first.
//
// With a window, the tiles of the first tokens are seen by every row and the
// others by a window's worth: their walks are split over several CTAs, and so
// are all walks when there are few; the last of a walk's CTAs to finish adds
// the parts in order.
//
// Waits are bounded as in paged_prompt.cu.
//
// Measured (B200): 6185 tokens in windows of 1024, 16 heads on 4 of 256: 77 us;
// 1650 clocks a 128 x 128 tile, 1250 of them the product, whose operands both
// come from shared memory beside the ring's refill.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "gemv.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace rt {

namespace {

constexpr int kTile = 128;     // positions, and rows, of a tile
constexpr int kSumGroups = 2;  // warpgroups that add
constexpr int kBufs = 4;       // score buffers in tensor memory
constexpr int kThreads = (kSumGroups * 4 + 4 + 1) * 32;
constexpr int kMaxParts = 16;  // CTAs that share a walk, at most

// Grid: `first_parts` CTAs for each item (position tile, sequence and KV head)
// below `first_items`, then `parts` for each other one.
struct MassWork {
    float* part;    // [item][kMaxParts][128]
    uint32_t* cnt;  // [item], zero between calls
    int64_t first_items;
    int first_parts, parts;
    float scale2;   // scale * log2(e)
};

template <int D>
struct MCfg {
    static constexpr int kChunk = kTile * 128;  // 64 columns of 128 rows
    static constexpr int kOperand = (D / 64) * kChunk;
    static constexpr int SPT = D == 256 ? 2 : 1;                  // ring stages of a query tile
    static constexpr int SD = D / SPT;                            // columns of a stage
    static constexpr int kStage = (SD / 64) * kChunk;
    static constexpr int NST = D == 256 ? 4 : D == 128 ? 5 : 8;
    static constexpr int kOffRing = kOperand;
    static constexpr int kOffRow = kOffRing + NST * kStage;  // [adding warp][128] - log-sums of the tile's rows
    static constexpr int kOffTotal = kOffRow + kSumGroups * 4 * kTile * 4;  // [128] the second group's totals
    static constexpr int kOffBar = kOffTotal + kTile * 4;
    static constexpr int kBars = 2 * NST + 2 * kBufs + 2;
    static constexpr int kOffMisc = kOffBar + kBars * 8;
    static constexpr int kSmem = kOffMisc + 16 + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <typename T, int D, bool TMAQ>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_mass_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const PagedKv kv, const PagedAttn a, const MassWork wk) {
    using C = MCfg<D>;
    constexpr int NST = C::NST, SPT = C::SPT;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];

    // ---- the positions of this CTA and the rows that see one of them ----
    const int G = a.G;
    const int64_t bhs = static_cast<int64_t>(kv.nseq) * kv.nkv;
    int64_t item = blockIdx.x;
    int part, parts;
    if (item < wk.first_items * wk.first_parts) {
        parts = wk.first_parts;
        part = static_cast<int>(item % parts);
        item /= parts;
    } else {
        item -= wk.first_items * wk.first_parts;
        parts = wk.parts;
        part = static_cast<int>(item % parts);
        item = item / parts + wk.first_items;
    }
    const int j0 = static_cast<int>(item / bhs) * kTile;
    const int b = static_cast<int>(item % bhs) / kv.nkv, h = static_cast<int>(item % bhs) % kv.nkv;
    const int64_t q_first = a.q_start[b];
    const int all = a.q_start[b + 1] - static_cast<int>(q_first), len = kv.len(b);
    if (all <= 0 || q_first < 0) return;
    const int m = static_cast<int>(min(static_cast<int64_t>(min(all, a.max_new)), a.rows - q_first));  // tokens computed
    const int pos0 = len - all;
    const int j_end = min(j0 + kTile, min(len, a.mass_cap));  // positions whose total is kept
    const int i_lo = max(0, j0 - pos0);
    int i_hi = m - 1;
    if (a.window > 0 && j0 >= a.sinks)
        i_hi = static_cast<int>(min(static_cast<int64_t>(i_hi), static_cast<int64_t>(j_end) - 1 + a.window - 1 - pos0));
    if (j_end <= j0 || i_hi < i_lo) return;
    // rows * G fits 32 bits (checked by the caller)
    const int all_tiles = ((i_hi + 1 - i_lo) * G + kTile - 1) / kTile;
    parts = min(parts, all_tiles);
    if (part >= parts) return;
    const int tile0 = static_cast<int>(static_cast<int64_t>(all_tiles) * part / parts);
    const int n = static_cast<int>(static_cast<int64_t>(all_tiles) * (part + 1) / parts) - tile0;
    const int r_begin = i_lo * G + tile0 * kTile, r_end = (i_hi + 1) * G;

    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    uint8_t* ring = sm + C::kOffRing;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::kOffBar);
    uint64_t* empty = full + NST;
    uint64_t* s_full = empty + NST;
    uint64_t* s_free = s_full + kBufs;
    uint64_t* k_full = s_free + kBufs;
    uint64_t* drain = k_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::kOffMisc);
    volatile int* abort = reinterpret_cast<volatile int*>(sm + C::kOffMisc + 4);
    int* joined = reinterpret_cast<int*>(sm + C::kOffMisc + 8);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, tid = threadIdx.x & 127;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(&full[s], TMAQ ? 1 : 4);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kBufs; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_free[s], 4);
        }
        mbar_init(k_full, 1);
        mbar_init(drain, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 0) tc::alloc(tmem_slot, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;
    float total = 0.f;

    if (warp == kSumGroups * 4 + 4) {
        // ---- the keys, then the products ----
        if (lane == 0) mbar_arrive_expect_tx(k_full, C::kOperand);
        __syncwarp();
        const int rows = min(1 << kv.page_log2, kTile), boxes = kTile / rows;
        for (int i = lane; i < boxes * (D / 64); i += 32) {
            const int chunk = i / boxes, box = i % boxes, p = j0 + box * rows;
            int page = -1;
            if (p < len) page = kv.table[b * kv.table_stride + (p >> kv.page_log2)];
            if (static_cast<uint32_t>(page) >= static_cast<uint64_t>(kv.num_pages)) page = static_cast<int>(kv.num_pages);
            tc::tma_4d(sm + chunk * C::kChunk + box * rows * 128, &tm_k, 64 * chunk, p & ((1 << kv.page_log2) - 1), h, page,
                       k_full);
        }
        __syncwarp();
        constexpr uint32_t kId = tc::idesc_f16(BF16, kTile, false);
        bool ok = tc::warp_wait(k_full, 0u, abort);
        for (int i = 0; i < n && ok; ++i) {
            const int buf = i % kBufs;
            ok = i < kBufs || tc::warp_wait(&s_free[buf], static_cast<uint32_t>(i / kBufs - 1) & 1u, abort);
            const uint32_t st = tc::uniform(tmem + buf * kTile);
#pragma unroll
            for (int sp = 0; sp < SPT; ++sp) {
                const int e = i * SPT + sp, s = e % NST;
                ok = ok && tc::warp_wait(&full[s], static_cast<uint32_t>(e / NST) & 1u, abort);
                if (!ok) break;
                tc::fence_after();
                const uint32_t kb = tc::uniform(tc::desc_lo(smem_u32(sm) + sp * C::kStage, 16));
                const uint32_t qb = tc::uniform(tc::desc_lo(smem_u32(ring + s * C::kStage), 16));
                if (tc::elect()) {
#pragma unroll
                    for (int k = 0; k < C::SD / 16; ++k) {
                        const uint32_t at = (k >> 2) * C::kChunk + (k & 3) * 32;
                        tc::mma_ss(st, tc::desc_sw128(kb, at), tc::desc_sw128(qb, at), kId, sp > 0 || k > 0);
                    }
                    tc::commit(&empty[s]);
                    if (sp == SPT - 1) tc::commit(&s_full[buf]);
                }
                __syncwarp();
            }
        }
        if (!ok) tc::give_up(abort, a.err);
        if (tc::elect()) tc::commit(drain);
        __syncwarp();
        (void)mbar_wait_timed(drain, 0u);
        (void)mbar_wait_timed(k_full, 0u);
        __syncwarp();
    } else if (warp >= kSumGroups * 4) {
        // ---- query rows into the ring ----
        bool ok = true;
        if constexpr (TMAQ) {
            if (warp == kSumGroups * 4 && lane == 0) {
                int done = 0;
                for (int e = 0; e < n * SPT && ok; ++e) {
                    const int s = e % NST;
                    ok = e < NST || tc::wait_phase(&empty[s], static_cast<uint32_t>(e / NST - 1) & 1u, abort);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&full[s], C::kStage);
                    const int tok = (r_begin + (e / SPT) * kTile) / G;  // tiles begin with a token
#pragma unroll
                    for (int c = 0; c < C::SD / 64; ++c)
                        tc::tma_3d(ring + s * C::kStage + c * C::kChunk, &tm_q, (e % SPT) * C::SD + 64 * c, h * G,
                                   static_cast<int>(q_first) + tok, &full[s]);
                    ++done;
                }
                // no copy may still be landing when the CTA exits
                for (int e = max(0, done - NST); e < done; ++e)
                    (void)mbar_wait_timed(&full[e % NST], static_cast<uint32_t>(e / NST) & 1u);
            }
            __syncwarp();
        } else {
            // gathered, one stage ahead of the one that is handed over
            constexpr int CPR = C::SD / 8;      // 16-byte chunks of a row of a stage
            constexpr int RPI = 32 / CPR;       // rows of a warp-wide copy
            const int row0 = (warp & 3) * 32;   // this warp's rows of a tile
            for (int e = 0; e <= n * SPT; ++e) {
                if (e < n * SPT) {
                    const int s = e % NST;
                    ok = ok && (e < NST || tc::warp_wait(&empty[s], static_cast<uint32_t>(e / NST - 1) & 1u, abort));
                    if (!ok) break;
                    // rows past the end repeat the last one (their weight is 0)
                    const int rho = min(r_begin + (e / SPT) * kTile + row0 + lane, r_end - 1), tok = rho / G;
                    const int64_t off = (q_first + tok) * a.q_row + (h * G + rho - tok * G) * a.q_head;
                    const int ch = lane % CPR;
                    const T* src = static_cast<const T*>(a.q) + (e % SPT) * C::SD + ch * 8;
                    const uint32_t dst = smem_u32(ring + s * C::kStage) + (ch >> 3) * C::kChunk;
#pragma unroll 8
                    for (int x = 0; x < 32 / RPI; ++x) {
                        const int r = x * RPI + lane / CPR, row = row0 + r;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + row * 128 + (((ch & 7) ^ (row & 7)) << 4)),
                                     "l"(src + __shfl_sync(0xffffffffu, off, r))
                                     : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (e > 0) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[(e - 1) % NST]);
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        if (!ok) tc::give_up(abort, a.err);
    } else {
        // ---- thread = position ----
        const int grp = warp >> 2, j = j0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
        // a warp's own copy of the tile's rows: minus the log-sum (powers of two;
        // -inf for none, whose weight is then 0)
        float* rz = reinterpret_cast<float*>(sm + C::kOffRow) + warp * kTile;
        float next_z[4];
        auto load_rows = [&](int i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int rho = min(r_begin + i * kTile + lane + 32 * e, r_end - 1), tok = rho / G;
                next_z[e] = a.lse[(q_first + tok) * a.lse_row + h * G + rho - tok * G];
            }
        };
        // rows of the tokens that see position j: [see, until)
        // (counts of tokens are cut to those of the call before they are multiplied: positions times G pass 32 bits)
        const int see = min(max(0, j - pos0), i_hi + 1) * G;
        const int until = a.window > 0 && j >= a.sinks
                              ? static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(i_hi) + 1, static_cast<int64_t>(j) + a.window - pos0))) * G
                              : r_end;
        load_rows(grp);
        bool ok = true;
        for (int i = grp; i < n; i += kSumGroups) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e) rz[lane + 32 * e] = next_z[e] == -INFINITY ? -INFINITY : next_z[e] * -1.44269504088896341f;
            __syncwarp();
            if (i + kSumGroups < n) load_rows(i + kSumGroups);
            const int buf = i % kBufs;
            ok = tc::warp_wait(&s_full[buf], static_cast<uint32_t>(i / kBufs) & 1u, abort);
            if (!ok) break;
            tc::fence_after();
            const int r0 = r_begin + i * kTile;
            // columns [c_see, c_until) of this tile are rows that see position j
            const int c_see = see - r0, c_until = until - r0;
            const bool masked = __any_sync(0xffffffffu, c_see > 0 || c_until < kTile);
            const float2 sc = make_float2(wk.scale2, wk.scale2);
            float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
            for (int c = 0; c < kTile; c += 64) {
                float x[64];
                tc::ld32(tmem + lanes + buf * kTile + c, x);
                tc::ld32(tmem + lanes + buf * kTile + c + 32, x + 32);
                tc::wait_ld();
                tc::tie32(x);
                tc::tie32(x + 32);
                if (c > 0) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[buf]);
                }
                auto add = [&](auto with_mask) {
#pragma unroll
                    for (int e = 0; e < 64; e += 4) {
                        const float4 z = *reinterpret_cast<const float4*>(rz + c + e);
                        float2 w0 = ffma2(make_float2(x[e], x[e + 1]), sc, make_float2(z.x, z.y));
                        float2 w1 = ffma2(make_float2(x[e + 2], x[e + 3]), sc, make_float2(z.z, z.w));
                        if constexpr (decltype(with_mask)::value) {
                            // behind the log-sum, which is NaN where a row has a NaN
                            auto see = [&](float v, int at) { return at < c_see || at >= c_until ? -INFINITY : v; };
                            w0 = make_float2(see(w0.x, c + e), see(w0.y, c + e + 1));
                            w1 = make_float2(see(w1.x, c + e + 2), see(w1.y, c + e + 3));
                        }
                        part[0] = tc::add2(part[0], make_float2(tc::ex2(w0.x), tc::ex2(w0.y)));
                        part[1] = tc::add2(part[1], make_float2(tc::ex2(w1.x), tc::ex2(w1.y)));
                    }
                };
                if (masked) add(std::true_type());
                else add(std::false_type());
            }
            total += (part[0].x + part[0].y) + (part[1].x + part[1].y);
        }
        if (!ok) tc::give_up(abort, a.err);
        if (grp == 1) reinterpret_cast<float*>(sm + C::kOffTotal)[tid] = total;
    }
    tc::fence_before();
    __syncthreads();
    if (warp < 4) {
        const int j = j0 + threadIdx.x;
        float sum = total + reinterpret_cast<const float*>(sm + C::kOffTotal)[threadIdx.x];
        bool write = j < j_end && !*abort;
        if (parts > 1) {
            float* pp = wk.part + item * kMaxParts * kTile + threadIdx.x;
            __stcg(pp + part * kTile, sum);
            __threadfence();
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (threadIdx.x == 0) {
                *joined = atomicAdd(&wk.cnt[item], 1u) == static_cast<uint32_t>(parts - 1);
                if (*joined) wk.cnt[item] = 0u;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            write = write && *joined;
            if (write) {
                __threadfence();
                sum = 0.f;
                for (int q = 0; q < parts; ++q) sum += __ldcg(pp + q * kTile);
            }
        }
        if (write) a.mass[b * a.mass_seq + h * a.mass_head + j] += sum;
    }
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, 512);
    }
}

// The queries as a 3-D tensor (column, head, token); boxes of 128 / G tokens x
// G heads x 64 columns.  False where there is no such map.
bool query_map(const PagedKv& kv, const PagedAttn& a, CUtensorMap* out) {
    const TmapEncodeFn encode = tmap_encoder();
    if (!encode || kTile % a.G != 0 || a.q_row == 0 || (a.nq > 1 && a.q_head == 0)) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(kv.D), static_cast<cuuint64_t>(a.nq), static_cast<cuuint64_t>(a.rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.nq > 1 ? a.q_head : kv.D) * 2, static_cast<cuuint64_t>(a.q_row) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.G), static_cast<cuuint32_t>(kTile / a.G)}, estr[3] = {1, 1, 1};
    return encode(out, kv.type == kPagedF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                  const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool TMAQ>
cudaError_t launch(const PagedKv& kv, const PagedAttn& a, const CUtensorMap& tq, MassWork wk, int num_sms, cudaStream_t s) {
    using C = MCfg<D>;
    auto kernel = paged_prompt_mass_kernel<T, D, TMAQ>;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < 64) done[dev] = true;
    }
    CUtensorMap tk;
    if (!paged_pool_map(kv, kv.k, &tk)) return cudaErrorInvalidValue;
    const int64_t cap = std::min<int64_t>(static_cast<int64_t>(kv.width) << kv.page_log2, a.mass_cap);
    const int64_t bhs = static_cast<int64_t>(kv.nseq) * kv.nkv, tiles = (cap + kTile - 1) / kTile, items = tiles * bhs;
    if (items == 0) return cudaSuccess;
    auto share = [&](int64_t walks) {  // CTAs of a walk when there are so many
        return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxParts, num_sms / walks)));
    };
    wk.parts = share(items);
    wk.first_items = a.window > 0 ? std::min<int64_t>(tiles, (static_cast<int64_t>(a.sinks) + kTile - 1) / kTile) * bhs : 0;
    wk.first_parts = wk.first_items > 0 ? std::max(wk.parts, share(wk.first_items)) : 1;
    const int64_t grid = wk.first_items * wk.first_parts + (items - wk.first_items) * wk.parts;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    kernel<<<static_cast<unsigned>(grid), kThreads, C::kSmem, s>>>(tk, tq, kv, a, wk);
    return cudaGetLastError();
}

template <typename T>
cudaError_t by_dim(const PagedKv& kv, const PagedAttn& a, const MassWork& wk, int num_sms, cudaStream_t s) {
    CUtensorMap tq = {};
    if (query_map(kv, a, &tq)) {
        if (kv.D == 64) return launch<T, 64, true>(kv, a, tq, wk, num_sms, s);
        if (kv.D == 128) return launch<T, 128, true>(kv, a, tq, wk, num_sms, s);
        return launch<T, 256, true>(kv, a, tq, wk, num_sms, s);
    }
    if (kv.D == 64) return launch<T, 64, false>(kv, a, tq, wk, num_sms, s);
    if (kv.D == 128) return launch<T, 128, false>(kv, a, tq, wk, num_sms, s);
    return launch<T, 256, false>(kv, a, tq, wk, num_sms, s);
}

}  // namespace

cudaError_t paged_prompt_mass16_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s) {
    MassWork wk = {};
    wk.cnt = static_cast<uint32_t*>(workspace);
    wk.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + paged_counter_bytes(num_sms));
    wk.scale2 = a.scale * 1.44269504088896341f;
    static_assert(kMaxParts * kTile <= 2 * 128 * (128 + 4), "fits paged_prompt_part_bytes");
    return kv.type == kPagedF16 ? by_dim<__half>(kv, a, wk, num_sms, s) : by_dim<__nv_bfloat16>(kv, a, wk, num_sms, s);
}

}  // namespace rt
