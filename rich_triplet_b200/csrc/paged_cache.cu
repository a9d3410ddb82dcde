// paged_cache.cu -- writing a paged cache: new rows in (append) and a
// sequence's most attended rows to other pages (evict).
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace rt {

namespace {

// Eight consecutive elements as f32, 16-byte (f16, bf16) or 2 x 16-byte (f32) accesses.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = u;
}

// One CTA per new row; a thread moves eight elements of K and of V at a time.
// HBM-bound: 155 MB (f32 to f16, 16 heads of 128) in 26.5 us, 5.8 TB/s; three
// rows in 2.2 us.
template <typename S, typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedKv kv, const PagedRows a) {
    const int64_t r = blockIdx.x;
    int b = static_cast<int>(r);
    int64_t j = 0;
    if (a.q_start) {
        b = row_seq(a.q_start, kv.nseq, r);
        if (r < a.q_start[b]) return;
        j = static_cast<int64_t>(a.q_start[b + 1]) - r;
        if (j <= 0) return;
        j = kv.len(b) - j;
    } else {
        j = kv.len(b) - 1;
    }
    if (j < 0) return;
    const int64_t off = kv.row(b, static_cast<int>(j));
    if (off < 0) return;
    const int per = kv.D / 8;
    for (int i = threadIdx.x; i < kv.nkv * per; i += blockDim.x) {
        const int h = i / per, d = (i % per) * 8;
        const int64_t src = r * a.row_stride + h * a.head_stride + d, dst = off + h * kv.head_stride + d;
        float x[8], y[8];
        load8(static_cast<const S*>(a.k) + src, x);
        load8(static_cast<const S*>(a.v) + src, y);
        store8(static_cast<T*>(kv.k) + dst, x);
        store8(static_cast<T*>(kv.v) + dst, y);
    }
}

template <typename S>
cudaError_t append_to(const PagedKv& kv, const PagedRows& a, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(a.rows);
    const int threads = std::min(256, (kv.nkv * kv.D / 8 + 31) / 32 * 32);
    if (kv.type == kPagedF32) paged_append_kernel<S, float><<<grid, threads, 0, s>>>(kv, a);
    else if (kv.type == kPagedF16) paged_append_kernel<S, __half><<<grid, threads, 0, s>>>(kv, a);
    else paged_append_kernel<S, __nv_bfloat16><<<grid, threads, 0, s>>>(kv, a);
    return cudaGetLastError();
}

// ---- evict ----

constexpr int kKeysEach = 8;                  // keys a thread holds of a block
constexpr int kHeldBlocks = 4;                // blocks whose keys stay in registers
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // rank_key of -inf
constexpr uint32_t kKeptKey = 0xFFFFFFFFu;    // rank_key of the ends that are always kept

// Rank of a position with mass x as an unsigned number in the order of x, NaN
// as -inf; 0 past the end.  Adding 0 makes -0 and +0 equal.
__device__ __forceinline__ uint32_t rank_key(const PagedEvict& e, float x, uint32_t j, int len) {
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t key = x != x ? kLowestKey : (u >> 31) ? ~u : (u | 0x80000000u);
    const uint32_t n = len, from = max(0, len - e.recent), first = e.sinks;
    return j >= n ? 0u : (j < first || j >= from) ? kKeptKey : key;
}

// Exclusive prefix of `v` over the block's threads; `total` is the block's sum.
template <int kThreads>
__device__ __forceinline__ int block_prefix(int v, int* red, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    int w = lane < kThreads / 32 ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - v + (warp ? before : 0);
}

// One CTA per (sequence, KV head).  The keys are read once and stay in
// registers where a table row has room for at most kHeldBlocks blocks (HELD;
// else each pass reads them again).  Three passes over 11, 11 and 10 bits find the key of
// the last position kept, by a histogram in shared memory each; then the kept
// positions are written in order: a warp owns 256 consecutive positions of a
// block, so that ballots rank them inside the warp and one prefix over the
// warps ranks the warps.  Latency-bound: 8192 positions of 128
// rows in 10.3 us.
template <int kThreads, bool HELD>
__global__ void __launch_bounds__(kThreads) paged_select_kernel(const PagedKv kv, const PagedEvict e) {
    __shared__ int hist[2048];
    __shared__ int red[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    constexpr int kBlock = kThreads * kKeysEach;
    pdl_launch_dependents();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int len = kv.len(b), n = min(len, e.budget);
    const float* mass = e.mass + b * e.mass_seq + h * e.mass_head;
    float* mout = e.mass_out + b * e.mass_seq + h * e.mass_head;
    int32_t* kept = e.kept + (static_cast<int64_t>(b) * kv.nkv + h) * e.budget;
    if (h == 0 && tid == 0) e.new_lens[b] = n;
    const int blocks = static_cast<int>((static_cast<uint32_t>(len) + kBlock - 1) / kBlock);
    const bool all = len <= e.budget;
    // (unsigned: the last block may end past 2^31)
    auto position = [&](int blk, int i) { return static_cast<uint32_t>(blk) * kBlock + (warp * 256 + i * 32 + lane); };
    const uint32_t have = min(len, e.mass_cap);  // positions with mass
    auto load_keys = [&](int blk, uint32_t(&k)[kKeysEach]) {  // all loads before the first use
        float x[kKeysEach];
#pragma unroll
        for (int i = 0; i < kKeysEach; ++i) {
            const uint32_t j = position(blk, i);
            x[i] = j < have ? mass[j] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kKeysEach; ++i) k[i] = rank_key(e, x[i], position(blk, i), len);
    };
    uint32_t held[HELD ? kHeldBlocks : 1][kKeysEach];
    if (HELD) {
#pragma unroll
        for (int blk = 0; blk < kHeldBlocks; ++blk)
            if (blk < blocks) load_keys(blk, held[HELD ? blk : 0]);
    }
    // f(block, its keys) for every block
    auto for_blocks = [&](auto f) {
        if (HELD) {
#pragma unroll
            for (int blk = 0; blk < kHeldBlocks; ++blk)
                if (blk < blocks) f(blk, held[HELD ? blk : 0]);
        } else {
            for (int blk = 0; blk < blocks; ++blk) {
                load_keys(blk, held[0]);
                f(blk, held[0]);
            }
        }
    };
    uint32_t last = 0;                       // key of the last position kept by rank
    int want = n - e.sinks - e.recent;       // positions kept by rank; of those with key `last`, when it is known
    if (!all && want == 0) last = kKeptKey - 1;  // above every mass
    if (!all && want > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
#pragma unroll
            for (int i = tid; i < 2048; i += kThreads) hist[i] = 0;
            __syncthreads();
            for_blocks([&](int, const uint32_t(&k)[kKeysEach]) {
#pragma unroll
                for (int i = 0; i < kKeysEach; ++i)
                    if (k[i] != 0u && k[i] != kKeptKey &&
                        (pass == 0 || (k[i] >> (pass == 1 ? 21 : 10)) == (last >> (pass == 1 ? 21 : 10))))
                        atomicAdd(&hist[(k[i] >> shift) & (bins - 1)], 1);
            });
            __syncthreads();
            // thread t looks at kDigits digits from the top: the one in which the count passes `want`
            constexpr int kDigits = 2048 / kThreads;
            const int top = bins - 1 - tid * kDigits;
            int sum = 0;
            if (top >= 0)
#pragma unroll
                for (int i = 0; i < kDigits; ++i) sum += hist[top - i];
            int total;
            int above = block_prefix<kThreads>(sum, red, total);
            if (above < want && above + sum >= want) {
#pragma unroll
                for (int i = 0; i < kDigits; ++i) {
                    const int c = hist[top - i];
                    if (above < want && above + c >= want) {
                        s_prefix = last | static_cast<uint32_t>(top - i) << shift;
                        // all of the digit's keys are kept: keys from `prefix` on, without a later pass
                        s_want = want - above == c ? 0 : want - above;
                        if (s_want == 0) s_prefix -= 1u;
                    }
                    above += c;
                }
            }
            __syncthreads();
            last = s_prefix;
            want = s_want;
            __syncthreads();
            if (want == 0) break;
        }
    }
    int done = 0, equal = 0;  // kept so far; keys equal to `last` so far
    const uint32_t below = (1u << lane) - 1u;
    for_blocks([&](int blk, const uint32_t(&k)[kKeysEach]) {
        uint32_t keep[kKeysEach];
        int eq_base = 0;
        if (!all) {
            int eqs = 0;
#pragma unroll
            for (int i = 0; i < kKeysEach; ++i) eqs += __popc(__ballot_sync(0xffffffffu, k[i] == last));
            int total;
            // every lane adds its warp's count once: lane 0's carries it
            const int before = block_prefix<kThreads>(lane == 0 ? eqs : 0, red, total);
            eq_base = equal + __shfl_sync(0xffffffffu, before, 0);
            equal += total;
        }
        int kepts = 0;
#pragma unroll
        for (int i = 0; i < kKeysEach; ++i) {
            const uint32_t eq = __ballot_sync(0xffffffffu, !all && k[i] == last);
            const bool mine = k[i] != 0u && (all || k[i] == kKeptKey || k[i] > last ||
                                             (k[i] == last && eq_base + __popc(eq & below) < want));
            eq_base += __popc(eq);
            keep[i] = __ballot_sync(0xffffffffu, mine);
            kepts += __popc(keep[i]);
        }
        int total;
        const int before = block_prefix<kThreads>(lane == 0 ? kepts : 0, red, total);
        int at = done + __shfl_sync(0xffffffffu, before, 0);
        done += total;
#pragma unroll
        for (int i = 0; i < kKeysEach; ++i) {
            if (keep[i] >> lane & 1u) {
                const uint32_t j = position(blk, i);
                const int to = at + __popc(keep[i] & below);
                kept[to] = static_cast<int>(j);
                if (to < e.mass_cap) mout[to] = j < have ? mass[j] : 0.f;
            }
            at += __popc(keep[i]);
        }
    });
    for (int64_t i = n + tid; i < e.budget; i += kThreads) kept[i] = -1;
    for (int64_t i = n + tid; i < e.mass_cap; i += kThreads) mout[i] = 0.f;
}

// A warp moves the K and V of eight kept rows (row bytes 16 CPR), their page
// lookups and then their loads in flight together: HBM-bound, kept rows read
// and written once (32 x 4 x 2048 rows of 512 bytes, K and V: 94 us, 5.7 TB/s).
template <int CPR>
__global__ void __launch_bounds__(256) paged_gather_kernel(const PagedKv kv, const PagedEvict e) {
    constexpr int kRows = 8, kEach = kRows * CPR / 32, kBatch = kEach < 8 ? kEach : 8;
    const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
    const int first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kRows;
    const int n = min(kv.len(b), e.budget);
    pdl_wait();
    if (first >= n) return;
    const int64_t es = kv.type == kPagedF32 ? 4 : 2;
    int64_t src = -1, dst = -1;  // byte offsets of row `first + lane`
    const int i = first + lane;
    if (lane < kRows && i < n) {
        const int32_t p = e.dst[b * e.dst_stride + (i >> kv.page_log2)];
        const int64_t s = kv.row(b, e.kept[(static_cast<int64_t>(b) * kv.nkv + h) * e.budget + i]);
        if (s >= 0) src = (s + h * kv.head_stride) * es;
        if (static_cast<uint32_t>(p) < static_cast<uint64_t>(kv.num_pages))
            dst = (p * kv.page_stride + (i & ((1 << kv.page_log2) - 1)) * kv.slot_stride + h * kv.head_stride) * es;
    }
#pragma unroll
    for (int x0 = 0; x0 < kEach; x0 += kBatch) {
        uint4 k[kBatch], v[kBatch];
        int64_t to[kBatch];
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const int id = (x0 + x) * 32 + lane, r = id / CPR, at = (id % CPR) * 16;
            const int64_t s = __shfl_sync(0xffffffffu, src, r);
            to[x] = __shfl_sync(0xffffffffu, dst, r);
            if (to[x] >= 0) to[x] += at;
            k[x] = v[x] = make_uint4(0, 0, 0, 0);
            if (s >= 0) {
                k[x] = *reinterpret_cast<const uint4*>(static_cast<const char*>(kv.k) + s + at);
                v[x] = *reinterpret_cast<const uint4*>(static_cast<const char*>(kv.v) + s + at);
            }
        }
#pragma unroll
        for (int x = 0; x < kBatch; ++x)
            if (to[x] >= 0) {
                *reinterpret_cast<uint4*>(static_cast<char*>(kv.k) + to[x]) = k[x];
                *reinterpret_cast<uint4*>(static_cast<char*>(kv.v) + to[x]) = v[x];
            }
    }
}

}  // namespace

cudaError_t paged_append_launch(const PagedKv& kv, const PagedRows& r, cudaStream_t s) {
    return r.src_type == kPagedF32 ? append_to<float>(kv, r, s)
         : r.src_type == kPagedF16 ? append_to<__half>(kv, r, s) : append_to<__nv_bfloat16>(kv, r, s);
}

cudaError_t paged_evict_launch(const PagedKv& kv, const PagedEvict& e, cudaStream_t s) {
    const dim3 rows(kv.nkv, kv.nseq);
    // A small block's barriers cost less, a large one's threads hold fewer keys
    // each: 700 positions take 7.1 us in 256 threads and 9.2 in 1024, 8192 take
    // 17.4 and 10.7.  The lengths are on the device, so the room of a table row
    // decides: short sequences in wide tables run on the larger variants.
    const int64_t cap = static_cast<int64_t>(kv.width) << kv.page_log2;
    if (cap <= 256 * kKeysEach) paged_select_kernel<256, true><<<rows, 256, 0, s>>>(kv, e);
    else if (cap <= kHeldBlocks * 1024 * kKeysEach) paged_select_kernel<1024, true><<<rows, 1024, 0, s>>>(kv, e);
    else paged_select_kernel<1024, false><<<rows, 1024, 0, s>>>(kv, e);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(e.budget) + 63) / 64), kv.nkv, kv.nseq);
    switch (kv.D * (kv.type == kPagedF32 ? 4 : 2) / 16) {
        case 8: return rt_launch(paged_gather_kernel<8>, grid, 256, 0, s, true, kv, e);
        case 16: return rt_launch(paged_gather_kernel<16>, grid, 256, 0, s, true, kv, e);
        case 32: return rt_launch(paged_gather_kernel<32>, grid, 256, 0, s, true, kv, e);
        default: return rt_launch(paged_gather_kernel<64>, grid, 256, 0, s, true, kv, e);
    }
}

}  // namespace rt
