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
        float x[8];
        load8(static_cast<const S*>(a.k) + src, x);
        store8(static_cast<T*>(kv.k) + dst, x);
        load8(static_cast<const S*>(a.v) + src, x);
        store8(static_cast<T*>(kv.v) + dst, x);
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

constexpr int kSelThreads = 1024;

constexpr uint32_t kLowestKey = 0x007FFFFFu;  // rank_key of -inf

// Rank of a position as an unsigned number in the order of its mass: the kept
// ends above everything, NaN and positions without a mass as -inf.  Adding 0
// makes -0 and +0 equal.
__device__ __forceinline__ uint32_t rank_key(const PagedEvict& e, const float* mass, int j, int len) {
    if (j < e.sinks || j >= len - e.recent) return 0xFFFFFFFFu;
    if (j >= e.mass_cap) return kLowestKey;
    const float x = mass[j] + 0.f;
    if (x != x) return kLowestKey;
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of `v` over the block's threads; `total` is the block's sum.
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
    int w = lane < (blockDim.x >> 5) ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - v + (warp ? before : 0);
}

// One CTA per (sequence, KV head): the budget-th largest key by four passes of
// eight bits over the keys, then the kept positions in order.
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const PagedKv kv, const PagedEvict e) {
    __shared__ int hist[256];
    __shared__ int red[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int len = kv.len(b), n = min(len, e.budget);
    const float* mass = e.mass + b * e.mass_seq + h * e.mass_head;
    float* mout = e.mass_out + b * e.mass_seq + h * e.mass_head;
    int32_t* kept = e.kept + (static_cast<int64_t>(b) * kv.nkv + h) * e.budget;
    if (h == 0 && tid == 0) e.new_lens[b] = n;
    uint32_t prefix = 0;
    int want = n;  // of the keys that share `prefix`, this many are kept
    if (len > e.budget) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < len; j += kSelThreads) {
                const uint32_t key = rank_key(e, mass, j, len);
                if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1);
            }
            __syncthreads();
            // thread t < 256 looks at digit 255 - t: the digit in which the count from above passes `want`
            const int c = tid < 256 ? hist[255 - tid] : 0;
            int total;
            const int above = block_prefix(c, red, total);
            if (tid < 256 && above < want && above + c >= want) {
                s_prefix = prefix | (static_cast<uint32_t>(255 - tid) << shift);
                s_want = want - above;
            }
            __syncthreads();
            prefix = s_prefix;
            want = s_want;
            __syncthreads();
        }
    }
    int done = 0, equal = 0;  // kept so far; keys equal to the threshold so far
    for (int j0 = 0; j0 < len; j0 += kSelThreads) {
        const int j = j0 + tid;
        const uint32_t key = j < len ? rank_key(e, mass, j, len) : 0u;
        bool keep = j < len;
        if (len > e.budget) {
            const bool eq = j < len && key == prefix;
            int eqs;
            const int eq_before = block_prefix(eq, red, eqs);
            keep = j < len && (key > prefix || (eq && equal + eq_before < want));
            equal += eqs;
        }
        int kepts;
        const int at = done + block_prefix(keep, red, kepts);
        if (keep) {
            kept[at] = j;
            if (at < e.mass_cap) mout[at] = j < e.mass_cap ? mass[j] : 0.f;
        }
        done += kepts;
    }
    for (int i = n + tid; i < e.budget; i += kSelThreads) kept[i] = -1;
    for (int i = n + tid; i < e.mass_cap; i += kSelThreads) mout[i] = 0.f;
}

// One warp per kept row: its K and V to slot i of the destination pages.
__global__ void __launch_bounds__(256) paged_gather_kernel(const PagedKv kv, const PagedEvict e, int esize) {
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
    if (i >= min(kv.len(b), e.budget)) return;
    const int j = e.kept[(static_cast<int64_t>(b) * kv.nkv + h) * e.budget + i];
    const int64_t src = kv.row(b, j);
    const int32_t p = e.dst[b * e.dst_stride + (i >> kv.page_log2)];
    if (static_cast<uint32_t>(p) >= static_cast<uint64_t>(kv.num_pages)) return;
    const int64_t dst = p * kv.page_stride + (i & ((1 << kv.page_log2) - 1)) * kv.slot_stride;
    const int words = kv.D * esize / 16;
    for (int w = lane; w < words; w += 32) {
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (src >= 0) {
            x = reinterpret_cast<const uint4*>(static_cast<const char*>(kv.k) + (src + h * kv.head_stride) * esize)[w];
            y = reinterpret_cast<const uint4*>(static_cast<const char*>(kv.v) + (src + h * kv.head_stride) * esize)[w];
        }
        reinterpret_cast<uint4*>(static_cast<char*>(kv.k) + (dst + h * kv.head_stride) * esize)[w] = x;
        reinterpret_cast<uint4*>(static_cast<char*>(kv.v) + (dst + h * kv.head_stride) * esize)[w] = y;
    }
}

}  // namespace

cudaError_t paged_append_launch(const PagedKv& kv, const PagedRows& r, cudaStream_t s) {
    return r.src_type == kPagedF32 ? append_to<float>(kv, r, s)
         : r.src_type == kPagedF16 ? append_to<__half>(kv, r, s) : append_to<__nv_bfloat16>(kv, r, s);
}

cudaError_t paged_evict_launch(const PagedKv& kv, const PagedEvict& e, cudaStream_t s) {
    paged_select_kernel<<<dim3(kv.nkv, kv.nseq), kSelThreads, 0, s>>>(kv, e);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    paged_gather_kernel<<<dim3((e.budget + 7) / 8, kv.nkv, kv.nseq), 256, 0, s>>>(kv, e, kv.type == kPagedF32 ? 4 : 2);
    return cudaGetLastError();
}

}  // namespace rt
