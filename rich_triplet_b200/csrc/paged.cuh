// paged.cuh -- operators over a paged key-value cache (rt_paged_*,
// include/rt_cuda.h): the cache as kernels see it and the launchers.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <cuda.h>  // CUtensorMap
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace rt {

enum PagedType : int { kPagedF32 = 0, kPagedF16 = 1, kPagedBF16 = 2 };

constexpr int kPagedMaxGroup = 16;  // query heads per KV head

// One layer's cache and the call's sequences (rt_paged_kv).
struct PagedKv {
    void* k;
    void* v;
    int64_t page_stride, head_stride, slot_stride;  // elements
    int64_t num_pages;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    int width, nseq, nkv, D;
    int page_log2;
    int type;  // PagedType

    __device__ __forceinline__ int len(int b) const {
        const int64_t cap = static_cast<int64_t>(width) << page_log2;
        const int n = lens[b];
        return n < 0 ? 0 : (n > cap ? static_cast<int>(cap) : n);
    }
    // Element offset of head 0's row of position j of sequence b; -1 when its
    // page number lies outside the pool.
    __device__ __forceinline__ int64_t row(int b, int j) const {
        const int32_t p = table[b * table_stride + (j >> page_log2)];
        if (static_cast<uint32_t>(p) >= static_cast<uint64_t>(num_pages)) return -1;
        return p * page_stride + (j & ((1 << page_log2) - 1)) * slot_stride;
    }
};

// What a token at the end of n positions sees: the first `sinks` positions and
// those from w0 on, counted without the gap between them.
struct Visible {
    int sinks, w0, n;
    __device__ __forceinline__ int pos(int c) const { return c < sinks ? c : w0 + c - sinks; }
};

__device__ __forceinline__ Visible visible(int n, int window, int sinks) {
    Visible v;
    v.w0 = window > 0 && n > window ? n - window : 0;
    v.sinks = sinks < v.w0 ? sinks : v.w0;
    v.n = v.sinks + n - v.w0;
    return v;
}

struct PagedRows {
    const void* k;
    const void* v;
    int64_t row_stride, head_stride, rows;
    int src_type;
    const int32_t* q_start;
};

struct PagedAttn {
    const void* q;
    void* out;
    int64_t q_row, q_head, out_row, out_head;
    float* lse;
    int64_t lse_row;
    int64_t rows;
    int nq, G;
    int window, sinks, max_new;
    float scale;
    int mass_cap;
    const int32_t* q_start;
    float* mass;
    int64_t mass_seq, mass_head;
    int* err;
};

struct PagedEvict {
    const float* mass;
    float* mass_out;
    int64_t mass_seq, mass_head;
    int mass_cap, budget, sinks, recent;
    const int32_t* dst;
    int64_t dst_stride;
    int32_t* kept;
    int32_t* new_lens;
};

// The sequence whose rows hold row r: the last b with q_start[b] <= r.
__device__ __forceinline__ int row_seq(const int32_t* q_start, int nseq, int64_t r) {
    int lo = 0, hi = nseq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (q_start[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

cudaError_t paged_append_launch(const PagedKv& kv, const PagedRows& r, cudaStream_t s);
// Fixed workspace of a stream: counters (zero before its first call; every
// call leaves them zero), then partial results.
size_t paged_workspace_bytes(int num_sms);
size_t paged_counter_bytes(int num_sms);
uint64_t paged_decode_scratch(const PagedKv& kv, const PagedAttn& a);
cudaError_t paged_decode_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, void* scratch, int num_sms,
                                cudaStream_t s);
cudaError_t paged_prompt32_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s);
size_t paged_prompt_part_bytes(int num_sms);
bool paged_pool_map(const PagedKv& kv, void* pool, CUtensorMap* out);
cudaError_t paged_prompt_mass16_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s);
cudaError_t paged_prompt16_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s);
cudaError_t paged_prompt_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s);
cudaError_t paged_evict_launch(const PagedKv& kv, const PagedEvict& e, cudaStream_t s);

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace rt
