// paged_attn.cu -- attention of several new tokens per sequence over a paged
// cache (rt_paged_prompt).
//
// One warp per (query row, head): lane l holds the dims l, l + 32, ... of the
// query and of the output, and walks the visible positions with a running
// maximum and sum (f32).
#include <math.h>

#include "common.cuh"
#include "paged.cuh"

namespace rt {

namespace {

// Row r's sequence and the positions its token sees (n of them up to and with itself).
__device__ __forceinline__ bool row_token(const PagedKv& kv, const PagedAttn& a, int64_t r, int& b, int& n) {
    b = row_seq(a.q_start, kv.nseq, r);
    const int64_t first = a.q_start[b], count = a.q_start[b + 1] - first, i = r - first;
    if (i < 0 || i >= count || i >= a.max_new) return false;
    n = static_cast<int>(kv.len(b) - count + i + 1);
    if (n < 0) n = 0;
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attend_kernel(const PagedKv kv, const PagedAttn a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t r = blockIdx.x;
    const int head = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (head >= a.nq) return;
    int b, n;
    if (!row_token(kv, a, r, b, n)) return;
    const int64_t hoff = (head / a.G) * kv.head_stride;
    const T* qr = static_cast<const T*>(a.q) + r * a.q_row + head * a.q_head;
    float q[E], acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = to_f32(qr[lane + 32 * i]) * a.scale;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const Visible vis = visible(n, a.window, a.sinks);
    for (int c = 0; c < vis.n; ++c) {
        const int64_t off = kv.row(b, vis.pos(c));
        const T* kr = static_cast<const T*>(kv.k) + off + hoff;
        const T* vr = static_cast<const T*>(kv.v) + off + hoff;
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) d += off < 0 ? 0.f : q[i] * to_f32(kr[lane + 32 * i]);
        d = warp_sum(d);
        const float mn = fmaxf(m, d);
        const float corr = m == -INFINITY ? 0.f : expf(m - mn), p = expf(d - mn);
        l = l * corr + p;
        m = mn;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = acc[i] * corr + (off < 0 ? 0.f : p * to_f32(vr[lane + 32 * i]));
    }
    T* o = static_cast<T*>(a.out) + r * a.out_row + head * a.out_head;
    const float inv = vis.n > 0 ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[lane + 32 * i] = from_f32<T>(acc[i] * inv);
    if (a.lse && lane == 0) a.lse[r * a.lse_row + head] = vis.n > 0 ? m + logf(l) : -INFINITY;
}

// One warp per (sequence, KV head, position): the position's weights over the
// sequence's new tokens and the G heads, added in that order.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_mass_kernel(const PagedKv kv, const PagedAttn a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
    const int len = kv.len(b);
    if (j >= len || j >= a.mass_cap) return;
    const int64_t first = a.q_start[b], all = a.q_start[b + 1] - first;
    const int64_t count = min(min(all, static_cast<int64_t>(a.max_new)), a.rows - first);
    const int64_t t0 = len - all;  // position of the first new token
    const int64_t off = kv.row(b, j);
    float k[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
        k[i] = off < 0 ? 0.f : to_f32(static_cast<const T*>(kv.k)[off + h * kv.head_stride + lane + 32 * i]);
    float sum = 0.f;
    for (int64_t i = t0 > j ? 0 : j - t0; i < count; ++i) {
        if (a.window > 0 && j <= t0 + i - a.window && j >= a.sinks) break;
        for (int g = 0; g < a.G; ++g) {
            const int head = h * a.G + g;
            const T* qr = static_cast<const T*>(a.q) + (first + i) * a.q_row + head * a.q_head;
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) d += k[e] * (to_f32(qr[lane + 32 * e]) * a.scale);
            d = warp_sum(d);
            sum += expf(d - a.lse[(first + i) * a.lse_row + head]);
        }
    }
    if (lane == 0) a.mass[b * a.mass_seq + h * a.mass_head + j] += sum;
}

template <typename T>
cudaError_t attend(const PagedKv& kv, const PagedAttn& a, cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.rows), (a.nq + 3) / 4);
    if (kv.D == 64) paged_attend_kernel<T, 64><<<grid, 128, 0, s>>>(kv, a);
    else if (kv.D == 128) paged_attend_kernel<T, 128><<<grid, 128, 0, s>>>(kv, a);
    else paged_attend_kernel<T, 256><<<grid, 128, 0, s>>>(kv, a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t mass(const PagedKv& kv, const PagedAttn& a, cudaStream_t s) {
    const int64_t cap = static_cast<int64_t>(kv.width) << kv.page_log2;
    const int64_t n = cap < a.mass_cap ? cap : a.mass_cap;
    if (n == 0) return cudaSuccess;
    const dim3 grid(static_cast<unsigned>((n + 3) / 4), kv.nkv, kv.nseq);
    if (kv.D == 64) paged_mass_kernel<T, 64><<<grid, 128, 0, s>>>(kv, a);
    else if (kv.D == 128) paged_mass_kernel<T, 128><<<grid, 128, 0, s>>>(kv, a);
    else paged_mass_kernel<T, 256><<<grid, 128, 0, s>>>(kv, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t paged_prompt_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s) {
    cudaError_t e = kv.type == kPagedF32 ? attend<float>(kv, a, s) : paged_prompt16_launch(kv, a, workspace, num_sms, s);
    if (e != cudaSuccess || !a.mass) return e;
    return kv.type == kPagedF32 ? mass<float>(kv, a, s) : paged_prompt_mass16_launch(kv, a, workspace, num_sms, s);
}

}  // namespace rt
