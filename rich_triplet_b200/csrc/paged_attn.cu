// paged_attn.cu -- which kernels a prompt runs on (rt_paged_prompt), and the
// weight totals of f32 caches.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace rt {

namespace {

// One warp per (sequence, KV head, position): the position's weights over the
// sequence's new tokens and the G heads, added in that order, 64 tokens to a
// partial sum.  Bound by the warp sums (one for each score); f32 totals of long
// prompts are the one path here that is not made fast.
template <int D>
__global__ void __launch_bounds__(128) paged_mass32_kernel(const PagedKv kv, const PagedAttn a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
    const int len = kv.len(b);
    if (j >= len || j >= a.mass_cap) return;
    const int64_t first = a.q_start[b], all = a.q_start[b + 1] - first;
    if (first < 0) return;
    const int64_t count = min(min(all, static_cast<int64_t>(a.max_new)), a.rows - first);
    const int64_t t0 = len - all;  // position of the first new token
    const int64_t off = kv.row(b, j);
    float k[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
        k[i] = off < 0 ? 0.f : static_cast<const float*>(kv.k)[off + h * kv.head_stride + lane + 32 * i];
    float sum = 0.f, part = 0.f;
    for (int64_t i = t0 > j ? 0 : j - t0; i < count; ++i) {
        if (a.window > 0 && j <= t0 + i - a.window && j >= a.sinks) break;
        for (int g = 0; g < a.G; ++g) {
            const int head = h * a.G + g;
            const float* qr = static_cast<const float*>(a.q) + (first + i) * a.q_row + head * a.q_head;
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) d += k[e] * (qr[lane + 32 * e] * a.scale);
            d = warp_sum(d);
            const float z = a.lse[(first + i) * a.lse_row + head];
            if (z != -INFINITY) part += expf(d - z);  // else the row has no weight at all
        }
        if ((i & 63) == 63) {
            sum += part;
            part = 0.f;
        }
    }
    if (lane == 0) a.mass[b * a.mass_seq + h * a.mass_head + j] += sum + part;
}

cudaError_t mass32(const PagedKv& kv, const PagedAttn& a, cudaStream_t s) {
    const int64_t cap = static_cast<int64_t>(kv.width) << kv.page_log2;
    const int64_t n = cap < a.mass_cap ? cap : a.mass_cap;
    if (n == 0) return cudaSuccess;
    const dim3 grid(static_cast<unsigned>((n + 3) / 4), kv.nkv, kv.nseq);
    if (kv.D == 64) paged_mass32_kernel<64><<<grid, 128, 0, s>>>(kv, a);
    else if (kv.D == 128) paged_mass32_kernel<128><<<grid, 128, 0, s>>>(kv, a);
    else paged_mass32_kernel<256><<<grid, 128, 0, s>>>(kv, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t paged_prompt_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s) {
    const cudaError_t e = kv.type == kPagedF32 ? paged_prompt32_launch(kv, a, workspace, num_sms, s)
                                               : paged_prompt16_launch(kv, a, workspace, num_sms, s);
    if (e != cudaSuccess || !a.mass) return e;
    return kv.type == kPagedF32 ? mass32(kv, a, s) : paged_prompt_mass16_launch(kv, a, workspace, num_sms, s);
}

}  // namespace rt
