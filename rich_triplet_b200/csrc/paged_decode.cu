// paged_decode.cu -- attention of one new token per sequence over a paged cache
// (rt_paged_decode): the kernel of paged_decode_core.cuh, and the weight totals
// from the scores that it stores on the way.
#include "paged_decode_core.cuh"

namespace rt {

namespace {

// mass[b][h][j] += the position's weights over the G heads, from the stored scores.
__global__ void __launch_bounds__(256) paged_decode_mass_kernel(const PagedKv kv, const PagedAttn a, const DecWork wk) {
    const int c = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    const Visible vis = visible(kv.len(b), a.window, a.sinks);
    if (c >= vis.n) return;
    const int j = vis.pos(c);
    if (j >= a.mass_cap) return;
    float sum = 0.f;
    for (int g = 0; g < a.G; ++g) {
        const int64_t row = static_cast<int64_t>(b) * a.nq + h * a.G + g;
        const float2 nm = wk.norm[row];
        const float w = exp2f(wk.scores[row * wk.score_stride + c] - nm.x) * nm.y;
        sum += nm.y != 0.f ? w : 0.f;  // 0: no weight at all
    }
    a.mass[b * a.mass_seq + h * a.mass_head + j] += sum;
}

template <typename T, int D>
cudaError_t by_group(const PagedKv& kv, const PagedAttn& a, const DecWork& wk, int grid, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (a.G <= 4) return launch<T, D, 1, true, false>(kv, a, wk, grid, s);
    }
    if (a.G <= 8) return launch<T, D, 1, false, false>(kv, a, wk, grid, s);
    return launch<T, D, 2, false, false>(kv, a, wk, grid, s);
}

template <typename T>
cudaError_t by_dim(const PagedKv& kv, const PagedAttn& a, const DecWork& wk, int grid, cudaStream_t s) {
    if (kv.D == 64) return by_group<T, 64>(kv, a, wk, grid, s);
    if (kv.D == 128) return by_group<T, 128>(kv, a, wk, grid, s);
    return by_group<T, 256>(kv, a, wk, grid, s);
}

}  // namespace

size_t paged_workspace_bytes(int num_sms) {
    const size_t grid = decode_grid(num_sms);
    return paged_counter_bytes(num_sms) +
           std::max(grid * 2 * kPagedMaxGroup * (256 + 4) * sizeof(float), paged_prompt_part_bytes(num_sms));
}

size_t paged_counter_bytes(int num_sms) { return (decode_grid(num_sms) * sizeof(uint32_t) + 255) / 256 * 256; }

// Scores of a (sequence, head): at most the positions that a token can see.
static int64_t score_stride(const PagedKv& kv, const PagedAttn& a) {
    const int64_t cap = static_cast<int64_t>(kv.width) << kv.page_log2;
    return a.window > 0 ? std::min<int64_t>(cap, static_cast<int64_t>(a.window) + a.sinks) : cap;
}

// All ones where it passes 2^62 bytes.
uint64_t paged_decode_scratch(const PagedKv& kv, const PagedAttn& a) {
    if (!a.mass) return 0;
    const int64_t each = static_cast<int64_t>(sizeof(float2)) + score_stride(kv, a) * static_cast<int64_t>(sizeof(float));
    if (a.rows > (int64_t{1} << 62) / a.nq / each) return UINT64_MAX;
    const uint64_t rows = static_cast<uint64_t>(a.rows) * a.nq;
    return (rows * sizeof(float2) + 255) / 256 * 256 + (rows * score_stride(kv, a) * sizeof(float) + 255) / 256 * 256;
}

cudaError_t paged_decode_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, void* scratch, int num_sms,
                                cudaStream_t s) {
    DecWork wk = {};
    wk.cnt = static_cast<uint32_t*>(workspace);
    wk.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + paged_counter_bytes(num_sms));
    wk.scale2 = a.scale * 1.44269504088896341f;
    if (a.mass) {
        const size_t rows = static_cast<size_t>(a.rows) * a.nq;
        wk.norm = static_cast<float2*>(scratch);
        wk.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + (rows * sizeof(float2) + 255) / 256 * 256);
        wk.score_stride = score_stride(kv, a);
    }
    const int grid = decode_grid(num_sms);
    const cudaError_t e = kv.type == kPagedF32 ? by_dim<float>(kv, a, wk, grid, s)
                        : kv.type == kPagedF16 ? by_dim<__half>(kv, a, wk, grid, s)
                                               : by_dim<__nv_bfloat16>(kv, a, wk, grid, s);
    if (e != cudaSuccess || !a.mass) return e;
    const int64_t n = wk.score_stride;
    if (n == 0) return cudaSuccess;
    return rt_launch(paged_decode_mass_kernel, dim3(static_cast<unsigned>((n + 255) / 256), kv.nkv, kv.nseq), 256, 0, s, true, kv, a, wk);
}

}  // namespace rt
