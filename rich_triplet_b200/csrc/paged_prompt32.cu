// paged_prompt32.cu -- prompts over f32 caches, on the decode kernel
// (paged_decode_core.cuh, FEW).
//
// f32 rows have no 16-bit form for tcgen05, so their split tf32 products run
// here, 16 (token, head) rows to a pass over the positions.  (16-bit caches
// stay on the tcgen05 kernel also for few rows: 5 x 8 tokens over 2050
// positions, 8 query heads on 4, took 29 us in this form and 23.5 there, whose
// CTAs have fewer partial outputs to join.)
#include "paged_decode_core.cuh"

namespace rt {

namespace {

template <int D>
cudaError_t by_rows(const PagedKv& kv, const PagedAttn& a, const DecWork& wk, int grid, cudaStream_t s) {
    if (std::min<int64_t>(a.max_new, a.rows) * a.G <= 8) return launch<float, D, 1, false, true>(kv, a, wk, grid, s);
    return launch<float, D, 2, false, true>(kv, a, wk, grid, s);
}

}  // namespace

cudaError_t paged_prompt32_launch(const PagedKv& kv, const PagedAttn& a, void* workspace, int num_sms, cudaStream_t s) {
    DecWork wk = {};
    wk.cnt = static_cast<uint32_t*>(workspace);
    wk.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + paged_counter_bytes(num_sms));
    wk.scale2 = a.scale * 1.44269504088896341f;
    const int grid = decode_grid(num_sms);
    if (kv.D == 64) return by_rows<64>(kv, a, wk, grid, s);
    if (kv.D == 128) return by_rows<128>(kv, a, wk, grid, s);
    return by_rows<256>(kv, a, wk, grid, s);
}

}  // namespace rt
