// paged_api.cu -- C ABI of the paged key-value cache (rt_paged_*,
// include/rt_cuda.h): argument checks, then the launchers of paged.cuh.
#include <math.h>

#include <mutex>
#include <utility>
#include <vector>

#include "paged.cuh"
#include "rt_internal.h"

using rt::fail;

namespace {

// The context's device is current while a call runs, and the caller's again after it.
struct DeviceScope {
    int before = -1;
    cudaError_t e;
    explicit DeviceScope(int device) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int paged_type(int fmt) {
    switch (fmt) {
        case RT_FMT_F32: return rt::kPagedF32;
        case RT_FMT_F16: return rt::kPagedF16;
        case RT_FMT_BF16: return rt::kPagedBF16;
        default: return -1;
    }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Every stride a multiple of 16 bytes and not negative.
template <typename... S>
bool strides_ok(int esize, S... s) {
    return ((s >= 0 && s * esize % 16 == 0) && ...);
}

// The stride of an extent of at most one is never used: its value is `unused`.
int64_t stride(int64_t extent, int64_t given, int64_t unused) { return extent > 1 ? given : unused; }

constexpr int64_t kMaxPositions = INT32_MAX - 256;  // of a sequence

bool page_size_ok(int page_size) { return page_size >= 8 && page_size <= 256 && (page_size & (page_size - 1)) == 0; }

// Whether n x m rows of `len` elements, at i * si + j * sj, lie apart: rows of
// one index hold those of the other between them.
bool apart(int64_t n, int64_t si, int64_t m, int64_t sj, int64_t len) {
    // the first stride spans all the rows of the second index (divided, so that nothing overflows)
    auto nested = [len](int64_t outer, int64_t so, int64_t inner, int64_t sn) {
        if (inner > 1 && sn < len) return false;
        if (outer <= 1) return true;
        return so >= len && (inner <= 1 || (so - len) / sn >= inner - 1);
    };
    return n <= 0 || m <= 0 || len <= 0 || nested(n, si, m, sj) || nested(m, sj, n, si);
}

// Whether a value of q is also one of out.  (Exact for equal strides; for
// unequal ones two ranges that meet count as shared.)
bool q_meets_out(const rt_paged_attn* a, int esize, int D) {
    auto span = [&](int64_t row, int64_t head) { return ((a->rows - 1) * row + (a->num_heads - 1) * head + D) * esize; };
    const intptr_t q = reinterpret_cast<intptr_t>(a->q), out = reinterpret_cast<intptr_t>(a->out);
    if (a->rows < 1 || q + span(a->q_row_stride, a->q_head_stride) <= out ||
        out + span(a->out_row_stride, a->out_head_stride) <= q)
        return false;
    const int64_t row = a->rows > 1 ? a->q_row_stride : 0, head = a->num_heads > 1 ? a->q_head_stride : 0;
    if ((a->rows > 1 && row != a->out_row_stride) || (a->num_heads > 1 && head != a->out_head_stride)) return true;
    for (int64_t h = 1 - a->num_heads; h < a->num_heads; ++h) {
        const int64_t d = (out - q) / esize - h * head;  // what row differences have to make up
        const int64_t r = row ? d / row : 0;
        for (int64_t i = r - 1; i <= r + 1; ++i)
            if (i > -a->rows && i < a->rows && d - i * row > -D && d - i * row < D) return true;
    }
    return false;
}

int make_kv(rt_ctx* ctx, const char* who, const rt_paged_kv* in, rt::PagedKv* out) {
    const int type = paged_type(in->fmt);
    if (type < 0) return fail(ctx, RT_E_FORMAT, "%s: cache format %d is not f32, f16 or bf16", who, in->fmt);
    if (in->head_dim != 64 && in->head_dim != 128 && in->head_dim != 256)
        return fail(ctx, RT_E_SHAPE, "%s: head_dim %d is not 64, 128 or 256", who, in->head_dim);
    if (!page_size_ok(in->page_size))
        return fail(ctx, RT_E_SHAPE, "%s: page_size %d is not a power of two in 8..256", who, in->page_size);
    if (in->kv_heads < 1 || in->kv_heads > 65535)
        return fail(ctx, RT_E_SHAPE, "%s: kv_heads %d out of range", who, in->kv_heads);
    if (in->num_pages < 1 || in->num_pages > INT32_MAX - 1)
        return fail(ctx, RT_E_SHAPE, "%s: num_pages %lld out of range", who, static_cast<long long>(in->num_pages));
    if (in->num_seqs < 0 || in->num_seqs > 65535)
        return fail(ctx, RT_E_SHAPE, "%s: num_seqs %d out of range (0..65535)", who, in->num_seqs);
    if (in->table_width < 0 || in->table_stride < 0 ||
        static_cast<int64_t>(in->table_width) * in->page_size > kMaxPositions ||
        static_cast<int64_t>(in->table_width) * in->page_size * in->num_seqs > (int64_t{1} << 44))
        return fail(ctx, RT_E_SHAPE, "%s: page table of width %d, row stride %lld", who, in->table_width,
                    static_cast<long long>(in->table_stride));
    const int esize = type == rt::kPagedF32 ? 4 : 2;
    const int64_t page_stride = stride(in->num_pages, in->page_stride, in->head_dim),
                  head_stride = stride(in->kv_heads, in->head_stride, in->head_dim);
    if (!strides_ok(esize, page_stride, head_stride, in->slot_stride))
        return fail(ctx, RT_E_INVAL, "%s: cache strides must be multiples of 16 bytes", who);
    if (in->slot_stride < in->head_dim || head_stride < in->head_dim || page_stride < in->head_dim)
        return fail(ctx, RT_E_SHAPE, "%s: the rows of the cache overlap", who);
    if (in->num_seqs > 0) {
        if (!in->k || !in->v || !in->lens || (in->table_width > 0 && !in->page_table))
            return fail(ctx, RT_E_INVAL, "%s: null cache pointer", who);
        if (!aligned(in->k) || !aligned(in->v)) return fail(ctx, RT_E_INVAL, "%s: the pools must be 16-byte aligned", who);
    }
    int lg = 3;
    while ((1 << lg) < in->page_size) ++lg;
    *out = rt::PagedKv{in->k,          in->v,           page_stride,     head_stride,     in->slot_stride,
                       in->num_pages,  in->page_table,  in->table_stride, in->lens,       in->table_width,
                       in->num_seqs,   in->kv_heads,    in->head_dim,    lg,              type};
    return RT_OK;
}

int make_attn(rt_ctx* ctx, const char* who, const rt_paged_kv* kv, const rt_paged_attn* in, bool prompt,
              rt::PagedAttn* out) {
    const int esize = kv->fmt == RT_FMT_F32 ? 4 : 2;
    if (in->num_heads < 1 || in->num_heads % kv->kv_heads || in->num_heads / kv->kv_heads > rt::kPagedMaxGroup)
        return fail(ctx, RT_E_SHAPE, "%s: %d query heads over %d KV heads (a multiple, at most %d each)", who,
                    in->num_heads, kv->kv_heads, rt::kPagedMaxGroup);
    if (!(in->scale > 0.f) || !isfinite(in->scale)) return fail(ctx, RT_E_INVAL, "%s: scale must be finite and > 0", who);
    if (in->window < 0 || in->sinks < 0) return fail(ctx, RT_E_INVAL, "%s: negative window or sinks", who);
    if (in->rows < 0 || in->rows > INT32_MAX / rt::kPagedMaxGroup)
        return fail(ctx, RT_E_SHAPE, "%s: rows %lld out of range", who, static_cast<long long>(in->rows));
    if (prompt) {
        if (in->max_new < 0) return fail(ctx, RT_E_INVAL, "%s: negative max_new", who);
        if (in->rows > 0 && !in->q_start) return fail(ctx, RT_E_INVAL, "%s: null q_start", who);
        if (kv->fmt == RT_FMT_F32 && in->rows * (in->num_heads / kv->kv_heads) > (1 << 25))
            return fail(ctx, RT_E_SHAPE, "%s: at most 2^25 rows x query heads to a KV head over an f32 cache", who);
    } else {
        if (in->q_start) return fail(ctx, RT_E_INVAL, "%s: q_start belongs to rt_paged_prompt", who);
        if (in->rows != kv->num_seqs)
            return fail(ctx, RT_E_SHAPE, "%s: %lld rows for %d sequences", who, static_cast<long long>(in->rows), kv->num_seqs);
    }
    const int64_t D = kv->head_dim, q_row = stride(in->rows, in->q_row_stride, D), q_head = stride(in->num_heads, in->q_head_stride, D),
                  out_row = stride(in->rows, in->out_row_stride, D), out_head = stride(in->num_heads, in->out_head_stride, D);
    if (in->rows > 0 && (!in->q || !in->out)) return fail(ctx, RT_E_INVAL, "%s: null q or out", who);
    if (!aligned(in->q) || !aligned(in->out) ||
        !strides_ok(esize, q_row, q_head, out_row, out_head))
        return fail(ctx, RT_E_INVAL, "%s: q and out must be 16-byte aligned with strides in multiples of 16 bytes", who);
    if (!apart(in->rows, in->out_row_stride, in->num_heads, in->out_head_stride, kv->head_dim))
        return fail(ctx, RT_E_SHAPE, "%s: the rows of out overlap", who);
    if (in->lse && in->lse_row_stride < in->num_heads) return fail(ctx, RT_E_SHAPE, "%s: lse rows overlap", who);
    if (in->mass && (in->mass_cap < 0 || in->mass_seq_stride < 0 || in->mass_head_stride < 0))
        return fail(ctx, RT_E_SHAPE, "%s: negative mass size or stride", who);
    if (prompt && in->mass && q_meets_out(in, esize, kv->head_dim))
        return fail(ctx, RT_E_INVAL, "%s: out overlaps q, which the totals read again", who);
    if (in->mass && !apart(kv->num_seqs, in->mass_seq_stride, kv->kv_heads, in->mass_head_stride, in->mass_cap))
        return fail(ctx, RT_E_SHAPE, "%s: the rows of mass overlap", who);
    *out = rt::PagedAttn{in->q, in->out, q_row, q_head, out_row, out_head,
                         in->lse, in->lse_row_stride, in->rows, in->num_heads, in->num_heads / kv->kv_heads,
                         in->window, in->sinks, in->max_new, in->scale, in->mass_cap, prompt ? in->q_start : nullptr,
                         in->mass, in->mass_seq_stride, in->mass_head_stride, nullptr};
    return RT_OK;
}

// The prompt mass pass reads every row's lse: room for it when the caller takes none.
uint64_t scratch_need(const rt::PagedKv& kv, const rt::PagedAttn& a, bool prompt) {
    if (!prompt) return rt::paged_decode_scratch(kv, a);
    if (!a.mass || a.lse) return 0;
    return a.rows > INT64_MAX / 8 / a.nq ? UINT64_MAX : (static_cast<uint64_t>(a.rows) * a.nq * 4 + 255) / 256 * 256;
}

// A small number of this thread, another thread's once this one has ended.
int thread_number() {
    struct Numbers {
        std::mutex m;
        std::vector<bool> taken;
    };
    static Numbers* const all = new Numbers;  // outlives every thread
    struct Own {
        int n = 0;
        Own() {
            std::lock_guard<std::mutex> lock(all->m);
            while (n < static_cast<int>(all->taken.size()) && all->taken[n]) ++n;
            if (n == static_cast<int>(all->taken.size())) all->taken.push_back(true);
            else all->taken[n] = true;
        }
        ~Own() {
            std::lock_guard<std::mutex> lock(all->m);
            all->taken[n] = false;
        }
    };
    static thread_local Own own;
    return own.n;
}

// The workspace of this thread's calls on the stream, made on first use.  (Two
// threads may hold the same stream of a pool without knowing it: a graph that one
// captured there then shares nothing with the other's calls.)
int workspace(rt_ctx* ctx, const char* who, cudaStream_t s, void** out) {
    const std::pair<cudaStream_t, int> key(s, thread_number());
    auto it = ctx->paged_ws.find(key);
    if (it != ctx->paged_ws.end()) {
        *out = it->second;
        return RT_OK;
    }
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    RT_CHECK_CUDA(ctx, cudaStreamIsCapturing(s, &st));
    if (st != cudaStreamCaptureStatusNone)
        return fail(ctx, RT_E_STATE, "%s: the stream's workspace does not exist yet; make one call before the capture", who);
    void* p = nullptr;
    if (int rc = rt::dev_alloc(ctx, &p, rt::paged_workspace_bytes(ctx->num_sms), "paged workspace"); rc != RT_OK) return rc;
    const cudaError_t e = cudaMemsetAsync(p, 0, rt::paged_counter_bytes(ctx->num_sms), s);
    if (e != cudaSuccess) {
        cudaFree(p);
        return fail(ctx, RT_E_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    ctx->paged_ws[key] = p;
    *out = p;
    return RT_OK;
}

int attend(rt_ctx* ctx, const char* who, const rt_paged_kv* in, const rt_paged_attn* at, bool prompt, void* stream) {
    if (!ctx || !in || !at) return fail(ctx, RT_E_INVAL, "%s: null argument", who);
    rt::PagedKv kv;
    rt::PagedAttn a;
    if (int rc = make_kv(ctx, who, in, &kv); rc != RT_OK) return rc;
    if (int rc = make_attn(ctx, who, in, at, prompt, &a); rc != RT_OK) return rc;
    const uint64_t need = scratch_need(kv, a, prompt);
    if (need > at->scratch_bytes || (need && (!at->scratch || (reinterpret_cast<uintptr_t>(at->scratch) & 255))))
        return fail(ctx, RT_E_INVAL, "%s: needs %llu bytes of 256-byte aligned scratch", who,
                    static_cast<unsigned long long>(need));
    if (a.rows == 0 || kv.nseq == 0 || (prompt && a.max_new == 0)) return RT_OK;
    DeviceScope scope(ctx->device);
    RT_CHECK_CUDA(ctx, scope.e);
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    a.err = ctx->d_err;
    void* ws = nullptr;
    if (int rc = workspace(ctx, who, s, &ws); rc != RT_OK) return rc;
    if (!prompt) {
        RT_CHECK_CUDA(ctx, rt::paged_decode_launch(kv, a, ws, at->scratch, ctx->num_sms, s));
        return RT_OK;
    }
    if (a.mass && !a.lse) {
        a.lse = static_cast<float*>(at->scratch);
        a.lse_row = a.nq;
    }
    RT_CHECK_CUDA(ctx, rt::paged_prompt_launch(kv, a, ws, ctx->num_sms, s));
    return RT_OK;
}

}  // namespace

extern "C" {

int rt_paged_append(rt_ctx* ctx, const rt_paged_kv* in, const rt_paged_rows* r, void* stream) {
    const char* who = "rt_paged_append";
    if (!ctx || !in || !r) return fail(ctx, RT_E_INVAL, "%s: null argument", who);
    rt::PagedKv kv;
    if (int rc = make_kv(ctx, who, in, &kv); rc != RT_OK) return rc;
    const int st = paged_type(r->src_fmt);
    if (st < 0) return fail(ctx, RT_E_FORMAT, "%s: row format %d is not f32, f16 or bf16", who, r->src_fmt);
    if (r->rows < 0 || r->rows > INT32_MAX)
        return fail(ctx, RT_E_SHAPE, "%s: rows %lld out of range", who, static_cast<long long>(r->rows));
    if (!r->q_start && r->rows != in->num_seqs)
        return fail(ctx, RT_E_SHAPE, "%s: %lld rows for %d sequences", who, static_cast<long long>(r->rows), in->num_seqs);
    if (r->rows == 0 || in->num_seqs == 0) return RT_OK;
    const int64_t row = stride(r->rows, r->row_stride, in->head_dim), head = stride(in->kv_heads, r->head_stride, in->head_dim);
    if (!r->k || !r->v) return fail(ctx, RT_E_INVAL, "%s: null rows", who);
    if (!aligned(r->k) || !aligned(r->v) || !strides_ok(st == rt::kPagedF32 ? 4 : 2, row, head))
        return fail(ctx, RT_E_INVAL, "%s: rows must be 16-byte aligned with strides in multiples of 16 bytes", who);
    DeviceScope scope(ctx->device);
    RT_CHECK_CUDA(ctx, scope.e);
    const rt::PagedRows a{r->k, r->v, row, head, r->rows, st, r->q_start};
    RT_CHECK_CUDA(ctx, rt::paged_append_launch(kv, a, stream ? static_cast<cudaStream_t>(stream) : ctx->stream));
    return RT_OK;
}

int rt_paged_scratch(const rt_paged_kv* in, const rt_paged_attn* at, int32_t prompt, uint64_t* bytes) {
    if (!in || !at || !bytes) return RT_E_INVAL;
    if (!page_size_ok(in->page_size) || in->table_width < 0 ||
        static_cast<int64_t>(in->table_width) * in->page_size > kMaxPositions || at->rows < 0 || at->num_heads < 1 ||
        at->window < 0 || at->sinks < 0)
        return RT_E_SHAPE;
    rt::PagedKv kv = {};
    rt::PagedAttn a = {};
    kv.width = in->table_width;
    while ((1 << kv.page_log2) < in->page_size) ++kv.page_log2;
    a.rows = at->rows;
    a.nq = at->num_heads;
    a.window = at->window;
    a.sinks = at->sinks;
    a.mass = at->mass;
    a.lse = at->lse;
    *bytes = scratch_need(kv, a, prompt != 0);
    return *bytes == UINT64_MAX ? RT_E_SHAPE : RT_OK;
}

int rt_paged_decode(rt_ctx* ctx, const rt_paged_kv* kv, const rt_paged_attn* a, void* stream) {
    return attend(ctx, "rt_paged_decode", kv, a, false, stream);
}

int rt_paged_prompt(rt_ctx* ctx, const rt_paged_kv* kv, const rt_paged_attn* a, void* stream) {
    return attend(ctx, "rt_paged_prompt", kv, a, true, stream);
}

int rt_paged_evict(rt_ctx* ctx, const rt_paged_kv* in, const rt_paged_evict_args* e, void* stream) {
    const char* who = "rt_paged_evict";
    if (!ctx || !in || !e) return fail(ctx, RT_E_INVAL, "%s: null argument", who);
    rt::PagedKv kv;
    if (int rc = make_kv(ctx, who, in, &kv); rc != RT_OK) return rc;
    if (e->budget < 1 || e->sinks < 0 || e->recent < 0 || static_cast<int64_t>(e->sinks) + e->recent > e->budget)
        return fail(ctx, RT_E_INVAL, "%s: sinks %d + recent %d must lie in 0..budget %d", who, e->sinks, e->recent, e->budget);
    if (e->budget > kMaxPositions || e->mass_cap > kMaxPositions)
        return fail(ctx, RT_E_SHAPE, "%s: budget %d, mass_cap %d: at most %lld positions", who, e->budget, e->mass_cap,
                    static_cast<long long>(kMaxPositions));
    if (e->mass_cap < 0 || e->mass_seq_stride < 0 || e->mass_head_stride < 0)
        return fail(ctx, RT_E_SHAPE, "%s: negative mass size or stride", who);
    if (!apart(in->num_seqs, e->mass_seq_stride, in->kv_heads, e->mass_head_stride, e->mass_cap))
        return fail(ctx, RT_E_SHAPE, "%s: the rows of mass overlap", who);
    if (e->dst_stride < (static_cast<int64_t>(e->budget) + in->page_size - 1) / in->page_size)
        return fail(ctx, RT_E_SHAPE, "%s: %lld destination pages a row hold fewer than %d positions", who,
                    static_cast<long long>(e->dst_stride), e->budget);
    if (in->num_seqs == 0) return RT_OK;
    if (!e->mass || !e->mass_out || !e->dst_table || !e->kept || !e->new_lens)
        return fail(ctx, RT_E_INVAL, "%s: null argument", who);
    DeviceScope scope(ctx->device);
    RT_CHECK_CUDA(ctx, scope.e);
    const rt::PagedEvict a{e->mass, e->mass_out, e->mass_seq_stride, e->mass_head_stride, e->mass_cap, e->budget,
                           e->sinks, e->recent, e->dst_table, e->dst_stride, e->kept, e->new_lens};
    RT_CHECK_CUDA(ctx, rt::paged_evict_launch(kv, a, stream ? static_cast<cudaStream_t>(stream) : ctx->stream));
    return RT_OK;
}

}  // extern "C"
