// paged_torch.cpp -- Python module _paged_torch: the rt_paged_* calls on torch
// tensors.
//
// A serving step makes one such call per layer, and its smallest ones take a few
// microseconds on the GPU, so the argument checks, the output allocation and the
// packing of the C structs are done here rather than in Python (there they took
// 8 to 12 microseconds a call).  rich_triplet_b200/paged.py documents the
// functions and wraps them.
//
// Wrong types, shapes or devices raise ValueError; a negative status of the
// library is handed to the function that bind() was given, which raises RtError.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/rt_cuda.h"

namespace {

PyObject* g_make_context = nullptr;  // device index -> address of the process's rt_ctx there
PyObject* g_raise = nullptr;         // (status, message): raises
// The contexts that g_make_context gave, until forget(): every use of them, and
// of this array, is made with the interpreter's lock held.
constexpr int kDevices = 64;
rt_ctx* g_ctx[kDevices] = {};

bool value_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(PyExc_ValueError, fmt, ap);
    va_end(ap);
    return false;
}

rt_ctx* context(int index) {
    if (index >= 0 && index < kDevices && g_ctx[index]) return g_ctx[index];
    PyObject* h = g_make_context ? PyObject_CallFunction(g_make_context, "i", index) : nullptr;
    if (!h) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "_paged_torch is not bound");
        return nullptr;
    }
    rt_ctx* ctx = static_cast<rt_ctx*>(PyLong_AsVoidPtr(h));
    Py_DECREF(h);
    if (PyErr_Occurred()) return nullptr;
    if (index >= 0 && index < kDevices) g_ctx[index] = ctx;
    return ctx;
}

// True if `rc` is RT_OK; else the error is raised.
bool done(int rc, rt_ctx* ctx) {
    if (rc == RT_OK) return true;
    PyObject* r = g_raise ? PyObject_CallFunction(g_raise, "is", rc, ctx ? rt_last_error(ctx) : "") : nullptr;
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "rt_paged call failed");
    return false;
}

const at::Tensor* tensor(PyObject* o, const char* name) {
    if (PyErr_Occurred()) return nullptr;  // an argument before this one was refused
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s must be a tensor", name);
        return nullptr;
    }
    return &THPVariable_Unpack(o);
}

// Nothing here is differentiable: inputs that want gradients are refused, where
// gradients are recorded, instead of being cut out of them silently.
template <typename... T>
bool no_gradients(const char* who, const T*... t) {
    if (!at::GradMode::is_enabled() || !((t && t->requires_grad()) || ...)) return true;
    return value_error("%s is not differentiable: call it under torch.no_grad()", who);
}

// The stream that torch uses now on the device.  The default stream's handle is
// null, which the library takes for the context's own: it is named by CUDA's
// value for it.
void* stream_of(int index) {
    cudaStream_t s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
    return s ? static_cast<void*>(s) : static_cast<void*>(cudaStreamLegacy);
}

int format_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return RT_FMT_F32;
        case at::kHalf: return RT_FMT_F16;
        case at::kBFloat16: return RT_FMT_BF16;
        default: return -1;
    }
}

bool int32_rows(const at::Tensor& t, int index, int64_t n) {
    return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.get_device() == index && t.is_contiguous();
}

// Whether two tensors of the same sizes have the same strides (those of extents of one say nothing).
bool same_strides(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

struct Cache {
    rt_paged_kv kv;
    const at::Tensor *k, *v;
    at::ScalarType type;
    int index;
};

// k_pages, v_pages, page_table, lens: sizes checked as far as the library cannot.
bool get_cache(PyObject* const* a, Cache* c) {
    const at::Tensor *k = tensor(a[0], "k_pages"), *v = tensor(a[1], "v_pages"), *table = tensor(a[2], "page_table"),
                     *lens = tensor(a[3], "lens");
    if (!k || !v || !table || !lens) return false;
    if (k->dim() != 4 || k->sizes() != v->sizes() || !same_strides(*k, *v))
        return value_error("paged: k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim] with the same strides");
    c->type = k->scalar_type();
    c->index = k->is_cuda() ? k->get_device() : -1;
    const int fmt = format_of(c->type);
    if (fmt < 0 || v->scalar_type() != c->type) return value_error("paged: pools must be f32, f16 or bf16, of one type");
    if (c->index < 0 || !v->is_cuda() || v->get_device() != c->index) return value_error("paged: pools must be on one GPU");
    if (k->stride(3) != 1) return value_error("paged: the rows of the pools must be contiguous");
    if (table->dim() != 2 || table->scalar_type() != at::kInt || table->get_device() != c->index ||
        (table->size(1) > 1 && table->stride(1) != 1))
        return value_error("paged: page_table must be [sequences, width] int32 with contiguous rows, on the pools' GPU");
    const int64_t n = table->size(0), width = table->size(1);
    if (!int32_rows(*lens, c->index, n)) return value_error("paged: lens must be [%lld] int32, contiguous, on the pools' GPU", n);
    if (n > INT32_MAX || width > INT32_MAX || k->size(1) > INT32_MAX || k->size(2) > INT32_MAX || k->size(3) > INT32_MAX)
        return value_error("paged: a size does not fit 32 bits");
    c->k = k;
    c->v = v;
    rt_paged_kv& kv = c->kv;
    kv.k = k->data_ptr();
    kv.v = v->data_ptr();
    kv.page_stride = k->stride(0);
    kv.head_stride = k->stride(1);
    kv.slot_stride = k->stride(2);
    kv.num_pages = k->size(0);
    kv.fmt = fmt;
    kv.kv_heads = static_cast<int32_t>(k->size(1));
    kv.head_dim = static_cast<int32_t>(k->size(3));
    kv.page_size = static_cast<int32_t>(k->size(2));
    kv.page_table = static_cast<const int32_t*>(table->data_ptr());
    kv.table_stride = n > 1 ? table->stride(0) : width;  // the stride of an extent of one is arbitrary
    kv.table_width = static_cast<int32_t>(width);
    kv.num_seqs = static_cast<int32_t>(n);
    kv.lens = static_cast<const int32_t*>(lens->data_ptr());
    return true;
}

bool get_starts(PyObject* o, const Cache& c, const char* who, const int32_t** out) {
    const at::Tensor* t = tensor(o, "q_start");
    if (!t) return false;
    if (!int32_rows(*t, c.index, static_cast<int64_t>(c.kv.num_seqs) + 1))
        return value_error("%s: q_start must be [%lld] int32, contiguous, on the pools' GPU", who,
                           static_cast<long long>(c.kv.num_seqs) + 1);
    *out = static_cast<const int32_t*>(t->data_ptr());
    return true;
}

bool get_int(PyObject* o, const char* name, int32_t* out) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < INT32_MIN || v > INT32_MAX) return value_error("%s does not fit 32 bits", name);
    *out = static_cast<int32_t>(v);
    return true;
}

// append(k_pages, v_pages, page_table, lens, k, v, q_start or None)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7) return PyErr_Format(PyExc_TypeError, "append takes 7 arguments");
    try {
        Cache c;
        if (!get_cache(a, &c)) return nullptr;
        const at::Tensor *k = tensor(a[4], "k"), *v = tensor(a[5], "v");
        if (!k || !v || !no_gradients("kv_append", k, v, c.k, c.v)) return nullptr;
        if (k->dim() != 3 || v->sizes() != k->sizes() || !same_strides(*k, *v) || k->size(1) != c.kv.kv_heads ||
            k->size(2) != c.kv.head_dim || k->stride(2) != 1) {
            value_error("kv_append: k and v must be [rows, %d, %d] with the same strides and contiguous rows",
                        c.kv.kv_heads, c.kv.head_dim);
            return nullptr;
        }
        rt_paged_rows r;
        r.src_fmt = format_of(k->scalar_type());
        if (r.src_fmt < 0 || v->scalar_type() != k->scalar_type() || !k->is_cuda() || !v->is_cuda() ||
            k->get_device() != c.index || v->get_device() != c.index) {
            value_error("kv_append: k and v must be f32, f16 or bf16 on the pools' GPU");
            return nullptr;
        }
        r.k = k->data_ptr();
        r.v = v->data_ptr();
        r.row_stride = k->stride(0);
        r.head_stride = k->stride(1);
        r.rows = k->size(0);
        r.q_start = nullptr;
        if (a[6] != Py_None && !get_starts(a[6], c, "kv_append", &r.q_start)) return nullptr;
        rt_ctx* ctx = context(c.index);
        if (!ctx || !done(rt_paged_append(ctx, &c.kv, &r, stream_of(c.index)), ctx)) return nullptr;
        Py_RETURN_NONE;
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// attend(k_pages, v_pages, page_table, lens, q, q_start or None, max_new, scale,
//        window, sinks, mass or None, out or None) -> (out, lse)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 12) return PyErr_Format(PyExc_TypeError, "attend takes 12 arguments");
    try {
        Cache c;
        if (!get_cache(a, &c)) return nullptr;
        const bool prompt = a[5] != Py_None;
        const char* who = prompt ? "attend_prompt" : "attend_decode";
        const at::Tensor* q = tensor(a[4], "q");
        if (!q) return nullptr;
        if (q->dim() != 3 || q->size(2) != c.kv.head_dim || q->scalar_type() != c.type || !q->is_cuda() ||
            q->get_device() != c.index || q->stride(2) != 1) {
            value_error("%s: q must be [rows, heads, %d] of the pools' type with contiguous rows on the pools' GPU", who,
                        c.kv.head_dim);
            return nullptr;
        }
        const int64_t rows = q->size(0), heads = q->size(1);
        if (!prompt && rows != c.kv.num_seqs) {
            value_error("%s: %lld query rows, but lens has %d sequences", who, static_cast<long long>(rows), c.kv.num_seqs);
            return nullptr;
        }
        rt_paged_attn t = {};
        if (prompt && !get_starts(a[5], c, who, &t.q_start)) return nullptr;
        if (!get_int(a[6], "max_new", &t.max_new) || !get_int(a[8], "window", &t.window) || !get_int(a[9], "sinks", &t.sinks))
            return nullptr;
        t.scale = static_cast<float>(PyFloat_AsDouble(a[7]));
        if (PyErr_Occurred()) return nullptr;
        at::Tensor out;
        if (a[11] == Py_None) {
            out = at::empty(q->sizes(), q->options());
        } else {
            const at::Tensor* o = tensor(a[11], "out");
            if (!o) return nullptr;
            if (o->sizes() != q->sizes() || o->scalar_type() != c.type || !o->is_cuda() || o->get_device() != c.index ||
                o->stride(2) != 1) {
                value_error("%s: out must be like q, with contiguous rows, on the pools' GPU", who);
                return nullptr;
            }
            out = *o;
        }
        const at::Tensor* m = a[10] == Py_None ? nullptr : tensor(a[10], "mass");
        if (PyErr_Occurred() || !no_gradients(who, q, c.k, c.v, m, a[11] == Py_None ? nullptr : &out)) return nullptr;
        at::Tensor lse = at::empty({rows, heads}, q->options().dtype(at::kFloat)), scratch;
        t.q = q->data_ptr();
        t.out = out.data_ptr();
        t.q_row_stride = q->stride(0);
        t.q_head_stride = q->stride(1);
        t.out_row_stride = out.stride(0);
        t.out_head_stride = out.stride(1);
        t.lse = static_cast<float*>(lse.data_ptr());
        t.lse_row_stride = heads;
        t.rows = rows;
        t.num_heads = static_cast<int32_t>(std::min<int64_t>(heads, INT32_MAX));
        if (m) {
            if (m->dim() != 3 || m->scalar_type() != at::kFloat || !m->is_cuda() || m->get_device() != c.index ||
                m->size(0) != c.kv.num_seqs || m->size(1) != c.kv.kv_heads || (m->size(2) > 1 && m->stride(2) != 1)) {
                value_error("%s: mass must be [%d, %d, positions] float32 with contiguous rows on the pools' GPU", who,
                            c.kv.num_seqs, c.kv.kv_heads);
                return nullptr;
            }
            t.mass = static_cast<float*>(m->data_ptr());
            t.mass_cap = static_cast<int32_t>(std::min<int64_t>(m->size(2), INT32_MAX));
            t.mass_seq_stride = m->stride(0);
            t.mass_head_stride = m->stride(1);
            uint64_t need = 0;
            if (rt_paged_scratch(&c.kv, &t, prompt, &need) == RT_OK && need) {  // else the call below refuses
                // freed when this call returns: only later work of this stream takes its place
                scratch = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
                t.scratch = scratch.data_ptr();
                t.scratch_bytes = need;
            }
        }
        rt_ctx* ctx = context(c.index);
        if (!ctx) return nullptr;
        void* s = stream_of(c.index);
        if (!done(prompt ? rt_paged_prompt(ctx, &c.kv, &t, s) : rt_paged_decode(ctx, &c.kv, &t, s), ctx)) return nullptr;
        return Py_BuildValue("NN", THPVariable_Wrap(out), THPVariable_Wrap(lse));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// evict(k_pages, v_pages, page_table, lens, mass, dst_table, budget, sinks,
//       recent) -> (kept, new_lens, mass)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9) return PyErr_Format(PyExc_TypeError, "evict takes 9 arguments");
    try {
        Cache c;
        if (!get_cache(a, &c)) return nullptr;
        const at::Tensor *m = tensor(a[4], "mass"), *dst = tensor(a[5], "dst_table");
        if (!m || !dst || !no_gradients("kv_evict", m, c.k, c.v)) return nullptr;
        rt_paged_evict_args e = {};
        if (!get_int(a[6], "budget", &e.budget) || !get_int(a[7], "sinks", &e.sinks) || !get_int(a[8], "recent", &e.recent))
            return nullptr;
        if (m->dim() != 3 || m->scalar_type() != at::kFloat || !m->is_cuda() || m->get_device() != c.index ||
            m->size(0) != c.kv.num_seqs || m->size(1) != c.kv.kv_heads || !m->is_contiguous() || m->size(2) > INT32_MAX) {
            value_error("kv_evict: mass must be a contiguous [%d, %d, positions] float32 tensor on the pools' GPU",
                        c.kv.num_seqs, c.kv.kv_heads);
            return nullptr;
        }
        if (dst->dim() != 2 || dst->size(0) != c.kv.num_seqs || dst->scalar_type() != at::kInt || !dst->is_cuda() ||
            dst->get_device() != c.index || !dst->is_contiguous() || dst->size(1) * c.kv.page_size < e.budget) {
            value_error("kv_evict: dst_table must be a contiguous int32 [%d, pages for %d positions] on the pools' GPU",
                        c.kv.num_seqs, e.budget);
            return nullptr;
        }
        const auto ints = dst->options();
        at::Tensor kept = at::empty({c.kv.num_seqs, c.kv.kv_heads, std::max(e.budget, 0)}, ints);
        at::Tensor lens = at::empty({c.kv.num_seqs}, ints), mass = at::empty(m->sizes(), m->options());
        e.mass = static_cast<const float*>(m->data_ptr());
        e.mass_out = static_cast<float*>(mass.data_ptr());
        e.mass_seq_stride = m->size(1) * m->size(2);
        e.mass_head_stride = m->size(2);
        e.mass_cap = static_cast<int32_t>(m->size(2));
        e.dst_table = static_cast<const int32_t*>(dst->data_ptr());
        e.dst_stride = dst->size(1);
        e.kept = static_cast<int32_t*>(kept.data_ptr());
        e.new_lens = static_cast<int32_t*>(lens.data_ptr());
        rt_ctx* ctx = context(c.index);
        if (!ctx || !done(rt_paged_evict(ctx, &c.kv, &e, stream_of(c.index)), ctx)) return nullptr;
        return Py_BuildValue("NNN", THPVariable_Wrap(kept), THPVariable_Wrap(lens), THPVariable_Wrap(mass));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

bool get_index(PyObject* const* a, Py_ssize_t n, int* out) {
    if (n != 1) {
        PyErr_SetString(PyExc_TypeError, "one device index is wanted");
        return false;
    }
    const long v = PyLong_AsLong(a[0]);
    *out = static_cast<int>(v);
    return !(v == -1 && PyErr_Occurred());
}

// sync(index): rt_sync of the device's context, if there is one
PyObject* sync(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int index;
    if (!get_index(a, n, &index)) return nullptr;
    rt_ctx* ctx = index >= 0 && index < kDevices ? g_ctx[index] : nullptr;
    if (ctx && !done(rt_sync(ctx), ctx)) return nullptr;
    Py_RETURN_NONE;
}

// forget(index): the next call on the device asks for its context again
PyObject* forget(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int index;
    if (!get_index(a, n, &index)) return nullptr;
    if (index >= 0 && index < kDevices) g_ctx[index] = nullptr;
    Py_RETURN_NONE;
}

// bind(make_context, raise_error)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "bind takes 2 arguments");
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(g_make_context, a[0]);
    Py_XSETREF(g_raise, a[1]);
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, "rt_paged_append"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, "rt_paged_decode, rt_paged_prompt"},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(evict)), METH_FASTCALL, "rt_paged_evict"},
    {"sync", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sync)), METH_FASTCALL, "rt_sync"},
    {"forget", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(forget)), METH_FASTCALL, "drop a device's context"},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, "set the context factory and the error raiser"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged_torch", "rt_paged_* on torch tensors", -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_torch() { return PyModule_Create(&g_module); }
