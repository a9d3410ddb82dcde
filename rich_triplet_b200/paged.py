"""Paged key-value cache: append, attention of new tokens, eviction.

The operators take torch tensors on the GPU and only enqueue work, on the
current CUDA stream of the tensors' device, like torch's own operators; the
context behind them (one per thread and device, as ops.default_context) keeps
one workspace per stream.  They run the rt_paged_* entry points of
include/rt_cuda.h, whose comments define them; the reference has one
contiguous cache per layer instead (Gemma3LayerKvCache,
src/transformer4.rs:1794-1864).

One layer's cache is two pools of pages, ``k_pages`` and ``v_pages``
``[num_pages, kv_heads, page_size, head_dim]`` (f32, f16 or bf16, any strides
that keep rows whole), a page table ``[sequences, width]`` (int32) and the
sequences' lengths ``[sequences]`` (int32, new tokens included).  Position j of
sequence b is slot ``j % page_size`` of page ``page_table[b, j // page_size]``.

    kv_append      new key and value rows to their sequences' last positions
    attend_decode  one new token per sequence attends to its cached positions
    attend_prompt  several new tokens per sequence attend, causally
    kv_evict       trim sequences to the positions that carry the most weight

``PagePool`` hands out page numbers; ``PagedKvCache`` keeps pools for several
layers, the page table and the lengths of a set of sequences, and calls the
operators.  Wrong types, shapes or devices raise ValueError, failures inside
the library RtError.
"""

import ctypes
import threading

import torch

from ._lib import (RT_FMT_BF16, RT_FMT_F16, RT_FMT_F32, RT_OK, RT_PAGED_ATTN, RT_PAGED_EVICT, RT_PAGED_KV,
                   RT_PAGED_ROWS, check, lib)
from .ops import Context

_FMT = {torch.float32: RT_FMT_F32, torch.float16: RT_FMT_F16, torch.bfloat16: RT_FMT_BF16}
_I32, _F32 = torch.int32, torch.float32
_pack_kv, _pack_rows, _pack_attn, _pack_evict = (s.pack for s in (RT_PAGED_KV, RT_PAGED_ROWS, RT_PAGED_ATTN,
                                                                  RT_PAGED_EVICT))


class _Contexts(threading.local):
    """This thread's library contexts, by device."""

    def __init__(self):
        self.made = {}

    def get(self, index):
        ctx = self.made.get(index)
        if ctx is None:
            before = torch.cuda.current_device()
            ctx = self.made[index] = Context(index)
            torch.cuda.set_device(before)
        return ctx


_contexts = _Contexts()


def context(device):
    """This thread's library context on a GPU: its sync() waits for the
    context's own stream and raises RtError if a kernel of any stream reported
    that a bounded wait gave up."""
    device = torch.device(device)
    return _contexts.get(device.index if device.index is not None else torch.cuda.current_device())


def _run(fn, index, kv, args):
    """Call fn(context, kv, args, current stream)."""
    ctx = _contexts.get(index)
    # the default stream has handle 0, which the library takes for the context's
    # own stream: it is named by CUDA's value for it (cudaStreamLegacy, 1)
    rc = fn(ctx.h, kv, args, torch._C._cuda_getCurrentRawStream(index) or 1)
    if rc != RT_OK:
        check(rc, ctx.h)


def _cache(k_pages, v_pages, page_table, lens):
    """(packed rt_paged_kv, shape of the pools, format, device index, sequences):
    sizes checked as far as the library cannot."""
    shape, strides, dtype, index = k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != strides:
        raise ValueError(f"paged: k_pages {tuple(shape)} and v_pages {tuple(v_pages.shape)} must be "
                         "[num_pages, kv_heads, page_size, head_dim] with the same strides")
    fmt = _FMT.get(dtype)
    if fmt is None or v_pages.dtype is not dtype:
        raise ValueError(f"paged: pools must be f32, f16 or bf16, got {dtype} and {v_pages.dtype}")
    if index < 0 or v_pages.get_device() != index:
        raise ValueError(f"paged: pools must be on one GPU, got {k_pages.device} and {v_pages.device}")
    num_pages, heads, page, d = shape
    ps, hs, ss, one = strides
    if one != 1:
        raise ValueError("paged: the rows of the pools must be contiguous")
    tshape = page_table.shape
    if len(tshape) != 2 or page_table.dtype is not _I32 or page_table.get_device() != index or \
            (tshape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("paged: page_table must be [sequences, width] int32 with contiguous rows, on the pools' GPU")
    n, width = tshape
    if lens.dtype is not _I32 or lens.shape != tshape[:1] or lens.get_device() != index or not lens.is_contiguous():
        raise ValueError(f"paged: lens must be [{n}] int32, contiguous, on the pools' GPU")
    kv = _pack_kv(k_pages.data_ptr(), v_pages.data_ptr(), ps, hs, ss, num_pages, fmt, heads, d, page,
                  page_table.data_ptr(), max(page_table.stride(0), width), width, n, lens.data_ptr())
    return kv, shape, dtype, index, n


def _starts(q_start, index, n, who):
    if q_start.dtype is not _I32 or q_start.shape != (n + 1,) or q_start.get_device() != index or \
            not q_start.is_contiguous():
        raise ValueError(f"{who}: q_start must be [{n + 1}] int32, contiguous, on the pools' GPU")
    return q_start.data_ptr()


def kv_append(k_pages, v_pages, k, v, page_table, lens, q_start=None):
    """New key and value rows ``k``, ``v`` [rows, kv_heads, head_dim] (f32, f16
    or bf16) into the cache, rounded to its type.  Without ``q_start`` row b is
    the last position of sequence b; with it ([sequences + 1] int32) rows
    q_start[b] .. q_start[b + 1] - 1 are the last positions of sequence b."""
    kv, shape, _, index, n = _cache(k_pages, v_pages, page_table, lens)
    ks, strides, dtype = k.shape, k.stride(), k.dtype
    if len(ks) != 3 or v.shape != ks or v.stride() != strides or ks[1] != shape[1] or ks[2] != shape[3] or \
            strides[2] != 1:
        raise ValueError(f"kv_append: k {tuple(ks)} and v {tuple(v.shape)} must be [rows, {shape[1]}, {shape[3]}] with "
                         "the same strides and contiguous rows")
    fmt = _FMT.get(dtype)
    if fmt is None or v.dtype is not dtype or k.get_device() != index or v.get_device() != index:
        raise ValueError("kv_append: k and v must be f32, f16 or bf16 on the pools' GPU")
    start = 0 if q_start is None else _starts(q_start, index, n, "kv_append")
    _run(lib().rt_paged_append, index, kv,
         _pack_rows(k.data_ptr(), v.data_ptr(), strides[0], strides[1], ks[0], fmt, start))


def _attend(who, prompt, q, k_pages, v_pages, page_table, lens, q_start, max_new, scale, window, sinks, mass, out):
    kv, shape, dtype, index, n = _cache(k_pages, v_pages, page_table, lens)
    qs, strides = q.shape, q.stride()
    if len(qs) != 3 or qs[2] != shape[3] or q.dtype is not dtype or q.get_device() != index or strides[2] != 1:
        raise ValueError(f"{who}: q must be [rows, heads, {shape[3]}] {dtype} with contiguous rows on the pools' GPU, "
                         f"got {tuple(qs)} {q.dtype} on {q.device}")
    rows, heads, _ = qs
    if prompt:
        start = _starts(q_start, index, n, who)
    elif rows != n:
        raise ValueError(f"{who}: {rows} query rows, but lens has {n} sequences")
    else:
        start = 0
    if out is None:
        out = q.new_empty(qs)
    elif out.shape != qs or out.dtype is not dtype or out.get_device() != index or out.stride(2) != 1:
        raise ValueError(f"{who}: out must be {tuple(qs)} {dtype} with contiguous rows on the pools' GPU")
    lse = q.new_empty((rows, heads), dtype=_F32)
    L = lib()
    os0, os1, _ = out.stride()
    head = (q.data_ptr(), out.data_ptr(), strides[0], strides[1], os0, os1, lse.data_ptr(), heads, rows, heads, window,
            sinks, max_new, scale)
    scratch = None
    if mass is None:
        args = _pack_attn(*head, 0, start, 0, 0, 0, 0, 0)
    else:
        ms = mass.shape
        if len(ms) != 3 or mass.dtype is not _F32 or mass.get_device() != index or ms[0] != n or ms[1] != shape[1] or \
                (ms[2] > 1 and mass.stride(2) != 1):
            raise ValueError(f"{who}: mass must be [{n}, {shape[1]}, positions] float32 with contiguous rows on the "
                             "pools' GPU")
        tail = (ms[2], start, mass.data_ptr(), mass.stride(0), mass.stride(1))
        args = _pack_attn(*head, *tail, 0, 0)
        need = ctypes.c_uint64()
        check(L.rt_paged_scratch(kv, args, int(prompt), ctypes.byref(need)))
        if need.value:
            # freed when this call returns: only later work of this stream takes its place
            scratch = q.new_empty(need.value, dtype=torch.uint8)
            args = _pack_attn(*head, *tail, scratch.data_ptr(), need.value)
    _run(L.rt_paged_prompt if prompt else L.rt_paged_decode, index, kv, args)
    return out, lse


def attend_decode(q, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None, out=None):
    """Attention of one new token per sequence, at its last position: ``q``
    [sequences, heads, head_dim] in the cache's type -> (out like q, lse
    [sequences, heads] f32).  Head h reads KV head h // (heads / kv_heads).
    With ``window`` > 0 a token sees the last ``window`` positions, its own
    among them, and the first ``sinks``.  ``mass`` [sequences, kv_heads,
    positions] f32: every visible position's attention weight, summed over the
    query heads of its KV head, is added to it."""
    return _attend("attend_decode", False, q, k_pages, v_pages, page_table, lens, None, 0, scale, window, sinks, mass,
                   out)


def attend_prompt(q, q_start, max_new, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None,
                  out=None):
    """Attention of several new tokens per sequence: rows q_start[b] ..
    q_start[b + 1] - 1 of ``q`` [rows, heads, head_dim] are the last tokens of
    sequence b, and each sees the positions up to its own (window, sinks and
    mass as for attend_decode).  ``max_new`` bounds the tokens of a sequence;
    rows beyond it are left as they are.  Returns (out, lse [rows, heads])."""
    return _attend("attend_prompt", True, q, k_pages, v_pages, page_table, lens, q_start, int(max_new), scale, window,
                   sinks, mass, out)


def kv_evict(k_pages, v_pages, page_table, lens, mass, dst_table, *, budget, sinks=0, recent=0):
    """Trim every sequence to ``budget`` positions, each KV head on its own:
    its first ``sinks``, its last ``recent`` and, of the others, those of the
    largest ``mass`` (equal ones: the lower position) are copied in order to
    the pages of ``dst_table`` [sequences, >= ceil(budget / page_size)] int32,
    which must not be in use.  Returns (kept positions [sequences, kv_heads,
    budget] int32, -1 after the last; new lengths [sequences] int32; the kept
    positions' mass in a tensor like ``mass``, zero after the last)."""
    kv, shape, _, index, n = _cache(k_pages, v_pages, page_table, lens)
    heads, page = shape[1], shape[2]
    ms = mass.shape
    if len(ms) != 3 or mass.dtype is not _F32 or mass.get_device() != index or ms[0] != n or ms[1] != heads or \
            not mass.is_contiguous():
        raise ValueError(f"kv_evict: mass must be a contiguous [{n}, {heads}, positions] float32 tensor on the pools' "
                         "GPU")
    ds = dst_table.shape
    if len(ds) != 2 or ds[0] != n or dst_table.dtype is not _I32 or dst_table.get_device() != index or \
            not dst_table.is_contiguous() or ds[1] * page < budget:
        raise ValueError(f"kv_evict: dst_table must be a contiguous [{n}, >= {-(-budget // page)}] int32 tensor on the "
                         "pools' GPU")
    kept = lens.new_empty((n, heads, max(budget, 0)))
    new_lens = torch.empty_like(lens)
    mass_out = torch.empty_like(mass)
    _run(lib().rt_paged_evict, index, kv,
         _pack_evict(mass.data_ptr(), mass_out.data_ptr(), heads * ms[2], ms[2], ms[2], budget, sinks, recent,
                     dst_table.data_ptr(), ds[1], kept.data_ptr(), new_lens.data_ptr()))
    return kept, new_lens, mass_out
