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

from ._lib import (RT_FMT_BF16, RT_FMT_F16, RT_FMT_F32, RtPagedAttn, RtPagedEvict, RtPagedKv, RtPagedRows, check, lib)
from .ops import Context

_FMT = {torch.float32: RT_FMT_F32, torch.float16: RT_FMT_F16, torch.bfloat16: RT_FMT_BF16}

_tls = threading.local()


def _context(device):
    """This thread's context on `device`."""
    made = getattr(_tls, "contexts", None)
    if made is None:
        made = _tls.contexts = {}
    index = device.index if device.index is not None else torch.cuda.current_device()
    ctx = made.get(index)
    if ctx is None:
        before = torch.cuda.current_device()
        ctx = made[index] = Context(index)
        torch.cuda.set_device(before)
    return ctx


def _stream(device):
    # 0 is the legacy default stream; the library takes a null stream as the
    # context's own, so it is named by CUDA's handle for it (cudaStreamLegacy)
    return torch.cuda.current_stream(device).cuda_stream or 1


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _int32(t, device, shape, name):
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name}: need a contiguous int32 tensor {shape} on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _cache(k_pages, v_pages, page_table, lens):
    """RtPagedKv of a cache, its sizes checked as far as the library cannot."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
        raise ValueError(f"paged: k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must be "
                         "[num_pages, kv_heads, page_size, head_dim] with the same strides")
    fmt, device = _FMT.get(k_pages.dtype), k_pages.device
    if fmt is None or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"paged: pools must be f32, f16 or bf16, got {k_pages.dtype} and {v_pages.dtype}")
    if device.type != "cuda" or v_pages.device != device:
        raise ValueError(f"paged: pools must be on one GPU, got {device} and {v_pages.device}")
    if k_pages.stride(3) != 1 and k_pages.shape[3] > 1:
        raise ValueError("paged: the rows of the pools must be contiguous")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("paged: page_table must be [sequences, width] int32 with contiguous rows, on the pools' GPU")
    n, width = page_table.shape
    _int32(lens, device, (n,), "paged: lens")
    num_pages, heads, page, d = k_pages.shape
    ps, hs, ss, _ = k_pages.stride()
    return RtPagedKv(k_pages.data_ptr(), v_pages.data_ptr(), ps, hs, ss, num_pages, fmt, heads, d, page,
                     page_table.data_ptr(), max(page_table.stride(0), width), width, n, lens.data_ptr())


def kv_append(k_pages, v_pages, k, v, page_table, lens, q_start=None):
    """New key and value rows ``k``, ``v`` [rows, kv_heads, head_dim] (f32, f16
    or bf16) into the cache, rounded to its type.  Without ``q_start`` row b is
    the last position of sequence b; with it ([sequences + 1] int32) rows
    q_start[b] .. q_start[b + 1] - 1 are the last positions of sequence b."""
    c = _cache(k_pages, v_pages, page_table, lens)
    device = k_pages.device
    if k.dim() != 3 or k.shape != v.shape or k.stride() != v.stride() or k.shape[1:] != (c.kv_heads, c.head_dim) or \
            k.stride(2) != 1:
        raise ValueError(f"kv_append: k {tuple(k.shape)} and v {tuple(v.shape)} must be [rows, {c.kv_heads}, "
                         f"{c.head_dim}] with the same strides and contiguous rows")
    fmt = _FMT.get(k.dtype)
    if fmt is None or v.dtype != k.dtype or k.device != device or v.device != device:
        raise ValueError("kv_append: k and v must be f32, f16 or bf16 on the pools' GPU")
    if q_start is not None:
        _int32(q_start, device, (c.num_seqs + 1,), "kv_append: q_start")
    ctx = _context(device)
    r = RtPagedRows(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.shape[0], fmt,
                    q_start.data_ptr() if q_start is not None else None)
    check(lib().rt_paged_append(ctx.h, ctypes.byref(c), ctypes.byref(r), _stream(device)), ctx.h)


def _attend(who, prompt, q, k_pages, v_pages, page_table, lens, q_start, max_new, scale, window, sinks, mass, out):
    c = _cache(k_pages, v_pages, page_table, lens)
    device = k_pages.device
    if q.dim() != 3 or q.shape[2] != c.head_dim or q.dtype != k_pages.dtype or q.device != device or \
            (q.stride(2) != 1 and c.head_dim > 1):
        raise ValueError(f"{who}: q must be [rows, heads, {c.head_dim}] {k_pages.dtype} with contiguous rows on "
                         f"{device}, got {tuple(q.shape)} {q.dtype} on {q.device}")
    rows, heads, d = q.shape
    if out is None:
        out = torch.empty((rows, heads, d), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or out.stride(2) != 1:
        raise ValueError(f"{who}: out must be {tuple(q.shape)} {q.dtype} with contiguous rows on {device}")
    lse = torch.empty((rows, heads), dtype=torch.float32, device=device)
    a = RtPagedAttn(q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                    lse.data_ptr(), heads, rows, heads, window, sinks, max_new, scale, 0,
                    q_start.data_ptr() if prompt else None, None, 0, 0, None, 0)
    L = lib()
    ctx = _context(device)
    scratch = None
    if mass is not None:
        if mass.dim() != 3 or mass.dtype != torch.float32 or mass.device != device or \
                mass.shape[:2] != (c.num_seqs, c.kv_heads) or (mass.shape[2] > 1 and mass.stride(2) != 1):
            raise ValueError(f"{who}: mass must be [{c.num_seqs}, {c.kv_heads}, positions] float32 with contiguous "
                             f"rows on {device}")
        a.mass, a.mass_cap = mass.data_ptr(), mass.shape[2]
        a.mass_seq_stride, a.mass_head_stride = mass.stride(0), mass.stride(1)
        n = ctypes.c_uint64()
        check(L.rt_paged_scratch(ctypes.byref(c), ctypes.byref(a), int(prompt), ctypes.byref(n)), None)
        if n.value:
            # freed when this call returns, and reused by later work of this stream only
            scratch = torch.empty(n.value, dtype=torch.uint8, device=device)
            a.scratch, a.scratch_bytes = scratch.data_ptr(), n.value
    fn = L.rt_paged_prompt if prompt else L.rt_paged_decode
    check(fn(ctx.h, ctypes.byref(c), ctypes.byref(a), _stream(device)), ctx.h)
    return out, lse


def attend_decode(q, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None, out=None):
    """Attention of one new token per sequence, at its last position: ``q``
    [sequences, heads, head_dim] in the cache's type -> (out like q, lse
    [sequences, heads] f32).  Head h reads KV head h // (heads / kv_heads).
    With ``window`` > 0 a token sees the last ``window`` positions, its own
    among them, and the first ``sinks``.  ``mass`` [sequences, kv_heads,
    positions] f32: every visible position's attention weight, summed over the
    query heads of its KV head, is added to it."""
    if q.shape[0] != lens.shape[0]:
        raise ValueError(f"attend_decode: {q.shape[0]} query rows, but lens has {lens.shape[0]} sequences")
    return _attend("attend_decode", False, q, k_pages, v_pages, page_table, lens, None, 0, scale, window, sinks, mass,
                   out)


def attend_prompt(q, q_start, max_new, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None,
                  out=None):
    """Attention of several new tokens per sequence: rows q_start[b] ..
    q_start[b + 1] - 1 of ``q`` [rows, heads, head_dim] are the last tokens of
    sequence b, and each sees the positions up to its own (window, sinks and
    mass as for attend_decode).  ``max_new`` bounds the tokens of a sequence;
    rows beyond it are left as they are.  Returns (out, lse [rows, heads])."""
    _int32(q_start, k_pages.device, (lens.shape[0] + 1,), "attend_prompt: q_start")
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
    c = _cache(k_pages, v_pages, page_table, lens)
    device = k_pages.device
    if mass.dim() != 3 or mass.dtype != torch.float32 or mass.device != device or \
            mass.shape[:2] != (c.num_seqs, c.kv_heads) or not mass.is_contiguous():
        raise ValueError(f"kv_evict: mass must be a contiguous [{c.num_seqs}, {c.kv_heads}, positions] float32 tensor "
                         f"on {device}")
    if dst_table.dim() != 2 or dst_table.shape[0] != c.num_seqs or dst_table.dtype != torch.int32 or \
            dst_table.device != device or not dst_table.is_contiguous() or \
            dst_table.shape[1] * c.page_size < budget:
        raise ValueError(f"kv_evict: dst_table must be a contiguous [{c.num_seqs}, >= {-(-budget // c.page_size)}] "
                         f"int32 tensor on {device}")
    kept = torch.empty((c.num_seqs, c.kv_heads, budget), dtype=torch.int32, device=device)
    new_lens = torch.empty_like(lens)
    mass_out = torch.empty_like(mass)
    e = RtPagedEvict(mass.data_ptr(), mass_out.data_ptr(), mass.stride(0), mass.stride(1), mass.shape[2], budget,
                     sinks, recent, dst_table.data_ptr(), dst_table.shape[1], kept.data_ptr(), new_lens.data_ptr())
    ctx = _context(device)
    check(lib().rt_paged_evict(ctx.h, ctypes.byref(c), ctypes.byref(e), _stream(device)), ctx.h)
    return kept, new_lens, mass_out
