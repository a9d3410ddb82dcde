"""Paged key-value cache: append, attention of new tokens, eviction.

The operators take torch tensors on the GPU and only enqueue work, on the
current CUDA stream of the tensors' device, like torch's own operators; the
context behind them, one per device for all threads of the process, keeps one
workspace per thread and stream.  They run the rt_paged_* entry points of
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
the library RtError.  Nothing here is differentiable, the framework trains
nothing: tensors that require gradients are refused unless under
torch.no_grad().

Over f16 and bf16 caches attend_prompt rounds each attention weight to the
cache's type before it multiplies the values, the sum of the weights being that
of the unrounded ones; attend_decode multiplies them in two parts.  Scores, sums,
lse and mass are 32 bits wide everywhere.
"""

import threading

import torch

from ._lib import RT_E_STATE, RtError, lib
from .ops import Context

lib()  # raises if the library has not been built
try:
    from . import _paged_torch as _ext
except ImportError as e:
    raise RuntimeError("rich_triplet_b200/_paged_torch.so is missing or does not load: run rich_triplet_b200.build() "
                       f"({e})") from e


class _DeviceContext(Context):
    """The library context of all paged calls on one device, made on first use
    and kept for the life of the process: the workspaces that captured graphs use
    belong to it, whichever thread captured them.  Calls, and sync(), use it with
    the interpreter's lock held, so threads may share it."""

    def sync(self):
        """Waits for all streams of the device and raises RtError if a kernel
        reported that a bounded wait gave up since the last sync()."""
        torch.cuda.synchronize(self.device)
        self.check()

    def check(self):
        """The same for kernels that have finished, without waiting for streams."""
        _ext.sync(self.device)

    def close(self):
        """Frees the context and the workspaces of its streams: no captured graph
        may run afterwards.  The next call makes a new one."""
        if self.h:
            if _made.get(self.device) is self:
                del _made[self.device]
                _ext.forget(self.device)
            torch.cuda.synchronize(self.device)
            super().close()


_made = {}
_making = threading.Lock()


def _context(index):
    with _making:
        ctx = _made.get(index)
        if ctx is None:
            if torch.cuda.is_current_stream_capturing():
                raise RtError(RT_E_STATE, "the paged operators' context does not exist yet; make one call before the capture")
            before = torch.cuda.current_device()
            ctx = _DeviceContext(index)
            torch.cuda.set_device(before)
            _made[index] = ctx
        return ctx


def _raise(rc, message):
    raise RtError(rc, message)


_ext.bind(lambda index: _context(index).h.value, _raise)


def context(device):
    """The library context behind the calls on a GPU: its sync() waits for the
    device and raises RtError if a kernel reported that a bounded wait gave up."""
    device = torch.device(device)
    return _context(device.index if device.index is not None else torch.cuda.current_device())


def kv_append(k_pages, v_pages, k, v, page_table, lens, q_start=None):
    """New key and value rows ``k``, ``v`` [rows, kv_heads, head_dim] (f32, f16
    or bf16) into the cache, rounded to its type.  Without ``q_start`` row b is
    the last position of sequence b; with it ([sequences + 1] int32) rows
    q_start[b] .. q_start[b + 1] - 1 are the last positions of sequence b."""
    _ext.append(k_pages, v_pages, page_table, lens, k, v, q_start)


def attend_decode(q, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None, out=None):
    """Attention of one new token per sequence, at its last position: ``q``
    [sequences, heads, head_dim] in the cache's type -> (out like q, lse
    [sequences, heads] f32).  Head h reads KV head h // (heads / kv_heads).
    With ``window`` > 0 a token sees the last ``window`` positions, its own
    among them, and the first ``sinks``.  ``mass`` [sequences, kv_heads,
    positions] f32: every visible position's attention weight, summed over the
    query heads of its KV head, is added to it."""
    return _ext.attend(k_pages, v_pages, page_table, lens, q, None, 0, scale, window, sinks, mass, out)


def attend_prompt(q, q_start, max_new, k_pages, v_pages, page_table, lens, *, scale, window=0, sinks=0, mass=None,
                  out=None):
    """Attention of several new tokens per sequence: rows q_start[b] ..
    q_start[b + 1] - 1 of ``q`` [rows, heads, head_dim] are the last tokens of
    sequence b, and each sees the positions up to its own (window, sinks and
    mass as for attend_decode).  ``max_new`` bounds the tokens of a sequence;
    rows beyond it are left as they are.  Returns (out, lse [rows, heads])."""
    if q_start is None:  # the binding would take it for a decode step
        raise ValueError("attend_prompt: q_start must be a tensor")
    return _ext.attend(k_pages, v_pages, page_table, lens, q, q_start, max_new, scale, window, sinks, mass, out)


def kv_evict(k_pages, v_pages, page_table, lens, mass, dst_table, *, budget, sinks=0, recent=0):
    """Trim every sequence to ``budget`` positions, each KV head on its own:
    its first ``sinks``, its last ``recent`` and, of the others, those of the
    largest ``mass`` (equal ones: the lower position) are copied in order to
    the pages of ``dst_table`` [sequences, >= ceil(budget / page_size)] int32,
    which must not be in use.  Returns (kept positions [sequences, kv_heads,
    budget] int32, -1 after the last; new lengths [sequences] int32; the kept
    positions' mass in a tensor like ``mass``, zero after the last)."""
    return _ext.evict(k_pages, v_pages, page_table, lens, mass, dst_table, budget, sinks, recent)


class PagePool:
    """Page numbers 0 .. num_pages - 1, handed out and taken back on the host."""

    def __init__(self, num_pages):
        self.num_pages = int(num_pages)
        self._free = list(range(self.num_pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    def take(self, n):
        if n > len(self._free):
            raise ValueError(f"PagePool: {n} pages wanted, {len(self._free)} of {self.num_pages} free")
        return [self._free.pop() for _ in range(n)]

    def give(self, pages):
        self._free.extend(pages)


class PagedKvCache:
    """The paged caches of several layers that keep the same positions of a set
    of sequences: one pool of keys and one of values per layer, one page table
    and one list of lengths for all of them.

    ``totals`` keeps a running total of every cached position's attention
    weight per layer ([layers, sequences, kv_heads, max_len] f32), which decode
    and prompt add to and evict ranks by.  Lengths and the table live on the
    host and are copied to the device when they change; the operators run on
    torch's current stream."""

    def __init__(self, layers, sequences, num_pages, page_size, kv_heads, head_dim, max_len, dtype=torch.bfloat16,
                 device="cuda", totals=False):
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.page_size, self.max_len, self.device = page_size, max_len, self.k.device
        self.pool = PagePool(num_pages)
        self.lens = [0] * sequences
        self._gone = [(0, 0)] * sequences  # table entries [from, to) whose pages drop() gave back
        width = -(-max_len // page_size)
        self._table = torch.full((sequences, width), -1, dtype=torch.int32)
        self.page_table = self._table.to(self.device)
        self.lens_device = torch.zeros(sequences, dtype=torch.int32, device=self.device)
        self.mass = None
        if totals:
            self.mass = torch.zeros((layers, sequences, kv_heads, max_len), dtype=torch.float32, device=self.device)

    def _upload(self, table=True):
        if table:
            self.page_table.copy_(self._table)
        self.lens_device.copy_(torch.tensor(self.lens, dtype=torch.int32))

    def extend(self, counts):
        """Room for counts[b] new tokens of every sequence b: lengths grow and
        pages are taken from the pool."""
        if any(c < 0 for c in counts):
            raise ValueError(f"PagedKvCache.extend: negative counts {list(counts)}")
        wanted = [n + c for n, c in zip(self.lens, counts)]
        if len(counts) != len(self.lens) or max(wanted) > self.max_len:
            raise ValueError(f"PagedKvCache.extend: lengths {wanted} for {len(self.lens)} sequences of at most "
                             f"{self.max_len} positions")
        need = [range(-(-n // self.page_size), -(-w // self.page_size)) for n, w in zip(self.lens, wanted)]
        pages = self.pool.take(sum(len(r) for r in need))
        for b, r in enumerate(need):
            for p in r:
                self._table[b, p] = pages.pop()
        self.lens = wanted
        self._upload(table=any(need))

    def drop(self, window, sinks=0):
        """Give back the pages that no later token sees: before the window of
        the next one, and past the first ``sinks`` positions (none with a window
        of 0, which sees everything)."""
        if window < 0 or sinks < 0:
            raise ValueError(f"PagedKvCache.drop: negative window {window} or sinks {sinks}")
        if window == 0:
            return
        first, given = -(-sinks // self.page_size), []
        for b, n in enumerate(self.lens):
            end = max(0, n + 1 - window) // self.page_size
            lo, hi = self._gone[b]
            for p in (*range(first, min(lo, end)), *range(max(hi, first), end)):
                page = int(self._table[b, p])
                if page >= 0:
                    given.append(page)
                    self._table[b, p] = -1
            if first < end and (lo == hi or first <= hi and lo <= end):  # else two gaps: the older one is remembered
                self._gone[b] = (first, end) if lo == hi else (min(lo, first), max(hi, end))
        if given:
            self.pool.give(given)
            self.page_table.copy_(self._table)

    def append(self, layer, k, v, q_start=None):
        kv_append(self.k[layer], self.v[layer], k, v, self.page_table, self.lens_device, q_start)

    def decode(self, layer, q, *, scale, window=0, sinks=0):
        mass = None if self.mass is None else self.mass[layer]
        return attend_decode(q, self.k[layer], self.v[layer], self.page_table, self.lens_device, scale=scale,
                             window=window, sinks=sinks, mass=mass)

    def prompt(self, layer, q, q_start, max_new, *, scale, window=0, sinks=0):
        mass = None if self.mass is None else self.mass[layer]
        return attend_prompt(q, q_start, max_new, self.k[layer], self.v[layer], self.page_table, self.lens_device,
                             scale=scale, window=window, sinks=sinks, mass=mass)

    def evict(self, budget, sinks=0, recent=0):
        """Trim every sequence of every layer that is longer than ``budget``
        positions to so many by its totals (kv_evict); its old pages go back to the
        pool.  Returns the kept positions of each layer.  Sequences take turns
        where the pool has too few free pages for all of them; with none to spare
        one is trimmed through a copy of its rows outside the pool."""
        if self.mass is None:
            raise ValueError("PagedKvCache.evict: the cache was made without totals")
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"PagedKvCache.evict: sinks {sinks} + recent {recent} must lie in 0..budget {budget}")
        layers, _, heads = self.mass.shape[:3]
        each = -(-budget // self.page_size)
        at = torch.arange(budget, dtype=torch.int32, device=self.device)
        kept = torch.where(at < self.lens_device[:, None, None], at, -1).repeat(layers, 1, heads, 1)
        left = [b for b, n in enumerate(self.lens) if n > budget]
        while left:
            now = max(1, self.pool.free_pages // each)
            self._trim(left[:now], kept, each, dict(budget=budget, sinks=sinks, recent=recent))
            left = left[now:]
        return list(kept)

    def _trim(self, seqs, kept, each, limits):
        """Trims sequences `seqs` into `each` pages each: free ones, or, for one
        sequence, as many of its own as are wanting."""
        own = [[int(p) for p in self._table[b] if p >= 0] for b in seqs]
        short = max(0, each * len(seqs) - self.pool.free_pages)
        if short > (len(own[0]) if len(seqs) == 1 else 0):
            raise ValueError(f"PagedKvCache.evict: {short} more pages wanted than are free")
        taken = self.pool.take(each * len(seqs) - short)
        try:
            pages = torch.tensor(taken + own[0][:short], dtype=torch.int32).view(len(seqs), each)
            dst = pages.to(self.device)
            rows = slice(None) if len(seqs) == len(self.lens) else torch.tensor(seqs, device=self.device)
            lens = self.lens_device[rows]
            if short:  # the sequence's pages and `each` more, in pools of their own
                at = torch.tensor(own[0], device=self.device)
                table = torch.full_like(self._table[seqs], -1)
                table[self._table[seqs] >= 0] = torch.arange(len(own[0]), dtype=torch.int32)
                table = table.to(self.device)
                spare = torch.arange(len(own[0]), len(own[0]) + each, dtype=torch.int32, device=self.device).view(1, -1)
            done = []
            for k, v, mass in zip(self.k, self.v, self.mass):
                if not short:
                    done.append(kv_evict(k, v, self.page_table[rows], lens, mass[rows], dst, **limits))
                else:
                    room = [torch.cat([x[at], x.new_zeros((each, *x.shape[1:]))]) for x in (k, v)]
                    done.append((*kv_evict(*room, table, lens, mass[rows], spare, **limits),
                                 *(x[len(own[0]):] for x in room)))
        except Exception:
            self.pool.give(taken)  # the sequences still have theirs
            raise
        for i, (got, _, mass, *moved) in enumerate(done):
            kept[i, rows] = got
            self.mass[i, rows] = mass
            for x, rest in zip((self.k, self.v), moved):
                x[i, dst[0].long()] = rest
        kept_own = own[0][:short]
        self.pool.give([p for ids in own for p in ids if p not in kept_own])
        for b, ids in zip(seqs, pages):
            self.lens[b] = limits["budget"]
            self._table[b] = -1
            self._table[b, :each] = ids
            self._gone[b] = (0, 0)
        self._upload()
