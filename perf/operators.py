"""Measured cases of the paged key-value cache operators.

Four operators work on one layer's paged cache: pools of pages
``[num_pages, kv_heads, page_size, head_dim]`` for keys and for values, a page
table ``[sequences, pages per sequence]`` and the sequences' lengths.

append   rows of new keys and values, rounded to the cache's type, go to their
         sequences' last positions;
decode   one new token per sequence attends to its cached positions: all of
         them, or a sliding window and a few first tokens that stay visible;
         optionally each cached position's attention weight, summed over the
         query heads of its key-value head, is added to a running total;
prompt   the same for several new tokens per sequence, each of which sees the
         positions up to its own;
evict    of every key-value head's positions the first few, the most recent and
         those with the largest running totals are kept, up to a budget, and
         copied in order to other pages.

``own = False`` runs them as elementary torch operations in 32 bits;
``own = True`` makes the calls of ``rich_triplet_b200.paged``.  Sizes are those
of this repository's configurations: 4 query heads on 1 key-value head and 8 on
4, both 256 wide (the 1B and 4B models), 32 on 16, 128 wide (27B), 16 on 4, 256
wide (the hybrid engine), 2 on 1, 128 wide (the tests' model), and 8 on 1, 64
wide, generic.
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(4, 1, 256), (8, 4, 256), (32, 16, 128), (16, 4, 256), (2, 1, 128), (8, 1, 64)]


# ---- cases ------------------------------------------------------------------


def _case(op, name=None, **given):
    """A case with every field that its operator reads."""
    c = {"op": op, "dtype": "bf16", "nq": 8, "nkv": 4, "D": 256, "page": 64, "layout": "head", "B": 1, "len": 1,
         "ragged": False}
    if op in ("append", "prompt"):
        c["new"] = 1
    if op in ("decode", "prompt"):
        c.update(window=0, sinks=0, mass=False)
    if op == "evict":
        c.update(budget=1, sinks=4, recent=0)
    if op == "append":
        c["src"] = "f32"
    assert all(k in c for k in given), given
    c.update(given)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step's new rows of a handful of chats: the smallest call, only latency
        _case("append", "append one row each", B=3, len=513, page=16, ragged=True),
        # prompts of several users enter the cache together (27B heads, rows as the f32 projections give them)
        _case("append", "append prompts", dtype="f16", nq=32, nkv=16, D=128, page=32, layout="slot", B=9, len=2048,
              new=1999, ragged=True),
        # a single chat near its start
        _case("decode", "decode one short", page=16, len=301),
        # a single long document: one row, split over the length
        _case("decode", "decode one long", B=1, len=131071, page=64),
        # many chats at the many-sequence benchmark's depth, in its f32 cache
        _case("decode", "decode 64 in f32", dtype="f32", B=64, len=4096, page=32, ragged=True),
        # long chats on the 27B heads whose weights are gathered for eviction
        _case("decode", "decode with totals", dtype="f16", nq=32, nkv=16, D=128, page=16, layout="slot", B=11,
              len=8209, ragged=True, mass=True),
        # a local layer late in long chats: 1024 positions and 4 first ones
        _case("decode", "decode in a window", B=64, len=32768, page=64, ragged=True, window=1024, sinks=4),
        # speculative verify: 8 drafted tokens a chat over a filled cache
        _case("prompt", "verify 8 tokens", B=5, len=2050, new=8, page=32, ragged=True),
        # prompts of several users through a local layer, their weights gathered for eviction
        _case("prompt", "prompts in a window with totals", dtype="f16", nq=16, nkv=4, D=256, page=64, B=3, len=4001,
              new=4001, ragged=True, window=1024, sinks=4, mass=True),
        # one long document on the 27B heads, every position visible: the most arithmetic
        _case("prompt", "one long prompt", nq=32, nkv=16, D=128, page=128, B=1, len=8192, new=8192),
        # one chat trimmed a little
        _case("evict", "evict one", page=16, len=700, budget=512, sinks=4, recent=64),
        # many long chats trimmed to a quarter at once
        _case("evict", "evict many", B=32, len=8192, page=64, ragged=True, budget=2048, sinks=4, recent=256),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "evict"])
    nq, nkv, d = rng.choice(HEADS)
    dtype = rng.choice(["f16", "bf16"]) if op == "prompt" else rng.choice(["f32", "f16", "bf16"])
    c = _case(op, dtype=dtype, nq=nq, nkv=nkv, D=d, page=rng.choice([8, 16, 32, 64, 128, 256]),
              layout=rng.choice(["head", "slot"]), ragged=rng.random() < 0.6)
    c["B"] = _log_int(rng, 1, 64)
    # cached values: at most those of 64 sequences of 4096 positions on 4 heads 256 wide
    most = max(16, (64 * 4096 * 4 * 256) // (c["B"] * nkv * d))
    if op == "append":
        c["src"] = rng.choice(["f32", dtype])
        c["len"] = _log_int(rng, 2, min(8192, most))
        c["new"] = min(c["len"], rng.choice([1, _log_int(rng, 1, 2048)]))
    elif op == "decode":
        c["len"] = _log_int(rng, 1, min(131072, most))
    elif op == "prompt":
        # score values: at most half of those of one sequence of 8192 tokens on 32 heads
        most = min(most, int(math.sqrt(32 * 8192 * 8192 / 2 / (c["B"] * nq))))
        c["len"] = _log_int(rng, 2, min(8192, most))
        c["new"] = c["len"] if rng.random() < 0.5 else _log_int(rng, 1, min(c["len"], 64))
    else:
        c["len"] = _log_int(rng, 32, min(32768, max(32, most)))
        c["budget"] = max(16, c["len"] // rng.choice([2, 3, 4, 8]))
        c["recent"] = c["budget"] // rng.choice([2, 4, 8])
    if op in ("decode", "prompt"):
        c["mass"] = rng.random() < 0.4
        if rng.random() < 0.5:
            c["window"] = _log_int(rng, 8, 2048)
            c["sinks"] = rng.choice([0, 1, 4, 16])
    return c


def _lengths(c):
    """(lengths with the new tokens, new tokens) of every sequence."""
    r = random.Random(c["len"] * 1000 + c["B"])
    low = {"evict": c.get("budget", 1) + 1}.get(c["op"], 1)
    n = [c["len"]] + [r.randint(min(low, c["len"]), c["len"]) if c["ragged"] else c["len"] for _ in range(c["B"] - 1)]
    new = [min(x, c.get("new", 1)) for x in n]
    if c["ragged"] and c["op"] in ("append", "prompt"):
        new = [new[0]] + [r.randint(1, x) for x in new[1:]]
    return n, new


def _seen(n, c):
    """How many positions the token at the end of n positions sees."""
    w, s = c["window"], c["sinks"]
    return n if not w or n <= w else w + min(s, n - w)


# ---- inputs -----------------------------------------------------------------


def prepare(c, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    pick = random.Random(seed)
    dt = DTYPES[c["dtype"]]
    B, nq, nkv, D, P = c["B"], c["nq"], c["nkv"], c["D"], c["page"]
    lens, new = _lengths(c)
    width = -(-max(lens) // P)
    used = [-(-n // P) for n in lens]
    spare = -(-c["budget"] // P) if c["op"] == "evict" else 0
    pages = sum(used) + B * spare + 3
    order = list(range(pages))
    pick.shuffle(order)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
        at += u

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    # values have channel means, as a model's do
    means = torch.randn(nkv, 1, D, generator=gen, device=dev) * 0.5

    def pool(add):
        shape = (pages, nkv, P, D) if c["layout"] == "head" else (pages, P, nkv, D)
        x = torch.empty(shape, device=dev, dtype=dt)
        x = x if c["layout"] == "head" else x.transpose(1, 2)
        for i in range(0, pages, 512):
            part = torch.randn(min(512, pages - i), nkv, P, D, generator=gen, device=dev)
            x[i:i + 512] = part + add
        return x

    s = {"case": c, "k_pages": pool(0.0), "v_pages": pool(means), "page_table": table.to(dev),
         "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_len": max(lens), "max_new": max(new)}
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] if c["op"] in ("append", "prompt") else B
    if c["op"] in ("append", "prompt"):
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if c["op"] in ("append", "decode", "prompt"):
        # queries, keys and values as a fused projection leaves them: slices of one row
        qkv = normal(rows, (nq + 2 * nkv) * D, dtype=DTYPES[c.get("src", c["dtype"])])
        s["q"] = qkv[:, :nq * D].view(rows, nq, D)
        s["k"] = qkv[:, nq * D:(nq + nkv) * D].view(rows, nkv, D)
        s["v"] = qkv[:, (nq + nkv) * D:].view(rows, nkv, D)
        s["scale"] = 1.0 / math.sqrt(D)
    if c.get("mass") or c["op"] == "evict":
        # running totals of earlier steps: a few positions hold most of the weight
        m = torch.rand(B, nkv, max(lens), generator=gen, device=dev).pow(8) * 4
        s["mass"] = m * (torch.arange(max(lens), device=dev) < s["lens"][:, None, None])
    if c["op"] == "evict":
        s["dst_table"] = torch.tensor(order[at:at + B * spare], dtype=torch.int32, device=dev).view(B, spare)
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    c = s["case"]
    return (_run_own if own else _run_plain)[c["op"]](s, c)


def _own_append(s, c):
    from rich_triplet_b200 import paged

    paged.kv_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["page_table"], s["lens"], q_start=s["q_start"])
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _own_decode(s, c):
    from rich_triplet_b200 import paged

    mass = s["mass"].clone() if c["mass"] else None
    out, lse = paged.attend_decode(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lens"], scale=s["scale"],
                                   window=c["window"], sinks=c["sinks"], mass=mass)
    return {"out": out, "lse": lse, "mass": mass}


def _own_prompt(s, c):
    from rich_triplet_b200 import paged

    mass = s["mass"].clone() if c["mass"] else None
    out, lse = paged.attend_prompt(s["q"], s["q_start"], s["max_new"], s["k_pages"], s["v_pages"], s["page_table"],
                                   s["lens"], scale=s["scale"], window=c["window"], sinks=c["sinks"], mass=mass)
    return {"out": out, "lse": lse, "mass": mass}


def _own_evict(s, c):
    from rich_triplet_b200 import paged

    kept, lens, mass = paged.kv_evict(s["k_pages"], s["v_pages"], s["page_table"], s["lens"], s["mass"],
                                      s["dst_table"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"])
    return {"kept": kept, "lens": lens, "mass": mass, "k": s["k_pages"], "v": s["v_pages"]}


def _places(table, pos, page):
    """(page, slot) of positions [B, ...] in the page table [B, width]."""
    flat = pos.reshape(pos.shape[0], -1).long()
    return table.long().gather(1, flat // page).clamp(min=0).view(pos.shape), (flat % page).view(pos.shape)


def _row_places(s, page):
    """(page, slot) of every new row."""
    rows = torch.arange(s["k"].shape[0], device=s["k"].device)
    b = torch.searchsorted(s["q_start"], rows.int(), right=True) - 1
    pos = s["lens"][b] - (s["q_start"][b + 1] - rows)
    return s["page_table"][b, pos // page].long(), (pos % page).long()


def _plain_append(s, c):
    pg, slot = _row_places(s, c["page"])
    s["k_pages"][pg, :, slot] = s["k"].to(s["k_pages"].dtype)
    s["v_pages"][pg, :, slot] = s["v"].to(s["v_pages"].dtype)
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _softmax(score, ok):
    """Weights and log of the sum of exponentials over the last axis, 0 and -inf where nothing is visible."""
    score = score.masked_fill(~ok, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    return e / total.clamp(min=1e-30), (top + torch.log(total)).squeeze(-1)


def _plain_decode(s, c):
    B, nq, nkv, D, w, k0 = c["B"], c["nq"], c["nkv"], c["D"], c["window"], c["sinks"]
    lens = s["lens"].long()[:, None]
    # the positions that may be visible: all, or the first few and a window
    at = torch.arange(min(s["max_len"], w + k0) if w else s["max_len"], device=lens.device)[None, :]
    pos = torch.where(at < k0, at, (lens - w).clamp(min=k0) - k0 + at) if w else at.expand(B, -1)
    ok = pos < lens
    pos = torch.where(ok, pos, torch.zeros_like(pos))
    pg, slot = _places(s["page_table"], pos, c["page"])
    k = s["k_pages"][pg, :, slot].permute(0, 2, 1, 3).float()
    v = s["v_pages"][pg, :, slot].permute(0, 2, 1, 3).float()
    q = s["q"].view(B, nkv, nq // nkv, D).float()
    p, lse = _softmax(q @ k.transpose(-1, -2) * s["scale"], ok[:, None, None, :])
    out = (p @ v).view(B, nq, D).to(s["q"].dtype)
    mass = None
    if c["mass"]:
        where = pos[:, None, :].expand(-1, nkv, -1)
        mass = s["mass"].scatter_add(2, where, p.sum(2))
    return {"out": out, "lse": lse.view(B, nq), "mass": mass}


def _plain_prompt(s, c):
    B, nq, nkv, D, w, k0 = c["B"], c["nq"], c["nkv"], c["D"], c["window"], c["sinks"]
    lens, start = s["lens"].long(), s["q_start"].long()
    dev = lens.device
    n = start[1:] - start[:-1]
    i = torch.arange(s["max_new"], device=dev)[None, :]
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    j = torch.arange(s["max_len"], device=dev)
    pg, slot = _places(s["page_table"], j[None, :].expand(B, -1), c["page"])
    k = s["k_pages"][pg, :, slot].permute(0, 2, 1, 3).float()
    v = s["v_pages"][pg, :, slot].permute(0, 2, 1, 3).float()
    q = s["q"].float()[row].view(B, -1, nkv, nq // nkv, D).permute(0, 2, 3, 1, 4)
    at = (lens - n)[:, None] + i
    ok = (j <= at[..., None]) & (i < n[:, None])[..., None]
    if w:
        ok &= (j > at[..., None] - w) | (j < k0)
    p, lse = _softmax(q @ k[:, :, None].transpose(-1, -2) * s["scale"], ok[:, None, None])
    out = (p @ v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(B, -1, nq, D)
    lse = lse.permute(0, 3, 1, 2).reshape(B, -1, nq)
    rows = torch.arange(s["q"].shape[0], device=dev)
    b = torch.searchsorted(s["q_start"], rows.int(), right=True) - 1
    at = rows - start[b]
    mass = s["mass"] + p.sum((2, 3)) if c["mass"] else None
    return {"out": out[b, at].to(s["q"].dtype), "lse": lse[b, at], "mass": mass}


def _plain_evict(s, c):
    nkv, n, recent = c["nkv"], c["budget"], c["recent"]
    lens = s["lens"].long()[:, None, None]
    at = torch.arange(s["mass"].shape[2], device=lens.device)
    rank = torch.where((at < c["sinks"]) | (at >= lens - recent), math.inf, s["mass"])
    rank = torch.where(at < lens, rank, -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :n].sort(-1).values
    new = lens.clamp(max=n)
    ok = torch.arange(n, device=lens.device) < new
    kept = torch.where(ok, kept, 0)
    pg, slot = _places(s["page_table"], kept, c["page"])
    to = torch.arange(n, device=lens.device)
    dpg, dslot = s["dst_table"].long()[:, to // c["page"]], to % c["page"]
    h = torch.arange(nkv, device=lens.device)[None, :, None]
    dpg, dslot = dpg[:, None, :], dslot[None, None, :]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[dpg, h, dslot] = torch.where(ok[..., None], pages[pg, h, slot], pages[dpg, h, dslot])
    mass = torch.zeros_like(s["mass"])
    mass[..., :n] = torch.where(ok, s["mass"].gather(2, kept), 0.0)
    return {"kept": torch.where(ok, kept, -1).int(), "lens": new.view(-1).int(), "mass": mass, "k": s["k_pages"],
            "v": s["v_pages"]}


_run_own = {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt, "evict": _own_evict}
_run_plain = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "evict": _plain_evict}


# ---- what a pass cannot do without -------------------------------------------


def work(c):
    lens, new = _lengths(c)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    es, B, nq, nkv, D = size[c["dtype"]], c["B"], c["nq"], c["nkv"], c["D"]
    table = 4 * sum(-(-n // c["page"]) for n in lens) + 4 * B
    if c["op"] == "append":
        return {"bytes": sum(new) * 2 * nkv * D * (size[c["src"]] + es) + table, "flops": 0}
    if c["op"] == "evict":
        # totals read, kept totals, indices and rows written, kept rows read
        kept = sum(min(n, c["budget"]) for n in lens) * nkv
        return {"bytes": sum(lens) * nkv * 4 + B * nkv * max(lens) * 4 + kept * (4 + 4 * D * es) + table, "flops": 0}
    rows = sum(new) if c["op"] == "prompt" else B
    if c["op"] == "decode":
        pairs = seen = sum(_seen(n, c) for n in lens)
    else:
        pairs = sum(_seen(p + 1, c) for n, m in zip(lens, new) for p in range(n - m, n))
        # positions that some new token sees: from the first token's window on, and the first few
        first = [max(0, n - m + 1 - c["window"]) if c["window"] else 0 for n, m in zip(lens, new)]
        seen = sum(n - f + min(c["sinks"], f) for n, f in zip(lens, first))
    moved = rows * nq * (2 * D * es + 4) + seen * nkv * 2 * D * es + table
    if c["mass"]:
        moved += 2 * 4 * B * nkv * max(lens)
    return {"bytes": moved, "flops": 4 * pairs * nq * D}


# ---- the definition, in 64 bits -----------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    dev = s["k_pages"].device
    lens, new = _lengths(c)
    P, G = c["page"], c["nq"] // c["nkv"]
    table = s["page_table"].tolist()

    def cached(pool, b, h):
        ids = torch.tensor(table[b][:-(-lens[b] // P)], device=dev)
        return pool[ids, h].reshape(-1, c["D"])[:lens[b]].double()

    if c["op"] == "append":
        got = {}
        for x in "kv":
            pool, rows = s[x + "_pages"].double(), s[x].double()
            r = 0
            for b in range(c["B"]):
                p = torch.arange(lens[b] - new[b], lens[b], device=dev)
                ids = torch.tensor(table[b], device=dev)[p // P]
                pool[ids, :, p % P] = rows[r:r + new[b]]
                r += new[b]
            got[x] = pool
        return got
    if c["op"] == "evict":
        got = {"k": s["k_pages"].double(), "v": s["v_pages"].double(), "kept": None, "lens": None,
               "mass": torch.zeros_like(s["mass"], dtype=torch.float64)}
        dst = s["dst_table"].tolist()
        for b in range(c["B"]):
            n, m = lens[b], min(lens[b], c["budget"])
            i = torch.arange(m, device=dev)
            to = torch.tensor(dst[b], device=dev)[i // P]
            for h in range(c["nkv"]):
                total = s["mass"][b, h, :n].double()
                score = total.clone()
                score[:c["sinks"]] = math.inf
                score[n - c["recent"]:] = math.inf
                # larger totals first, the lower position first among equal ones
                keep = torch.argsort(-score, stable=True)[:m].sort().values
                got["mass"][b, h, :m] = total[keep]
                for x in "kv":
                    got[x][to, h, i % P] = cached(s[x + "_pages"], b, h)[keep]
        return got
    rows = s["q"].shape[0]
    out = torch.zeros(rows, c["nq"], c["D"], dtype=torch.float64, device=dev)
    lse = torch.full((rows, c["nq"]), -math.inf, dtype=torch.float64, device=dev)
    mass = s["mass"].double() if c["mass"] else None
    r = 0
    for b in range(c["B"]):
        n, m = lens[b], new[b] if c["op"] == "prompt" else 1
        here = torch.arange(n - m, n, device=dev)[:, None]
        there = torch.arange(n, device=dev)[None, :]
        hidden = there > here
        if c["window"]:
            hidden = hidden | ((there <= here - c["window"]) & (there >= c["sinks"]))
        for h in range(c["nkv"]):
            k, v = cached(s["k_pages"], b, h), cached(s["v_pages"], b, h)
            for g in range(h * G, h * G + G):
                x = (s["q"][r:r + m, g].double() @ k.T) * s["scale"]
                x[hidden] = -math.inf
                z = torch.logsumexp(x, -1)
                p = torch.exp(x - z[:, None])
                out[r:r + m, g] = p @ v
                lse[r:r + m, g] = z
                if mass is not None:
                    mass[b, h, :n] += p.sum(0)
        r += m
    return {"out": out, "lse": lse, "mass": mass}
