"""Gemma 3 over paged caches (rich_triplet_b200.paged_model) against the decode
engine, and its caches' bookkeeping.

Tolerances: the projections of a prompt run on fp16 tensor cores (3e-4 relative
L2 each), as the many-sequence engine's, so logits get the same bar, 2e-3, with
an f32 cache.  A 16-bit cache rounds every key, value, query and attention
output once, 2^-12 (f16) or 2^-9 (bf16) of their size in the root mean square
at each of 6 layers' attentions: 5e-3 and 2e-2 bound a few of those.
"""

import numpy as np
import pytest
import torch

from rich_triplet_b200.decode import CudaDecodeContext
from rich_triplet_b200.model import Config4, synth_gemma3, synth_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    cfg = Config4.tiny()
    return cfg, synth_gemma3(cfg, seed=1234)


def rel(a, b):
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b.astype(np.float64)))


@pytest.mark.parametrize("dtype,bar", [(torch.float32, 2e-3), (torch.float16, 5e-3), (torch.bfloat16, 2e-2)])
def test_logits_are_the_engines(tiny, dtype, bar):
    from rich_triplet_b200.paged_model import PagedGemma3

    cfg, w = tiny
    prompts = [list(synth_tokens(5, b, n, cfg.vocab_size)) for b, n in enumerate((37, 1, 20))]
    follow = [list(synth_tokens(6, b, 6, cfg.vocab_size)) for b in range(3)]
    model = PagedGemma3(w, 3, 64, page_size=8, dtype=dtype)
    got = [model.step(prompts).cpu().numpy()]
    for i in range(4):
        got.append(model.step([[f[i]] for f in follow]).cpu().numpy())
    got.append(model.step([f[4:6] for f in follow]).cpu().numpy())  # two tokens at once on a filled cache
    for b in range(3):
        dec = CudaDecodeContext(w, 64)
        want = [dec.prefill(prompts[b])]
        n = len(prompts[b])
        for i in range(6):
            want.append(dec.decode_step(follow[b][i], n + i))
        dec.close()
        want = want[:5] + [want[6]]
        for i, (g, x) in enumerate(zip(got, want)):
            assert rel(g[b], x) < bar, (b, i)
    model.ctx.sync()


def test_trimmed_caches(tiny):
    """Local layers keep their window's pages and the first ones', global layers
    their budget; a budget that nothing exceeds changes nothing."""
    from rich_triplet_b200.paged_model import PagedGemma3

    cfg, w = tiny
    prompts = [list(synth_tokens(7, b, n, cfg.vocab_size)) for b, n in enumerate((60, 9))]
    plain = PagedGemma3(w, 2, 128, page_size=8, dtype=torch.float16, sinks=2)
    wide = PagedGemma3(w, 2, 128, page_size=8, dtype=torch.float16, sinks=2, budget=100, recent=8)
    tight = PagedGemma3(w, 2, 128, page_size=8, dtype=torch.float16, sinks=2, budget=24, recent=8)
    models = (plain, wide, tight)
    logits = [m.step(prompts) for m in models]
    for i in range(20):
        tok = [[3 + i], [50 + i]]
        logits = [m.step(tok) for m in models]
    torch.cuda.synchronize()
    assert torch.equal(logits[0], logits[1])
    assert torch.isfinite(logits[2]).all()
    assert plain.position == [80, 29]
    assert plain.caches[1].lens == [80, 29] and max(tight.caches[1].lens) < 24 + 8
    local = plain.caches[0]
    for b, n in enumerate(plain.position):
        held = {p for p in range(local.page_table.shape[1]) if int(local.page_table[b, p]) >= 0}
        first = (n + 1 - cfg.sliding_window) // 8
        assert held == {0} | set(range(first, -(-n // 8)))
    for m in models:
        for c in m.caches:
            used = [int(p) for p in c.page_table.flatten() if p >= 0]
            assert len(set(used)) == len(used) and len(used) + c.pool.free_pages == c.pool.num_pages
        m.ctx.sync()


def test_pool_and_cache_refuse():
    from rich_triplet_b200.paged import PagedKvCache, PagePool

    p = PagePool(3)
    assert sorted(p.take(3)) == [0, 1, 2]
    with pytest.raises(ValueError, match="1 pages wanted"):
        p.take(1)
    c = PagedKvCache(1, 2, 4, 8, 1, 64, 32)
    with pytest.raises(ValueError, match="extend"):
        c.extend([33, 1])
    with pytest.raises(ValueError, match="pages wanted"):
        c.extend([32, 32])
    with pytest.raises(ValueError, match="without totals"):
        c.evict(8)
