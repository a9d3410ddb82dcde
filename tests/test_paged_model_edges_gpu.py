"""Edges of Gemma 3 over paged caches (rich_triplet_b200.paged_model): streams,
refused steps, errors reported by kernels."""

import pytest
import torch

from rich_triplet_b200.model import Config4, synth_gemma3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    cfg = Config4.tiny()
    return cfg, synth_gemma3(cfg, seed=1234)


def test_logits_are_complete_on_the_callers_stream(tiny):
    """The head's product is held back on the model's stream; the caller reads the
    logits on its own, without a synchronisation, and writes into them."""
    from rich_triplet_b200.paged_model import PagedGemma3

    cfg, w = tiny
    held = torch.randn(4096, 4096, device="cuda") * 1e-3
    models = [PagedGemma3(w, 2, 32, page_size=8, dtype=torch.float16) for _ in range(2)]
    linear = models[1]._linear

    def late(layer, x):
        if layer is models[1].head:
            y = held
            for _ in range(30):
                y = y @ held
            x = x + y.sum() * 0
        return linear(layer, x)

    models[1]._linear = late
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            want = models[0].step([[3, 4, 5], [6]])
            torch.cuda.synchronize()
            got = models[1].step([[3, 4, 5], [6]])
            seen = got.clone()
            got.zero_()
        torch.cuda.synchronize()
        assert torch.equal(seen, want) and not torch.equal(seen, got)


def test_tokens_and_positions_out_of_range_are_refused(tiny):
    """Both index device tensors: refused on the host, and nothing has changed."""
    from rich_triplet_b200.paged_model import PagedGemma3

    cfg, w = tiny
    model = PagedGemma3(w, 2, 16, page_size=8, dtype=torch.float16)
    other = PagedGemma3(w, 2, 16, page_size=8, dtype=torch.float16)
    for m in (model, other):
        m.step([[1, 2, 3], [4]])
    for bad in ([[cfg.vocab_size], [0]], [[0], [-1]], [[0], [5, 10 ** 12]]):
        with pytest.raises(ValueError, match="vocabulary"):
            model.step(bad)
    with pytest.raises(ValueError, match="pass position 16"):
        model.step([[1] * 14, [1]])
    with pytest.raises(ValueError, match="at least one token"):
        model.step([[1], []])
    assert model.position == [3, 1]
    tok = [[5], [6]]
    assert torch.equal(model.step(tok), other.step(tok))
    model.step([[1] * 12, [1]])  # up to the last position
    assert model.position == [16, 3]


def test_a_wait_that_gave_up_is_reported(tiny, monkeypatch):
    """The attention kernels report to the paged operators' context: the next step
    and sync() ask it (here a stand-in for its error word)."""
    from rich_triplet_b200 import paged
    from rich_triplet_b200._lib import RT_E_TIMEOUT, RtError
    from rich_triplet_b200.paged_model import PagedGemma3

    cfg, w = tiny
    model = PagedGemma3(w, 1, 16, page_size=8, dtype=torch.float16)
    model.step([[1, 2, 3]])
    model.sync()
    asked = []

    def gave_up(self):
        asked.append(self)
        raise RtError(RT_E_TIMEOUT, "a kernel reported error word 1 (bounded wait gave up)")

    with monkeypatch.context() as m:
        m.setattr(paged._DeviceContext, "check", gave_up)
        with pytest.raises(RtError, match="gave up"):
            model.step([[4]])
        with pytest.raises(RtError, match="gave up"):
            model.sync()
        with pytest.raises(RtError, match="gave up"):
            paged.context("cuda").sync()
    assert asked == [paged.context("cuda")] * 3
    assert model.position == [3] and model.caches[0].lens == [3]  # refused before the step
    model.step([[4]])
    model.sync()
