"""Gemma 3 over paged caches: many sequences with prompts of their own lengths,
caches that grow by pages, local layers that keep a window and a few first
tokens, global layers trimmed by attention weight.

    python -m rich_triplet_b200.paged_model --seqs 4 --prompt 600 --steps 64 --budget 512

runs a synthetic model (4B widths, few layers) and prints what it did.  The
projections are QLinear layers over the same Q4_K weights as the decode engines
(Gemma3Block::forward_cached, src/transformer4.rs:1954-1964); attention and
caches are rich_triplet_b200.paged; norms, RoPE and the gate are torch
operations.  A step runs on the context's stream, after the work of the caller's
current stream, which waits for it.  Without eviction and with no first tokens
its logits are the engine's (CudaDecodeContext).
"""

import argparse
import time

import numpy as np
import torch

from . import paged
from .model import Config4, Gemma3Weights, MatBf16, Q4KMat, synth_gemma3, synth_tokens
from .ops import Context
from .paged import PagedKvCache
from .qlinear import QLinear


class PagedGemma3:
    """Decode and prompt steps of ``sequences`` sequences.  ``sinks``: first
    tokens that stay visible to the local layers.  ``budget`` > 0: the global
    layers' caches are trimmed to it when they exceed it by ``page_size``."""

    def __init__(self, weights: Gemma3Weights, sequences, max_len, page_size=32, dtype=torch.bfloat16, sinks=0,
                 budget=0, recent=64, ctx: Context = None):
        if budget and not (0 <= sinks and 0 <= recent and sinks + recent <= budget):
            raise ValueError(f"PagedGemma3: sinks {sinks} + recent {recent} must lie in 0..budget {budget}")
        cfg = self.cfg = weights.cfg
        self.ctx = ctx or Context(0)
        self.stream = torch.cuda.ExternalStream(self.ctx.stream_ptr)
        self.sinks, self.budget, self.recent, self.page_size, self.dtype = sinks, budget, recent, page_size, dtype
        self.max_len = max_len
        H, D, F = cfg.hidden_size, cfg.head_dim, cfg.intermediate_size
        nq, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        shapes = {"q": (nq * D, H), "k": (nkv * D, H), "v": (nkv * D, H), "o": (H, nq * D), "gate": (F, H), "up": (F, H),
                  "down": (H, F)}
        with torch.cuda.stream(self.stream):
            def vec(a):
                return 1.0 + torch.tensor(np.ascontiguousarray(a, dtype=np.float32)).cuda()

            self.proj = [{n: QLinear.from_q4k(self.ctx, Q4KMat(r, c, getattr(L, n)), r, c)
                          for n, (r, c) in shapes.items()} for L in weights.layers]
            self.norm = [{n: vec(getattr(L, n)) for n in ("attn_norm", "post_attn_norm", "pre_ffn_norm", "post_ffn_norm",
                                                          "q_norm", "k_norm")} for L in weights.layers]
            self.final_norm = vec(weights.final_norm)
            bits = torch.tensor(weights.embed.view(np.int16)).cuda()
            self.embed = bits.view(torch.bfloat16).view(cfg.vocab_size, H)
            self.head = QLinear.from_bf16(self.ctx, MatBf16(cfg.vocab_size, H, weights.embed))
            self.rope = {g: self._rope_table(g, max_len) for g in (False, True)}
            groups = [[i for i in range(cfg.num_hidden_layers) if cfg.is_global_layer(i) == g] for g in (False, True)]
            pages = sequences * (-(-max_len // page_size) + (-(-budget // page_size) if budget else 0))
            self.caches = [PagedKvCache(len(g), sequences, pages, page_size, nkv, D, max_len, dtype,
                                        totals=bool(i and budget)) if g else None for i, g in enumerate(groups)]
            self.place = {layer: (i, at) for i, g in enumerate(groups) for at, layer in enumerate(g)}
        self.position = [0] * sequences

    def _rope_table(self, is_global, n):
        """cos and sin [n, head_dim / 2] (apply_rope_at_offset, src/transformer4.rs:2742-2772)."""
        c = self.cfg
        theta, scale = (c.rope_theta_global, c.rope_freq_scale_global) if is_global else \
            (c.rope_theta_local, c.rope_freq_scale_local)
        f32 = np.float32
        inv = f32(1.0) / np.power(f32(theta), np.arange(0, c.head_dim, 2, dtype=f32) / f32(c.head_dim))
        angle = (np.arange(n, dtype=f32) * f32(scale))[:, None] * inv[None, :]
        return torch.tensor(np.cos(angle)).cuda(), torch.tensor(np.sin(angle)).cuda()

    def _rms(self, x, weight):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.cfg.rms_norm_eps) * weight

    def _linear(self, layer, x):
        x = x.contiguous()
        y = torch.empty((x.shape[0], layer.out_features), dtype=torch.float32, device=x.device)
        layer.forward_device(x.data_ptr(), x.shape[0], y.data_ptr())
        return y

    def step(self, tokens):
        """One step for every sequence: tokens[b] is a list of new token ids (one
        each: a decode step; else a prompt step).  Returns the logits of each
        sequence's last new token ([sequences, vocab] f32, on the device), for use
        on the caller's current stream."""
        caller = torch.cuda.current_stream(self.stream.device)
        self.stream.wait_stream(caller)
        with torch.cuda.stream(self.stream):
            logits = self._step(tokens)
        # the head's product may still run when the host gets here
        caller.wait_stream(self.stream)
        logits.record_stream(caller)
        return logits

    def sync(self):
        """Waits for the steps so far; raises RtError if one of their kernels
        reported that a bounded wait gave up (as the next step would)."""
        self.stream.synchronize()
        self.ctx.sync()
        paged.context(self.stream.device).check()

    def _step(self, tokens):
        cfg, D = self.cfg, self.cfg.head_dim
        nq, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        counts = [len(t) for t in tokens]
        if len(tokens) != len(self.position) or min(counts) < 1:
            raise ValueError(f"PagedGemma3.step: at least one token for each of {len(self.position)} sequences")
        flat = np.concatenate(tokens).astype(np.int64)
        if flat.min() < 0 or flat.max() >= cfg.vocab_size:
            raise ValueError(f"PagedGemma3.step: tokens from {flat.min()} to {flat.max()}, vocabulary of {cfg.vocab_size}")
        if max(p + c for p, c in zip(self.position, counts)) > self.max_len:
            raise ValueError(f"PagedGemma3.step: {counts} tokens after {self.position} pass position {self.max_len}")
        decode = max(counts) == 1
        starts = np.concatenate([[0], np.cumsum(counts)])
        q_start = None if decode else torch.tensor(starts, dtype=torch.int32).cuda()
        ids = torch.tensor(flat).cuda()
        at = torch.tensor(np.concatenate([np.arange(p, p + c) for p, c in zip(self.position, counts)])).cuda()
        # those copies waited for the last step: its kernels' reports are there
        paged.context(self.stream.device).check()
        for c in self.caches:
            if c is not None:
                c.extend(counts)
        x = self.embed[ids].float() * float(np.sqrt(np.float32(cfg.hidden_size)))
        scale = 1.0 / float(np.sqrt(cfg.query_pre_attn_scalar))
        for i, (proj, norm) in enumerate(zip(self.proj, self.norm)):
            is_global = cfg.is_global_layer(i)
            group, layer = self.place[i]
            cache = self.caches[group]
            cos, sin = (t[at][:, None, :] for t in self.rope[is_global])

            def head(y, heads, weight):
                y = self._rms(y.view(-1, heads, D), weight)
                a, b = y[..., :D // 2], y[..., D // 2:]
                return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

            h = self._rms(x, norm["attn_norm"])
            q = head(self._linear(proj["q"], h), nq, norm["q_norm"]).to(self.dtype)
            k = head(self._linear(proj["k"], h), nkv, norm["k_norm"])
            v = self._linear(proj["v"], h).view(-1, nkv, D)
            cache.append(layer, k, v, q_start)
            see = dict(scale=scale) if is_global else dict(scale=scale, window=cfg.sliding_window or 0, sinks=self.sinks)
            o, _ = cache.decode(layer, q, **see) if decode else cache.prompt(layer, q, q_start, max(counts), **see)
            x = x + self._rms(self._linear(proj["o"], o.float().view(-1, nq * D)), norm["post_attn_norm"])
            h = self._rms(x, norm["pre_ffn_norm"])
            h = torch.nn.functional.gelu(self._linear(proj["gate"], h), approximate="tanh") * self._linear(proj["up"], h)
            x = x + self._rms(self._linear(proj["down"], h), norm["post_ffn_norm"])
        for b, c in enumerate(counts):
            self.position[b] += c
        if cfg.sliding_window and self.caches[0] is not None:
            self.caches[0].drop(cfg.sliding_window, self.sinks)
        trim = self.caches[1]
        if self.budget and trim is not None and max(trim.lens) >= self.budget + self.page_size:
            trim.evict(self.budget, self.sinks, self.recent)
        last = torch.tensor(starts[1:] - 1).cuda()
        return self._linear(self.head, self._rms(x[last], self.final_norm))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--layers", type=int, default=6)
    ap.add_argument("--prompt", type=int, default=600, help="longest prompt; the others are shorter")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=512, help="positions the global layers keep (0: all)")
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--seed", type=int, default=1234)
    a = ap.parse_args(argv)

    cfg = Config4.gemma3_4b(vocab_size=262144).with_layers(a.layers)
    model = PagedGemma3(synth_gemma3(cfg, seed=a.seed), a.seqs, a.prompt + a.steps + 1, sinks=a.sinks, budget=a.budget,
                        recent=max(0, min(64, a.budget - a.sinks)))
    prompts = [list(synth_tokens(a.seed, b, max(1, a.prompt * (b + 1) // a.seqs), cfg.vocab_size)) for b in range(a.seqs)]
    out = [[] for _ in prompts]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    logits = model.step(prompts)
    model.sync()
    t1 = time.perf_counter()
    for _ in range(a.steps):
        tok = logits.argmax(-1).tolist()
        for o, t in zip(out, tok):
            o.append(t)
        logits = model.step([[t] for t in tok])
    model.sync()
    t2 = time.perf_counter()
    kept = "no global layer" if model.caches[1] is None else f"global layers hold {model.caches[1].lens}"
    print(f"paged_model: {a.seqs} sequences, {a.layers} layers, prompts {[len(p) for p in prompts]}: prompt step "
          f"{(t1 - t0) * 1e3:.1f} ms, {a.steps} decode steps {(t2 - t1) / a.steps * 1e3:.2f} ms each; positions "
          f"{model.position}, {kept}; first tokens {[o[:4] for o in out]}", flush=True)


if __name__ == "__main__":
    main()
