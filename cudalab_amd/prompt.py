"""Prompt driver: prompts of unequal length through every layer of a Llama-shaped
model (7B or 70B) on one GPU, INT8 weights and a quantized paged cache, and then
trees of drafted tokens checked against it.  No counterpart in the reference (it
excludes model integration: README.md:34-35).

The weights are the decode driver's (`decode.DecodeModel`, INT8), so a model keeps
one copy for prompts and for single tokens, and the data flow between projections is
its own: norms of the layer, residual adds and the SwiGLU product are not modelled,
the down projection takes up's output.  Per call

  place     pages, positions and slots of the packed tokens (once for all layers)
and in every layer
  quantize_tokens   the layer's input, once for q, k and v
  forward           q, k, v
  qk_norm_rope      each head of q and k, and their rotation, in place
  append_rows       k and v into the layer's cache
  prompt            attention of the prompts over their own tokens, or
  forward(tree=)    of the drafts over the cache and their ancestors
  quantize_tokens, forward   o; gate and up; down

`accept` closes the caches up behind the drafts that were kept.

Usage: python -m cudalab_amd.prompt [--model 7b|70b] [--layers N] [--batch 4]
       [--tokens 2048] [--drafts 16] [--cache-bits 8|4] [--steps 5] [--warmup 2]
"""
from __future__ import annotations

import argparse
import json
import sys

import torch

from .build import build
from .decode import HEAD_DIM, MODELS, PAGE, ROPE_BASE, DecodeModel, time_steps
from .kvcache import KVCache


class PromptModel:
    """Weights, caches with room for `room` tokens of each of `batch` sequences, and
    the sequences' lengths, all on `device`."""

    def __init__(self, batch: int, room: int, layers: int, seed: int = 7,
                 device: str = "cuda", hidden: int = 4096, inter: int = 11008,
                 kv: int | None = None, cache_bits: int = 8):
        self.weights = DecodeModel("qgemv", layers, seed, device, hidden, inter, kv)
        self.gemm, self.att = build("qgemm"), build("attention")
        self.batch, self.room, self.device = batch, room, device
        self.heads = self.weights.kv // HEAD_DIM
        cols = -(-room // PAGE)
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def norm():
            return 1 + torch.randn(HEAD_DIM, generator=g, device=device).half() / 8

        self.norms = [(norm(), norm()) for _ in range(layers)]
        self.caches = [KVCache.empty(batch * cols, self.heads, HEAD_DIM, PAGE, cache_bits, device)
                       for _ in range(layers)]
        self.free = torch.randperm(batch * cols, generator=g, device=device).int()
        self.table = torch.full((batch, cols), -1, dtype=torch.int32, device=device)
        angle = (torch.arange(room, device=device)[:, None] * ROPE_BASE **
                 (-torch.arange(0, HEAD_DIM, 2, device=device) / HEAD_DIM))
        self.cos, self.sin = angle.cos(), angle.sin()
        self.clear()

    def clear(self) -> None:
        """No tokens, all pages free."""
        self.lengths = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        self.taken = torch.zeros(1, dtype=torch.int32, device=self.device)
        # pages of each sequence: drafts that were given up leave theirs to the next
        self.held = torch.zeros_like(self.lengths)

    def _product(self, name: str, layer: int, quantized) -> torch.Tensor:
        return self.gemm.forward(*quantized, *self.weights.layers[layer].w[name])

    def _layers(self, x, positions, slots, attend):
        """All layers over packed x (rows, hidden); (the last layer's output, the
        keys and values that went into each cache)."""
        kept = []
        for i, (cache, norm) in enumerate(zip(self.caches, self.norms)):
            inp = self.gemm.quantize_tokens(x)
            q, k, v = (self._product(n, i, inp).view(x.size(0), -1, HEAD_DIM)
                       for n in ("q", "k", "v"))
            self.att.qk_norm_rope_into(q, k, q, k, *norm, self.cos, self.sin, positions)
            self.att.append_rows(cache, k, v, slots)
            kept.append((k, v))
            o = self._product("o", i, self.gemm.quantize_tokens(
                attend(cache, q, k, v).view(x.size(0), -1)))
            inp = self.gemm.quantize_tokens(o)
            self._product("gate", i, inp)
            up = self._product("up", i, inp)
            x = self._product("down", i, self.gemm.quantize_tokens(up))
        return x, kept

    def prompt(self, x: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
        """The first counts[b] tokens of each sequence (0 for one that has some: these
        would see nothing that is in the caches), packed in x (rows, hidden) fp16;
        rows behind the last sequence are carried along and belong to none."""
        p = self.att.place(self.table, self.lengths, counts, x.size(0), PAGE, self.free,
                           self.taken, held=self.held)
        self.lengths, self.taken, self.held = p.lengths, p.taken, p.held
        return self._layers(x, p.positions, p.slots, lambda cache, q, k, v:
                            self.att.prompt(q, k, v, p.offsets))[0]

    def check(self, x: torch.Tensor, tree: torch.Tensor, depth: torch.Tensor) -> torch.Tensor:
        """T drafted tokens behind each sequence, x (batch, T, hidden): token t is at
        depth[b, t] (int32, 0 behind the context) and sees the context and the tokens
        of its bits (tree int64 (batch, T, ceil(T / 64)))."""
        rows, T = x.size(0) * x.size(1), x.size(1)
        counts = torch.full_like(self.lengths, T)
        p = self.att.place(self.table, self.lengths, counts, rows, PAGE, self.free, self.taken,
                           held=self.held)
        self.taken, self.held = p.taken, p.held
        positions = (self.lengths[:, None] + depth).view(-1)

        def attend(cache, q, k, v):
            return self.att.forward(q.view(self.batch, T, -1, HEAD_DIM), cache, self.table,
                                    p.lengths, tree=tree)

        y, self.drafts = self._layers(x.view(rows, -1), positions, p.slots, attend)
        return y.view(x.shape)

    def accept(self, keep: torch.Tensor) -> None:
        """Of the last check's tokens those with keep[b, t], in their order, become
        the sequences' next ones, as many as `room` has places for."""
        rank = keep.long().cumsum(1) - 1
        at = self.lengths.long()[:, None] + rank
        keep = keep & (at < self.room)
        page = self.table.long().gather(1, (at // PAGE).clamp(0, self.table.size(1) - 1))
        slots = torch.where(keep, page * PAGE + at % PAGE, -1).view(-1)
        for cache, (k, v) in zip(self.caches, self.drafts):
            self.att.append_rows(cache, k, v, slots)
        self.lengths = self.lengths + keep.sum(1, dtype=torch.int32)


def chains(batch: int, drafts: int, width: int, device: str = "cuda"):
    """(tree, depth) of `width` chains side by side: token t continues token
    t - width."""
    seen, depth = [], []
    for t in range(drafts):
        seen.append((seen[t - width] if t >= width else 0) | 1 << t)
        depth.append(t // width)
    words = [[(m >> 64 * w & 2 ** 64 - 1) - (2 ** 64 if m >> 64 * w & 2 ** 63 else 0)
              for w in range((drafts + 63) // 64)] for m in seen]
    tree = torch.tensor(words, dtype=torch.int64, device=device).expand(batch, -1, -1)
    return (tree.contiguous(),
            torch.tensor(depth, dtype=torch.int32, device=device).expand(batch, -1).contiguous())


def lengths_of(batch: int, tokens: int) -> list[int]:
    """Prompt lengths from `tokens` down to about half of it."""
    return [tokens - (b * tokens // (2 * batch)) for b in range(batch)]


def run(model: str = "7b", layers: int | None = None, batch: int = 4, tokens: int = 2048,
        drafts: int = 16, cache_bits: int = 8, steps: int = 5, warmup: int = 2) -> dict:
    cfg = MODELS[model]
    layers = cfg["layers"] if layers is None else layers
    m = PromptModel(batch, tokens + drafts, layers, hidden=cfg["hidden"], inter=cfg["inter"],
                    kv=cfg["kv"], cache_bits=cache_bits)
    lens = lengths_of(batch, tokens)
    counts = torch.tensor(lens, dtype=torch.int32, device="cuda")
    x = torch.randn(sum(lens), cfg["hidden"], device="cuda").half()
    weights = sum(n * k for _, n, k in m.weights.proj)

    def prompt():
        m.clear()
        m.prompt(x, counts)

    res = {"model": model, "layers": layers, "batch": batch, "prompt_lengths": lens,
           "cache_bits": cache_bits,
           "note": "INT8 weights and activations; norms, residuals and SwiGLU between the "
                   "projections are not modelled"}
    us = time_steps(prompt, steps, warmup)
    res["prompt"] = {"us_per_step": round(us, 1), "us_per_layer": round(us / layers, 2),
                     "tokens_per_s": round(sum(lens) / us * 1e6),
                     "int8_TOPS": round(2 * sum(lens) * weights * layers / us / 1e6, 1)}
    if drafts:
        tree, depth = chains(batch, drafts, 4)
        y = torch.randn(batch, drafts, cfg["hidden"], device="cuda").half()
        us = time_steps(lambda: m.check(y, tree, depth), steps, warmup)
        res["check"] = {"drafts": drafts, "us_per_step": round(us, 1),
                        "us_per_layer": round(us / layers, 2),
                        "GBps_of_weights": round(weights * layers / us / 1e3, 1)}
    return res


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--model", choices=tuple(MODELS), default="7b")
    ap.add_argument("--layers", type=int, default=None,
                    help="layers (default: the model's, 32 for 7b, 80 for 70b)")
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=2048,
                    help="tokens of the longest prompt; the others are shorter")
    ap.add_argument("--drafts", type=int, default=16,
                    help="drafted tokens a sequence, four chains side by side (0: none)")
    ap.add_argument("--cache-bits", type=int, choices=(8, 4), default=8)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=2)
    a = ap.parse_args(argv)
    from . import _capi
    print(f"library: {_capi.version()}", flush=True)   # the build that ran
    if min(a.batch, a.tokens, a.steps) < 1 or a.drafts < 0 or a.warmup < 0 \
            or (a.layers is not None and a.layers < 1):
        print("prompt: --batch, --tokens, --steps and --layers must be >= 1, --drafts and "
              "--warmup >= 0", file=sys.stderr)
        return 2
    if not torch.cuda.is_available():
        print("prompt: no GPU visible", file=sys.stderr)
        return 1
    print(json.dumps(run(a.model, a.layers, a.batch, a.tokens, a.drafts, a.cache_bits, a.steps,
                         a.warmup)), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
