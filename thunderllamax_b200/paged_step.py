"""One decoder layer of a paged serving step, and a small serving loop around it.

A step takes the new tokens of a batch of requests, prompt chunks and single tokens
alike: the plan gives every request the pages it needs (once a step), then per layer

    append k, v -> attention over the pages (* sigmoid(gate)) -> o-projection (Q6_K)
    -> residual add + RMS norm -> int8 tokens -> W4A8 gate/up + SiLU -> down (Q6_K)

all on the device and stream-ordered.  The projections in front (q, k, v, gate with
their norms and rotary) are the caller's; Plan.positions holds every token's position.

    python -m thunderllamax_b200.paged_step        # a few requests from admission to release
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops, paged, prefill


@dataclass(frozen=True)
class LayerShape:
    heads: int = 24
    kv_heads: int = 4
    head_dim: int = 256
    dim: int = 5120
    ffn: int = 17408


class PagedLayer:
    """The layer behind the projections for up to `tokens` new tokens a step, with its own
    pages (the block tables are shared by all layers).  weights: tiled o, down (Q6_K), gate,
    up (IQ3_XXS) and the fp32 norm weight; synthetic ones if not given."""

    def __init__(self, tokens: int, pages: int, page_size: int, shape: LayerShape = LayerShape(), cache="int8",
                 weights: dict = None, seed: int = 0):
        from .verify import synth_tiled

        ops.require_device()
        self.shape = s = shape
        self.tokens = int(tokens)
        wide = s.heads * s.head_dim
        self.w = weights if weights is not None else {
            "o": synth_tiled("q6_k", s.dim, wide, seed + 1), "gate": synth_tiled("iq3_xxs", s.ffn, s.dim, seed + 2),
            "up": synth_tiled("iq3_xxs", s.ffn, s.dim, seed + 3), "down": synth_tiled("q6_k", s.dim, s.ffn, seed + 4),
            "norm": torch.ones(s.dim, dtype=torch.float32, device="cuda"),
        }
        self.cache = paged.PagedCache.empty(pages, page_size, s.kv_heads, s.head_dim, cache)
        self.attention = paged.PagedAttention(s.heads, s.kv_heads, s.head_dim)
        self.ws_o = prefill.PrefillWorkspace(self.tokens, wide)
        self.ws_ffn = prefill.PrefillWorkspace(self.tokens, s.dim)
        self.ws_down = prefill.PrefillWorkspace(self.tokens, s.ffn)
        self.lut = prefill.lut8()

    def __call__(self, plan: paged.Plan, table: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 residual: torch.Tensor, gate: torch.Tensor = None, max_new: int = None):
        """q, gate [tokens][heads][head_dim], k, v [tokens][kv_heads][head_dim] fp16 -> the
        FFN's output y [tokens][dim] fp32; residual [tokens][dim] fp32 is updated in place with
        the attention's output (y is the next layer's norm's to add)."""
        s, n = self.shape, q.shape[0]
        if n > self.tokens:
            raise ops.TLXError(f"{n} rows for a layer of {self.tokens}")
        self.cache.append(k, v, plan.slots)
        ao = self.attention(self.cache, table, plan.q_start, plan.kv_len, q, gate=gate, max_new=max_new)
        o = prefill.gemm("q6_k", self.w["o"], ao.view(n, -1), s.dim, self.ws_o)
        _, xq, sx = prefill.add_rms_norm_q8(o, residual, self.w["norm"], out=residual)
        act = prefill.w4a8_gate_up(self.w["gate"], self.w["up"], xq, sx, s.ffn, self.ws_ffn, lut=self.lut)
        return prefill.gemm("q6_k", self.w["down"], act, s.dim, self.ws_down)

    def errors(self) -> int:
        """The error bits of the layer's bounded waits; synchronous."""
        return self.attention.error() | self.ws_o.error() | self.ws_ffn.error() | self.ws_down.error()


def serve(layer: PagedLayer, prompts, new_tokens: int, chunk: int, pages: int, page_size: int, seed: int = 0):
    """Requests with prompts of the given lengths, from admission to release: prompts in
    chunks of at most `chunk` tokens beside the single tokens of the requests that already
    generate.  Rows are random (no projections here).  Returns (steps, tokens)."""
    s, r = layer.shape, len(prompts)
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(-(-(p + new_tokens) // page_size) for p in prompts)
    table = paged.PageTable(r, width, pages, page_size)
    done, steps, tokens = [0] * r, 0, 0
    end = [p + new_tokens for p in prompts]
    while any(d < e for d, e in zip(done, end)):
        new = [min(chunk, p - d) if d < p else min(1, e - d) for d, p, e in zip(done, prompts, end)]
        n = sum(new)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        # a finished request is planned empty: with its cached length it would take its pages again
        cached = [d if d < e else 0 for d, e in zip(done, end)]
        plan = table.plan(i32(cached), i32(new), paged.Plan(r, n))
        rows = lambda h: torch.randn((n, h, s.head_dim), generator=g, device="cuda").half()
        residual = torch.randn((n, s.dim), generator=g, device="cuda")
        layer(plan, table.table, rows(s.heads), rows(s.kv_heads), rows(s.kv_heads), residual, gate=rows(s.heads),
              max_new=max(new))
        if int(plan.status.max()):
            raise ops.TLXError(f"the pool ran out of pages: {plan.status.tolist()}")
        done = [d + x for d, x in zip(done, new)]
        finished = [int(d >= e) for d, e in zip(done, end)]
        table.release(i32(finished))
        steps, tokens = steps + 1, tokens + n
    if layer.errors() or int(table.n_free) != pages:
        raise ops.TLXError("the serving loop left an error or a page behind")
    return steps, tokens


def main():
    prompts, new_tokens, chunk, page_size = [1000, 37, 513, 1, 260], 20, 256, 64
    pages = sum(-(-(p + new_tokens) // page_size) for p in prompts)
    layer = PagedLayer(tokens=chunk * len(prompts), pages=pages, page_size=page_size)
    steps, tokens = serve(layer, prompts, new_tokens, chunk, pages, page_size)
    print(f"served {len(prompts)} requests: {tokens} tokens in {steps} steps, all pages returned")


if __name__ == "__main__":
    main()
