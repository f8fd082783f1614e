"""One decoded token of each of a batch of sequences through one layer: the
attention half (head norms, rotation, paged cache, attention), the router and
the routed experts, as a serving loop would call them.

    python examples/decode_layer.py            # a few steps on synthetic weights, with timings

The projections are plain torch products; everything else is libsabah_rt.so.
"""
from __future__ import annotations

import os
import sys
import time
from dataclasses import dataclass

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from sabah_moe_accelerator_b200 import ops, rt

IQ3_S = rt.QTYPE["IQ3_S"]


@dataclass
class Layer:
    """Weights of one layer. Projections [in, out] float32; experts as quantised banks."""
    heads: int
    kv_heads: int
    head_dim: int
    experts: int
    used: int
    ff: int
    qkv: torch.Tensor        # [d_model, (heads + 2 kv_heads) head_dim]
    out: torch.Tensor        # [heads head_dim, d_model]
    q_weight: torch.Tensor   # [head_dim]
    k_weight: torch.Tensor
    router: torch.Tensor     # [d_model, experts]
    gate: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor


class PagedCache:
    """Pages of one layer's keys and values, and the sequences' block table.
    Sequence b owns pages b * width .. (b + 1) * width - 1 here; a server hands
    pages out as sequences grow."""

    def __init__(self, seqs: int, max_len: int, kv_heads: int, head_dim: int, page: int = 16,
                 dtype: torch.dtype = torch.bfloat16):
        self.page, width = page, -(-max_len // page)
        shape = (seqs * width, page, kv_heads, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
        self.table = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def grow(self):
        """Room for one more token per sequence: (positions int32, slots int64) of it."""
        pos = self.lens.clone()
        self.lens += 1
        page = self.table.gather(1, (pos // self.page).long()[:, None])[:, 0]
        return pos, page.long() * self.page + pos % self.page


def rms(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def decode_layer(x: torch.Tensor, layer: Layer, cache: PagedCache, table: torch.Tensor, positions: torch.Tensor,
                 slots: torch.Tensor):
    """x [sequences, d_model] float32 -> (the next x, router ids, weights, logits)."""
    B, d_model = x.shape
    H, K, D = layer.heads, layer.kv_heads, layer.head_dim
    qkv = (rms(x) @ layer.qkv).view(B, H + 2 * K, D)
    q = ops.qk_norm_rope(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], layer.q_weight, layer.k_weight, table, positions,
                         cache=(cache.k, cache.v, slots))
    a = ops.attend_paged(q, cache.k, cache.v, cache.table, cache.lens)
    x = x + a.view(B, H * D) @ layer.out
    h = rms(x)
    logits = h @ layer.router
    ids, w = ops.route_topk(logits, layer.used)
    y = ops.moe_block_ids(layer.gate, layer.up, layer.down, ids, w, h, d_model, layer.ff, layer.experts, IQ3_S, IQ3_S,
                          IQ3_S)
    return x + y, ids, w, logits


def synthetic_layer(d_model=2048, ff=768, heads=16, kv_heads=2, head_dim=128, experts=64, used=10, seed=0) -> Layer:
    g = torch.Generator("cuda").manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale

    def bank(rows, k, n):
        return ops.synth_rows(experts * rows, k, IQ3_S, seed=100 * seed + n)

    return Layer(heads, kv_heads, head_dim, experts, used, ff,
                 qkv=rnd(d_model, (heads + 2 * kv_heads) * head_dim, scale=d_model ** -0.5),
                 out=rnd(heads * head_dim, d_model, scale=(heads * head_dim) ** -0.5),
                 q_weight=1 + rnd(head_dim, scale=0.1), k_weight=1 + rnd(head_dim, scale=0.1),
                 router=rnd(d_model, experts, scale=d_model ** -0.5),
                 gate=bank(ff, d_model, 1), up=bank(ff, d_model, 2), down=bank(d_model, ff, 3))


def main(seqs: int = 4, steps: int = 64) -> None:
    ops.init(0)
    layer = synthetic_layer()
    cache = PagedCache(seqs, steps + 8, layer.kv_heads, layer.head_dim)
    table = ops.rope_table(steps + 8, layer.head_dim)
    x = torch.randn(seqs, 2048, device="cuda")
    for step in range(steps + 8):
        if step == 8:
            torch.cuda.synchronize()
            t = time.perf_counter()
        positions, slots = cache.grow()
        y, ids, w, _ = decode_layer(x, layer, cache, table, positions, slots)
        x = rms(y)   # stands in for the next token's embedding
    torch.cuda.synchronize()
    print("%d sequences, %d steps of one layer: %.1f us a step; experts of the last token: %s"
          % (seqs, steps, (time.perf_counter() - t) / steps * 1e6, ids[0].tolist()))


if __name__ == "__main__":
    main()
