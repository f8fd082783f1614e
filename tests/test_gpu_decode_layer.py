"""The operators around the experts together, as examples/decode_layer.py calls
them: steps of one layer against the same chain in 64 bits."""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest
import torch

import attn_oracle as o
from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_steps_of_a_layer_match_the_chain_in_64_bits(gpu_rt, orc):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_layer as ex
    from sabah_moe_accelerator_b200 import ops, rt
    B, steps, d_model, ff = 3, 21, 256, 256
    layer = ex.synthetic_layer(d_model, ff, heads=8, kv_heads=2, head_dim=64, experts=16, used=4, seed=3)
    cache = ex.PagedCache(B, steps, 2, 64, page=16, dtype=torch.float16)
    table = ops.rope_table(steps, 64)
    g = torch.Generator("cuda").manual_seed(1)
    W = {n: getattr(layer, n).cpu().double() for n in ("qkv", "out", "router")}
    banks = [getattr(layer, n).cpu().numpy().reshape(16, -1) for n in ("gate", "up", "down")]
    rms = lambda x: x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    for step in range(steps):
        x = torch.randn(B, d_model, device="cuda", generator=g)
        if step == 5:   # sequences of different lengths: the first restarts
            cache.lens[0] = 0
        positions, slots = cache.grow()
        y, ids, w, logits = ex.decode_layer(x, layer, cache, table, positions, slots)
        # the chain, from the same x; the cache of earlier tokens as the device holds it
        xd = x.cpu().double()
        qkv = (rms(xd) @ W["qkv"]).view(B, 12, 64)
        q = o.norm_rope(qkv[:, :8], layer.q_weight, table, positions, "halves", None, 1e-6)
        k = o.norm_rope(qkv[:, 8:10], layer.k_weight, table, positions, "halves", None, 1e-6)
        flat_k, flat_v = cache.k.flatten(0, 1)[slots].cpu(), cache.v.flatten(0, 1)[slots].cpu()
        assert o.rel_l2(flat_k, k) <= 2.0 ** -11 + 1e-4 and o.rel_l2(flat_v, qkv[:, 10:]) <= 2.0 ** -11 + 1e-4
        a, _ = o.attend(q, cache.k, cache.v, cache.table, cache.lens)
        xd = xd + a.view(B, -1) @ W["out"]
        h = rms(xd)
        # four fp32 products of 256 to 512 terms in a row: 1e-4 leaves a factor of ten and more
        assert o.rel_l2(logits, h @ W["router"]) <= 1e-4
        want_ids, want_w = o.route(logits, 4, True)
        assert torch.equal(ids.cpu().long(), want_ids) and o.rel_l2(w, want_w) <= 2e-6
        moe = [orc.moe_block_f64(*banks, ids[b].cpu().numpy(), w[b].cpu().numpy(), h[b].numpy().astype(np.float32),
                                 d_model, ff, 21, 21, 21) for b in range(B)]
        assert o.rel_l2(y, xd + torch.from_numpy(np.stack(moe))) <= 1e-4
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0


def test_the_example_runs(gpu_rt, capsys):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_layer as ex
    ex.main(seqs=2, steps=4)
    assert "us a step" in capsys.readouterr().out
