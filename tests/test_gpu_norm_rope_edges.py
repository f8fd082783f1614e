"""Head norms, rotation and cache write (ops.qk_norm_rope) where values are out of
the ordinary, against the formula in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import attn_oracle as o
from test_gpu_norm_rope import BF, EPS, F32, HF, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_rt):
    from sabah_moe_accelerator_b200 import ops
    return ops


def call(ops, a, pairing):
    """(q_out, k_out, the cache's rows of k)."""
    kc, vc, slots = a["cache"]
    k_out = torch.empty(a["k"].shape, dtype=a["k"].dtype, device="cuda")
    q = ops.qk_norm_rope(*[a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table", "positions")], eps=EPS,
                         pairing=pairing, pair_axis=a["pair_axis"], cache=a["cache"], k_out=k_out)
    return q.clone(), k_out, kc.flatten(0, 1)[slots]


@pytest.mark.parametrize("pairing", ["halves", "pairs"])
@pytest.mark.parametrize("T,D,rope", [(12, 64, 32), (12, 64, 0), (12, 96, 24), (12, 90, 30), (12, 256, 64), (3000, 128, 64),
                                      (3000, 256, 32)])
@pytest.mark.parametrize("act,cache", [(F32, HF), (BF, BF), (HF, HF)])
def test_what_is_not_turned_does_not_mix(ops, T, D, rope, act, cache, pairing):
    """Without norms, an infinity or NaN past the rotated part stays where it is: every
    other value keeps its bits, in the outputs and in the cache."""
    a = make(ops, T, 4, 2, D, rope, act, cache)
    a["q_weight"] = a["k_weight"] = None
    clean = call(ops, a, pairing)
    marks = {}
    for i, (at, x) in enumerate(((rope, math.inf), (D - 1, math.nan), (rope + (D - rope) // 2, -math.inf))):
        for n in ("q", "k"):
            a[n][2 + i, i % 2, at] = x
        marks[2 + i, i % 2, at] = x
    got = call(ops, a, pairing)
    for x, y in zip(got, clean):
        changed = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
        for (t, h, at), v in marks.items():
            changed[t, h, at] = True
            assert x[t, h, at].isnan() if math.isnan(v) else x[t, h, at] == v, (t, h, at)
        assert torch.equal(x[~changed], y[~changed])


@pytest.mark.parametrize("pairing", ["halves", "pairs"])
@pytest.mark.parametrize("D,rope", [(64, 32), (90, 30), (256, 64)])
def test_an_infinity_under_a_norm(ops, D, rope, pairing):
    """x * rsqrt(inf): zeros beside it, NaN itself and what the rotation mixes with it."""
    a = make(ops, 12, 4, 2, D, rope, F32, HF)
    a["q"][3, 1, rope + 1], a["q"][5, 0, 1], a["q"][7, 2, D - 1] = math.inf, -math.inf, math.nan
    q = call(ops, a, pairing)[0].cpu().double()
    want = o.norm_rope(a["q"], a["q_weight"], a["table"], a["positions"], pairing, a["pair_axis"], EPS)
    assert torch.equal(q.isnan(), want.isnan()) and not q.isinf().any()
    keep = ~want.isnan()
    assert o.rel_l2(q[keep], want[keep]) <= o.TOL[F32] and (q[3, 1][~want[3, 1].isnan()] == 0).all()
