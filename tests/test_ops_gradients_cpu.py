"""The operators around the experts have no derivatives: a tensor that would lose one
is refused, before anything that needs a GPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from test_ops_wrapped_cpu import calls


@pytest.fixture(scope="module")
def ops(rtlib):
    from sabah_moe_accelerator_b200 import ops
    return ops


@pytest.mark.parametrize("which", range(3))
def test_reverse_and_forward_mode(ops, which):
    f = calls(ops)[which]
    with pytest.raises(ValueError, match="no gradient"):
        f(torch.zeros(4, 8, requires_grad=True))
    with pytest.raises(ValueError, match="no gradient"):
        f(torch.nn.Parameter(torch.zeros(4, 8)))
    with fw.dual_level(), pytest.raises(ValueError, match="no forward gradient"):
        f(fw.make_dual(torch.zeros(4, 8), torch.ones(4, 8)))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):   # nothing is lost: the next check speaks
        f(torch.zeros(4, 8, requires_grad=True))


def test_weights_values_caches_tables_and_outputs(ops):
    q, w, i = torch.zeros(2, 2, 8), torch.ones(8, requires_grad=True), torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(4, 16, 2, 8, dtype=torch.float16)
    slots, block = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 1, dtype=torch.int32)

    def refused(call, *a, **kw):
        with pytest.raises(ValueError, match="no gradient"):
            call(*a, **kw)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call(*a, **kw)

    need = lambda t: t.clone().requires_grad_()  # noqa: E731
    good = dict(q=q, k=q, v=q, q_weight=w.detach(), k_weight=w.detach(), table=torch.zeros(4, 4, 2), positions=i)
    for n in ("q", "k", "v", "q_weight", "k_weight", "table"):
        refused(ops.qk_norm_rope, **{**good, n: need(good[n])}, cache=(c, c, slots))
    refused(ops.qk_norm_rope, **good, cache=(need(c), c, slots))
    refused(ops.qk_norm_rope, **good, cache=(c, need(c), slots))
    refused(ops.qk_norm_rope, **good, q_out=need(q))
    refused(ops.qk_norm_rope, **good, k_out=need(q))
    refused(ops.attend_paged, q, need(c), c, block, i)
    refused(ops.attend_paged, q, c, need(c), block, i)
    refused(ops.attend_paged, q, c, c, block, i, out=need(q))
    refused(ops.attend_paged, q, c, c, block, i, lse=torch.zeros(2, 2, requires_grad=True))
    refused(ops.route_topk, torch.zeros(2, 8), 2, w=torch.zeros(2, 2, requires_grad=True))
