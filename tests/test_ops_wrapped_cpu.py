"""Tensors that the operators around the experts cannot read as they lie in memory:
refused before anything else is looked at, so the refusals are testable without a GPU."""
from __future__ import annotations

import pytest
import torch

from torch._subclasses import FakeTensorMode


@pytest.fixture(scope="module")
def ops(rtlib):
    from sabah_moe_accelerator_b200 import ops
    return ops


def calls(ops):
    """One call of each operator of one float tensor x [4, 8]."""
    i32 = torch.int32

    def norm_rope(x):
        q = x.view(2, 2, 8)
        return ops.qk_norm_rope(q, q, None, None, None, None, None)[0]

    def attend(x):
        c = torch.zeros(4, 16, 1, 8, dtype=torch.float16)
        return ops.attend_paged(x.view(2, 2, 8), c, c, torch.zeros(2, 1, dtype=i32), torch.zeros(2, dtype=i32))

    def route(x):
        return ops.route_topk(x, 2)[1]

    return norm_rope, attend, route


@pytest.mark.parametrize("which", range(3))
def test_transforms_are_refused(ops, which):
    f = calls(ops)[which]
    x = torch.zeros(3, 4, 8)
    with pytest.raises(ValueError, match="plain tensor"):
        torch.vmap(f)(x)
    with pytest.raises(ValueError, match="plain tensor"):
        torch.func.jvp(f, (x[0],), (x[0],))
    with pytest.raises(ValueError, match="plain tensor"):
        torch.func.grad(lambda y: f(y).sum())(x[0])


@pytest.mark.parametrize("which", range(3))
def test_fake_tensors_are_refused(ops, which):
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.zeros(4, 8)
        with pytest.raises(ValueError, match="plain tensor"):
            calls(ops)[which](x)


def test_every_argument_is_looked_at(ops):
    """A batched tensor in any place, beside plain ones."""
    x, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(2, 2, 8), torch.zeros(4, 16, 2, 8, dtype=torch.float16)

    def refused(f, t):
        with pytest.raises(ValueError, match="plain tensor"):
            torch.vmap(f)(torch.stack((t, t)))

    refused(lambda t: ops.route_topk(x, 2, ids=t)[1], torch.zeros(2, 2, dtype=torch.int32))
    refused(lambda t: ops.route_topk(x, 2, w=t)[1], torch.zeros(2, 2))
    attend = (q, c, c, torch.zeros(2, 1, dtype=torch.int32), i)
    for n in range(5):
        refused(lambda t, n=n: ops.attend_paged(*attend[:n], t, *attend[n + 1:]), attend[n])
    for name, t in (("out", q), ("lse", torch.zeros(2, 2)), ("workspace", torch.zeros(64, dtype=torch.uint8))):
        refused(lambda t, name=name: ops.attend_paged(*attend, **{name: t}), t)
    slots = torch.zeros(2, dtype=torch.int64)
    args = (q, q, q, torch.ones(8), torch.ones(8), torch.zeros(4, 4, 2), i)
    for n in range(7):
        refused(lambda t, n=n: ops.qk_norm_rope(*args[:n], t, *args[n + 1:], cache=(c, c, slots)), args[n])
    for n in range(3):
        refused(lambda t, n=n: ops.qk_norm_rope(*args, cache=tuple(t if m == n else (c, c, slots)[m] for m in range(3))),
                (c, c, slots)[n])
    for name, t in (("pair_axis", torch.zeros(4, dtype=torch.uint8)), ("q_out", q), ("k_out", q)):
        refused(lambda t, name=name: ops.qk_norm_rope(*args, **{name: t}), t)


@pytest.mark.parametrize("which", range(3))
def test_memory_that_does_not_hold_the_values_is_refused(ops, which):
    """A view that reads as the negative of its memory; zeros without memory."""
    f = calls(ops)[which]
    with pytest.raises(ValueError, match="hold its values"):
        f(torch._neg_view(torch.ones(4, 8)))
    with pytest.raises(ValueError, match="hold its values"):
        f(torch._efficientzerotensor((4, 8)))


def test_what_is_neither_true_nor_false(ops):
    """renorm is asked for its truth; what it raises is what the caller gets."""
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.route_topk(torch.zeros(4, 8), 2, renorm=torch.zeros(2))


@pytest.mark.parametrize("which", range(3))
def test_plain_tensors_under_a_dispatch_mode_are_plain(ops, which):
    """A mode that watches torch's own operations is none of a tensor's doing."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Watch(), pytest.raises(ValueError, match="CUDA"):   # the next check speaks
        calls(ops)[which](torch.zeros(4, 8))


@pytest.mark.parametrize("which", range(3))
def test_other_layouts_are_refused(ops, which):
    with pytest.raises(ValueError, match="plain tensor"):
        if which == 2:
            ops.route_topk(torch.zeros(4, 8).to_sparse(), 2)
        else:
            s, x = torch.zeros(2, 2, 8).to_sparse(), torch.zeros(2, 2, 8)
            ops.qk_norm_rope(x, s, None, None, None, None, None) if which else ops.attend_paged(s, x, x, x, x)
    functional = torch.func.functionalize(calls(ops)[which])
    with pytest.raises(ValueError, match="plain tensor"):
        functional(torch.zeros(4, 8))
