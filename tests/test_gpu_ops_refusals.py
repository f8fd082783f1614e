"""Arguments that the operators around the experts refuse, on CUDA tensors that
nothing else is wrong with; after each refusal a good call is good."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_rt):
    from sabah_moe_accelerator_b200 import ops
    return ops


def args_of(ops):
    """name -> (call(**tensors), its tensors)."""
    g = torch.Generator("cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    T, H, K, D = 3, 4, 2, 64
    caches = dict(k_cache=rnd(4, 16, K, D).half(), v_cache=rnd(4, 16, K, D).half())

    def norm_rope(k_cache, v_cache, slots, **a):
        return ops.qk_norm_rope(**a, cache=(k_cache, v_cache, slots))

    i32 = torch.int32
    return {
        "norm_rope": (norm_rope, dict(
            q=rnd(T, H, D), k=rnd(T, K, D), v=rnd(T, K, D), q_weight=rnd(D), k_weight=rnd(D), table=ops.rope_table(8, D),
            positions=torch.arange(T, device="cuda", dtype=i32), slots=torch.arange(T, device="cuda"),
            q_out=rnd(T, H, D), k_out=rnd(T, K, D), **caches)),
        "attend": (ops.attend_paged, dict(
            q=rnd(T, H, D), block_table=torch.arange(T, device="cuda", dtype=i32).view(T, 1),
            lens=torch.tensor([1, 9, 16], device="cuda", dtype=i32), out=rnd(T, H, D), lse=rnd(T, H),
            workspace=torch.zeros(1 << 24, device="cuda", dtype=torch.uint8), **caches)),
        "route": (lambda **a: ops.route_topk(a.pop("logits"), 2, **a), dict(
            logits=rnd(T, 8), w=rnd(T, 2), ids=torch.zeros(T, 2, device="cuda", dtype=i32))),
    }


EVERY = [(op, n) for op, names in (
    ("norm_rope", "q k v q_weight k_weight table positions k_cache v_cache slots q_out k_out"),
    ("attend", "q k_cache v_cache block_table lens out lse workspace"), ("route", "logits ids w")) for n in names.split()]


@pytest.mark.parametrize("op,name", EVERY)
def test_batched_tensors(ops, op, name):
    call, a = args_of(ops)[op]
    call(**a)
    x = torch.stack((a[name], a[name]))
    with pytest.raises(ValueError, match=name + ".*plain tensor"):
        torch.vmap(lambda t: call(**{**a, name: t}))(x)
    call(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("op", ["norm_rope", "attend", "route"])
def test_functional_transforms(ops, op):
    call, a = args_of(ops)[op]
    name = "logits" if op == "route" else "q"
    first = lambda y: y[0] if isinstance(y, tuple) else y  # noqa: E731
    f = lambda t: first(call(**{**a, name: t}))  # noqa: E731
    with pytest.raises(ValueError, match="plain tensor"):
        torch.func.jvp(f, (a[name],), (a[name],))
    with pytest.raises(ValueError, match="plain tensor"):
        torch.func.grad(lambda t: f(t).sum())(a[name])
    call(**a)
    torch.cuda.synchronize()


FLOATS = [(op, n) for op, n in EVERY if n not in ("positions", "slots", "block_table", "lens", "workspace", "ids")]


@pytest.mark.parametrize("op,name", FLOATS)
def test_memory_that_does_not_hold_the_values(ops, op, name):
    """A view that reads as the negative of its memory; a storage that was freed."""
    call, a = args_of(ops)[op]
    with pytest.raises(ValueError, match=name + ".*hold its values"):
        call(**{**a, name: torch._neg_view(a[name])})
    gone = a[name].clone()
    gone.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match=name + ".*hold its values"):
        call(**{**a, name: gone})
    call(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("op,name", FLOATS)
def test_what_would_lose_a_gradient(ops, op, name):
    import torch.autograd.forward_ad as fw
    call, a = args_of(ops)[op]
    wants = {**a, name: a[name].clone().requires_grad_()}
    with pytest.raises(ValueError, match=name + ".*no gradient"):
        call(**wants)
    with torch.no_grad():
        call(**wants)
    with fw.dual_level(), pytest.raises(ValueError, match=name + ".*no forward gradient"):
        call(**{**a, name: fw.make_dual(a[name], torch.ones_like(a[name]))})
    call(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("op", ["norm_rope", "attend", "route"])
def test_a_dispatch_mode_changes_nothing(ops, op):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    call, a = args_of(ops)[op]
    want = call(**a)
    want = [t.clone() for t in (want if isinstance(want, tuple) else (want,))]
    with Watch():
        got = call(**a)
    assert all(torch.equal(x, y) for x, y in zip(got if isinstance(got, tuple) else (got,), want))
