"""What the operators around the experts check and refuse without a GPU."""
from __future__ import annotations

import math

import pytest
import torch

import attn_oracle as o


@pytest.fixture(scope="module")
def ops(rtlib):
    from sabah_moe_accelerator_b200 import ops
    return ops


def test_cpu_tensors_are_refused(ops):
    q, c = torch.zeros(1, 2, 64), torch.zeros(4, 16, 1, 64, dtype=torch.float16)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attend_paged(q, c, c, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(q, q, None, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.route_topk(torch.zeros(2, 8), 2)


@pytest.mark.parametrize("bad", [3, "x", None, [1.0]])
def test_what_is_no_tensor_is_refused(ops, bad):
    with pytest.raises(ValueError, match="tensor"):
        ops.route_topk(bad, 2)
    with pytest.raises(ValueError, match="tensor"):
        ops.attend_paged(bad, bad, bad, bad, bad)
    with pytest.raises(ValueError, match="tensor"):
        ops.qk_norm_rope(bad, bad, None, None, None, None, None)


def test_shapes_are_checked_before_anything_is_launched(ops):
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        ops.route_topk(x[0], 2)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(x, x, None, None, None, None, None)
    with pytest.raises(ValueError, match="pairing"):
        ops.qk_norm_rope(x, x, None, None, None, None, None, pairing="other")
    with pytest.raises(ValueError, match="caches"):
        ops.attend_paged(torch.zeros(1, 2, 64), x, x, x, x)


def test_the_abi_refuses_before_init(rtlib):
    from sabah_moe_accelerator_b200 import rt
    if rt.device_count():
        pytest.skip("the runtime may be initialised")
    assert rtlib.sabah_route_topk(None, 0, 0, 1, 8, 2, 1, 1.0, None, None, None) == -1
    assert "sabah_rt_init" in rt.last_error()
    assert rtlib.sabah_attend_paged(*[None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, 1, 0, 16, None, 0, 0, None, 1, 1, 1, 64,
                                      1.0, 0, None, None, None, 0, None]) == -1
    assert rtlib.sabah_qk_norm_rope(*[None, 0, 0, 1, None, 0, 0, None, 0, 0, 1, 1, 64, 0, None, None, 1e-6, None, 0, 0, 0,
                                      None, 0, None, None, None, None, 0, 0, 0, None, 0, 0, 0, 0, 0, 0, None, None]) == -1


def test_workspace_of_what_does_not_exist_is_empty(rtlib):
    for args in ((0, 1, 64), (1, 0, 64), (8, 8, 0), (8, 8, 257)):
        assert rtlib.sabah_attend_paged_workspace(*args) == 0


def test_rope_table(ops):
    t = ops.rope_table(4097, 64, 1e6, device="cpu")
    assert t.shape == (4097, 32, 2) and t.dtype == torch.float32
    for pos, i in ((0, 0), (1, 0), (4096, 0), (4096, 31), (77, 5)):
        a = pos * 1e6 ** (-2 * i / 64)
        assert abs(t[pos, i, 0] - math.cos(a)) < 1e-7 and abs(t[pos, i, 1] - math.sin(a)) < 1e-7


def test_the_oracle_against_torch(ops):
    """The 64-bit forms that the GPU tests compare with, on dense inputs torch can do."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, 16, generator=g, dtype=torch.float64)
    k, v = (torch.randn(6, 5, 2, 16, generator=g, dtype=torch.float64) for _ in range(2))
    table, lens = torch.tensor([[3, 1, 5], [0, 4, 2]], dtype=torch.int32), torch.tensor([13, 6], dtype=torch.int32)
    out, lse = o.attend(q, k, v, table, lens, window=7)
    for b, n in enumerate(lens.tolist()):
        lo = max(0, n - 7)
        kk, vv = (c[table[b].long()].flatten(0, 1)[lo:n].repeat_interleave(2, 1) for c in (k, v))
        s = torch.einsum("hd,jhd->hj", q[b], kk) / 4
        assert torch.allclose(out[b], torch.einsum("hj,jhd->hd", torch.softmax(s, -1), vv))
        assert torch.allclose(lse[b], torch.logsumexp(s, -1))
    x, w = torch.randn(3, 2, 8, generator=g, dtype=torch.float64), torch.rand(8, generator=g)
    t = ops.rope_table(9, 6, device="cpu")
    pos = torch.tensor([0, 8, 3], dtype=torch.int32)
    y = o.norm_rope(x, w, t, pos, "pairs", None, 1e-6)
    z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    turn = torch.view_as_complex(t.double()[pos.long()])[:, None]
    want = torch.view_as_real(torch.view_as_complex(z[..., :6].reshape(3, 2, 3, 2).contiguous()) * turn).flatten(-2)
    assert torch.allclose(y[..., :6], want) and torch.equal(y[..., 6:], z[..., 6:])
    ids, p = o.route(torch.tensor([[0.0, 2.0, 2.0, -1.0]]), 3, False, 2.0)
    assert ids.tolist() == [[1, 2, 0]] and torch.allclose(p, 2 * torch.softmax(torch.tensor([0.0, 2, 2, -1]), 0)[ids[0]].double())
