"""The router's choice (ops.route_topk) against a Python sort in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import attn_oracle as o

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(gpu_rt):
    from sabah_moe_accelerator_b200 import ops
    return ops


def check(ops, x, K, renorm=True, scale=1.0):
    ids, w = ops.route_topk(x, K, renorm=renorm, scale=scale)
    want_ids, want_w = o.route(x, K, renorm, scale)
    assert torch.equal(ids.cpu().long(), want_ids)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    # a weight is one exp and one quotient of sums of at most 2048 positive terms
    assert o.rel_l2(w, want_w) <= 2e-6
    return ids, w


def logits(T, E, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(T, E, device="cuda", generator=g).mul(2).to(dtype)


@pytest.mark.parametrize("dtype", [F32, HF, BF])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,K", [(1, 512, 10), (64, 512, 10), (3, 8, 2), (129, 161, 6), (40, 128, 8), (17, 1000, 16),
                                   (2, 2048, 32), (5, 1, 1), (7, 31, 31), (9, 33, 32), (2, 2047, 1), (33, 60, 4),
                                   (11, 256, 8), (6, 513, 7), (500, 64, 6)])
def test_sizes(ops, T, E, K, dtype, renorm):
    check(ops, logits(T, E, dtype), K, renorm, 1.0 if renorm else 2.5)


def test_many_tokens(ops):
    check(ops, logits(4099, 512, BF), 10)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_ties_go_to_the_lowest_index(ops, dtype):
    x = torch.zeros(6, 300, dtype=dtype, device="cuda")
    x[1, 100:110] = 1
    x[2, ::7] = -3
    x[3] = torch.tensor([1.0, -1.0], device="cuda", dtype=dtype).repeat(150)
    x[4, :150] = -0.0                                   # -0 and +0 are one value
    x[5] = torch.arange(300, device="cuda") // 32
    check(ops, x, 10)
    check(ops, x, 32, False)


def test_strided_rows(ops):
    wide = logits(20, 700, F32)
    check(ops, wide[:, 5:517], 10)
    check(ops, logits(20, 700, BF)[::2, 3:514], 10)
    check(ops, logits(20, 704, HF)[:, 8:520], 10)


def test_wide_range(ops):
    x = logits(12, 512, F32) * 40
    check(ops, x, 10)
    check(ops, x * 1e30, 10)
    check(ops, x * 1e-30, 10)
    check(ops, x, 10, False)
    check(ops, x - 3e38, 8)


def test_masked_experts(ops):
    x = logits(8, 512, F32)
    x[0, 100:] = -math.inf
    x[1, 3:] = -math.inf            # three left of ten: the rest follow by index with weight 0
    x[2, :505] = -math.inf
    x[3] = -3.4028234663852886e38   # the type's lowest value masks, all ties
    x[3, 7] = 1.0
    ids, w = check(ops, x, 10)
    assert (w[1, 3:] == 0).all() and ids[1, 3:].tolist() == list(range(3, 10))
    for renorm in (True, False):
        x[4] = -math.inf            # nothing left: no weight anywhere
        ids, w = ops.route_topk(x, 10, renorm=renorm)
        assert (w[4] == 0).all() and ids[4].tolist() == list(range(10))
        assert torch.isfinite(w).all()


def test_nan_and_infinity_stay_in_their_row(ops):
    x = logits(5, 512, F32)
    want = ops.route_topk(x, 10)
    x[1, 17] = math.nan
    x[3, 200] = math.inf
    ids, w = ops.route_topk(x, 10)
    assert w[1].isnan().all() and w[3].isnan().any() and ids[3, 0] == 200 and 17 not in ids[1]
    assert ((ids >= 0) & (ids < 512)).all()
    for t in (0, 2, 4):
        assert torch.equal(ids[t], want[0][t]) and torch.equal(w[t], want[1][t])
    x[:] = math.nan
    ids, w = ops.route_topk(x, 10)
    assert w.isnan().all() and ids[0].tolist() == list(range(10))


def test_given_outputs_no_tokens_streams_capture(ops):
    x = logits(30, 512, F32)
    want = ops.route_topk(x, 10)
    ids, w = torch.empty_like(want[0]), torch.empty_like(want[1])
    got = ops.route_topk(x, 10, ids=ids, w=w)
    assert got[0] is ids and torch.equal(ids, want[0]) and torch.equal(w, want[1])
    assert ops.route_topk(x[:0], 10)[0].shape == (0, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.route_topk(x, 10, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.route_topk(x, 10, ids=ids, w=w)
    ids.zero_()
    g.replay()
    assert torch.equal(ids, want[0])


def test_refusals(ops):
    from sabah_moe_accelerator_b200 import rt
    x = logits(4, 64, F32)
    bad = [(x, 0), (x, 65), (logits(4, 64, F32), 33), (logits(2, 2049, F32), 4), (x.double(), 4), (x.cpu(), 4),
           (x.t(), 4), (x.int(), 4)]
    for y, k in bad:
        with pytest.raises((ValueError, rt.SabahCudaError)):
            ops.route_topk(y, k)
    with pytest.raises(ValueError):
        ops.route_topk(x, 4, ids=torch.empty(4, 4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.route_topk(x, 4, w=torch.empty(4, 5, device="cuda"))
    check(ops, x, 4)


@pytest.mark.parametrize("dtype", [F32, HF, BF])
@pytest.mark.parametrize("E", [64, 124, 128, 304, 512, 1024])
def test_ties_in_whole_chunks(ops, dtype, E):
    x = torch.zeros(7, E, dtype=dtype, device="cuda")
    x[1, E - 40:] = 1
    x[2, ::9] = 2
    x[3] = torch.arange(E, device="cuda") // 50
    x[4, 1::2] = -0.0
    x[5, 5] = 3
    x[5, 9:60] = 2.5
    x[6, :33] = 1                                        # one more than lanes
    for K in (1, 10, 32):
        check(ops, x, K)
        check(ops, x, K, False)


@pytest.mark.parametrize("dtype", [HF, BF])
def test_every_16_bit_value_ranks_where_it_belongs(ops, dtype):
    """Subnormals, zeros and the largest values, in rows of 512."""
    bits = torch.randperm(65536, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    x = (bits - ((bits > 32767) * 65536)).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x.float())]
    x = x[:x.numel() // 512 * 512].view(-1, 512).cuda()
    ids, _ = ops.route_topk(x, 32)
    want, _ = o.route(x, 32, True)
    assert torch.equal(ids.cpu().long(), want)
    tiny = x.clone()
    tiny[tiny.float().abs() > 1e-3] = 0                  # only small ones are left to choose
    ids, _ = ops.route_topk(tiny, 32)
    assert torch.equal(ids.cpu().long(), o.route(tiny, 32, True)[0])


@pytest.mark.parametrize("dtype", [F32, HF, BF])
@pytest.mark.parametrize("E", [512, 301, 128])
def test_every_kind_of_nan(ops, dtype, E):
    x = logits(6, E, dtype)
    ints = {F32: torch.int32, HF: torch.int16, BF: torch.int16}[dtype]
    for t, payload in enumerate((-1, torch.iinfo(ints).max)):   # all bits set, with and without the sign
        x.view(ints)[t, 7] = payload
        x.view(ints)[t + 2, E - 1] = payload
    ids, w = ops.route_topk(x, 10)
    assert w[:4].isnan().all() and not w[4:].isnan().any()
    assert not (ids[:2] == 7).any() and not (ids[2:4] == E - 1).any() and ((ids >= 0) & (ids < E)).all()
    x[0, 1:] = x[0, 7]                                    # one number among NaNs
    ids, w = ops.route_topk(x, 10)
    assert ids[0].tolist() == list(range(10)) and w[0].isnan().all()


def test_no_gradient(ops):
    with pytest.raises(ValueError, match="gradient"):
        ops.route_topk(logits(2, 64, F32).requires_grad_(), 4)
