"""Head norms, rotation and cache write in one pass (ops.qk_norm_rope) against
the formula in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import attn_oracle as o

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


@pytest.fixture(scope="module")
def ops(gpu_rt):
    from sabah_moe_accelerator_b200 import ops
    return ops


def make(ops, T, n_q, n_kv, D, rope, act, cache=HF, axes=1, page=16, heads_first=False, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    qkv = rnd(T, (n_q + 2 * n_kv) * D).mul(1.5).to(act)
    q, k, v = (qkv[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in
               ((0, n_q), (n_q, n_q + n_kv), (n_q + n_kv, n_q + 2 * n_kv)))
    pages = -(-T // page) + 2
    shape = (pages, n_kv, page, D) if heads_first else (pages, page, n_kv, D)
    kc, vc = (rnd(*shape).to(cache) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    return dict(q=q, k=k, v=v, q_weight=1 + 0.3 * rnd(D), k_weight=1 + 0.3 * rnd(D),
                table=ops.rope_table(5000, rope, 1e6) if rope else None,
                positions=torch.randint(0, 5000, (axes, T) if axes > 1 else (T,), device="cuda", generator=g).int(),
                pair_axis=(torch.arange(rope // 2, device="cuda") * 7 % axes).to(torch.uint8) if axes > 1 else None,
                cache=(kc, vc, torch.randperm(pages * page, device="cuda", generator=g)[:T].contiguous()))


def check(ops, a, pairing="halves"):
    from sabah_moe_accelerator_b200 import rt
    args = [a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table", "positions")]
    kc, vc, slots = a["cache"]
    kw, vw = kc.cpu().double(), vc.cpu().double()
    k_out = torch.empty(a["k"].shape, dtype=a["k"].dtype, device="cuda")
    q = ops.qk_norm_rope(*args, eps=EPS, pairing=pairing, pair_axis=a["pair_axis"], cache=a["cache"], k_out=k_out)
    q2, k2 = ops.qk_norm_rope(*args, eps=EPS, pairing=pairing, pair_axis=a["pair_axis"])
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0
    assert torch.equal(q, q2) and torch.equal(k_out, k2)
    tol = o.TOL[a["q"].dtype]
    want_q = o.norm_rope(a["q"], a["q_weight"], a["table"], a["positions"], pairing, a["pair_axis"], EPS)
    want_k = o.norm_rope(a["k"], a["k_weight"], a["table"], a["positions"], pairing, a["pair_axis"], EPS)
    assert o.rel_l2(q, want_q) <= tol and o.rel_l2(k_out, want_k) <= tol
    page = kc.shape[1]
    live = slots.cpu() >= 0
    at = slots.cpu()[live]
    kw[at // page, at % page], vw[at // page, at % page] = want_k[live], a["v"].cpu().double()[live]
    rows = torch.zeros(kc.shape[:2], dtype=torch.bool)
    rows[at // page, at % page] = True
    if len(at):
        assert o.rel_l2(kc.cpu()[rows], kw[rows]) <= o.TOL[kc.dtype]
        assert torch.equal(vc.cpu()[rows], a["v"].cpu()[live][torch.argsort(at)].to(vc.dtype))
    assert torch.equal(kc.cpu()[~rows].double(), kw[~rows]) and torch.equal(vc.cpu()[~rows].double(), vw[~rows])
    return q


@pytest.mark.parametrize("pairing", ["halves", "pairs"])
@pytest.mark.parametrize("act,cache", [(BF, BF), (HF, HF), (F32, HF), (F32, BF), (BF, HF)])
@pytest.mark.parametrize("T,n_q,n_kv,D,rope", [(1, 16, 2, 256, 64), (64, 32, 8, 128, 128), (37, 5, 1, 64, 32)])
def test_types(ops, T, n_q, n_kv, D, rope, act, cache, pairing):
    check(ops, make(ops, T, n_q, n_kv, D, rope, act, cache), pairing)


@pytest.mark.parametrize("pairing", ["halves", "pairs"])
@pytest.mark.parametrize("D,rope", [(2, 2), (6, 4), (8, 8), (18, 10), (40, 40), (72, 24), (80, 20), (96, 96), (100, 50),
                                    (120, 8), (130, 130), (160, 160), (192, 64), (222, 100), (254, 254), (256, 0), (64, 0)])
def test_odd_sizes(ops, D, rope, pairing):
    check(ops, make(ops, 19, 3, 2, D, rope, F32), pairing)
    check(ops, make(ops, 19, 3, 2, D, rope, BF, BF), pairing)


@pytest.mark.parametrize("T", [1, 2, 3, 31, 500, 2049, 8191])
def test_token_counts(ops, T):
    check(ops, make(ops, T, 32 if T < 3000 else 7, 8 if T < 3000 else 1, 128, 128, BF, BF))


@pytest.mark.parametrize("T,n_q,n_kv", [(5, 131, 9), (1, 1, 1024), (700, 50, 33)])
def test_many_heads(ops, T, n_q, n_kv):
    check(ops, make(ops, T, n_q, n_kv, 64, 64, BF, BF))


@pytest.mark.parametrize("D,rope,pairing", [(64, 32, "pairs"), (80, 80, "halves"), (192, 128, "halves"), (256, 256, "pairs")])
@pytest.mark.parametrize("act", [F32, HF])
def test_many_rows(ops, D, rope, pairing, act):
    check(ops, make(ops, 5003, 6, 5, D, rope, act, HF, axes=2), pairing)


@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("D,rope,pairing", [(80, 80, "pairs"), (128, 64, "halves"), (90, 30, "halves")])
def test_axes(ops, axes, D, rope, pairing):
    check(ops, make(ops, 65, 6, 2, D, rope, HF, HF, axes=axes), pairing)


@pytest.mark.parametrize("page", [1, 7, 24, 128])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages_and_orders(ops, page, heads_first):
    check(ops, make(ops, 150, 4, 2, 64, 64, BF, BF, page=page, heads_first=heads_first))


def test_padding_tokens_write_nothing(ops):
    a = make(ops, 50, 4, 2, 64, 64, BF, BF)
    a["cache"][2][torch.arange(0, 50, 3)] = -1
    check(ops, a)
    a["cache"][2][:] = -1
    check(ops, a)


def test_without_norms_or_rotation(ops):
    a = make(ops, 20, 4, 2, 64, 64, F32)
    for name in ("q_weight", "k_weight"):
        check(ops, dict(a, **{name: None}))
    b = dict(a, q_weight=None, k_weight=None, table=None, positions=None)
    assert torch.equal(check(ops, b), a["q"].contiguous())       # nothing to do: the same bits


def test_unaligned_rows(ops):
    """Views whose rows start at an odd element."""
    a = make(ops, 20, 4, 2, 64, 64, BF, BF)
    wide = torch.zeros(20, 8 * 64 + 3, dtype=BF, device="cuda")
    for n, (i, j) in {"q": (0, 4), "k": (4, 6), "v": (6, 8)}.items():
        wide[:, 1 + 64 * i:1 + 64 * j] = a[n].reshape(20, -1)
        a[n] = wide[:, 1 + 64 * i:1 + 64 * j].unflatten(1, (j - i, 64))
    check(ops, a)
    base = torch.zeros(65, device="cuda")
    base[1:] = a["q_weight"]
    check(ops, dict(a, q_weight=base[1:]))


def test_in_place(ops):
    for act, D, rope in ((BF, 128, 128), (F32, 90, 30)):
        a = make(ops, 33, 4, 2, D, rope, act)
        q, k = a["q"].contiguous(), a["k"].contiguous()
        args = (a["q_weight"], a["k_weight"], a["table"], a["positions"])
        want = ops.qk_norm_rope(q, k, None, *args)
        got = ops.qk_norm_rope(q, k, None, *args, q_out=q, k_out=k)
        assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_zeros_and_large_values(ops):
    a = make(ops, 8, 4, 2, 64, 64, F32)
    a["q"][0], a["q"][1], a["k"][2] = 0, 1e15, 1e-20
    a["q"][3, 1], a["k"][4, 0] = a["q"][3, 1] * 1e-3, a["k"][4, 0] * 1e4
    q = check(ops, a)
    assert (q[0] == 0).all()
    a["q"][5, 2, 3], a["k"][6, 1, 9] = math.nan, math.inf
    q2, k2 = ops.qk_norm_rope(a["q"], a["k"], None, a["q_weight"], a["k_weight"], a["table"], a["positions"])
    assert q2[5, 2].isnan().all() and torch.isfinite(q2[5, [0, 1, 3]]).all() and k2[6, 1].isnan().any()
    assert torch.equal(q2[:5], q[:5]) and torch.isfinite(k2[6, 0]).all()


def test_q_or_k_alone(ops):
    a = make(ops, 9, 4, 2, 64, 64, BF)
    args = (a["q_weight"], a["k_weight"], a["table"], a["positions"])
    want = ops.qk_norm_rope(a["q"], a["k"], None, *args)
    q, k = ops.qk_norm_rope(a["q"], a["k"][:, :0], None, *args)
    assert torch.equal(q, want[0]) and k.shape == (9, 0, 64)
    q, k = ops.qk_norm_rope(a["q"][:, :0], a["k"], None, *args)
    assert torch.equal(k, want[1]) and q.shape == (9, 0, 64)


def test_no_tokens(ops):
    a = make(ops, 4, 4, 2, 64, 64, BF)
    q, k = ops.qk_norm_rope(a["q"][:0], a["k"][:0], None, a["q_weight"], a["k_weight"], a["table"],
                            a["positions"][:0].contiguous())
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_cache_past_32_bits(ops):
    a = make(ops, 70, 4, 2, 128, 128, BF, BF)
    want_k = torch.empty(70, 2, 128, dtype=BF, device="cuda")
    args = [a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table", "positions")]
    ops.qk_norm_rope(*args, cache=a["cache"], k_out=want_k)
    n = (5 << 30) // (64 * 2 * 128 * 2)
    kc, vc = (torch.empty((n, 64, 2, 128), dtype=BF, device="cuda") for _ in range(2))
    slots = torch.arange(70, device="cuda") + (n - 2) * 64
    ops.qk_norm_rope(*args, cache=(kc, vc, slots))
    assert torch.equal(kc[n - 2:].flatten(0, 1)[:70], want_k)
    assert torch.equal(vc[n - 2:].flatten(0, 1)[:70], a["v"])


def test_side_stream_and_capture(ops):
    a = make(ops, 300, 8, 2, 128, 128, BF, BF)
    args = [a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table", "positions")]
    want = ops.qk_norm_rope(*args, cache=a["cache"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.qk_norm_rope(*args, cache=a["cache"], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out, g = torch.empty_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.qk_norm_rope(*args, cache=a["cache"], q_out=out)
    out.zero_()
    g.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("what", ["position past the table", "negative position", "slot past the cache", "axis"])
def test_bad_index(ops, what):
    from sabah_moe_accelerator_b200 import rt
    a = make(ops, 12, 4, 2, 64, 32, BF, BF, axes=2)
    args = [a[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table")]
    kc, vc, slots = a["cache"]
    pos, axis = a["positions"].clone(), a["pair_axis"].clone()
    want = ops.qk_norm_rope(*args, pos, pair_axis=axis, cache=(kc.clone(), vc.clone(), slots))
    if what == "position past the table":
        pos[0, 5] = 5000
    elif what == "negative position":
        pos[1, 5] = -1
    elif what == "slot past the cache":
        slots[5] = kc.shape[0] * kc.shape[1]
    else:
        axis[3] = 2
    before = kc.clone()
    got = ops.qk_norm_rope(*args, pos, pair_axis=axis, cache=(kc, vc, slots))
    torch.cuda.synchronize()
    with pytest.raises(rt.SabahCudaError, match="out of range"):
        ops.qk_norm_rope(*args, pos, pair_axis=axis, cache=(kc, vc, slots))
    rt.lib().sabah_rt_device_error()
    if what == "slot past the cache":
        assert torch.equal(got, want)
        rows = torch.ones(kc.shape[0] * kc.shape[1], dtype=torch.bool, device="cuda")
        rows[slots[torch.arange(12, device="cuda") != 5]] = False
        assert torch.equal(kc.flatten(0, 1)[rows], before.flatten(0, 1)[rows])
    elif what == "axis":
        assert got[..., 3].isnan().all() and torch.equal(got[..., 4:16], want[..., 4:16])
    else:
        assert got[5].isnan().any() and torch.equal(got[:5], want[:5]) and torch.equal(got[6:], want[6:])


def test_refusals(ops):
    from sabah_moe_accelerator_b200 import rt
    a = make(ops, 12, 4, 2, 64, 64, BF, BF)

    def refused(pairing="halves", **kw):
        b = dict(a, **kw)
        with pytest.raises((ValueError, rt.SabahCudaError)):
            ops.qk_norm_rope(*[b[n] for n in ("q", "k", "v", "q_weight", "k_weight", "table", "positions")],
                             pairing=pairing, pair_axis=b["pair_axis"], cache=b["cache"])

    kc, vc, slots = a["cache"]
    refused(pairing="other")
    refused(k=a["k"].float())
    refused(k=a["k"][:5])
    refused(v=None)
    refused(v=a["v"].half())
    refused(q_weight=a["q_weight"].half())
    refused(k_weight=a["k_weight"][:32])
    refused(table=a["table"].double())
    refused(table=ops.rope_table(50, 66))                         # rotates more than there is
    refused(positions=None)
    refused(positions=a["positions"].long())
    refused(positions=a["positions"][:5])
    refused(positions=torch.zeros(5, 12, dtype=torch.int32, device="cuda"))   # five axes
    refused(pair_axis=torch.zeros(5, dtype=torch.uint8, device="cuda"))
    refused(cache=(kc, vc, slots.int()))
    refused(cache=(kc, vc, slots[:5]))
    refused(cache=(kc.float(), vc.float(), slots))
    refused(cache=(kc, vc.half(), slots))
    refused(cache=(kc[:, :, :1], vc[:, :, :1], slots))
    refused(cache=(kc.cpu(), vc.cpu(), slots))
    refused(q=a["q"].cpu(), k=a["k"].cpu())
    refused(q=a["q"].transpose(1, 2).contiguous().transpose(1, 2))
    z = torch.zeros(12, 2, 258, dtype=BF, device="cuda")
    refused(q=z, k=z, v=z, q_weight=None, k_weight=None, cache=None)          # a head of 258
    refused(q=z[..., :63], k=z[..., :63], v=None, q_weight=None, k_weight=None, table=None, cache=None)
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0
    check(ops, a)


def test_too_many_heads_are_refused(ops):
    from sabah_moe_accelerator_b200 import rt
    q = torch.zeros(1, 16385, 2, device="cuda", dtype=BF)
    one = ops.qk_norm_rope(q[:, :16384], q[:, :16384], None, None, None, None, None)
    assert one[0].shape == (1, 16384, 2)
    for a, b in ((q, q[:, :4]), (q[:, :4], q)):
        with pytest.raises(rt.SabahCudaError, match="geometry"):
            ops.qk_norm_rope(a, b, None, None, None, None, None)
