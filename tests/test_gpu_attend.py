"""Attention of one new token over a paged cache (ops.attend_paged) against the
formula in 64 bits: lengths from zero and one, pages that no tile divides,
shared heads, windows, poisoned memory outside the window, strides, refusals."""
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


def make(lens, heads, kv_heads, dim, page, act, cache, heads_first=False, seed=0, q_scale=2.0, width=None, window=0):
    """A pool with every page in random order; NaN in every row outside the windows, -1 in
    every table entry outside them."""
    g = torch.Generator("cuda").manual_seed(seed)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    k, v = (torch.randn(shape, device="cuda", generator=g).to(cache) for _ in range(2))
    if heads_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(pages, device="cuda", generator=g).int()
    width = max(used + [1]) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    live = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        first = lo // page
        if n > lo:
            table[b, first:used[b]] = order[at + first:at + used[b]]
            j = torch.arange(lo, n, device="cuda")
            live[table[b, j // page].long(), j % page] = True
        at += used[b]
    k[~live], v[~live] = math.nan, math.nan
    q = (torch.randn(len(lens), heads, dim, device="cuda", generator=g) * q_scale).to(act)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(ops, t, window=0, scale=None, **kw):
    q, k, v, table, lens = t
    lse = torch.empty(q.shape[:2], device="cuda")
    out = ops.attend_paged(q, k, v, table, lens, window=window, scale=scale, lse=lse, **kw)
    torch.cuda.synchronize()
    from sabah_moe_accelerator_b200 import rt
    assert rt.lib().sabah_rt_device_error() == 0
    want, want_lse = o.attend(q, k, v, table, lens, scale, window)
    assert out.dtype == q.dtype and torch.isfinite(out).all()
    # one sequence at a time, so that a short one is not lost in the norm of all
    for b, n in enumerate(lens.tolist()):
        assert o.rel_l2(out[b], want[b]) <= o.TOL[q.dtype], (b, n)
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
        else:
            assert o.rel_l2(lse[b], want_lse[b]) <= 2e-5, (b, n)
    return out


TYPES = [(BF, BF), (HF, HF), (F32, HF), (F32, BF)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (32, 8, 128), (8, 8, 64), (6, 2, 96), (3, 1, 80)])
def test_types_and_heads(ops, act, cache, heads, kv_heads, dim):
    check(ops, make([0, 1, 2, 15, 16, 17, 31, 33, 100, 257, 700], heads, kv_heads, dim, 16, act, cache))


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 104, 112, 120, 136, 160, 176, 192, 200, 248])
@pytest.mark.parametrize("act,cache", [(BF, BF), (F32, HF)])
def test_odd_head_sizes(ops, dim, act, cache):
    check(ops, make([5, 64, 130], 4, 2, dim, 16, act, cache))


@pytest.mark.parametrize("page", [1, 2, 3, 8, 15, 16, 17, 24, 64, 100, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_page_sizes_and_orders(ops, page, heads_first):
    check(ops, make([1, 47, 48, 49, 300, 0, 1025], 8, 2, 128, page, F32, HF, heads_first))


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 9, 12, 15, 16, 17, 24, 33, 64])
@pytest.mark.parametrize("act,cache", [(HF, HF), (F32, BF)])
def test_group_sizes(ops, group, act, cache):
    check(ops, make([1, 90, 400], 2 * group, 2, 64, 16, act, cache))


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 4096])
@pytest.mark.parametrize("page", [16, 24])
def test_window(ops, window, page):
    check(ops, make([0, 1, 16, 17, 99, 100, 101, 1000, 5000], 12, 4, 64, page, F32, BF, window=window), window)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("lens", [[20000], [1, 30011], [4097] * 9, [9000, 3, 0, 12345, 64]])
def test_long(ops, lens, act, cache):
    check(ops, make(lens, 8, 1, 128, 32, act, cache, q_scale=3.0))
    check(ops, make(lens, 4, 2, 256, 64, act, cache, seed=1))


def test_many_sequences(ops):
    lens = [(37 * i) % 70 for i in range(5003)]
    check(ops, make(lens, 2, 1, 64, 16, BF, BF))


@pytest.mark.parametrize("width", [0, 1, 7, 600])
def test_table_widths(ops, width):
    lens = [0, 0] if width == 0 else [0, 1, min(100, 16 * width)]
    check(ops, make(lens, 4, 2, 64, 16, HF, HF, width=width))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("q_scale", [0.0, 1e-3, 30.0])
def test_flat_and_sharp(ops, act, cache, q_scale):
    """All scores equal; nearly equal; one key that takes all."""
    q, k, v, table, lens = make([1, 500, 3000], 4, 1, 64, 16, act, cache, q_scale=q_scale)
    check(ops, (q, k, v, table, lens))


def test_one_key_far_above_a_long_flat_tail(ops):
    """The tail's sum matters although each of its weights is e^-12 of the largest."""
    for act, cache in TYPES:
        q, k, v, table, lens = make([6000], 2, 1, 64, 16, act, cache, q_scale=0.0)
        q[..., 0] = 8.0
        live = torch.isfinite(k[..., 0])
        k[..., 0] = torch.where(live, 0, k[..., 0])
        k[table[0, 3], 5, 0, 0] = 12.0   # score 12 among zeros
        v += 1.0                          # a mean that the tail carries
        check(ops, (q, k, v, table, lens))


def test_extreme_scores_do_not_overflow(ops):
    for sign in (1, -1):
        q, k, v, table, lens = make([40, 700], 2, 1, 64, 16, F32, BF)
        check(ops, (q * 0 + sign * 300.0, k, v, table, lens))
        check(ops, (q * 3e4, k, v, table, lens))


def test_tiny_and_huge_queries_in_an_f16_cache(ops):
    """f32 queries outside f16's range."""
    q, k, v, table, lens = make([40, 700], 4, 2, 64, 16, F32, HF)
    check(ops, (q * 1e6, k, v, table, lens), scale=1e-7)
    check(ops, (q * 1e-9, k, v, table, lens), scale=1e8)
    q[:, 0] *= 1e5   # heads of very different size
    q[:, 1] *= 1e-5
    check(ops, (q, k, v, table, lens))


def test_infinities_and_nan_in_valid_places(ops):
    """What the formula makes of them, in the sequence that holds them and no other."""
    from sabah_moe_accelerator_b200 import rt
    q, k, v, table, lens = make([50, 50, 50, 50], 2, 1, 64, 16, BF, BF)
    clean = ops.attend_paged(q, k, v, table, lens)
    v[table[0, 1], 3, 0, 7] = math.nan
    v[table[1, 1], 3, 0, 7] = math.inf
    k[table[2, 0], 2, 0, 0] = math.nan
    out = ops.attend_paged(q, k, v, table, lens)
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0
    assert out[0, :, 7].isnan().all() and out[1, :, 7].isinf().all() and out[2].isnan().all()
    keep = torch.arange(64, device="cuda") != 7
    assert torch.equal(out[:2][..., keep], clean[:2][..., keep]) and torch.equal(out[3], clean[3])


def test_strided_queries_and_cache_slices(ops):
    """Queries inside a fused projection's rows; caches that are slices of wider pools."""
    q, k, v, table, lens = make([3, 77, 260], 8, 2, 128, 16, BF, BF)
    fused = torch.full((3, 8 * 128 + 328), math.nan, dtype=BF, device="cuda")
    fused[:, 8:8 + 8 * 128] = q.view(3, -1)
    qv = fused[:, 8:8 + 8 * 128].view(3, 8, 128)
    pool = torch.full((k.shape[0], 16, 2, 3, 128), math.nan, dtype=BF, device="cuda")
    pool[:, :, :, 0], pool[:, :, :, 2] = k, v
    got = check(ops, (qv, pool[:, :, :, 0], pool[:, :, :, 2], table, lens))
    assert torch.equal(got, ops.attend_paged(q, k, v, table, lens))
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    assert torch.equal(got, ops.attend_paged(q, k, v, wide[:, 2:2 + table.shape[1]], lens))


def test_offsets_past_32_bits(ops):
    """Pages that lie beyond 4 GiB of the cache."""
    q, k, v, table, lens = make([40, 1000], 4, 2, 128, 64, BF, BF)
    n = (5 << 30) // (64 * 2 * 128 * 2)
    kb, vb = (torch.empty((n, 64, 2, 128), dtype=BF, device="cuda") for _ in range(2))
    kb[n - k.shape[0]:], vb[n - k.shape[0]:] = k, v
    far = torch.where(table >= 0, table + n - k.shape[0], table)
    assert torch.equal(ops.attend_paged(q, kb, vb, far, lens), ops.attend_paged(q, k, v, table, lens))


def test_same_bits_every_time_and_on_any_stream(ops):
    t = make([9000, 17, 40000, 0, 333], 16, 2, 128, 16, F32, HF)
    first = check(ops, t)
    side = torch.cuda.Stream()
    for i in range(20):
        assert torch.equal(ops.attend_paged(*t), first)
        side.wait_stream(torch.cuda.current_stream())
        got = ops.attend_paged(*t, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, first)


def test_two_streams_at_once(ops):
    """Calls that overlap have workspaces of their own."""
    ts = [make([30000 + 7 * i], 16, 2, 128, 16, BF, BF, seed=i) for i in range(2)]
    want = [ops.attend_paged(*t) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attend_paged(*ts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_graph_capture(ops):
    q, k, v, table, lens = make([600, 5000, 1], 16, 2, 128, 16, BF, BF, width=400)
    out = torch.empty_like(q)
    ops.attend_paged(q, k, v, table, lens, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attend_paged(q, k, v, table, lens, out=out)
    lens -= torch.tensor([1, 4000, 0], dtype=torch.int32, device="cuda")   # the replay reads the lengths anew
    want = ops.attend_paged(q, k, v, table, lens)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_own_workspace(ops):
    from sabah_moe_accelerator_b200 import rt
    t = make([7000, 80], 16, 2, 256, 16, BF, BF)
    n = rt.lib().sabah_attend_paged_workspace(16, 2, 256)
    ws = torch.full((n + 16,), 0xff, dtype=torch.uint8, device="cuda")
    got = check(ops, t, workspace=ws[:n])
    assert torch.equal(got, ops.attend_paged(*t)) and (ws[n:] == 0xff).all()
    if n:
        with pytest.raises(rt.SabahCudaError, match="workspace"):
            ops.attend_paged(*t, workspace=ws[:n - 16])


def test_lse_joins_two_parts(ops):
    """Attention over [0, a) and over [a, n) joined by their lse is attention over [0, n)."""
    q, k, v, table, lens = make([1600], 4, 2, 64, 16, F32, HF)
    parts = []
    for tab, n in ((table[:, :40], 640), (table[:, 40:], 960)):
        lse = torch.empty(1, 4, device="cuda")
        n = torch.tensor([n], dtype=torch.int32, device="cuda")
        parts.append((ops.attend_paged(q, k, v, tab, n, lse=lse).double(), lse.double()))
    w = torch.softmax(torch.stack([p[1] for p in parts]), 0)
    got = sum(a[..., None] * p[0] for a, p in zip(w, parts))
    assert o.rel_l2(got, o.attend(q, k, v, table, lens)[0]) <= 4e-5


def test_no_sequences(ops):
    q, k, v, table, lens = make([5], 4, 2, 64, 16, BF, BF)
    assert ops.attend_paged(q[:0], k, v, table[:0], lens[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("what", ["page past the pool", "negative page", "length past the table", "negative length"])
def test_bad_index_is_nan_there_and_an_error(ops, what):
    from sabah_moe_accelerator_b200 import rt
    q, k, v, table, lens = make([50, 900, 50, 20000], 4, 2, 64, 16, BF, BF)
    good = ops.attend_paged(q, k, v, table, lens)
    for b in (1, 3):
        t2, l2 = table.clone(), lens.clone()
        if what == "page past the pool":
            t2[b, 30] = k.shape[0]
        elif what == "negative page":
            t2[b, 0] = -1
        elif what == "length past the table":
            l2[b] = 16 * table.shape[1] + 1
        else:
            l2[b] = -1
        lse = torch.zeros(4, 4, device="cuda")
        out = ops.attend_paged(q, k, v, t2, l2, lse=lse)
        torch.cuda.synchronize()
        with pytest.raises(rt.SabahCudaError, match="out of range"):
            ops.attend_paged(q, k, v, table, lens)
        assert rt.lib().sabah_rt_device_error() == 0
        assert out[b].isnan().all() and lse[b].isnan().all()
        rest = [i for i in range(4) if i != b]
        assert torch.equal(out[rest], good[rest])


def test_refusals(ops):
    from sabah_moe_accelerator_b200 import rt
    q, k, v, table, lens = make([50, 90], 4, 2, 64, 16, BF, BF)
    call = ops.attend_paged

    def refused(*a, **kw):
        with pytest.raises((ValueError, rt.SabahCudaError)):
            call(*a, **kw)

    refused(q.half(), k, v, table, lens)                         # f16 over bf16
    refused(q.double(), k, v, table, lens)
    refused(q, k.float(), v.float(), table, lens)
    refused(q, k, v.half(), table, lens)
    refused(q, k, v[:, :8], table, lens)
    refused(q[:, :3], k, v, table, lens)                         # 3 heads over 2
    refused(q[..., :32], k, v, table, lens)
    refused(q, k, v, table[:1], lens)
    refused(q, k, v, table.long(), lens)
    refused(q, k, v, table, lens.long())
    refused(q, k, v, table, lens[:1])
    refused(q, k, v, table, lens.cpu())
    refused(q.cpu(), k.cpu(), v.cpu(), table.cpu(), lens.cpu())
    refused(q, k, v, table, lens, window=-1)
    refused(q, k, v, table, lens, out=torch.empty_like(q)[:, :, :32])
    refused(q, k, v, table, lens, out=torch.empty(2, 4, 64, device="cuda"))
    refused(q, k, v, table, lens, lse=torch.empty(2, 4, device="cuda", dtype=BF))
    refused(q, k.transpose(2, 3), v.transpose(2, 3), table, lens)
    odd = torch.empty(k.numel() + 8, dtype=BF, device="cuda")
    refused(q, odd[1:1 + k.numel()].view(k.shape), v, table, lens)      # rows at 2 bytes past 16
    k12 = torch.zeros(4, 16, 2, 12, dtype=BF, device="cuda")
    refused(q[..., :12], k12, k12, table, lens)                  # 12 is no multiple of 8
    k264 = torch.zeros(4, 16, 2, 264, dtype=BF, device="cuda")
    refused(torch.zeros(2, 4, 264, dtype=BF, device="cuda"), k264, k264, table, lens)
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0
    check(ops, (q, k, v, table, lens))                           # and the next good call is good


def test_more_sequences_than_one_launch_holds_some_of_them_long(ops):
    """Launches of a call share the workspace one after another."""
    lens = [(13 * i) % 60 for i in range(2500)]
    lens[3], lens[1000], lens[1030], lens[2400] = 9000, 5000, 7001, 3333
    check(ops, make(lens, 4, 1, 64, 16, F32, HF))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_constant_values_keep_their_sum(ops, act, cache, dim):
    """One warp adds up thousands of equal products: a sum that is cut off instead of rounded drifts."""
    q, k, v, table, lens = make([3000] * 620, 4, 2, dim, 16, act, cache, q_scale=0.0)
    v[torch.isfinite(v)] = 1.0 + 2.0 ** -6
    out = ops.attend_paged(q, k, v, table, lens)
    assert o.rel_l2(out, torch.full(out.shape, 1.0 + 2.0 ** -6, dtype=torch.float64)) <= o.TOL[act]


def test_no_pages_at_all(ops):
    z = torch.zeros(0, 16, 2, 64, dtype=BF, device="cuda")
    q = torch.randn(3, 4, 64, device="cuda").to(BF)
    table, lens = torch.zeros(3, 5, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    lse = torch.zeros(3, 4, device="cuda")
    assert (ops.attend_paged(q, z, z, table, lens, lse=lse) == 0).all() and (lse == -math.inf).all()


def test_heads_that_share_their_memory(ops):
    q, k, v, table, lens = make([50, 900], 4, 1, 64, 16, BF, BF)
    check(ops, (q, k.expand(-1, -1, 2, -1), v.expand(-1, -1, 2, -1), table, lens))


def test_more_refusals(ops):
    from sabah_moe_accelerator_b200 import rt
    q, k, v, table, lens = make([50, 90], 4, 2, 64, 16, BF, BF)
    with pytest.raises(ValueError, match="gradient"):
        ops.attend_paged(q.requires_grad_(), k, v, table, lens)
    q = q.detach()
    flat = torch.empty(q.numel() + 1, dtype=BF, device="cuda")
    with pytest.raises(rt.SabahCudaError):                     # an output at an odd element
        ops.attend_paged(q, k, v, table, lens, out=flat[1:].view(q.shape))
    with pytest.raises(ValueError):
        ops.attend_paged(q, k, v, table, lens, window=1 << 40)
    wide = torch.zeros(2, 1, dtype=torch.int32, device="cuda").expand(2, 1 << 28)
    with pytest.raises((ValueError, rt.SabahCudaError)):         # 2^32 keys per sequence
        ops.attend_paged(q, k, v, wide, lens)
    assert rt.lib().sabah_rt_device_error() == 0
    check(ops, (q, k, v, table, lens))
