"""Attention of one new token (ops.attend_paged) where scores, values or waits are
out of the ordinary, against the formula in 64 bits."""
from __future__ import annotations

import math
import os
import subprocess
import sys

import pytest
import torch

import attn_oracle as o
from conftest import ROOT
from test_gpu_attend import BF, F32, HF, TYPES, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_rt):
    from sabah_moe_accelerator_b200 import ops
    return ops


def same(got, want, tol):
    """NaN and infinities where the formula has them, the finite values within tol."""
    got, want = got.detach().cpu().double(), want.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan().sum(), want.isnan().sum())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    keep = want.isfinite()
    assert o.rel_l2(got[keep], want[keep]) <= tol


def check(ops, q, k, v, table, lens):
    from sabah_moe_accelerator_b200 import rt
    lse = torch.empty(q.shape[:2], device="cuda")
    out = ops.attend_paged(q, k, v, table, lens, lse=lse)
    torch.cuda.synchronize()
    assert rt.lib().sabah_rt_device_error() == 0
    want, want_lse = o.attend(q, k, v, table, lens)
    for b in range(len(lens)):
        same(out[b], want[b], o.TOL[q.dtype])
        same(lse[b], want_lse[b], 2e-5)
    return out


def put(cache, table, b, keys, value, col=0):
    """Writes value into column col of the given keys of sequence b, in every head."""
    j = torch.as_tensor(keys, device="cuda")
    page = cache.shape[1]
    cache[table[b, j // page].long(), j % page, :, col] = value


# ---------------------------------------------------------------- scores of -inf
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,dim", [(4, 64), (12, 128), (4, 256), (16, 256)])
def test_keys_that_score_minus_infinity_weigh_nothing(ops, act, cache, heads, dim):
    """The first key, the first step, all but the last, and one in the middle, in sequences
    that stay whole and in ones that are cut between warps."""
    q, k, v, table, lens = make([2, 50, 60, 700, 3000, 3000], heads, 1, dim, 16, act, cache)
    q[..., 0] = q[..., 0].abs() + 1                      # of one sign: -inf times it is -inf
    for b, keys in enumerate(([0], [0], range(59), range(40), range(2000), [1500])):
        put(k, table, b, list(keys), -math.inf)
    check(ops, q, k, v, table, lens)


@pytest.mark.parametrize("act,cache", TYPES)
def test_no_key_left(ops, act, cache):
    """All scores -inf: 0 / 0, in that sequence alone."""
    q, k, v, table, lens = make([1, 40, 2500, 70], 4, 1, 128, 16, act, cache)
    q[..., 0] = q[..., 0].abs() + 1
    for b in range(3):
        put(k, table, b, range(int(lens[b])), -math.inf)
    lse = torch.empty(4, 4, device="cuda")
    out = ops.attend_paged(q, k, v, table, lens, lse=lse)
    assert out[:3].isnan().all()
    want, want_lse = o.attend(q[3:], k, v, table[3:], lens[3:])
    same(out[3:], want, o.TOL[act])
    same(lse[3:], want_lse, 2e-5)


@pytest.mark.parametrize("act,cache,heads", [(F32, HF, 4), (F32, BF, 4), (BF, BF, 16), (HF, HF, 16)])
def test_a_warp_s_whole_part_scores_minus_infinity(ops, act, cache, heads):
    """640 sequences over the same pages give each warp some hundred steps, so parts lie
    inside the 2,500 keys that score -inf, and their sums pass through memory several times."""
    q, k, v, table, lens = make([3000], heads, 1, 256, 16, act, cache)
    q[..., 0] = q[..., 0].abs() + 1
    put(k, table, 0, range(2500), -math.inf)
    want, want_lse = o.attend(q, k, v, table, lens)
    n = 640
    lse = torch.empty(n, heads, device="cuda")
    out = ops.attend_paged(q.expand(n, -1, -1), k, v, table.expand(n, -1), lens.expand(n).contiguous(), lse=lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    tol = o.TOL[act]
    for got, w, t in ((out, want, tol), (lse, want_lse, 2e-5)):
        err = (got.double() - w.cuda()).flatten(1).norm(dim=1) / w.norm()
        assert float(err.max()) <= t


@pytest.mark.parametrize("act,cache", TYPES)
def test_nan_stays_however_little_it_weighs(ops, act, cache):
    """A NaN value or score before keys that outweigh it by more than fp32 can tell."""
    q, k, v, table, lens = make([60, 60, 2000], 4, 1, 64, 16, act, cache, q_scale=0.0)
    q[..., 0] = 8.0
    for b, at in enumerate((40, 40, 1999)):
        put(k, table, b, range(int(lens[b])), 0.0)
        put(k, table, b, [at], 400.0)                    # a score of 400 among zeros
    put(v, table, 0, [0], math.nan, col=7)
    put(k, table, 1, [0], math.nan)
    put(v, table, 2, [3], math.nan, col=9)
    out = ops.attend_paged(q, k, v, table, lens)
    want, _ = o.attend(q, k, v, table, lens)
    assert want[0, :, 7].isnan().all() and want[1].isnan().all() and want[2, :, 9].isnan().all()
    for b in range(3):
        same(out[b], want[b], o.TOL[act])


# ---------------------------------------------------------------- a wait that runs out
STALL = "SABAH_TEST_ATTEND_STALL"


def stall(ops, act, cache, heads, kv, dim):
    from sabah_moe_accelerator_b200 import rt
    short, long = [1, 40, 0, 7, 96, 33] * 40, [30000, 5, 20000]
    for lens in (long, short + long):
        t = make(lens, heads, kv, dim, 16, act, cache)
        lse_ok = torch.empty(len(lens), heads, device="cuda")
        want = ops.attend_paged(*t, lse=lse_ok)
        assert torch.isfinite(want).all()
        hurt = 0
        for w in (3, 400):
            lse, out = torch.full_like(lse_ok, 7.0), torch.full_like(want, 7.0)
            os.environ[STALL] = str(w)
            ops.attend_paged(*t, lse=lse, out=out)
            torch.cuda.synchronize()
            os.environ[STALL] = "-1"
            code = rt.lib().sabah_rt_device_error()
            lost = out.isnan()
            rows = lost.all(-1)
            assert torch.equal(rows, lost.any(-1)) and torch.equal(rows, lse.isnan())
            assert torch.equal(out[~lost], want[~lost]) and torch.equal(lse[~rows], lse_ok[~rows])
            assert code == (2 if rows.any() else 0)   # a warp beyond the list's parts has nothing to wait for
            hurt += int(rows.any())
        assert hurt
        assert torch.equal(ops.attend_paged(*t), want)
    assert rt.lib().sabah_rt_device_error() == 0


def test_a_wait_that_runs_out_gives_nan_there_and_an_error():
    """With the test switch SABAH_TEST_ATTEND_STALL=w, warp w's first wait is for bytes that
    no load brings. After its limit, under a second, the warp gives up, lets its
    loads arrive and makes NaN of the rows that it owes, whole or cut; every other row is
    what it was, the error word is set, and the next call is clean. The switch is looked
    for at a process's first call."""
    env = dict(os.environ, **{STALL: "-1"})
    env["PYTHONPATH"] = os.pathsep.join((ROOT, os.path.join(ROOT, "tests"), env.get("PYTHONPATH", "")))
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], cwd=ROOT, env=env, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "stall ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


if __name__ == "__main__":
    from sabah_moe_accelerator_b200 import ops as _ops
    _ops.init(0)
    for _case in ((BF, BF, 16, 2, 256), (F32, HF, 8, 2, 128), (HF, HF, 40, 2, 64)):
        stall(_ops, *_case)
    print("stall ok")
