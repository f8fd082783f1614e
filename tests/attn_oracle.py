"""Plain 64-bit forms of the operators around the experts, for the tests: loops
over sequences and heads, straight from the formulas."""
from __future__ import annotations

import math

import torch


def attend(q, k_cache, v_cache, table, lens, scale=None, window=0):
    """(out, lse) float64 on the CPU."""
    q, table, lens = q.cpu().double(), table.cpu().long(), lens.cpu().tolist()
    B, H, D = q.shape
    page, n_kv = k_cache.shape[1], k_cache.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n == lo:
            continue
        j = torch.arange(lo, n)
        pages, rows = table[b, j // page].to(k_cache.device), (j % page).to(k_cache.device)
        k, v = (c[pages, rows].cpu().double() for c in (k_cache, v_cache))
        for h in range(H):
            g = h // (H // n_kv)
            s = k[:, g] @ q[b, h] * scale
            m = s.max()
            p = torch.exp(s - m)
            out[b, h] = p @ v[:, g] / p.sum()
            lse[b, h] = m + torch.log(p.sum())
    return out, lse


def norm_rope(x, weight, table, positions, pairing, pair_axis, eps):
    """x [T, heads, D] normed and turned, float64 on the CPU."""
    x = x.cpu().double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.cpu().double()
    if table is None:
        return x
    t, pos = table.cpu().double(), positions.cpu().long().reshape(-1, x.shape[0])
    y = x.clone()
    half = t.shape[1]
    for i in range(half):
        a, b = (i, i + half) if pairing == "halves" else (2 * i, 2 * i + 1)
        p = pos[int(pair_axis[i]) if pair_axis is not None else 0]
        c, s = t[p, i, 0][:, None], t[p, i, 1][:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def route(logits, n_used, renorm, scale=1.0):
    """(ids, w float64): Python's sort by (-logit, index)."""
    ids, w = [], []
    for row in logits.cpu().double().tolist():
        top = sorted(range(len(row)), key=lambda e: (-row[e], e))[:n_used]
        m = row[top[0]]
        over = top if renorm else range(len(row))
        total = sum(math.exp(row[e] - m) for e in over)
        ids.append(top)
        w.append([scale * math.exp(row[e] - m) / total for e in top])
    return torch.tensor(ids), torch.tensor(w, dtype=torch.float64)


def rel_l2(got, want):
    got, want = got.detach().cpu().double(), want.cpu().double()
    n = float(want.norm())
    return float((got - want).norm()) / n if n else float((got - want).norm())


# Half a unit in the last place of an output rounded once, plus the fp32 part:
# sums of a few hundred fp32 products and an exp, each within a few 2^-24 of
# terms that do not cancel far, stay below 2e-5.
TOL = {torch.float32: 2e-5, torch.float16: 2.0 ** -11 + 2e-5, torch.bfloat16: 2.0 ** -8 + 2e-5}
