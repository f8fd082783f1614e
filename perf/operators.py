"""The attention half and the router of a decode or prefill step, as cases to measure.

Three operators stand next to the routed experts of this package in every layer:

  norm_rope   per-head norms of queries and keys, the position rotation, and the
              write of keys and values into the paged cache, in one pass
  attend      attention of one new token per sequence over the paged cache
  route       softmax, top-k and renormalisation of the router's logits

`run` gives each in its plain form (elementary torch operations in 32 bits) or,
where `own` is true, through the package's entry points.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---------------------------------------------------------------- the cases
def attend(name, seqs, shortest, longest, heads, kv_heads, dim, page, act, cache, window=0, empties=False,
           heads_first=False):
    return {"name": name, "op": "attend", "seqs": seqs, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "act": act, "cache": cache, "window": window,
            "empties": empties, "heads_first": heads_first}


def norm_rope(name, tokens, heads, kv_heads, dim, rope, pairing, axes, page, act, cache, heads_first=False):
    return {"name": name, "op": "norm_rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rope": rope, "pairing": pairing, "axes": axes, "page": page, "act": act, "cache": cache,
            "heads_first": heads_first}


def route(name, tokens, experts, used, act, renorm):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "used": used, "act": act,
            "renorm": renorm}


def listed():
    return [
        # the first words of a chat: one sequence, a few tokens in the cache; all latency
        attend("attend one, 37 tokens", 1, 37, 37, 16, 2, 256, 16, "bf16", "bf16"),
        # one sequence with a long document before it: the cache's length is the only axis to split
        attend("attend one, 131071 tokens", 1, 131071, 131071, 16, 2, 256, 64, "bf16", "bf16"),
        # a serving batch of ragged lengths, activations in 32 bits as the experts' calls take them
        attend("attend 64 ragged", 64, 128, 8192, 32, 8, 128, 16, "f32", "f16"),
        # many short chats, one query head per key head, some slots of the batch empty
        attend("attend 256 short", 256, 16, 512, 8, 8, 64, 32, "f16", "f16", empties=True),
        # layers with a sliding window; pages that no tile size divides, a cache laid out head by head
        attend("attend 16 windowed", 16, 1024, 32768, 24, 4, 96, 24, "f32", "bf16", window=4096, heads_first=True),
        # one decoded token; a quarter of each head is rotated
        norm_rope("norm_rope 1 token", 1, 16, 2, 256, 64, "halves", 1, 16, "bf16", "bf16"),
        # one decoded token of each of 64 sequences, 32-bit activations
        norm_rope("norm_rope 64 tokens", 64, 32, 8, 128, 128, "halves", 1, 16, "f32", "f16"),
        # a prompt, of an odd length
        norm_rope("norm_rope 8191 tokens", 8191, 32, 8, 128, 128, "halves", 1, 64, "bf16", "bf16"),
        # an image's patches: time, height and width turn parts of each head
        norm_rope("norm_rope 2049 patches", 2049, 24, 4, 80, 80, "pairs", 3, 24, "f16", "f16", heads_first=True),
        # the router of one decoded token
        route("route 1 token", 1, 512, 10, "f32", True),
        # a small bank of experts with an odd count, without renormalisation
        route("route 511 tokens", 511, 161, 6, "f32", False),
        # the router over a long prompt's tokens; 16-bit logits tie often
        route("route 16384 tokens", 16384, 512, 10, "bf16", True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "norm_rope", "route"])
    act, cache = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16")])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 16])
    if op == "attend":
        most = sum(lengths(listed()[2])) * 8 * 128  # values of the largest listed cache
        seqs = _log(rng, 1, 256)
        longest = max(1, min(_log(rng, 1, 131072), most // (seqs * kv * dim)))
        window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
        c = attend("", seqs, max(1, longest // rng.choice([1, 4, 64])), longest, heads, kv, dim, page, act, cache,
                   window, rng.random() < 0.3, rng.random() < 0.3)
    elif op == "norm_rope":
        tokens = max(1, min(_log(rng, 1, 8192), 8192 * 48 * 128 // ((heads + 2 * kv) * dim * BYTES[act] // 2)))
        rope = rng.choice([dim, dim // 2, 32])
        c = norm_rope("", tokens, heads, kv, dim, rope, rng.choice(["halves", "pairs"]), rng.choice([1, 1, 3]), page,
                      act, cache, rng.random() < 0.3)
    else:
        experts = _log(rng, 8, 1024)
        c = route("", _log(rng, 1, 16384 * 512 // max(512, experts)), experts, rng.randint(1, min(16, experts)), act,
                  rng.random() < 0.7)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def lengths(case):
    """The sequences' lengths: spread over the logarithm of the range, the same ones for every seed."""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    v = [b if n == 1 else int(round(a * (b / a) ** ((i + 0.5) / n))) for i in range(n)]
    return [0 if case["empties"] and n > 1 and i % 16 == 3 else x for i, x in enumerate(v)]


def _cache(case, pages, gen):
    """A cache of pages x page x kv_heads x dim values, in either order of memory."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["heads_first"]:
        shape = (shape[0], shape[2], shape[1], shape[3])
    t = torch.randn(shape, device="cuda", dtype=TYPES[case["cache"]], generator=gen)
    return t.transpose(1, 2) if case["heads_first"] else t


def rope_table(positions, rope, theta=1e6):
    f = theta ** (-torch.arange(0, rope, 2, device="cuda", dtype=torch.float64) / rope)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    act = TYPES[case["act"]]
    if case["op"] == "attend":
        page = case["page"]
        lens = torch.tensor(lengths(case), device="cuda", dtype=torch.int32)
        lens = lens[torch.randperm(case["seqs"], device="cuda", generator=gen)].contiguous()
        width = max(1, -(-case["longest"] // page))
        used = (lens + page - 1) // page
        pages = sum(-(-n // page) for n in lengths(case)) + 1
        order = torch.randperm(pages, device="cuda", generator=gen).int()
        j = torch.arange(width, device="cuda", dtype=torch.int32)
        at = (used.cumsum(0) - used)[:, None] + j  # a sequence's pages lie anywhere in the pool
        s["table"] = torch.where(j < used[:, None], order[at.clamp(max=pages - 1)], -1).int()
        s["lens"] = lens
        s["k_cache"], s["v_cache"] = _cache(case, pages, gen), _cache(case, pages, gen)
        # normed keys and queries; the factor makes some keys stand out, as a trained head's do
        q = torch.randn(case["seqs"], case["heads"], case["dim"], device="cuda", generator=gen) * 2
        s["q"] = q.to(act)
        s["span"] = min(case["longest"], case["window"]) if case["window"] else case["longest"]
    elif case["op"] == "norm_rope":
        T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # one fused projection's rows: queries, keys and values side by side
        qkv = (torch.randn(T, (H + 2 * K) * D, device="cuda", generator=gen) * 1.5).to(act)
        s["q"], s["k"], s["v"] = (qkv[:, a * D:b * D].unflatten(1, (b - a, D))
                                  for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
        s["q_weight"] = 1 + 0.2 * torch.randn(D, device="cuda", generator=gen)
        s["k_weight"] = 1 + 0.2 * torch.randn(D, device="cuda", generator=gen)
        start = 4096
        s["rope_table"] = rope_table(start + 8192, case["rope"])
        pos = torch.arange(T, device="cuda", dtype=torch.int32)
        if case["axes"] == 3:
            side = max(1, math.isqrt(T))
            s["positions"] = start + torch.stack([pos // (side * side), pos // side % side, pos % side]).int()
            s["pair_axis"] = (torch.arange(case["rope"] // 2, device="cuda") % 3).to(torch.uint8)
        else:
            s["positions"], s["pair_axis"] = start + pos, None
        pages = -(-T // case["page"])
        order = torch.randperm(pages, device="cuda", generator=gen)
        t = torch.arange(T, device="cuda")
        s["slots"] = order[t // case["page"]] * case["page"] + t % case["page"]
        s["k_cache"], s["v_cache"] = _cache(case, pages, gen), _cache(case, pages, gen)
    else:
        s["logits"] = torch.randn(case["tokens"], case["experts"], device="cuda", generator=gen).mul(2).to(act)
    return s


# ---------------------------------------------------------------- one pass
_package = None


def package():
    global _package
    if _package is None:
        from sabah_moe_accelerator_b200 import ops
        ops.init(torch.cuda.current_device())
        _package = ops
    return _package


def run(s):
    if own:
        ops = package()
        if s["op"] == "attend":
            return ops.attend_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=s["window"])
        if s["op"] == "norm_rope":
            q = ops.qk_norm_rope(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["rope_table"],
                                 s["positions"], eps=EPS, pairing=s["pairing"], pair_axis=s["pair_axis"],
                                 cache=(s["k_cache"], s["v_cache"], s["slots"]))
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        ids, w = ops.route_topk(s["logits"], s["used"], renorm=s["renorm"])
        return {"ids": ids, "w": w}
    return {"attend": plain_attend, "norm_rope": plain_norm_rope, "route": plain_route}[s["op"]](s)


def plain_attend(s):
    B, H, D = s["q"].shape
    K, page = s["kv_heads"], s["page"]
    lens = s["lens"].long()
    first = (lens - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(lens)
    j = first[:, None] + torch.arange(s["span"], device="cuda")
    valid = j < lens[:, None]
    j = torch.where(valid, j, 0)
    pages = s["table"].long().gather(1, j // page).clamp(min=0)
    k = s["k_cache"][pages, j % page].float()  # [B, span, K, D]
    v = s["v_cache"][pages, j % page].float()
    v = torch.where(valid[:, :, None, None], v, 0)
    q = s["q"].float().view(B, K, H // K, D)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * D ** -0.5
    x = torch.where(valid[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2)) / torch.where(total == 0, 1, total)
    return out.reshape(B, H, D).to(s["q"].dtype)


def _turn(x, c, sn, rope, pairing):
    """x [T, heads, D] with its first `rope` values turned by (c, sn) [T, 1, rope / 2]."""
    r, rest = x[..., :rope], x[..., rope:]
    a, b = (r[..., :rope // 2], r[..., rope // 2:]) if pairing == "halves" else (r[..., 0::2], r[..., 1::2])
    y = (a * c - b * sn, a * sn + b * c)
    y = torch.cat(y, -1) if pairing == "halves" else torch.stack(y, -1).flatten(-2)
    return torch.cat([y, rest], -1)


def plain_norm_rope(s):
    def norm(x, w):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w

    t = s["rope_table"]
    if s["pair_axis"] is not None:
        i = torch.arange(s["rope"] // 2, device="cuda")
        t = t[s["positions"].long()[s["pair_axis"].long()], i[:, None]].transpose(0, 1)
    else:
        t = t[s["positions"].long()]
    c, sn = t[:, None, :, 0], t[:, None, :, 1]
    q = _turn(norm(s["q"], s["q_weight"]), c, sn, s["rope"], s["pairing"])
    k = _turn(norm(s["k"], s["k_weight"]), c, sn, s["rope"], s["pairing"])
    at = (s["slots"] // s["page"], s["slots"] % s["page"])
    s["k_cache"][at] = k.to(s["k_cache"].dtype)
    s["v_cache"][at] = s["v"].float().to(s["v_cache"].dtype)
    return {"q": q.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def plain_route(s):
    x = s["logits"].float()
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    top, ids = top[:, :s["used"]], ids[:, :s["used"]]
    e = torch.exp(top - top[:, :1])
    total = e.sum(-1, keepdim=True) if s["renorm"] else torch.exp(x - top[:, :1]).sum(-1, keepdim=True)
    return {"ids": ids.int(), "w": e / total}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "attend":
        keys = sum(min(n, case["window"]) if case["window"] else n for n in lengths(case))
        ends = 2 * case["seqs"] * case["heads"] * case["dim"] * BYTES[case["act"]]
        return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 * BYTES[case["cache"]] + ends + 8 * case["seqs"],
                "flops": 4 * keys * case["heads"] * case["dim"]}
    if case["op"] == "norm_rope":
        T, D, K = case["tokens"], case["dim"], case["kv_heads"]
        row = (2 * case["heads"] + 2 * K) * BYTES[case["act"]] + 2 * K * BYTES[case["cache"]]
        return {"bytes": T * (D * row + 4 * case["rope"] + 4 * case["axes"] + 8) + 8 * D,
                "flops": T * (case["heads"] + K) * (4 * D + 3 * case["rope"])}
    T, E = case["tokens"], case["experts"]
    return {"bytes": T * (E * BYTES[case["act"]] + 8 * case["used"]), "flops": 3 * T * E}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        B, H, D, K, page = case["seqs"], case["heads"], case["dim"], case["kv_heads"], case["page"]
        out = torch.zeros(B, H, D, device="cuda", dtype=torch.float64)
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - case["window"]) if case["window"] else 0
            if n == lo:
                continue
            rows = [s[c].index_select(0, s["table"][b, lo // page:-(-n // page)].long()).flatten(0, 1)
                    [lo - lo // page * page:n - lo // page * page] for c in ("k_cache", "v_cache")]
            for h in range(H):
                x = rows[0][:, h * K // H].double() @ s["q"][b, h].double() / math.sqrt(D)
                out[b, h] = torch.softmax(x, 0) @ rows[1][:, h * K // H].double()
        return out
    if case["op"] == "norm_rope":
        rope = case["rope"]
        half = torch.arange(rope // 2, device="cuda")
        first, second = (half, half + rope // 2) if case["pairing"] == "halves" else (2 * half, 2 * half + 1)
        p = s["positions"].long().view(case["axes"], -1)
        axis = half * 0 if s["pair_axis"] is None else s["pair_axis"].long()
        z = torch.view_as_complex(s["rope_table"].double()[p[axis].t(), half])[:, None]
        done = []
        for x, w in ((s["q"].double(), s["q_weight"].double()), (s["k"].double(), s["k_weight"].double())):
            y = w * x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + EPS)
            u = torch.complex(y[..., first], y[..., second]) * z
            y[..., first], y[..., second] = u.real, u.imag
            done.append(y)
        caches = []
        for name, new in (("k_cache", done[1]), ("v_cache", s["v"].double())):
            c = s[name].double().contiguous()
            c.view(-1, case["kv_heads"], case["dim"])[s["slots"]] = new
            caches.append(c)
        return {"q": done[0], "k_cache": caches[0], "v_cache": caches[1]}
    x = s["logits"].double()
    # an expert's rank: how many logits are larger, or as large and of a lower index
    E = case["experts"]
    if case["tokens"] * E * E < 1 << 24:
        rank = (x[:, None, :] > x[:, :, None]).sum(-1)
        low = torch.ones(E, E, device="cuda", dtype=torch.bool).tril(-1)
        rank += ((x[:, None, :] == x[:, :, None]) & low).sum(-1)
        ids = rank.argsort(-1)[:, :case["used"]]
    else:
        ids = torch.argsort(-x, dim=-1, stable=True)[:, :case["used"]]
    p = torch.softmax(x, -1).gather(1, ids)
    return {"ids": ids.int(), "w": p / p.sum(-1, keepdim=True) if case["renorm"] else p}
