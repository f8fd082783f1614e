"""PyTorch-facing wrappers over the C ABI.

torch provides device memory and the current stream; every computation runs in
libsabah_rt.so. Tensors are passed by data_ptr(), streams by cuda_stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import rt

_initialised_device = None


def init(device: int = 0) -> None:
    """sabah_rt_init once per process (re-initialising resets the hot tier)."""
    global _initialised_device
    if _initialised_device is None:
        torch.cuda.set_device(device)
        rt.check(rt.lib().sabah_rt_init(device), "sabah_rt_init")
        _initialised_device = device


def _stream(stream) -> int:
    """Raw stream handle for the C ABI. torch's default stream has handle 0,
    which the ABI reads as "the runtime's own stream"; it is passed as the
    explicit legacy-stream handle (cudaStreamLegacy = 1) instead."""
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream or 1


def _ptr(t) -> int:
    if isinstance(t, torch.Tensor):
        return t.data_ptr()
    return int(t.ctypes.data)   # numpy array (host-backed source)


def row_bytes(qt: int, k: int) -> int:
    return rt.row_bytes(qt, k)


def synth_rows(n_rows: int, k: int, qt: int, seed: int, sigma: float = 0.02, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
    """n_rows dense rows of k elements of type qt encoding N(0, sigma) weights."""
    nbytes = n_rows * rt.row_bytes(qt, k)
    if out is None:
        out = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    assert out.numel() >= nbytes and out.is_cuda
    rt.check(rt.lib().sabah_synth_rows(ctypes.c_void_p(out.data_ptr()), qt, n_rows, k, seed, sigma,
                                       ctypes.c_void_p(_stream(stream))), "synth_rows")
    return out


def mul_mat_id(source, expert_stride: int, row_stride: int, x: torch.Tensor, ids: torch.Tensor, rows: int,
               k: int, n_experts: int, qt: int, out: torch.Tensor | None = None, stream=None, ids_key=None):
    """MUL_MAT_ID through sabah_rt_mul_mat_id_v2 on dense tensors.

    source: the expert tensor (a CUDA uint8 tensor = resident bank, or a host
    numpy array = the hot-tier path). x: [T, x_rows, k] float32, ids: [T, n_ids]
    int32, out: [T, n_ids, rows] float32.
    """
    T, n_ids = ids.shape
    x_rows = x.shape[1]
    assert x.shape == (T, x_rows, k) and x.dtype == torch.float32 and x.is_contiguous()
    assert ids.dtype == torch.int32 and ids.is_contiguous()
    if out is None:
        out = torch.empty((T, n_ids, rows), dtype=torch.float32, device="cuda")
    rc = rt.mul_mat_id_v2(_ptr(source), expert_stride, row_stride, x.data_ptr(), k * 4, x_rows, x_rows * k * 4,
                          ids.data_ptr(), 4, n_ids * 4, n_ids, T, out.data_ptr(), rows * 4, n_ids * rows * 4,
                          rows, k, n_experts, qt, _stream(stream), ids_key)
    rt.check(rc, "sabah_rt_mul_mat_id_v2")
    return out


def moe_block_ids(gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, ids: torch.Tensor, w: torch.Tensor,
                  x: torch.Tensor, d_model: int, ff: int, n_experts: int, qt_gate: int, qt_up: int, qt_down: int,
                  out: torch.Tensor | None = None, h: torch.Tensor | None = None, accumulate: bool = False,
                  stream=None) -> torch.Tensor:
    """Fused routed block on device-resident banks: out (+)= sum_e w * Wd (silu(Wg x) * Wu x)."""
    T, n_used = ids.shape
    if out is None:
        out = torch.empty((T, d_model), dtype=torch.float32, device="cuda")
    if h is None:
        h = torch.empty((T, n_used, ff), dtype=torch.float32, device="cuda")
    gs = ff * rt.row_bytes(qt_gate, d_model)
    ds = d_model * rt.row_bytes(qt_down, ff)
    assert rt.row_bytes(qt_up, d_model) == rt.row_bytes(qt_gate, d_model)
    L = rt.lib()
    rc = L.sabah_moe_block_ids(ctypes.c_void_p(gate.data_ptr()), ctypes.c_void_p(up.data_ptr()),
                               ctypes.c_void_p(down.data_ptr()), gs, ds, n_experts,
                               ctypes.c_void_p(ids.data_ptr()), ctypes.c_void_p(w.data_ptr()),
                               ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(out.data_ptr()),
                               ctypes.c_void_p(h.data_ptr()), d_model, ff, n_used, T, qt_gate, qt_up, qt_down,
                               1 if accumulate else 0, ctypes.c_void_p(_stream(stream)))
    rt.check(rc, "sabah_moe_block_ids")
    return out


# ---------------------------------------------------------------------------
# the step around the experts: attention over a paged cache, the router
# ---------------------------------------------------------------------------
_ACT = {torch.float32: rt.ACT_F32, torch.float16: rt.ACT_F16, torch.bfloat16: rt.ACT_BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _empty(shape, dtype, like: torch.Tensor, stream) -> torch.Tensor:
    """Device memory that belongs to the stream the kernel runs on."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=like.device)


def _cache_shape(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor) -> tuple:
    """Shape and byte strides of a cache [pages, page_size, kv_heads, head_dim]."""
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "caches: two of [pages, page_size, kv_heads, head_dim]")
    _need(k_cache.dtype == v_cache.dtype and k_cache.dtype in (torch.float16, torch.bfloat16), "caches: f16 or bf16")
    _need(k_cache.device == v_cache.device == like.device, "caches: on the device of the other tensors")
    ks, vs = k_cache.stride(), v_cache.stride()
    _need(k_cache.numel() == 0 or (ks[3] == 1 and vs[3] == 1), "caches: head_dim must be dense")
    return k_cache.shape, (2 * ks[0], 2 * ks[1], 2 * ks[2]), (2 * vs[0], 2 * vs[1], 2 * vs[2])


def rope_table(n_positions: int, rope_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """[n_positions, rope_dim / 2, 2] float32 (cos, sin) of position * theta^(-2i / rope_dim),
    computed in 64 bits; lay it out once and pass it to qk_norm_rope."""
    f = theta ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64, device=device) / rope_dim)
    a = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, q_weight: torch.Tensor | None,
                 k_weight: torch.Tensor | None, table: torch.Tensor | None, positions: torch.Tensor | None, *,
                 eps: float = 1e-6, pairing: str = "halves", pair_axis: torch.Tensor | None = None,
                 cache: tuple | None = None, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 stream=None):
    """Per-head RMS norms of q and k, the position rotation and the cache write, in one launch.

    q [T, q_heads, D], k and v [T, kv_heads, D]: f32, f16 or bf16 with a dense
    last dimension (views of one fused projection will do). q_weight, k_weight
    [D] float32, or None for no norm. table: rope_table()'s, or None for no
    rotation; positions int32 [T] or [axes, T], and then pair_axis uint8
    [rope_dim / 2] names the axis of each pair. pairing: "halves" or "pairs".
    cache = (k_cache, v_cache, slots): pages [pages, page_size, kv_heads, D] of
    f16 or bf16 and the int64 row of each token (negative: none); returns q_out.
    Without a cache v is not read, and (q_out, k_out) is returned.
    """
    T, n_q, D = q.shape
    _need(k.dim() == 3 and k.shape[0] == T and k.shape[2] == D, "k: [tokens, kv_heads, head_dim] beside q")
    n_kv = k.shape[1]
    act = _ACT.get(q.dtype)
    _need(act is not None and k.dtype == q.dtype, "q and k: both f32, f16 or bf16")
    _need(q.is_cuda and k.device == q.device, "q and k: on one CUDA device")
    _need(pairing == "halves" or pairing == "pairs", 'pairing: "halves" or "pairs"')
    eb = q.element_size()
    qs, ks, vs = q.stride(), k.stride(), (0, 0, 1)
    _need(q.numel() == 0 or qs[2] == 1, "q: head_dim must be dense")
    _need(k.numel() == 0 or ks[2] == 1, "k: head_dim must be dense")
    for w in (q_weight, k_weight):
        _need(w is None or (w.shape == (D,) and w.dtype == torch.float32 and w.is_contiguous()
                            and w.device == q.device), "norm weights: dense float32 [head_dim] or None")
    n_pos = rope = axes = 0
    if table is not None:
        _need(table.dim() == 3 and table.shape[2] == 2 and table.dtype == torch.float32 and table.is_contiguous()
              and table.device == q.device, "table: dense float32 [positions, rope_dim / 2, 2]")
        n_pos, rope = table.shape[0], 2 * table.shape[1]
        _need(positions is not None and positions.dtype == torch.int32 and positions.is_contiguous()
              and positions.shape[-1:] == (T,) and positions.dim() <= 2 and positions.device == q.device,
              "positions: dense int32 [tokens] or [axes, tokens]")
        axes = positions.shape[0] if positions.dim() == 2 else 1
        _need(pair_axis is None or (pair_axis.shape == (rope // 2,) and pair_axis.dtype == torch.uint8
                                    and pair_axis.is_contiguous() and pair_axis.device == q.device),
              "pair_axis: dense uint8 [rope_dim / 2]")
    kc = vc = (0, 0, 0)
    n_pages = page_size = ctype = 0
    k_cache = v_cache = slots = None
    if cache is not None:
        k_cache, v_cache, slots = cache
        shape, kc, vc = _cache_shape(k_cache, v_cache, q)
        n_pages, page_size = shape[0], shape[1]
        _need(shape[2] == n_kv and shape[3] == D, "caches: kv_heads and head_dim as k's")
        _need(v is not None and v.shape == k.shape and v.dtype == k.dtype and v.device == k.device, "v: as k")
        vs = v.stride()
        _need(v.numel() == 0 or vs[2] == 1, "v: head_dim must be dense")
        _need(slots.shape == (T,) and slots.dtype == torch.int64 and slots.is_contiguous()
              and slots.device == q.device, "slots: dense int64 [tokens]")
        ctype = _ACT[k_cache.dtype]
    elif k_out is None:
        k_out = _empty((T, n_kv, D), q.dtype, q, stream)
    if q_out is None:
        q_out = _empty((T, n_q, D), q.dtype, q, stream)
    _need(q_out.shape == q.shape and q_out.dtype == q.dtype and q_out.is_contiguous() and q_out.device == q.device,
          "q_out: dense, as q")
    _need(k_out is None or (k_out.shape == k.shape and k_out.dtype == k.dtype and k_out.is_contiguous()
                            and k_out.device == k.device), "k_out: dense, as k")
    rc = rt.lib().sabah_qk_norm_rope(
        q.data_ptr(), eb * qs[0], eb * qs[1], n_q, k.data_ptr(), eb * ks[0], eb * ks[1],
        None if cache is None else v.data_ptr(), eb * vs[0], eb * vs[1], n_kv, T, D, act,
        None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
        None if table is None else table.data_ptr(), n_pos, rope, pairing == "pairs",
        None if table is None else positions.data_ptr(), axes,
        None if table is None or pair_axis is None else pair_axis.data_ptr(), q_out.data_ptr(),
        None if k_out is None else k_out.data_ptr(),
        None if cache is None else k_cache.data_ptr(), kc[0], kc[1], kc[2],
        None if cache is None else v_cache.data_ptr(), vc[0], vc[1], vc[2], n_pages, page_size, ctype,
        None if cache is None else slots.data_ptr(), _stream(stream))
    rt.check(rc, "sabah_qk_norm_rope")
    return q_out if cache is not None else (q_out, k_out)


def attend_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 lens: torch.Tensor, *, scale: float | None = None, window: int = 0,
                 out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of one new token per sequence over the paged cache.

    q [B, q_heads, D] f32 or the cache's type; caches [pages, page_size,
    kv_heads, D] f16 or bf16 (any order of memory with a dense D and rows at
    multiples of 16 bytes); block_table int32 [B, pages per sequence]; lens int32
    [B], the new token's own key included. window: only the last `window` keys
    (0: all). scale: 1 / sqrt(D) by default. lse: float32 [B, q_heads] to fill.
    workspace: uint8 memory of rt.lib().sabah_attend_paged_workspace(q_heads,
    kv_heads, D) bytes, by default from torch's allocator for each call.
    """
    B, H, D = q.shape
    act = _ACT.get(q.dtype)
    (n_pages, page_size, n_kv, cd), kc, vc = _cache_shape(k_cache, v_cache, q)
    _need(act is not None and (act == rt.ACT_F32 or q.dtype == k_cache.dtype), "q: f32 or the cache's type")
    _need(cd == D and n_kv > 0 and H % n_kv == 0, "q heads: a multiple of the cache's, of one head_dim")
    _need(q.is_cuda, "q: on a CUDA device")
    qs, eb = q.stride(), q.element_size()
    _need(q.numel() == 0 or qs[2] == 1, "q: head_dim must be dense")
    _need(block_table.dim() == 2 and block_table.shape[0] == B and block_table.dtype == torch.int32
          and (block_table.shape[1] <= 1 or block_table.stride(1) == 1) and block_table.device == q.device,
          "block_table: int32 [sequences, pages per sequence]")
    _need(lens.shape == (B,) and lens.dtype == torch.int32 and lens.is_contiguous() and lens.device == q.device,
          "lens: dense int32 [sequences]")
    if out is None:
        out = _empty((B, H, D), q.dtype, q, stream)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous() and out.device == q.device,
              "out: dense, as q")
    _need(lse is None or (lse.shape == (B, H) and lse.dtype == torch.float32 and lse.is_contiguous()
                          and lse.device == q.device), "lse: dense float32 [sequences, q_heads]")
    L = rt.lib()
    if workspace is None:
        workspace = _empty(L.sabah_attend_paged_workspace(H, n_kv, D), torch.uint8, q, stream)
    else:
        _need(workspace.is_contiguous() and workspace.device == q.device, "workspace: dense, on q's device")
    rc = L.sabah_attend_paged(
        q.data_ptr(), eb * qs[0], eb * qs[1], act, k_cache.data_ptr(), kc[0], kc[1], kc[2],
        v_cache.data_ptr(), vc[0], vc[1], vc[2], _ACT[k_cache.dtype], n_pages, page_size, block_table.data_ptr(),
        4 * block_table.stride(0), block_table.shape[1], lens.data_ptr(), B, H, n_kv, D,
        D ** -0.5 if scale is None else scale, window, out.data_ptr(), None if lse is None else lse.data_ptr(),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(stream))
    rt.check(rc, "sabah_attend_paged")
    return out


def route_topk(logits: torch.Tensor, n_used: int, *, renorm: bool = True, scale: float = 1.0,
               ids: torch.Tensor | None = None, w: torch.Tensor | None = None, stream=None):
    """(ids int32, w float32) [T, n_used] for moe_block_ids from router logits [T, n_experts].

    The n_used largest logits per token, ties to the lower index, in descending
    order; w is their softmax times scale, over the chosen (renorm) or all experts.
    """
    T, E = logits.shape
    act = _ACT.get(logits.dtype)
    _need(act is not None and logits.is_cuda, "logits: f32, f16 or bf16 on a CUDA device")
    _need(logits.numel() == 0 or E == 1 or logits.stride(1) == 1, "logits: experts must be dense")
    if ids is None:
        ids = _empty((T, n_used), torch.int32, logits, stream)
    if w is None:
        w = _empty((T, n_used), torch.float32, logits, stream)
    for t, dt in ((ids, torch.int32), (w, torch.float32)):
        _need(t.shape == (T, n_used) and t.dtype == dt and t.is_contiguous() and t.device == logits.device,
              "ids and w: dense int32 and float32 [tokens, n_used]")
    rc = rt.lib().sabah_route_topk(logits.data_ptr(), logits.element_size() * logits.stride(0), act, T, E, n_used,
                                   renorm, scale, ids.data_ptr(), w.data_ptr(), _stream(stream))
    rt.check(rc, "sabah_route_topk")
    return ids, w
