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
# the step around the experts: attention over a paged cache, the router. Inputs
# are checked (ValueError); outputs that are not given come from torch's
# allocator on the stream that the kernel runs on: the current one, or `stream`.
# ---------------------------------------------------------------------------
_native = None


def _ops():
    """The native side of these calls (csrc/sb_torch.cpp): argument checks, outputs, the current
    stream. Bound to the loaded runtime once."""
    global _native
    if _native is None:
        L = rt.lib()
        try:
            from . import _torch_ops
        except ImportError as e:
            raise rt.RuntimeUnavailable("could not load _torch_ops.so (%s): build it with make -C "
                                        "sabah_moe_accelerator_b200/csrc" % e)
        _torch_ops.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            L.sabah_qk_norm_rope, L.sabah_attend_paged, L.sabah_attend_paged_workspace, L.sabah_route_topk,
            L.sabah_rt_last_error)), rt.SabahCudaError)
        _native = _torch_ops
    return _native


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
    if pairing != "halves" and pairing != "pairs":
        raise ValueError('pairing: "halves" or "pairs"')
    k_cache, v_cache, slots = cache if cache is not None else (None, None, None)
    args = (q, k, v, q_weight, k_weight, table, positions, eps, pairing == "pairs", pair_axis, k_cache, v_cache, slots,
            q_out, k_out)
    if stream is None:
        return (_native or _ops()).norm_rope(*args)
    with torch.cuda.stream(stream):
        return _ops().norm_rope(*args)


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
    args = (q, k_cache, v_cache, block_table, lens, scale, window, out, lse, workspace)
    if stream is None:
        return (_native or _ops()).attend(*args)
    with torch.cuda.stream(stream):
        return _ops().attend(*args)


def route_topk(logits: torch.Tensor, n_used: int, *, renorm: bool = True, scale: float = 1.0,
               ids: torch.Tensor | None = None, w: torch.Tensor | None = None, stream=None):
    """(ids int32, w float32) [T, n_used] for moe_block_ids from router logits [T, n_experts].

    The n_used largest logits per token, ties to the lower index, in descending
    order; w is their softmax times scale, over the chosen (renorm) or all experts.
    """
    if stream is None:
        return (_native or _ops()).route(logits, n_used, renorm, scale, ids, w)
    with torch.cuda.stream(stream):
        return _ops().route(logits, n_used, renorm, scale, ids, w)
