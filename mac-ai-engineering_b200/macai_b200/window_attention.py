"""Causal softmax attention with a sliding window and first tokens that stay visible, the mixer of the layers that
alternate with the gated delta rule's, on B200 (C ABI gd_wattn_* in libgated_delta_b200.so):

    o = softmax(scale q k^T over the visible keys) v

Query i of T_q stands at position p = i + T_k - T_q (the queries are the last T_q positions) and sees key j when j <= p and
(j > p - window or j < sinks); a query that sees no key gets zeros. `window_attention` trains and prefills (tcgen05
products, probabilities rounded to the inputs' 16-bit type as the matrix instruction's operand, everything else float32);
`window_attention_step` is the single-token form over a cache. bfloat16 and float16. There is no CPU path: CUDA tensors
only.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
MAX_D = 256


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [B, T, heads, D] if the kernels can read it in place (adjacent channels, 16-byte aligned rows), else a copy."""
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(
        n <= 1 or (s >= 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride()[:3]))
    return t if ok else t.contiguous().clone() if t.is_contiguous() else t.contiguous()


def _strides(*ts):
    return (ctypes.c_longlong * (3 * len(ts)))(*[s for t in ts for s in t.stride()[:3]])


def _stream(t: torch.Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def _fwd(q, k, v, cu, window, sinks, scale):
    lib = _lib.load()
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1:3]
    o = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Tq), dtype=torch.float32, device=q.device)
    ws = torch.empty(64, dtype=torch.uint8, device=q.device)  # gd_wattn_workspace_bytes(..., for_backward=0)
    with torch.cuda.device(q.device):
        st = lib.gd_wattn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), _p(cu),
                              0 if cu is None else cu.numel() - 1, _DTYPES[q.dtype], B, Tq, Tk, H, HK, D,
                              _strides(q, k, v), window, sinks, scale, ws.data_ptr(), 64, _stream(q))
    _lib.check(st, "gd_wattn_fwd")
    return o, lse


@torch.library.custom_op("macai_b200::window_attention_fwd", mutates_args=(), device_types="cuda")
def window_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
                         window: int, sinks: int, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(o [B, Tq, H, D], lse [B, H, Tq] float32, the log2-sum of a row's exponentials); window 0: none."""
    return _fwd(q, k, v, cu_seqlens, window, sinks, scale)


@window_attention_fwd.register_fake
def _(q, k, v, cu_seqlens, window, sinks, scale):
    return q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)


@torch.library.custom_op("macai_b200::window_attention_bwd", mutates_args=(), device_types="cuda")
def window_attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                         do: torch.Tensor, cu_seqlens: Optional[torch.Tensor], window: int, sinks: int,
                         scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv), contiguous, in the inputs' dtype."""
    lib = _lib.load()
    q, k, v, do = _rows(q), _rows(k), _rows(v), _rows(do)
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1:3]
    dq, dk, dv = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    n = lib.gd_wattn_workspace_bytes(B, Tq, Tk, H, HK, D, window, sinks, cu_seqlens is not None, 1)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        st = lib.gd_wattn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), do.data_ptr(),
                              dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _p(cu_seqlens),
                              0 if cu_seqlens is None else cu_seqlens.numel() - 1, _DTYPES[q.dtype], B, Tq, Tk, H, HK, D,
                              _strides(q, k, v, do), window, sinks, scale, ws.data_ptr(), n, _stream(q))
    _lib.check(st, "gd_wattn_bwd")
    return dq, dk, dv


@window_attention_bwd.register_fake
def _(q, k, v, o, lse, do, cu_seqlens, window, sinks, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _setup_context(ctx, inputs, output):
    q, k, v, cu_seqlens, window, sinks, scale = inputs
    ctx.save_for_backward(q, k, v, cu_seqlens, *output)
    ctx.mask = (window, sinks, scale)
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])


def _backward(ctx, do, _):
    if do is None:
        return None, None, None, None, None, None, None
    q, k, v, cu_seqlens, o, lse = ctx.saved_tensors
    dq, dk, dv = window_attention_bwd(q, k, v, o, lse, do.to(q.dtype), cu_seqlens, *ctx.mask)
    return dq, dk, dv, None, None, None, None


window_attention_fwd.register_autograd(_backward, setup_context=_setup_context)


def _check_qkv(name, q, k, v):
    for x, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{name}: {x} must be [B, T, heads, D]")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name}: bfloat16 or float16, got {t.dtype} for {x}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name}: q, k and v must share one dtype and device")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"{name}: k and v [B, T_k, H_k, D] must agree with each other and with q's batch and head width")
    if q.shape[2] == 0 or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{name}: {q.shape[2]} query heads are no multiple of {k.shape[2]} key heads")
    if not 0 < q.shape[3] <= MAX_D or q.shape[3] % 8:
        raise NotImplementedError(f"{name}: head widths are multiples of 8 up to {MAX_D}, got {q.shape[3]}")


def _check_mask(name, window, sinks):
    if window is not None and (not isinstance(window, int) or window <= 0):
        raise ValueError(f"{name}: window must be a positive int or None, got {window!r}")
    if not isinstance(sinks, int) or sinks < 0:
        raise ValueError(f"{name}: sinks must be a non-negative int, got {sinks!r}")
    return min(window or 0, 0x3FFFFFFF), min(sinks, 0x3FFFFFFF)


def _check_cu(cu, q, k):
    """Packed rows' boundaries as the kernels read them (int32 on q's device); a list given on the host is checked."""
    if cu is None:
        return None
    if q.shape[0] != 1 or q.shape[1] != k.shape[1]:
        raise ValueError("window_attention: cu_seqlens needs batch size 1 and as many queries as keys")
    if not isinstance(cu, torch.Tensor) or cu.dim() != 1 or cu.numel() < 2 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError("window_attention: cu_seqlens must be an integer [N + 1] tensor")
    if not cu.is_cuda:
        c = cu.tolist()
        if c[0] != 0 or c[-1] != q.shape[1] or any(b < a for a, b in zip(c, c[1:])):
            raise ValueError(f"window_attention: cu_seqlens must rise from 0 to {q.shape[1]}, got {c}")
    return cu.to(device=q.device, dtype=torch.int32).contiguous()


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     scale: Optional[float] = None, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [B, T_q, H, D] for q [B, T_q, H, D] and k, v [B, T_k, H_k, D] (H a multiple of H_k: each key head serves
    H / H_k consecutive query heads), bfloat16 or float16, D a multiple of 8 up to 256. Each query sees its own position
    and those before it, of which the last `window` (None: all) and the first `sinks`. scale: of the scores, default
    D^-0.5. cu_seqlens: int [N + 1], the boundaries of N sequences packed along the tokens of one batch row, each on its
    own (positions count from its first token, also for `sinks`). Inputs may be strided views; gradients are the same
    bits every run."""
    _check_qkv("window_attention", q, k, v)
    w, s = _check_mask("window_attention", window, sinks)
    cu = _check_cu(cu_seqlens, q, k)
    if not q.is_cuda:
        raise RuntimeError("window_attention: CUDA tensors only (there is no CPU path)")
    scale = float(q.shape[3] ** -0.5 if scale is None else scale)
    if torch.compiler.is_compiling() or (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return window_attention_fwd(q, k, v, cu, w, s, scale)[0]
    return _fwd(q, k, v, cu, w, s, scale)[0]
