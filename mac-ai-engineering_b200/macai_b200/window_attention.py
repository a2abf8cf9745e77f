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
    n = lib.gd_wattn_workspace_bytes(B, Tq, Tk, H, HK, D, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        st = lib.gd_wattn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), _p(cu),
                              0 if cu is None else cu.numel() - 1, _DTYPES[q.dtype], B, Tq, Tk, H, HK, D,
                              _strides(q, k, v), window, sinks, scale, ws.data_ptr(), n, _stream(q))
    _lib.check(st, "gd_wattn_fwd")
    return o, lse


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


def window_attention(q, k, v, window=None, sinks=0, scale=None, cu_seqlens=None):
    _check_qkv("window_attention", q, k, v)
    w, s = _check_mask("window_attention", window, sinks)
    return _fwd(q, k, v, cu_seqlens, w, s, float(scale if scale is not None else q.shape[3] ** -0.5))[0]
