"""Causal softmax attention with a sliding window and first tokens that stay visible, the mixer of the layers that
alternate with the gated delta rule's, on B200 (C ABI gd_wattn_* in libgated_delta_b200.so):

    o = softmax(scale q k^T over the visible keys) v

Query i of T_q stands at position p = i + T_k - T_q (the queries are the last T_q positions) and sees key j when j <= p and
(j > p - window or j < sinks); a query that sees no key gets zeros. `window_attention` trains and prefills: tcgen05
products; the probabilities and the scores' gradients are rounded to the inputs' 16-bit type as the matrix instruction's
operands, everything else is float32. Masked scores are never used; a masked value's infinity or NaN still meets a weight of
0 in the products of its tile, as in the formula's matrix product, except across packed sequences, which stay apart.
`window_attention_step` is the single-token form over a cache. bfloat16 and float16. There is no CPU path: CUDA tensors
only.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._call import aligned, first_order, launch, like, recorded

_DTYPES = {torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
MAX_D = 256


@functools.lru_cache(maxsize=1024)
def _bwd_bytes(*sizes) -> int:
    return _lib.load().gd_wattn_workspace_bytes(*sizes, 1)


@functools.lru_cache(maxsize=1024)
def _step_bytes(*sizes) -> int:
    return _lib.load().gd_wattn_step_workspace_bytes(*sizes)


def _readable(t: torch.Tensor) -> bool:
    """Whether the kernels can read t [B, T, heads, D] in place: adjacent channels, 16-byte aligned rows of their own (an
    expanded dimension has the stride 0, which the tensor maps are not documented to take)."""
    if t.data_ptr() % 16:
        return False
    if t.is_contiguous():
        return True
    b, s, h, d = t.stride()
    B, T, H, _ = t.shape
    return (d == 1 and (B <= 1 or (b > 0 and b % 8 == 0)) and (T <= 1 or (s > 0 and s % 8 == 0))
            and (H <= 1 or (h > 0 and h % 8 == 0)))


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if _readable(t) else aligned(t)


def _strides(*ts):
    return (ctypes.c_longlong * (3 * len(ts)))(*[s for t in ts for s in t.stride()[:3]])


def _fwd(q, k, v, cu, window, sinks, scale, keep):
    """(o, o_low, lse) on readable inputs; keep: for the backward, o_low, what o's rounding took away, and lse (else None)."""
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1], k.shape[2]
    o = like(q)
    low = lse = None
    if keep:
        low, lse = like(q), torch.empty((B, H, Tq), dtype=torch.float32, device=q.device)
    launch("gd_wattn_fwd", q.get_device(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
           None if low is None else low.data_ptr(), None if lse is None else lse.data_ptr(),
           None if cu is None else cu.data_ptr(), 0 if cu is None else cu.numel() - 1, _DTYPES[q.dtype], B, Tq, Tk, H, HK, D,
           _strides(q, k, v), window, sinks, scale, None, 0)
    return o, low, lse


def _bwd(q, k, v, o, low, lse, do, cu, window, sinks, scale):
    """(dq, dk, dv), contiguous, on readable inputs."""
    B, Tq, H, D = q.shape
    Tk, HK = k.shape[1], k.shape[2]
    dq, dk, dv = like(q), like(k), like(v)
    n = _bwd_bytes(B, Tq, Tk, H, HK, D, window, sinks, cu is not None)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    launch("gd_wattn_bwd", q.get_device(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), low.data_ptr(),
           lse.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None if cu is None else cu.data_ptr(),
           0 if cu is None else cu.numel() - 1, _DTYPES[q.dtype], B, Tq, Tk, H, HK, D, _strides(q, k, v, do), window,
           sinks, scale, ws.data_ptr(), n)
    return dq, dk, dv


class WindowAttention(torch.autograd.Function):
    """`WindowAttention.apply(q, k, v, cu_seqlens or None, window (0: none), sinks, scale)` on readable inputs."""

    @staticmethod
    def forward(ctx, q, k, v, cu, window, sinks, scale):
        o, low, lse = _fwd(q, k, v, cu, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, o, low, lse, cu)
        ctx.args = (window, sinks, scale)
        return o

    @staticmethod
    @first_order
    def backward(ctx, do):
        q, k, v, o, low, lse, cu = ctx.saved_tensors
        return (*_bwd(q, k, v, o, low, lse, _rows(do), cu, *ctx.args), None, None, None, None)


def _check_qkv(name, q, k, v):
    for x, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{name}: {x} must be [B, T, heads, D]")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name}: bfloat16 or float16, got {t.dtype} for {x}")
        if t.dtype != q.dtype or t.get_device() != q.get_device():
            raise ValueError(f"{name}: q, k and v must share one dtype and device")
    if not q.is_cuda:
        raise RuntimeError(f"{name}: CUDA tensors only (there is no CPU path)")
    B, _, H, D = q.shape
    kb, _, HK, kd = k.shape
    if k.shape != v.shape or kb != B or kd != D:
        raise ValueError(f"{name}: k and v [B, T_k, H_k, D] must agree with each other and with q's batch and head width")
    if H == 0 or HK == 0 or H % HK:
        raise ValueError(f"{name}: {H} query heads are no multiple of {HK} key heads")
    if not 0 < D <= MAX_D or D % 8:
        raise NotImplementedError(f"{name}: head widths are multiples of 8 up to {MAX_D}, got {D}")


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
    and those before it, of which the last `window` (None: all) and the first `sinks`. scale: of the scores, any finite
    number, default D^-0.5. cu_seqlens: int [N + 1], the boundaries of N sequences packed along the tokens of one batch
    row, each on its own (positions count from its first token, also for `sinks`). A list on the host must rise from 0 to
    T; one on the device is not looked at by the host: rows before its first and behind its last boundary give zeros, in o
    and in the gradients, and a boundary below an earlier one counts as that one. Inputs may be strided views
    (expanded ones are copied); gradients are the same bits every run."""
    _check_qkv("window_attention", q, k, v)
    w, s = _check_mask("window_attention", window, sinks)
    cu = _check_cu(cu_seqlens, q, k)
    scale = float(q.shape[3] ** -0.5 if scale is None else scale)
    q_, k_, v_ = _rows(q), _rows(k), _rows(v)
    if recorded(q, k, v):
        return WindowAttention.apply(q_, k_, v_, cu, w, s, scale)
    return _fwd(q_, k_, v_, cu, w, s, scale, False)[0]


def window_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, lengths: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                          scale: Optional[float] = None) -> torch.Tensor:
    """One new token for each request: stores its key and value in the caches (in place) and returns its attention
    o [B, 1, H, D] over the visible positions, its own included. q [B, 1, H, D], k, v [B, 1, H_k, D], k_cache, v_cache
    [B, S, H_k, D] (any strides with adjacent channels and 16-byte aligned rows that share no memory), lengths int32 [B] on
    the device: the tokens in each request's cache before the call, which is the new token's position. The caller adds 1 to
    lengths after its last layer. A negative length marks an idle request: zeros, nothing stored.

    Position j stands in slot j while j < S, then in slot sinks + (j - sinks) mod (S - sinks): with S >= sinks + window the
    cache rolls, keeping its first `sinks` tokens, and requests may grow without limit; a smaller cache then shows the last
    S - sinks positions. No gradient. Nothing waits for the host."""
    _check_qkv("window_attention_step", q, k, v)
    w, s = _check_mask("window_attention_step", window, sinks)
    B, t, H, D = q.shape
    HK, index = k.shape[2], q.get_device()
    if t != 1 or k.shape[1] != 1:
        raise ValueError("window_attention_step: one token a request (q [B, 1, H, D], k and v [B, 1, H_k, D])")
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor) or k_cache.dim() != 4:
        raise ValueError("window_attention_step: k_cache and v_cache must be [B, S, H_k, D]")
    S = k_cache.shape[1]
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.shape != (B, S, HK, D) or S == 0 or c.dtype != q.dtype or c.get_device() != index:
            raise ValueError(f"window_attention_step: {name} must be [B, S, H_k, D] with k's batch, heads, width, dtype and "
                             "device")
        if not _readable(c):
            raise ValueError(f"window_attention_step: {name} needs adjacent channels and 16-byte aligned rows, each "
                             "with memory of its own (it is written in place)")
    if (not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != (B,)
            or lengths.get_device() != index or not lengths.is_contiguous()):
        raise ValueError("window_attention_step: lengths must be a contiguous int32 [B] on q's device")
    if recorded(q, k, v, k_cache, v_cache):
        raise RuntimeError("window_attention_step has no gradient: call it under torch.no_grad()")
    q, k, v = aligned(q), aligned(k), aligned(v)
    o = torch.empty_like(q)
    n = _step_bytes(B, S, H, HK, D, w, s)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    launch("gd_wattn_step", index, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
           lengths.data_ptr(), o.data_ptr(), _DTYPES[q.dtype], B, S, H, HK, D, _strides(k_cache, v_cache), w, s,
           float(D ** -0.5 if scale is None else scale), None if ws is None else ws.data_ptr(), n)
    increment_version((k_cache, v_cache))  # written through their pointers: autograd sees that saved ones have changed
    return o
