"""The gated feed-forward block of a decoder layer on B200 (C ABI gd_ff_* in libgated_delta_b200.so), the half of the layer
after its mixer:

    g = x w_gate^T,   u = x w_up^T,   h = silu(g) * u,   y = h w_down^T

`gated_feed_forward` trains, prefills, and takes the few tokens of a decoding step. tcgen05 products with float32 sums; the
activation and its gradient are taken in float32 as the products leave the tensor core, so neither g nor u is read again in
the forward, and the gradient of h never leaves the chip. h and the gradients of g and u are rounded to the inputs' 16-bit type
(the matrix instruction's operands); g and u are kept for the backward in 24 bits. bfloat16 and float16. There is no CPU path:
CUDA tensors only.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._call import first_order, launch, matrix, pitch, recorded, room

_DTYPES = {torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}


@functools.lru_cache(maxsize=1024)
def _bytes(*sizes) -> int:
    n = _lib.load().gd_ff_workspace_bytes(*sizes)
    if n == 0:
        raise NotImplementedError(f"gated_feed_forward: sizes (rows, D, F, O) = {sizes[:4]} are too large")
    return n


@functools.lru_cache(maxsize=1024)
def _longs(*x):
    return (ctypes.c_longlong * len(x))(*x)


def _sizes(x, wg, wd):
    return x.shape[0], x.shape[1], wg.shape[0], wd.shape[0]


def _fwd(x, wg, wu, wd, keep):
    """(y, kept) on matrices; keep: 24 bits of g and u, and behind them float16's two bounds, for the backward, else None."""
    n, D, F, O = _sizes(x, wg, wd)
    y = x.new_empty((n, O))
    if n == 0:
        return y, None
    kept = at = bounds = None
    if keep:
        words = 3 * n * (-(-F // 64) * 64)
        kept = x.new_empty(words + 8)
        at = kept.data_ptr()
        bounds = at + 2 * words if x.dtype == torch.float16 else None
    size = _bytes(n, D, F, O, 0)  # (a multiple of 256)
    ws = x.new_empty(size // 2)
    launch("gd_ff_fwd", x.get_device(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), at, bounds, y.data_ptr(),
           _DTYPES[x.dtype], n, D, F, O, _longs(pitch(x), pitch(wg), pitch(wu), pitch(wd)), ws.data_ptr(), size)
    return y, kept


def _bwd(x, wg, wu, wd, kept, dy, need):
    """(dx, dw_gate, dw_up, dw_down), contiguous, each None unless needed."""
    n, D, F, O = _sizes(x, wg, wd)
    out = [room(t) if yes else None for t, yes in zip((x, wg, wu, wd), need)]
    if n == 0:
        return tuple(None if t is None else t.zero_() for t in out)
    at = kept.data_ptr()
    size = _bytes(n, D, F, O, 1)
    ws = x.new_empty(size // 2)
    launch("gd_ff_bwd", x.get_device(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), at,
           at + 2 * (kept.numel() - 8) if x.dtype == torch.float16 else None, dy.data_ptr(),
           *[None if t is None else t.data_ptr() for t in out], _DTYPES[x.dtype], n, D, F, O,
           _longs(pitch(x), pitch(wg), pitch(wu), pitch(wd), pitch(dy)), ws.data_ptr(), size)
    return tuple(out)


class GatedFeedForward(torch.autograd.Function):
    """`GatedFeedForward.apply(x, w_gate, w_up, w_down)` on matrices (adjacent columns, aligned rows)."""

    @staticmethod
    def forward(ctx, x, wg, wu, wd):
        y, kept = _fwd(x, wg, wu, wd, True)
        ctx.save_for_backward(x, wg, wu, wd, kept)
        return y

    @staticmethod
    @first_order
    def backward(ctx, dy):
        return _bwd(*ctx.saved_tensors, matrix(dy), ctx.needs_input_grad)


def _refuse(name, x, w_gate, w_up, w_down):
    """The error for inputs that the block does not take."""
    for n, t, d in (("x", x, 1), ("w_gate", w_gate, 2), ("w_up", w_up, 2), ("w_down", w_down, 2)):
        if not isinstance(t, torch.Tensor) or t.dim() < d or (d == 2 and t.dim() != 2):
            return ValueError(f"{name}: {n} must be {'[..., D]' if d == 1 else 'a matrix'}")
        if t.dtype not in _DTYPES:
            return TypeError(f"{name}: bfloat16 or float16, got {t.dtype} for {n}")
        if t.dtype != x.dtype or t.get_device() != x.get_device():
            return ValueError(f"{name}: x and the weights must share one dtype and device")
    if not x.is_cuda:
        return RuntimeError(f"{name}: CUDA tensors only (there is no CPU path)")
    D, (F, d2), O = x.shape[-1], w_gate.shape, w_down.shape[0]
    if d2 != D or w_up.shape != w_gate.shape or w_down.shape[1] != F:
        return ValueError(f"{name}: w_gate and w_up [F, D] and w_down [O, F] must agree with x [..., D]; got {tuple(x.shape)}, "
                          f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    return NotImplementedError(f"{name}: D, F and O are multiples of 8, got {D}, {F}, {O}")


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """y [..., O] for x [..., D], w_gate and w_up [F, D] (as nn.Linear keeps them; halves of one [2 F, D] weight are read in
    place) and w_down [O, F], all bfloat16 or all float16, D, F and O multiples of 8. Gradients of all four come in their
    type, the same bits every run; those of frozen inputs are not formed. Up to 128 rows a call that records no gradient takes
    another kernel than one that does, and its last bits may differ. Views with adjacent columns and 16-byte aligned
    rows are read in place, others are copied."""
    name = "gated_feed_forward"
    try:
        dt, D, index = x.dtype, x.shape[-1], x.get_device()
        F, d2 = w_gate.shape
        O, f2 = w_down.shape
        ok = (x.is_cuda and dt in _DTYPES and w_gate.dtype == dt and w_up.dtype == dt and w_down.dtype == dt and d2 == D
              and w_up.shape == w_gate.shape and f2 == F and D > 0 and F > 0 and O > 0 and D % 8 == 0 and F % 8 == 0
              and O % 8 == 0 and w_gate.get_device() == index and w_up.get_device() == index and w_down.get_device() == index)
    except (AttributeError, IndexError, ValueError):
        ok = False
    if not ok:
        raise _refuse(name, x, w_gate, w_up, w_down)
    if recorded(x, w_gate, w_up, w_down):
        y = GatedFeedForward.apply(matrix(x), matrix(w_gate), matrix(w_up), matrix(w_down))
    else:
        y = _fwd(matrix(x), matrix(w_gate), matrix(w_up), matrix(w_down), False)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], O)
