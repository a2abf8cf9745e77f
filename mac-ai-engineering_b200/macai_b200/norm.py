"""The residual addition with its RMS norm on B200, the step that opens every layer of the decoder, one CUDA pass each
way (C ABI gd_rnorm_fwd / gd_rnorm_bwd / gd_rnorm_fp8 in libgated_delta_b200.so):

    s = x + residual                                   (rounded to x's dtype: the stream the next layer adds to)
    y = s * rsqrt(mean(s^2) + eps) * w'                (float32 from the rounded s, one rounding; w' = w, or 1 + w with
                                                        zero_centered=True, as Qwen3.5's RMSNorm keeps its weight)

`add_rms_norm` has a gradient: of x and the residual (one tensor, they are equal) in their dtype, and of the weight in
its dtype when it needs one, as a sum over rows in a fixed order (the same bits every run). `add_rms_norm_fp8` returns y
as float8_e4m3fn with a float32 scale for each group of channels, for 8-bit projections (no gradient). There is no CPU
path: CUDA tensors only.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._call import aligned, first_order, launch, recorded

_DTYPES = {torch.float32: _lib.GD_FLOAT32, torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
MAX_CHUNKS = 2048  # 16-byte chunks of a row (a width that fills no whole number of them takes two more)


def supported(x, residual, weight) -> bool:
    """The cases the kernels take: x [..., D] (and the residual, of its shape and dtype) in float32, float16 or
    bfloat16; weight [D] in x's dtype or float32; CUDA tensors; D up to 16,384 at 16 bits (16,375 where it is not a
    multiple of 8) and 8,192 at float32 (8,187 where it is not a multiple of 4)."""
    if not (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor)) or not x.is_cuda or x.dim() == 0:
        return False
    dt, d, index = x.dtype, x.shape[-1], x.get_device()
    if dt not in _DTYPES or d == 0:
        return False
    e = 4 if dt == torch.float32 else 8
    if (d // e if d % e == 0 else d // e + 2) > MAX_CHUNKS:
        return False
    if weight.shape != (d,) or (weight.dtype != dt and weight.dtype != torch.float32) or weight.get_device() != index:
        return False
    return residual is None or (isinstance(residual, torch.Tensor) and residual.dtype == dt
                                and residual.shape == x.shape and residual.get_device() == index)


def _fwd(x, residual, w, eps, zero_centered):
    """(y, s) on aligned inputs; s is None without a residual."""
    y = torch.empty_like(x)
    s = None if residual is None else torch.empty_like(x)
    d = x.shape[-1]
    launch("gd_rnorm_fwd", x.get_device(), x.data_ptr(), None if residual is None else residual.data_ptr(), w.data_ptr(),
           None if s is None else s.data_ptr(), y.data_ptr(), _DTYPES[x.dtype], _DTYPES[w.dtype], zero_centered,
           x.numel() // d, d, eps)
    return y, s


def _bwd(s, w, dy, ds, eps, zero_centered, need_dw):
    """(dx, dw); dw None unless asked for."""
    d = s.shape[-1]
    rows = s.numel() // d
    dx = torch.empty_like(s)
    dw = ws = None
    nbytes = 0
    if need_dw:
        dw = torch.empty_like(w)
        nbytes = _lib.load().gd_rnorm_workspace_bytes(rows, d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device)
    launch("gd_rnorm_bwd", s.get_device(), s.data_ptr(), w.data_ptr(), None if dy is None else dy.data_ptr(),
           None if ds is None else ds.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr(), _DTYPES[s.dtype],
           _DTYPES[w.dtype], zero_centered, rows, d, eps, None if ws is None else ws.data_ptr(), nbytes)
    return dx, dw


class AddRMSNorm(torch.autograd.Function):
    """`AddRMSNorm.apply(x, residual or None, w, eps, zero_centered)` on aligned inputs: (y, s), or y without a residual."""

    @staticmethod
    def forward(ctx, x, residual, w, eps, zero_centered):
        y, s = _fwd(x, residual, w, eps, zero_centered)
        ctx.save_for_backward(x if s is None else s, w)
        ctx.args = (eps, zero_centered, s is not None)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @first_order
    def backward(ctx, dy, ds=None):
        s, w = ctx.saved_tensors
        eps, zero_centered, has_residual = ctx.args
        if dy is None and ds is None:
            return None, None, None, None, None
        need_dw = ctx.needs_input_grad[2] and dy is not None
        dx, dw = _bwd(s, w, None if dy is None else aligned(dy), None if ds is None else aligned(ds), eps, zero_centered,
                      need_dw)
        return dx, (dx if has_residual else None), dw, None, None


_REFUSED = ("x [..., D] and the residual must be CUDA tensors of one float dtype and shape, the weight [D] in x's dtype "
            "or float32, D at most 16,384 (16 bits) or 8,192 (float32); there is no CPU path")


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                 zero_centered: bool = False):
    """(y, s) = the RMS norm of s = x + residual, and s. Without a residual s is x itself."""
    if not supported(x, residual, weight):
        raise ValueError("add_rms_norm: " + _REFUSED)
    x_, w = aligned(x), aligned(weight)
    r = None if residual is None else aligned(residual)
    if recorded(x, residual, weight):
        out = AddRMSNorm.apply(x_, r, w, float(eps), bool(zero_centered))
        return (out, x) if r is None else out
    y, s = _fwd(x_, r, w, float(eps), bool(zero_centered))
    return y, (x if r is None else s)


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                     group: Optional[int] = 128, zero_centered: bool = False):
    """(q, scale, s): q [..., D] float8_e4m3fn and scale [..., ceil(D / group)] float32 with y = q * scale, one scale for
    each `group` channels (a multiple of 8; None: for the whole row), scale = max |y| / 448 over them, at least the
    smallest normal number 2^-126, or 1 where y is all zero; s as add_rms_norm's. No gradient."""
    if not supported(x, residual, weight):
        raise ValueError("add_rms_norm_fp8: " + _REFUSED)
    if group is not None and (group <= 0 or group % 8):
        raise ValueError(f"add_rms_norm_fp8: group must be a positive multiple of 8 or None, got {group}")
    if recorded(x, residual, weight):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad(), or add_rms_norm")
    x_, w = aligned(x), aligned(weight)
    r = None if residual is None else aligned(residual)
    d = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((*x.shape[:-1], -(-d // group) if group else 1), dtype=torch.float32, device=x.device)
    s = x if r is None else torch.empty_like(x_)
    launch("gd_rnorm_fp8", x.get_device(), x_.data_ptr(), None if r is None else r.data_ptr(), w.data_ptr(),
           None if r is None else s.data_ptr(), q.data_ptr(), scale.data_ptr(), _DTYPES[x.dtype], _DTYPES[w.dtype],
           bool(zero_centered), x.numel() // d, d, group or 0, float(eps))
    return q, scale, s
