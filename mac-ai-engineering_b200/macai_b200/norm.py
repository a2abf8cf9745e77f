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

_DTYPES = {torch.float32: _lib.GD_FLOAT32, torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
MAX_CHUNKS = 2048  # 16-byte chunks of a row (a width that fills no whole number of them takes two more)


def supported(x, residual, weight) -> bool:
    """The cases the kernels take: x [..., D] (and the residual, of its shape and dtype) in float32, float16 or
    bfloat16; weight [D] in x's dtype or float32; CUDA tensors; D up to 16,384 at 16 bits (16,375 where it is not a
    multiple of 8) and 8,192 at float32 (8,187 where it is not a multiple of 4)."""
    ts = (x, weight) if residual is None else (x, residual, weight)
    if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in ts) or x.dim() == 0 or x.dtype not in _DTYPES:
        return False
    d = x.shape[-1]
    e = 4 if x.dtype == torch.float32 else 8
    chunks = d // e if d % e == 0 else d // e + 2
    return (0 < d and chunks <= MAX_CHUNKS and weight.dim() == 1 and weight.shape[0] == d
            and weight.dtype in (x.dtype, torch.float32) and weight.device == x.device
            and (residual is None or (residual.dtype == x.dtype and residual.shape == x.shape
                                      and residual.device == x.device)))


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous with a 16-byte aligned start (a copy only when the view is not)."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _fwd(x, residual, w, eps, zero_centered):
    y = torch.empty_like(x)
    s = torch.empty_like(x) if residual is not None else x.new_empty(0)
    d = x.shape[-1]
    with torch.cuda.device(x.device):
        st = _lib.load().gd_rnorm_fwd(x.data_ptr(), _p(residual), w.data_ptr(),
                                      s.data_ptr() if residual is not None else None, y.data_ptr(), _DTYPES[x.dtype],
                                      _DTYPES[w.dtype], zero_centered, x.numel() // d, d, eps,
                                      torch.cuda.current_stream(x.device).cuda_stream)
    if st:
        _lib.check(st, "gd_rnorm_fwd")
    return y, s


@torch.library.custom_op("macai_b200::rnorm_fwd", mutates_args=(), device_types="cuda")
def rnorm_fwd(x: torch.Tensor, residual: Optional[torch.Tensor], w: torch.Tensor, eps: float,
              zero_centered: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, s) in x's dtype and shape; s is empty without a residual."""
    return _fwd(x, residual, w, eps, zero_centered)


@rnorm_fwd.register_fake
def _(x, residual, w, eps, zero_centered):
    return torch.empty_like(x), torch.empty_like(x) if residual is not None else x.new_empty(0)


@torch.library.custom_op("macai_b200::rnorm_bwd", mutates_args=(), device_types="cuda")
def rnorm_bwd(s: torch.Tensor, w: torch.Tensor, dy: Optional[torch.Tensor], ds: Optional[torch.Tensor], eps: float,
              zero_centered: bool, need_dw: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dw): dx like s (of x and of the residual), dw an empty tensor unless asked for; a None cotangent is zero."""
    lib = _lib.load()
    d = s.shape[-1]
    rows = s.numel() // d
    dx = torch.empty_like(s)
    dw = torch.empty_like(w) if need_dw else w.new_empty(0)
    ws, nbytes = None, 0
    if need_dw:
        nbytes = lib.gd_rnorm_workspace_bytes(rows, d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device)
    with torch.cuda.device(s.device):
        st = lib.gd_rnorm_bwd(s.data_ptr(), w.data_ptr(), _p(dy), _p(ds), dx.data_ptr(),
                              dw.data_ptr() if need_dw else None, _DTYPES[s.dtype], _DTYPES[w.dtype], zero_centered,
                              rows, d, eps, _p(ws), nbytes, torch.cuda.current_stream(s.device).cuda_stream)
    _lib.check(st, "gd_rnorm_bwd")
    return dx, dw


@rnorm_bwd.register_fake
def _(s, w, dy, ds, eps, zero_centered, need_dw):
    return torch.empty_like(s), w.new_empty(w.shape[0] if need_dw else 0)


def _setup_context(ctx, inputs, output):
    x, residual, w, eps, zero_centered = inputs
    ctx.save_for_backward(x if residual is None else output[1], w)
    ctx.eps, ctx.zero_centered, ctx.has_residual = eps, zero_centered, residual is not None
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, ds):
    s, w = ctx.saved_tensors
    if not ctx.has_residual:
        ds = None  # the empty second output
    if dy is None and ds is None:
        return None, None, None, None, None
    need_dw = bool(ctx.needs_input_grad[2]) and dy is not None
    dy = None if dy is None else _aligned(dy.to(s.dtype))
    ds = None if ds is None else _aligned(ds.to(s.dtype))
    dx, dw = rnorm_bwd(s, w, dy, ds, ctx.eps, ctx.zero_centered, need_dw)
    return dx, (dx if ctx.has_residual else None), (dw if need_dw else None), None, None


rnorm_fwd.register_autograd(_backward, setup_context=_setup_context)

_REFUSED = ("x [..., D] and the residual must be CUDA tensors of one float dtype and shape, the weight [D] in x's dtype "
            "or float32, D at most 16,384 (16 bits) or 8,192 (float32); there is no CPU path")


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                 zero_centered: bool = False):
    """(y, s) = the RMS norm of s = x + residual, and s. Without a residual s is x itself."""
    if not supported(x, residual, weight):
        raise ValueError("add_rms_norm: " + _REFUSED)
    x_, w = _aligned(x), _aligned(weight)
    r = None if residual is None else _aligned(residual)
    recorded = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                            or (r is not None and r.requires_grad))
    y, s = (rnorm_fwd if recorded or torch.compiler.is_compiling() else _fwd)(x_, r, w, float(eps), bool(zero_centered))
    return y, (x if residual is None else s)


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                     group: Optional[int] = 128, zero_centered: bool = False):
    """(q, scale, s): q [..., D] float8_e4m3fn and scale [..., ceil(D / group)] float32 with y = q * scale, one scale for
    each `group` channels (a multiple of 8; None: for the whole row), scale = max |y| / 448 over them, or 1 where y is
    all zero; s as add_rms_norm's. No gradient."""
    if not supported(x, residual, weight):
        raise ValueError("add_rms_norm_fp8: " + _REFUSED)
    if group is not None and (group <= 0 or group % 8):
        raise ValueError(f"add_rms_norm_fp8: group must be a positive multiple of 8 or None, got {group}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad(), or add_rms_norm")
    x_, w = _aligned(x), _aligned(weight)
    r = None if residual is None else _aligned(residual)
    d = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((*x.shape[:-1], -(-d // group) if group else 1), dtype=torch.float32, device=x.device)
    s = x if r is None else torch.empty_like(x_)
    with torch.cuda.device(x.device):
        st = _lib.load().gd_rnorm_fp8(x_.data_ptr(), _p(r), w.data_ptr(), None if r is None else s.data_ptr(),
                                      q.data_ptr(), scale.data_ptr(), _DTYPES[x.dtype], _DTYPES[w.dtype],
                                      bool(zero_centered), x.numel() // d, d, group or 0, float(eps),
                                      torch.cuda.current_stream(x.device).cuda_stream)
    if st:
        _lib.check(st, "gd_rnorm_fp8")
    return q, scale, s
