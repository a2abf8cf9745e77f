"""Rotary positions on B200: queries and keys of a softmax-attention layer turned in one CUDA pass, each way (C ABI
gd_rotary in libgated_delta_b200.so). The first R channels of a head are pairs turned by the token's angles, the others
pass through:

    a' = a cos - b sin,  b' = b cos + a sin             (float32, one rounding)

with pairs (i, i + R/2) (half layout) or (2 i, 2 i + 1) (interleaved=True). The angles come from a table that a program
builds once (`rotary_table`, in float64: exact to float32 at every position) and shares between its layers; scalings for
long contexts are a matter of the table. The gradient is the turn by the opposite angles. There is no CPU path: CUDA
tensors only.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.GD_FLOAT32, torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> tuple[torch.Tensor, float]:
    """(angles per position [dim / 2] in float64, the factor on cos and sin). scaling, by its "type":
      None                the plain frequencies base^(-2 i / dim)
      "linear"            positions divided by "factor"
      "ntk"               the base raised to base * factor^(dim / (dim - 2)): the slowest pair slows by "factor", the
                          fastest keeps its speed
      "yarn"              pairs that turn more than "fast" (32) times within "original_length" positions keep their
                          speed, those that turn less than "slow" (1) times are slowed by "factor", in between a linear
                          ramp over the pair's index; cos and sin are multiplied by "attention_factor"
                          (default 0.1 ln factor + 1)"""
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be positive and even, got {dim}")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    freq = base ** (-i / dim)
    if scaling is None:
        return freq, 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 0.0))
    if factor <= 0:
        raise ValueError(f"rotary_frequencies: scaling needs a positive factor, got {scaling}")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        if dim == 2:
            return freq, 1.0
        return (base * factor ** (dim / (dim - 2))) ** (-i / dim), 1.0
    if kind == "yarn":
        length = float(scaling["original_length"])

        def pair(turns):  # the (fractional) pair that turns so often within the original length
            return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair(float(scaling.get("fast", 32.0)))), 0)
        high = min(math.ceil(pair(float(scaling.get("slow", 1.0)))), dim // 2 - 1)
        slowed = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq * (1 - slowed) + freq / factor * slowed, float(
            scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    raise ValueError(f"rotary_frequencies: unknown scaling type {kind!r}")


def rotary_table(positions: int, dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                 device="cuda") -> torch.Tensor:
    """[positions, dim / 2, 2] float32: cos and sin of every pair's angle at positions 0 .. positions - 1, computed in
    float64. Build it once."""
    freq, factor = rotary_frequencies(dim, base, scaling)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return torch.stack([angle.cos() * factor, angle.sin() * factor], -1).to(torch.float32)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _turn(q, k, table, positions, interleaved, inverse):
    B, T, H, D = q.shape
    oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k is None:
        ok, kp, okp, HK, ks = q.new_empty(0), None, None, 0, (0, 0, 0)
    else:
        ok = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        kp, okp, HK, ks = k.data_ptr(), ok.data_ptr(), k.shape[2], k.stride()
    qs = q.stride()
    pp, p64, pb = None, 0, 0
    if positions is not None:
        pp, p64 = positions.data_ptr(), positions.dtype == torch.int64
        pb = T if positions.dim() == 2 else 0
    with torch.cuda.device(q.device):
        st = _lib.load().gd_rotary(q.data_ptr(), kp, oq.data_ptr(), okp, table.data_ptr(), pp, p64, pb, table.shape[0],
                                   _DTYPES[q.dtype], B, T, H, HK, D, 2 * table.shape[1], qs[0], qs[1], qs[2], ks[0],
                                   ks[1], ks[2], interleaved, inverse,
                                   torch.cuda.current_stream(q.device).cuda_stream)
    if st:
        _lib.check(st, "gd_rotary")
    return oq, ok


@torch.library.custom_op("macai_b200::rotary", mutates_args=(), device_types="cuda")
def rotary_op(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor],
              interleaved: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, k) turned (contiguous); k's place is an empty tensor without it."""
    return _turn(_rows(q), None if k is None else _rows(k), table, positions, interleaved, inverse)


@rotary_op.register_fake
def _(q, k, table, positions, interleaved, inverse):
    return q.new_empty(q.shape), q.new_empty(0 if k is None else k.shape)


def _setup_context(ctx, inputs, output):
    q, k, table, positions, interleaved, inverse = inputs
    ctx.save_for_backward(table, positions)
    ctx.flags = (interleaved, inverse, k is not None)
    ctx.set_materialize_grads(False)


def _backward(ctx, dq, dk):
    table, positions = ctx.saved_tensors
    interleaved, inverse, has_k = ctx.flags
    if not has_k:
        dk = None  # the empty second output
    if dq is None and dk is None:
        return None, None, None, None, None, None
    if dq is None:
        return None, rotary_op(dk, None, table, positions, interleaved, not inverse)[0], None, None, None, None
    gq, gk = rotary_op(dq, dk, table, positions, interleaved, not inverse)
    return gq, (gk if dk is not None else None), None, None, None, None


rotary_op.register_autograd(_backward, setup_context=_setup_context)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
           interleaved: bool = False):
    """(q, k) with their first 2 * table.shape[1] channels turned. q [B, T, H, D], k [B, T, H_k, D] (or None) in one
    float dtype, with any strides as long as a head's channels are adjacent (views of a fused projection are read in
    place); table [P, R / 2, 2] from rotary_table; positions int32 or int64 [T] or [B, T] on the device (None: 0 .. T-1).
    A position outside the table is taken as its nearest row."""
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _DTYPES:
            raise ValueError(f"rotary: {name} must be [B, T, heads, D] in float32, float16 or bfloat16")
        if not t.is_cuda:
            raise RuntimeError("rotary: CUDA tensors only (there is no CPU path)")
    if k is not None and (k.dtype != q.dtype or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]
                          or k.device != q.device):
        raise ValueError("rotary: q and k must agree in dtype, device, batch, tokens and head width")
    if (not isinstance(table, torch.Tensor) or table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32
            or table.device != q.device or not table.is_contiguous() or 2 * table.shape[1] > q.shape[3]
            or table.shape[1] == 0 or table.shape[0] == 0 or table.data_ptr() % 8):
        raise ValueError("rotary: table must be a contiguous float32 [positions, R / 2, 2] on q's device with R at most "
                         "the head width")
    if positions is not None:
        if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
                or positions.device != q.device or tuple(positions.shape) not in ((q.shape[1],), tuple(q.shape[:2]))):
            raise ValueError("rotary: positions must be int32 or int64 [T] or [B, T] on q's device")
        positions = positions.contiguous()
    elif table.shape[0] < q.shape[1]:
        raise ValueError(f"rotary: the table has {table.shape[0]} positions, the call {q.shape[1]} tokens")
    interleaved = bool(interleaved)
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) \
            or torch.compiler.is_compiling():
        oq, ok = rotary_op(q, k, table, positions, interleaved, False)
    else:
        oq, ok = _turn(_rows(q), None if k is None else _rows(k), table, positions, interleaved, False)
    return oq, (None if k is None else ok)
