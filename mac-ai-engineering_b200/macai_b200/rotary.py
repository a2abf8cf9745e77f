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
from ._call import first_order, launch, like, recorded

_DTYPES = {torch.float32: _lib.GD_FLOAT32, torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> tuple[torch.Tensor, float]:
    """(angles per position [dim / 2] in float64, the factor on cos and sin). scaling, by its "type":
      None                the plain frequencies base^(-2 i / dim)
      "linear"            positions divided by "factor"
      "ntk"               the base raised to base * factor^(dim / (dim - 2)): the slowest pair slows by "factor", the
                          fastest keeps its speed
      "yarn"              pairs that turn more than "fast" (32) times within "original_length" positions keep their
                          speed, those that turn less than "slow" (1) times are slowed by "factor", in between a linear
                          ramp over the pair's index (which may end past the last pair); cos and sin are multiplied
                          by "attention_factor" (default 0.1 ln factor + 1)"""
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
        # bounded by dim - 1 as published: a ramp that ends past the last pair keeps its slope
        high = min(math.ceil(pair(float(scaling.get("slow", 1.0)))), dim - 1)
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
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _turn(q, k, table, positions, interleaved, inverse):
    """(q, k) turned, contiguous; None for a k of None."""
    q = _rows(q)
    B, T, H, D = q.shape
    qb, qt, qh, _ = q.stride()
    oq = like(q)
    ok = kp = okp = None
    HK = kb = kt = kh = 0
    if k is not None:
        k = _rows(k)
        ok = like(k)
        kp, okp, HK = k.data_ptr(), ok.data_ptr(), k.shape[2]
        kb, kt, kh, _ = k.stride()
    pp, p64, pb = None, 0, 0
    if positions is not None:
        pp, p64 = positions.data_ptr(), positions.dtype == torch.int64
        pb = T if positions.dim() == 2 else 0
    launch("gd_rotary", q.get_device(), q.data_ptr(), kp, oq.data_ptr(), okp, table.data_ptr(), pp, p64, pb,
           table.shape[0], _DTYPES[q.dtype], B, T, H, HK, D, 2 * table.shape[1], qb, qt, qh, kb, kt, kh, interleaved,
           inverse)
    return oq, ok


class Rotary(torch.autograd.Function):
    """`Rotary.apply(q, k or None, table, positions or None, interleaved)`: (q, k), or q without a k."""

    @staticmethod
    def forward(ctx, q, k, table, positions, interleaved):
        ctx.save_for_backward(table, positions)
        ctx.interleaved, ctx.has_k = interleaved, k is not None
        ctx.set_materialize_grads(False)
        oq, ok = _turn(q, k, table, positions, interleaved, False)
        return oq if k is None else (oq, ok)

    @staticmethod
    @first_order
    def backward(ctx, dq, dk=None):
        table, positions = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None
        if dq is None:
            return None, _turn(dk, None, table, positions, ctx.interleaved, True)[0], None, None, None
        gq, gk = _turn(dq, dk, table, positions, ctx.interleaved, True)
        return gq, gk, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
           interleaved: bool = False):
    """(q, k) with their first 2 * table.shape[1] channels turned. q [B, T, H, D], k [B, T, H_k, D] (or None) in one
    float dtype, with any strides as long as a head's channels are adjacent (views of a fused projection are read in
    place); table [P, R / 2, 2] from rotary_table; positions int32 or int64 [T] or [B, T] on the device (None: 0 .. T-1).
    A position outside the table is taken as its nearest row. The gradients are q's and k's; the table has none."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.dtype not in _DTYPES:
        raise ValueError("rotary: q must be [B, T, heads, D] in float32, float16 or bfloat16")
    if not q.is_cuda:
        raise RuntimeError("rotary: CUDA tensors only (there is no CPU path)")
    shape, index = q.shape, q.get_device()
    if k is not None and (not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype != q.dtype
                          or k.shape[:2] != shape[:2] or k.shape[3] != shape[3] or k.get_device() != index):
        raise ValueError("rotary: q and k [B, T, heads, D] must agree in dtype, device, batch, tokens and head width")
    if not isinstance(table, torch.Tensor) or table.dim() != 3 or table.dtype != torch.float32:
        raise ValueError("rotary: table must be float32 [positions, R / 2, 2]")
    P, half, two = table.shape
    if (two != 2 or P == 0 or half == 0 or 2 * half > shape[3] or table.get_device() != index
            or not table.is_contiguous() or table.data_ptr() % 8):
        raise ValueError("rotary: table must be a contiguous float32 [positions, R / 2, 2] on q's device with R at most "
                         "the head width")
    if positions is not None:
        if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
                or positions.get_device() != index
                or (positions.shape != shape[:2] and positions.shape != shape[1:2])):
            raise ValueError("rotary: positions must be int32 or int64 [T] or [B, T] on q's device")
        positions = positions.contiguous()
    elif P < shape[1]:
        raise ValueError(f"rotary: the table has {P} positions, the call {shape[1]} tokens")
    if recorded(table):
        raise RuntimeError("rotary: the table has no gradient: pass table.detach()")
    if recorded(q, k):
        out = Rotary.apply(q, k, table, positions, bool(interleaved))
        return (out, None) if k is None else out
    return _turn(q, k, table, positions, bool(interleaved), False)
