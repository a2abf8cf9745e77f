"""The gated delta rule's recurrent form on B200, for decoding (C ABI gd_rule_step in libgated_delta_b200.so): single tokens
and short runs over kept states, token after token, everything in float32:

    S <- exp(g) S,   d = beta (v - S^T k),   S <- S + k d^T,   o = S^T q        (q scaled by DK^-0.5)

`gated_delta_step` works on a pool of states in place, as a server keeps it; `recurrent_gated_delta_rule` is the drop-in for
transformers' torch_recurrent_gated_delta_rule (the reference's token-serial kernels, src/macai/gated_delta/_metal.py:37-77).
A call reads and writes each state once, however many tokens it runs, and a token has the same bits alone, in a run, and in any
batch; long rows belong to `chunk_gated_delta_rule`. No gradient, and no CPU path: CUDA tensors only.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.graph import increment_version

from .. import _lib
from .._call import aligned, launch, recorded

_DTYPES = {torch.float32: _lib.GD_FLOAT32, torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
MAX_WIDTH = 256


def _refuse(name, q, k, v, g, beta):
    """The error for inputs that `_inputs` does not take."""
    for x, t in (("query", q), ("key", k), ("value", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            return ValueError(f"{name}: {x} must be [B, T, heads, width]")
    if q.dtype not in _DTYPES:
        return TypeError(f"{name}: float32, float16 or bfloat16, got {q.dtype}")
    if not q.is_cuda:
        return RuntimeError(f"{name}: CUDA tensors only (there is no CPU path)")
    B, T, HK, DK = q.shape
    H, DV = v.shape[2], v.shape[3]
    if k.shape != q.shape or v.shape[:2] != q.shape[:2]:
        return ValueError(f"{name}: query and key [B, T, HK, DK] and value [B, T, H, DV] must agree; got {tuple(q.shape)}, "
                          f"{tuple(k.shape)}, {tuple(v.shape)}")
    if H == 0 or HK == 0 or H % HK:
        return ValueError(f"{name}: value heads ({H}) must be a multiple of key heads ({HK})")
    if DK == 0 or DV == 0 or DK % 32 or DV % 32:
        return ValueError(f"{name}: head widths must be multiples of 32; got DK={DK}, DV={DV}")
    if DK > MAX_WIDTH or DV > MAX_WIDTH:
        return NotImplementedError(f"{name}: head widths go up to {MAX_WIDTH}; got DK={DK}, DV={DV}")
    if B > 65535:
        return NotImplementedError(f"{name}: at most 65,535 requests a call, got {B}")
    for x, t in (("g", g), ("beta", beta)):
        if not isinstance(t, torch.Tensor) or t.shape != (B, T, H):
            return ValueError(f"{name}: {x} must be [B, T, H] = {(B, T, H)}")
    return ValueError(f"{name}: the inputs must be on one device")


def _inputs(name, q, k, v, g, beta):
    """(q, k, v, g, beta, B, T, H, HK, DK, DV) as the kernel reads them; raises for what it does not take."""
    try:
        B, T, HK, DK = q.shape
        _, _, H, DV = v.shape
        row, index, dt = (B, T, H), q.get_device(), q.dtype
        ok = (q.is_cuda and dt in _DTYPES and k.shape == q.shape and v.shape[:2] == q.shape[:2] and g.shape == row
              and beta.shape == row and HK > 0 and H > 0 and H % HK == 0 and 0 < DK <= MAX_WIDTH and 0 < DV <= MAX_WIDTH
              and DK % 32 == 0 and DV % 32 == 0 and B <= 65535 and k.get_device() == index and v.get_device() == index
              and g.get_device() == index and beta.get_device() == index)
    except (AttributeError, ValueError):
        ok = False
    if not ok:
        raise _refuse(name, q, k, v, g, beta)
    if k.dtype != dt:
        k = k.to(dt)
    if v.dtype != dt and v.dtype != torch.float32:
        v = v.float()  # (exact for any other type of 16 bits)
    if g.dtype != torch.float32:
        g = g.float()
    if beta.dtype != torch.float32:
        beta = beta.float()
    return aligned(q), aligned(k), aligned(v), g.contiguous(), beta.contiguous(), B, T, H, HK, DK, DV


def gated_delta_step(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, slots: Optional[torch.Tensor] = None, out_slots: Optional[torch.Tensor] = None,
                     use_qk_l2norm_in_kernel: bool = False) -> torch.Tensor:
    """T new tokens of each request over a pool of states: the output o [B, T, H, DV] in the query's dtype, the states
    carried on in place. query, key [B, T, HK, DK]; value [B, T, H, DV] in the query's dtype or float32 (H a multiple of
    HK: each key head serves H / HK consecutive value heads); g (log decay, <= 0) and beta [B, T, H]; state
    [S, H, DK, DV] float32, contiguous. Head widths are multiples of 32 up to 256.

    slots (int32 [B] on the device, default: request b has slot b): the slot whose state each request starts from, and,
    unless out_slots names others, the one that it leaves its state in. out_slots lets the state before the tokens stay,
    as drafted tokens need. A negative slot marks an idle request: its output is zeros. A request whose slot the pool does
    not have, or whose written slot another request of the call reads or writes, gets NaN. Neither of them changes a state;
    idle requests and those without a slot contest none.
    No gradient. Nothing waits for the host."""
    name = "gated_delta_step"
    q, k, v, g_, beta_, B, T, H, HK, DK, DV = _inputs(name, query, key, value, g, beta)
    index = q.get_device()
    if not isinstance(state, torch.Tensor) or state.dim() != 4 or state.shape != (state.shape[0], H, DK, DV):
        raise ValueError(f"{name}: state must be [S, H, DK, DV] with (H, DK, DV) = {(H, DK, DV)}")
    pool = state.data_ptr()
    if state.dtype != torch.float32 or state.get_device() != index or not state.is_contiguous() or pool % 16:
        raise ValueError(f"{name}: state must be float32, contiguous and 16-byte aligned on the query's device (it is "
                         "written in place)")
    if slots is None and out_slots is not None:
        raise ValueError(f"{name}: out_slots needs slots")
    for t in (slots, out_slots):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != (B,)
                              or t.get_device() != index or not t.is_contiguous()):
            raise ValueError(f"{name}: slots and out_slots must be contiguous int32 [B] on the query's device")
    if slots is None and state.shape[0] < B:
        raise ValueError(f"{name}: {B} requests need as many slots, the pool has {state.shape[0]}")
    if recorded(query, key, value, g, beta, state):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or train with chunk_gated_delta_rule")
    o = torch.empty_like(v) if v.dtype == q.dtype else q.new_empty((B, T, H, DV))
    at = None if slots is None else slots.data_ptr()
    launch("gd_rule_step", index, q.data_ptr(), k.data_ptr(), v.data_ptr(), g_.data_ptr(), beta_.data_ptr(), pool, pool, at,
           at if out_slots is None else out_slots.data_ptr(), o.data_ptr(), _DTYPES[q.dtype], _DTYPES[v.dtype], B, T, H, HK,
           DK, DV, state.shape[0], _lib.GD_L2NORM if use_qk_l2norm_in_kernel else 0)
    increment_version(state)  # written through its pointer: autograd sees that a saved one has changed
    return o


def recurrent_gated_delta_rule(query, key, value, g, beta, initial_state=None, output_final_state: bool = False,
                               use_qk_l2norm_in_kernel: bool = False, cu_seqlens=None):
    """Drop-in for transformers' torch_recurrent_gated_delta_rule: arguments as `chunk_gated_delta_rule`'s, any of the three
    float types; returns the output [B, T, H, DV] in the query's dtype and the final state (float32, a new tensor) when
    output_final_state, else None. cu_seqlens only None. No gradient."""
    name = "recurrent_gated_delta_rule"
    if cu_seqlens is not None:
        raise NotImplementedError(f"{name}: packed rows run through chunk_gated_delta_rule")
    q, k, v, g_, beta_, B, T, H, HK, DK, DV = _inputs(name, query, key, value, g, beta)
    if recorded(query, key, value, g, beta, initial_state):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or train with chunk_gated_delta_rule")
    s0 = None
    if initial_state is not None:
        if initial_state.shape != (B, H, DK, DV) or initial_state.get_device() != q.get_device():
            raise ValueError(f"{name}: initial_state must be [B, H, DK, DV] = {(B, H, DK, DV)} on the query's device")
        s0 = aligned(initial_state.float())
    sT = torch.empty((B, H, DK, DV), dtype=torch.float32, device=q.device) if output_final_state else None
    o = torch.empty_like(v) if v.dtype == q.dtype else q.new_empty((B, T, H, DV))
    launch("gd_rule_step", q.get_device(), q.data_ptr(), k.data_ptr(), v.data_ptr(), g_.data_ptr(), beta_.data_ptr(),
           None if s0 is None else s0.data_ptr(), None if sT is None else sT.data_ptr(), None, None, o.data_ptr(),
           _DTYPES[q.dtype], _DTYPES[v.dtype], B, T, H, HK, DK, DV, B, _lib.GD_L2NORM if use_qk_l2norm_in_kernel else 0)
    return o, sT
