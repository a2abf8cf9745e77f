"""How the operators of the softmax-attention layer's steps reach the C ABI: on the tensor's device and its current
stream, with as little host work as a call of a few microseconds can bear (a device guard only when another device is
current)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle without the Stream object around it


def launch(name: str, index: int, *args) -> None:
    """lib.<name>(*args, stream) with device `index` current; a failure status raises GatedDeltaError."""
    fn = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, name)


def like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of t's shape, dtype and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous with a 16-byte aligned start (a copy only when the view is not)."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def first_order(backward):
    """once_differentiable for an autograd function's backward, without its cost (a grad-mode switch) where no graph of the
    gradient is asked for."""
    guarded = once_differentiable(backward)

    def wrapper(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return wrapper


def has_tangent(*ts) -> bool:
    """Whether one of these inputs (None allowed) carries a forward-mode tangent (torch.autograd.forward_ad)."""
    if forward_ad._current_level < 0:  # no dual level is open
        return False
    return any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def refuse_tangents(name: str, *ts) -> None:
    """Raises where one of these inputs carries a forward-mode tangent: the custom ops would drop it in silence."""
    if has_tangent(*ts):
        raise NotImplementedError(f"{name}: no forward-mode derivative")


def recorded(*ts) -> bool:
    """Whether autograd has a part in a call with these inputs (None allowed): a gradient to record, or a tangent, which
    the autograd functions refuse (they have no forward-mode derivative)."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return has_tangent(*ts)
