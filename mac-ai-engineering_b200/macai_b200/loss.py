"""The softmax cross entropy of a decoder's vocabulary projection on B200, without ever keeping the logits (C ABI gd_xent_* in
libgated_delta_b200.so):

    loss_i = logsumexp_v(x_i . w_v) - x_i . w_label(i)

tcgen05 products of 16-bit operands with float32 sums, in runs of at most 768 terms that are added outside the tensor core
(whose adder cuts off instead of rounding: long sums would be shifted towards zero). The logits stay on the chip as float32:
the forward keeps a maximum and a sum of exponentials for every 128 of them, the backward forms them again, a piece of the
vocabulary at a time, and rounds their gradient to the inputs' 16-bit type (the matrix instruction's operand). bfloat16 and
float16. There is no CPU path: CUDA tensors only.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._call import first_order, launch, matrix, pitch, recorded, room

_DTYPES = {torch.float16: _lib.GD_FLOAT16, torch.bfloat16: _lib.GD_BFLOAT16}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


@functools.lru_cache(maxsize=1024)
def _bytes(*sizes) -> int:
    n = _lib.load().gd_xent_workspace_bytes(*sizes)
    if n == 0:
        raise NotImplementedError(f"linear_cross_entropy: sizes (rows, D, V) = {sizes[:3]} are too large")
    return n


def _fwd(x, w, labels, ignore, reduction, keep):
    """(loss, kept): kept, int32 for the backward (else None): the live rows' maxima and sums (as logarithms), 2 n, and which
    rows those are, 4 + 2 n."""
    n, D = x.shape
    loss = torch.empty(n if reduction == 0 else (), dtype=torch.float32, device=x.device)
    kept = lse = plan = None
    if n == 0:  # no row: torch's own results, a mean over nothing among them
        return loss.fill_(float("nan") if reduction == 1 else 0.0), kept
    if keep:
        kept = torch.empty(4 + 4 * n, dtype=torch.int32, device=x.device)
        lse = kept.data_ptr()
        plan = lse + 8 * n
    size = _bytes(n, D, w.shape[0], 0)  # (even)
    ws = x.new_empty(size // 2)
    launch("gd_xent_fwd", x.get_device(), x.data_ptr(), w.data_ptr(), labels.data_ptr(), labels.dtype == torch.int64,
           loss.data_ptr(), lse, plan, reduction, ignore, _DTYPES[x.dtype], n, D, w.shape[0], pitch(x), pitch(w), ws.data_ptr(),
           size)
    return loss, kept


def _bwd(x, w, kept, dloss, reduction, need):
    """(dx, dw), contiguous, each None unless needed."""
    n, D = x.shape
    V = w.shape[0]
    dx, dw = room(x) if need[0] else None, room(w) if need[1] else None
    if n == 0:
        return dx, None if dw is None else dw.zero_()
    size = _bytes(n, D, V, 1)
    ws = x.new_empty(size // 2)
    lse = kept.data_ptr()
    launch("gd_xent_bwd", x.get_device(), x.data_ptr(), w.data_ptr(), lse, lse + 8 * n, dloss.data_ptr(),
           None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), reduction, _DTYPES[x.dtype], n, D, V,
           pitch(x), pitch(w), ws.data_ptr(), size)
    return dx, dw


class LinearCrossEntropy(torch.autograd.Function):
    """`LinearCrossEntropy.apply(x, weight, labels, ignore_index, reduction)` on matrices; reduction 0 none, 1 mean, 2 sum."""

    @staticmethod
    def forward(ctx, x, w, labels, ignore, reduction):
        loss, kept = _fwd(x, w, labels, ignore, reduction, True)
        ctx.save_for_backward(x, w, kept)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @first_order
    def backward(ctx, dloss):
        dx, dw = _bwd(*ctx.saved_tensors, dloss.float().contiguous(), ctx.reduction, ctx.needs_input_grad)
        return dx, dw, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of the logits x weight^T, in float32: x [..., D] and weight [V, D] (as nn.Linear keeps it) both
    bfloat16 or both float16, D a multiple of 8, V any size; labels [...] int64 or int32. reduction "none": one loss for each
    row, in the labels' shape; "mean": over the rows that are not ignored (NaN if all are); "sum". A row with the label
    ignore_index has loss 0, a zero row in x's gradient and no part in the weight's, whatever it holds; any other label outside
    [0, V) gives NaN (nothing waits for the host to look). Gradients of x and weight come in their type, the same bits every
    run; a frozen one's is not formed.

    Ignored rows cost no products. The logits are never kept: beside the gradients a call holds the other rows of x and 8 bytes
    for each row and 128 columns; the backward at most 256 MiB (or 256 columns) of the logits' gradients, x's gradient once
    more, and float32 sums of it (with several pieces of 256 MiB one for each value, else at most 64 MiB)."""
    name = "linear_cross_entropy"
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{name}: reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int) or not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"{name}: ignore_index must be an int of 64 bits, got {ignore_index!r}")
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"{name}: x must be [..., D] and weight [V, D]")
    for n, t in (("x", x), ("weight", weight)):
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name}: bfloat16 or float16, got {t.dtype} for {n}")
    if not isinstance(labels, torch.Tensor) or labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: labels must be an int64 or int32 tensor")
    if weight.dtype != x.dtype or not x.get_device() == weight.get_device() == labels.get_device():
        raise ValueError(f"{name}: x and weight must share one dtype, and all inputs one device")
    if not x.is_cuda:
        raise RuntimeError(f"{name}: CUDA tensors only (there is no CPU path)")
    D, V = x.shape[-1], weight.shape[0]
    if weight.shape[1] != D or labels.shape != x.shape[:-1]:
        raise ValueError(f"{name}: weight [V, D] and labels [...] must agree with x [..., D]; got {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}, {tuple(labels.shape)}")
    if D == 0 or V == 0 or D % 8:
        raise NotImplementedError(f"{name}: D is a multiple of 8 and V at least 1, got {D}, {V}")
    r, lab = _REDUCTIONS[reduction], labels.reshape(-1).contiguous()
    if recorded(x, weight):
        loss = LinearCrossEntropy.apply(matrix(x), matrix(weight), lab, ignore_index, r)
    else:
        loss = _fwd(matrix(x), matrix(weight), lab, ignore_index, r, False)[0]
    return loss.view(labels.shape) if r == 0 else loss
