"""Expanded tensors (strides of 0) in window_attention and its step: inputs and cotangents give what their contiguous copies
give; a cache whose rows share memory is refused, since every request writes its own."""
import ctypes

import pytest
import torch

from macai_b200 import _lib
from test_gpu_window_attention import BF, DEV, _inputs, _run

gpu = pytest.mark.gpu
NUL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(256)


def test_the_c_abi_refuses_rows_that_share_memory():
    """Without a GPU: strides of 0 where the dimension has more than one entry, and caches that overlap themselves."""
    lib = _lib.load()
    B, T, H, HK, D = 2, 100, 4, 2, 64
    good = [T * H * D, H * D, D] + [T * HK * D, HK * D, D] * 2 + [T * H * D, H * D, D]
    for i in range(12):
        st = (ctypes.c_longlong * 12)(*good)
        st[i] = 0
        if i < 9:
            assert lib.gd_wattn_fwd(ONE, ONE, ONE, ONE, ONE, ONE, NUL, 0, _lib.GD_BFLOAT16, B, T, T, H, HK, D, st, 0, 0,
                                    0.125, NUL, 0, NUL) == _lib.GD_ERR_ALIGN, i
        assert lib.gd_wattn_bwd(ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, NUL, 0, _lib.GD_BFLOAT16, B, T, T, H, HK, D,
                                st, 0, 0, 0.125, ONE, 1 << 40, NUL) == _lib.GD_ERR_ALIGN, i
    S = 50

    def step(st):
        return lib.gd_wattn_step(ONE, ONE, ONE, ONE, ONE, ONE, ONE, _lib.GD_BFLOAT16, B, S, H, HK, D,
                                 (ctypes.c_longlong * 6)(*st), 0, 0, 0.125, ONE, 1 << 30, NUL)
    good = [S * HK * D, HK * D, D]
    for bad in ([0, HK * D, D], [S * HK * D, 0, D], [S * HK * D, HK * D, 0], [S * HK * D, HK * D, D // 2],
                [S * HK * D // 2, HK * D, D], [HK * D, HK * D, D], [D, HK * D, D]):
        assert step(bad + good) == _lib.GD_ERR_ALIGN and step(good + bad) == _lib.GD_ERR_ALIGN, bad


@gpu
def test_expanded_inputs_and_cotangents():
    B, T, H, HK, D = 3, 200, 4, 2, 64
    q, k, v, do = _inputs(B, T, T, H, HK, D, BF, 12)
    views = [  # over the batch, the heads, the tokens
        (q[:1].expand(B, T, H, D), k, v, do), (q, k[:1].expand(B, T, HK, D), v[:1].expand(B, T, HK, D), do),
        (q, k[:, :, :1].expand(B, T, HK, D), v[:, :, :1].expand(B, T, HK, D), do[:, :, :1].expand(B, T, H, D)),
        (q[:, :1].expand(B, T, H, D), k, v[:, :1].expand(B, T, HK, D), do[:, :1].expand(B, T, H, D)),
        (q, k, v, do[:1, :1].expand(B, T, H, D)), (q, k, v, do[:1, :1, :1, :1].expand(B, T, H, D))]
    for i, xs in enumerate(views):
        got = _run(*xs, window=70, sinks=2)
        want = _run(*(t.contiguous() for t in xs), window=70, sinks=2)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    from macai_b200.window_attention import window_attention
    x = q.clone().requires_grad_(True)
    window_attention(x, k, v, window=70).sum(1).float().square().sum().backward()   # its cotangent is expanded over the tokens
    o = window_attention(q, k, v, window=70)
    g = (2 * o.sum(1, keepdim=True).float()).to(BF).expand(B, T, H, D).contiguous()
    assert torch.equal(x.grad, _run(q, k, v, g, window=70)[1])


@gpu
def test_caches_that_share_rows_are_refused():
    from macai_b200.window_attention import window_attention_step
    q, k, v, _ = _inputs(3, 1, 1, 4, 2, 64, BF)
    L = torch.zeros(3, dtype=torch.int32, device=DEV)
    good = torch.zeros(3, 32, 2, 64, dtype=BF, device=DEV)
    flat = torch.zeros(3 * 32 * 2 * 64, dtype=BF, device=DEV)
    for bad in (good[:1].expand(3, 32, 2, 64), good[:, :1].expand(3, 32, 2, 64), good[:, :, :1].expand(3, 32, 2, 64)):
        for pair in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="own"):
                window_attention_step(q, k, v, *pair, L)
    overlapping = flat.as_strided((3, 32, 2, 64), (64, 128, 64, 1))
    with pytest.raises((ValueError, _lib.GatedDeltaError)):
        window_attention_step(q, k, v, overlapping, good, L)
    alone = good[:1].expand(1, 32, 2, 64)
    window_attention_step(q[:1], k[:1], v[:1], alone, good[:1].clone(), L[:1])
