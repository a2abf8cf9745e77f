"""add_rms_norm_fp8 where a group's largest |y| is near the ends of float32: scale = max |y| / 448, at least the smallest
normal number 2^-126 (1 where all are zero), and the codes are those of y / scale. With y's fp32 chain to 5e-6 of its size,
a code is within half a step of e4m3, 2^-4 of y or 2^-10 of the scale."""
import pytest
import torch

from oracle import layer_steps_f64 as ref

gpu = pytest.mark.gpu
DEV = "cuda"


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,group", [(256, 128), (256, None), (256, 24), (2048, 128), (1111, 64), (203, None)])
@pytest.mark.parametrize("size", [1e-45, 1e-41, 1e-38, 3e-37, 5e-36, 6e-36, 1e-30, 1e30, 2e37, 7e37])
def test_groups_of_tiny_and_huge_values(D, group, dt, size):
    from macai_b200.norm import add_rms_norm_fp8
    g = torch.Generator().manual_seed(D)
    x = torch.randn(5, D, generator=g).clamp(-2.5, 2.5).to(dt).to(DEV)
    x[:, 1::3] = 0                                          # zeros among them: codes 0, not NaN
    w = torch.ones(D, device=DEV)
    w[:D // 2] = size                                       # tiny and ordinary groups side by side
    q, scale, _ = add_rms_norm_fp8(x, None, w, 1e-6, group)
    y, _ = ref.rms_norm(x, None, w)
    n = group or D
    tops = torch.stack([c.abs().amax(-1) for c in y.split(n, -1)], -1)
    want = torch.where(tops > 0, (tops / 448.0).clamp_min(2.0 ** -126), torch.ones_like(tops))
    # y itself is fp32: below 2^-126 it stands in steps of 2^-149
    assert ((scale.double() - want).abs() <= 5e-6 * want + 2.0 ** -149).all()
    sc = scale.double().repeat_interleave(n, -1)[:, :D]
    back = q.float().double() * sc
    assert torch.isfinite(back).all()
    assert ((back - y).abs() <= (2.0 ** -4 + 1e-5) * y.abs() + 2.0 ** -10 * sc + 2.0 ** -148).all()
