"""Rotary positions (macai_b200.rotary) against the float64 turn.

Tolerance: two products and a sum in fp32 (three roundings of 2^-24 relative to |a| + |b|), then the output's rounding, at
most u = 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32) of the result or half the spacing of fp16's
subnormals (2^-25); channels past the turned part are the same bits."""
import math

import pytest
import torch

from oracle import layer_steps_f64 as ref

gpu = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DEV = "cuda"


def _close(got, want, x, R):
    size = x.double().abs()
    size = size + size[..., :R].amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert (err <= U[got.dtype] * want.abs() + 2.0 ** -25 * (got.dtype == torch.float16) + 4 * 2.0 ** -24 * size).all(), err.max().item()
    assert torch.equal(got[..., R:], x[..., R:])


@gpu
@pytest.mark.parametrize("dt", list(U))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,HK,D,R", [(1, 1, 1, 1, 2, 2), (2, 1, 16, 2, 256, 64), (3, 37, 4, 2, 128, 128),
                                          (1, 100, 3, 1, 72, 18), (2, 65, 2, 2, 80, 20), (1, 9, 5, 1, 33, 6),
                                          (2, 50, 8, 4, 96, 24)])
def test_turn_and_gradient(dt, interleaved, B, T, H, HK, D, R):
    from macai_b200.rotary import rotary, rotary_table
    g = torch.Generator().manual_seed(T * D)
    q, k = (torch.randn(B, T, h, D, generator=g).to(dt).to(DEV).requires_grad_(True) for h in (H, HK))
    dq, dk = (torch.randn(B, T, h, D, generator=g).to(dt).to(DEV) for h in (H, HK))
    table = rotary_table(5000, R, device=DEV)
    for pos in (None, torch.randint(0, 5000, (B, T), generator=g).to(DEV),
                torch.randint(0, 5000, (T,), generator=g).to(DEV, torch.int32)):
        oq, ok = rotary(q, k, table, pos, interleaved)
        p = torch.arange(T, device=DEV) if pos is None else pos
        for x, o in ((q, oq), (k, ok)):
            _close(o.detach(), ref.rotary(x.detach(), table, p, interleaved), x.detach(), R)
        gq, gk = torch.autograd.grad([oq, ok], [q, k], [dq, dk])
        for x, o in ((dq, gq), (dk, gk)):
            _close(o, ref.rotary(x, table, p, interleaved, inverse=True), x, R)


@gpu
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_views_of_a_fused_projection(offset):
    """q and k read in place through their strides, also where the view's start is not 16-byte aligned."""
    from macai_b200.rotary import rotary, rotary_table
    B, T, H, HK, D, R = 2, 40, 4, 2, 64, 16
    qkv = torch.randn(B, T, (H + 2 * HK) * D + offset, device=DEV).to(torch.bfloat16)
    q = qkv[..., offset:offset + H * D].unflatten(-1, (H, D))
    k = qkv[..., offset + H * D:offset + (H + HK) * D].unflatten(-1, (HK, D))
    table = rotary_table(T, R, device=DEV)
    oq, ok = rotary(q, k, table)
    for x, o in ((q, oq), (k, ok)):
        assert o.is_contiguous()
        _close(o, ref.rotary(x, table, torch.arange(T, device=DEV)), x, R)
    t = qkv[..., :2 * H * D].unflatten(-1, (H, 2 * D))[..., ::2]     # channels not adjacent: copied first
    o, none = rotary(t, None, table)
    assert none is None
    _close(o, ref.rotary(t, table, torch.arange(T, device=DEV)), t, R)
    o, _ = rotary(q.transpose(1, 2)[:, :3].transpose(1, 2)[:, 3:], None, table)
    _close(o, ref.rotary(q[:, 3:, :3], table, torch.arange(T - 3, device=DEV)), q[:, 3:, :3], R)


@gpu
def test_only_one_gradient_and_gradient_by_differences():
    from macai_b200.rotary import rotary, rotary_table
    q, k = torch.randn(1, 3, 2, 8, device=DEV).requires_grad_(True), torch.randn(1, 3, 1, 8, device=DEV).requires_grad_(True)
    table = rotary_table(9, 4, device=DEV)
    oq, ok = rotary(q, k, table)
    gk, = torch.autograd.grad(ok.sum(), [k])
    want = ref.rotary(torch.ones_like(k), table, torch.arange(3, device=DEV), inverse=True)
    assert (gk.double() - want).abs().max() < 1e-6
    oq, ok = rotary(q, None, table)
    w = torch.randn_like(q)
    gq, = torch.autograd.grad(oq, [q], w)
    for at in ((0, 2, 1, 0), (0, 1, 0, 3), (0, 2, 0, 7)):
        e = torch.zeros_like(q, dtype=torch.float64)
        e[at] = 1e-3
        p = torch.arange(3, device=DEV)
        d = ((ref.rotary(q.detach().double() + e, table, p) - ref.rotary(q.detach().double() - e, table, p)) * w.double()).sum() / 2e-3
        assert abs(float(d) - float(gq[at])) < 1e-5  # the turn is linear: differences are exact to rounding


@gpu
def test_positions_outside_the_table_take_its_nearest_row():
    from macai_b200.rotary import rotary, rotary_table
    q = torch.randn(1, 4, 1, 16, device=DEV)
    table = rotary_table(10, 16, device=DEV)
    far = torch.tensor([-5, 10, 2 ** 40, -2 ** 40], device=DEV)
    o, _ = rotary(q, None, table, far)
    near, _ = rotary(q, None, table, torch.tensor([0, 9, 9, 0], device=DEV))
    assert torch.equal(o, near)


def test_tables():
    """Scalings by their definitions, on the CPU."""
    from macai_b200.rotary import rotary_frequencies, rotary_table
    f, a = rotary_frequencies(64)
    assert a == 1 and torch.allclose(f, 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))
    assert torch.allclose(rotary_frequencies(64, scaling={"type": "linear", "factor": 4})[0], f / 4)
    n = rotary_frequencies(64, scaling={"type": "ntk", "factor": 4})[0]
    assert math.isclose(n[0], f[0]) and math.isclose(n[-1], f[-1] / 4, rel_tol=1e-12)
    y, att = rotary_frequencies(64, scaling={"type": "yarn", "factor": 4, "original_length": 4096})
    turns = f * 4096 / (2 * math.pi)
    assert torch.allclose(y[turns > 40], f[turns > 40]) and torch.allclose(y[turns < 0.8], f[turns < 0.8] / 4)
    assert ((y <= f * (1 + 1e-12)) & (y >= f / 4 * (1 - 1e-12))).all() and math.isclose(att, 0.1 * math.log(4) + 1)
    t = rotary_table(100001, 8, device="cpu")
    assert t.shape == (100001, 4, 2) and abs(float(t[100000, 0, 0]) - math.cos(100000.0)) < 1e-7
    for bad in ({"type": "yarn", "factor": 0}, {"type": "other", "factor": 2}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=bad)
    with pytest.raises(ValueError):
        rotary_frequencies(7)


@gpu
def test_refusals_and_no_tokens():
    from macai_b200.rotary import rotary, rotary_table
    q, k = torch.randn(1, 4, 2, 16, device=DEV), torch.randn(1, 4, 1, 16, device=DEV)
    table = rotary_table(8, 16, device=DEV)
    for bad in ((q, k.half(), table), (q, k[:, :3], table), (q[0], k, table), (q, k, table.double()),
                (q, k, rotary_table(8, 32, device=DEV)), (q, k, table[:3]), (q, k, table, torch.arange(4)),
                (q, k, table, torch.arange(3, device=DEV)), (q, k, table, torch.arange(4, device=DEV).float())):
        with pytest.raises(ValueError):
            rotary(*bad)
    with pytest.raises(RuntimeError, match="CPU"):
        rotary(q.cpu(), None, table)
    assert rotary(q[:, :0], k[:, :0], table)[0].shape == (1, 0, 2, 16)
