"""The residual RMS norm (macai_b200.norm) against its float64 definition.

Tolerances. u = the unit roundoff of the output's type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32): the last rounding is off by at
most u |y|, or half the spacing of the subnormals (2^-25 in fp16: ETA). What comes before it is fp32: a sum of D squares in chains of at most 16 + 37 additions, a division, a root
and three products, under 80 roundings of 2^-24 each, so 5e-6 relative to the terms that are added; dw adds up to
rows / CTAs + 64 terms in a chain, under 160 here: 1e-5 of the sum of the terms' sizes."""
import pytest
import torch

from oracle import layer_steps_f64 as ref

gpu = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ETA = {torch.float16: 2.0 ** -25}
TYPES = list(U)
DEV = "cuda"


def _inputs(rows, D, dt, wt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, res, dy, ds = (torch.randn(rows, D, generator=g).to(dt).to(DEV) for _ in range(4))
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(wt).to(DEV)
    return x, res, w, dy, ds


def _close(got, want, size, u, rel):
    err = (got.double() - want).abs()
    bad = err > u * want.abs() + ETA.get(got.dtype, 1e-30) + rel * size
    assert not bad.any(), (err[bad].max().item(), int(bad.sum()))


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (1, 2048), (5, 64), (700, 96), (33, 1111), (4, 8184), (2, 8190),
                                    (1300, 264), (9, 2056), (2, 8192)])
@pytest.mark.parametrize("wt32,zero_centered", [(False, False), (True, True)])
def test_forward_and_backward(dt, rows, D, wt32, zero_centered):
    from macai_b200.norm import add_rms_norm, supported
    wt = torch.float32 if wt32 else dt
    x, res, w, dy, ds = _inputs(rows, D, dt, wt, rows + D)
    if not supported(x, res, w):
        assert dt == torch.float32 and D > 8184
        with pytest.raises(ValueError):
            add_rms_norm(x, res, w)
        return
    for t in (x, res, w):
        t.requires_grad_(True)
    y, s = add_rms_norm(x, res, w, 1e-5, zero_centered)
    want, s64 = ref.rms_norm(x.detach(), res.detach(), w.detach(), 1e-5, zero_centered)
    assert torch.equal(s, s64)
    _close(y, want, want.abs(), U[dt], 5e-6)
    dx, dres, dw = torch.autograd.grad([y, s], [x, res, w], [dy, ds])
    wx, ww, bx, bw = ref.rms_norm_backward(s64, w.detach(), dy, ds, 1e-5, zero_centered)
    _close(dx, wx, bx, U[dt], 5e-6)
    assert torch.equal(dx, dres)
    _close(dw, ww, bw, U[wt], 1e-5)
    again = torch.autograd.grad(add_rms_norm(x, res, w, 1e-5, zero_centered), [x, w], [dy, ds])
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)  # the same bits every run


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16384, 16361])
def test_widest_rows(dt, D):
    from macai_b200.norm import add_rms_norm
    x, res, w, dy, ds = _inputs(3, D, dt, dt)
    x.requires_grad_(True), w.requires_grad_(True)
    y, s = add_rms_norm(x, res, w)
    want, s64 = ref.rms_norm(x.detach(), res, w.detach())
    _close(y, want, want.abs(), U[dt], 5e-6)
    dx, dw = torch.autograd.grad([y, s], [x, w], [dy, ds])
    wx, ww, bx, bw = ref.rms_norm_backward(s64, w.detach(), dy, ds)
    _close(dx, wx, bx, U[dt], 5e-6)
    _close(dw, ww, bw, U[dt], 1e-5)


@gpu
def test_many_rows_share_ctas():
    """More rows than resident CTAs: the persistent backward's loop, its partial rows and their sum."""
    from macai_b200.norm import add_rms_norm
    x, res, w, dy, ds = _inputs(20011, 136, torch.bfloat16, torch.float32)
    x.requires_grad_(True), w.requires_grad_(True)
    y, s = add_rms_norm(x, res, w)
    dx, dw = torch.autograd.grad([y, s], [x, w], [dy, ds])
    want, s64 = ref.rms_norm(x.detach(), res, w.detach())
    wx, ww, bx, bw = ref.rms_norm_backward(s64, w.detach(), dy, ds)
    _close(y, want, want.abs(), 2.0 ** -8, 5e-6)
    _close(dx, wx, bx, 2.0 ** -8, 5e-6)
    _close(dw, ww, bw, 2.0 ** -24, 1e-5)


@gpu
def test_without_residual_and_missing_cotangents():
    from macai_b200.norm import add_rms_norm
    x, res, w, dy, ds = _inputs(37, 200, torch.bfloat16, torch.bfloat16)
    x.requires_grad_(True), w.requires_grad_(True), res.requires_grad_(True)
    y, s = add_rms_norm(x, None, w)
    assert s is x
    zero = torch.zeros_like(ds)
    want, _ = ref.rms_norm(x.detach(), None, w.detach())
    _close(y, want, want.abs(), 2.0 ** -8, 5e-6)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    wx, ww, bx, bw = ref.rms_norm_backward(x.detach(), w.detach(), dy, zero)
    _close(dx, wx, bx, 2.0 ** -8, 5e-6)
    _close(dw, ww, bw, 2.0 ** -8, 1e-5)
    y, s = add_rms_norm(x, res, w)
    s64 = s.detach()
    dx, = torch.autograd.grad(y, [res], dy, retain_graph=True)   # no gradient into s
    wx, ww, bx, _ = ref.rms_norm_backward(s64, w.detach(), dy, zero)
    _close(dx, wx, bx, 2.0 ** -8, 5e-6)
    dx, = torch.autograd.grad(s, [x], ds)                        # only through s
    assert torch.equal(dx, ds)


@gpu
def test_gradient_against_differences():
    """fp32, central differences of the float64 definition at the kernel's inputs: h = 1e-4, error O(h^2) and the
    kernel's own 5e-6."""
    from macai_b200.norm import add_rms_norm
    x, res, w, dy, ds = _inputs(2, 24, torch.float32, torch.float32)
    x.requires_grad_(True), w.requires_grad_(True)
    y, s = add_rms_norm(x, res, w)
    dx, dw = torch.autograd.grad([y, s], [x, w], [dy, ds])

    def value(xx, ww):
        s64 = xx + res.double()
        yy = s64 / torch.sqrt((s64 * s64).mean(-1, keepdim=True) + 1e-6) * ww
        return float((yy * dy.double()).sum() + (s64 * ds.double()).sum())
    h = 1e-4
    for i in (0, 7, 23):
        e = torch.zeros(2, 24, dtype=torch.float64, device=DEV)
        e[1, i] = h
        d = (value(x.detach().double() + e, w.detach().double()) - value(x.detach().double() - e, w.detach().double())) / (2 * h)
        assert abs(d - float(dx[1, i])) < 1e-5 * (1 + abs(d))
        e = torch.zeros(24, dtype=torch.float64, device=DEV)
        e[i] = h
        d = (value(x.detach().double(), w.detach().double() + e) - value(x.detach().double(), w.detach().double() - e)) / (2 * h)
        assert abs(d - float(dw[i])) < 1e-5 * (1 + abs(d))


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,D,group", [(1, 128, 128), (5, 4096, 128), (700, 2048, 128), (3, 1111, 64), (2, 200, None),
                                          (9, 2056, 32), (4, 96, 24), (7, 72, 8), (1, 5, 8), (2, 8184, None),
                                          (1500, 264, 256)])
def test_fp8(dt, rows, D, group):
    """Scales to 5e-6 (fp32 chain); codes: the nearest e4m3 to y / scale, where a quotient within 1e-5 of the middle of
    two codes may go either way."""
    from macai_b200.norm import add_rms_norm_fp8
    x, res, w, _, _ = _inputs(rows, D, dt, torch.float32, rows * D)
    x[0] = -res[0]                      # an all-zero row: scale 1, codes 0
    q, scale, s = add_rms_norm_fp8(x, res, w, 1e-6, group)
    y, s64 = ref.rms_norm(x, res, w)
    assert torch.equal(s, s64) and q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    ws, ratio = ref.fp8_scales(y, group)
    assert scale.shape == ws.shape
    assert ((scale.double() - ws).abs() <= 5e-6 * ws).all()
    assert (scale[0] == 1).all() and (q[0].float() == 0).all()
    lo = (ratio * (1 - 1e-5)).float().clamp(-448, 448).to(torch.float8_e4m3fn).float()
    hi = (ratio * (1 + 1e-5)).float().clamp(-448, 448).to(torch.float8_e4m3fn).float()
    got = q.float()
    assert ((got == lo) | (got == hi)).all()


@gpu
def test_infinities_and_nan_stay_in_their_row():
    from macai_b200.norm import add_rms_norm, add_rms_norm_fp8
    x, res, w, _, _ = _inputs(6, 100, torch.bfloat16, torch.bfloat16)
    x[2, 50], x[4, 99] = float("nan"), float("inf")
    y, s = add_rms_norm(x, res, w)
    clean = [0, 1, 3, 5]
    want, _ = ref.rms_norm(x[clean], res[clean], w)
    _close(y[clean], want, want.abs(), 2.0 ** -8, 5e-6)
    assert y[2].isnan().all() and y[4, 99].isnan() and s[4, 99].isinf()
    q, scale, _ = add_rms_norm_fp8(x, res, w, group=None)
    assert q[2].float().isnan().all() and not q[clean].float().isnan().any() and not scale[clean].isnan().any()


@gpu
def test_no_rows_views_and_streams():
    from macai_b200.norm import add_rms_norm
    x, res, w, dy, _ = _inputs(8, 64, torch.bfloat16, torch.bfloat16)
    e = x[:0].requires_grad_(True)
    w.requires_grad_(True)
    y, s = add_rms_norm(e, res[:0], w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, [e, w], dy[:0])
    assert dx.shape == (0, 64) and (dw == 0).all()
    w = w.detach()
    base = torch.randn(8, 130, device=DEV).to(torch.bfloat16)
    y, s = add_rms_norm(base[:, 1:65], None, w)                      # a view of unaligned rows
    want, _ = ref.rms_norm(base[:, 1:65], None, w)
    _close(y, want, want.abs(), 2.0 ** -8, 5e-6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, s2 = add_rms_norm(x, res, w)
    torch.cuda.current_stream().wait_stream(side)
    y1, s1 = add_rms_norm(x, res, w)
    assert torch.equal(y1, y2) and torch.equal(s1, s2)
    assert add_rms_norm(x.view(2, 4, 64), res.view(2, 4, 64), w)[0].shape == (2, 4, 64)


@gpu
def test_refusals():
    from macai_b200.norm import add_rms_norm, add_rms_norm_fp8
    x, res, w, _, _ = _inputs(4, 64, torch.bfloat16, torch.bfloat16)
    for a in ((x, res.float(), w), (x, res[:2], w), (x, res, w[:32]), (x, res, w.half()), (x.double(), None, w.double()),
              (x.cpu(), None, w.cpu())):
        with pytest.raises(ValueError):
            add_rms_norm(*a)
    for group in (0, -8, 12):
        with pytest.raises(ValueError):
            add_rms_norm_fp8(x, res, w, group=group)
    with pytest.raises(RuntimeError, match="no gradient"):
        add_rms_norm_fp8(x.requires_grad_(True), res, w)
