"""Scales of the scores that are zero or negative (macai_b200.window_attention), against the float64 formulas. The negative
scale -c is the scale c with -q (exact in 16 bits), so the bounds are those of the positive scale: results o, dk and dv are
the same, dq changes its sign."""
import pytest
import torch

from oracle import layer_steps_f64 as ref
from test_gpu_window_attention import BF, DEV, F, HF, U, _bounds, _check, _inputs, _run

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,Tq,Tk,H,HK,D,w,s", [(1, 300, 300, 2, 1, 64, 100, 3), (2, 200, 333, 4, 2, 128, None, 0),
                                                (1, 400, 400, 2, 2, 256, 150, 130), (1, 130, 50, 2, 1, 80, 20, 0)])
@pytest.mark.parametrize("c", [0.3, 0.011, 1e-30])
def test_negative_scales(B, Tq, Tk, H, HK, D, w, s, c, dt):
    q, k, v, do = _inputs(B, Tq, Tk, H, HK, D, dt, 5)
    c = min(c, 2.4 * D ** -0.5)      # scores of the size that the bounds' f was derived for
    o, dq, dk, dv = _run(q, k, v, do, window=w, sinks=s, scale=-c)
    _check((o, -dq, dk, dv), *_bounds(-q, k, v, do, w, s, c), c)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_zero_scale(D):
    """Every visible key weighs the same; q and k have no gradient."""
    q, k, v, do = _inputs(1, 300, 300, 2, 1, D, BF, 6)
    o, dq, dk, dv = _run(q, k, v, do, window=77, sinks=2, scale=0.0)
    res, tol = _bounds(q, k, v, do, 77, 2, 0.0)
    _check((o, dq, dk, dv), res, tol, D)
    assert (dq == 0).all() and (dk == 0).all()


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_packed_rows_and_the_step(scale):
    from macai_b200.window_attention import window_attention, window_attention_step
    q, k, v, do = _inputs(1, 300, 300, 4, 2, 64, BF, 7)
    o = window_attention(q, k, v, window=50, sinks=1, scale=scale, cu_seqlens=torch.tensor([0, 90, 300]))
    for a, b in ((0, 90), (90, 300)):
        r = ref.attention(q[:, a:b], k[:, a:b], v[:, a:b], 50, 1, scale)
        A = ref.attention(q[:, a:b], k[:, a:b], v[:, a:b].abs(), 50, 1, scale)
        assert ((o[:, a:b].double() - r).abs() <= U[BF] * r.abs() + (U[BF] + F) * A).all()
    kc, vc = k[:, :200].clone(), v[:, :200].clone()
    L = torch.tensor([150], dtype=torch.int32, device=DEV)
    one = [t[:, 150:151] for t in (q, k, v)]
    ro, _, _ = ref.attention_step(*one, kc, vc, L, 50, 1, scale)
    A, _, _ = ref.attention_step(*one[:2], one[2].abs(), kc, vc.abs(), L, 50, 1, scale)
    o = window_attention_step(*one, kc, vc, L, 50, 1, scale)
    assert ((o.double() - ro).abs() <= U[BF] * ro.abs() + (U[BF] + F) * A).all()
