"""float16's range in window_attention's gradients.

P is rounded as 2^15 P (exact scaling; P <= 1), so nothing above 2^-29 loses bits and below that the error is at most 2^-40.
dS is rounded as F dS with a power of two F such that 2 F max ||do|| max ||v|| lies in [2^13, 2^15] (it bounds F |dS|, by
Cauchy and Schwarz): besides u |dS| it is within 2^-25 / F <= 2^-37 max ||do|| max ||v||. Added to the bounds of the other
attention tests:  dv: sum_i 2^-40 |do|,  dq: scale sum_j 2^-37 M |k|,  dk: scale sum_i 2^-37 M |q|."""
import pytest
import torch

from oracle import layer_steps_f64 as ref
from test_gpu_window_attention import DEV, HF, _bounds, _check, _inputs, _run

gpu = pytest.mark.gpu


def _wider(tol, q, k, v, do, window, sinks, scale):
    H, HK = q.shape[2], k.shape[2]
    seen = ref.visible(q.shape[1], k.shape[1], window, sinks, q.device).double()
    M = float(do.double().norm(dim=-1).max() * v.double().norm(dim=-1).max())
    for h in range(H):
        c = h * HK // H
        for b in range(q.shape[0]):
            tol[1][b, :, h] += scale * 2.0 ** -37 * M * (seen @ k[b, :, c].double().abs())
            tol[2][b, :, c] += scale * 2.0 ** -37 * M * (seen.T @ q[b, :, h].double().abs())
            tol[3][b, :, c] += 2.0 ** -40 * (seen.T @ do[b, :, h].double().abs())
    return tol


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_values_and_tiny_cotangents(D):
    """|do| of 1e-4 and |v| up to 60,000: dS is a moderate number, whatever do's scale alone would make of it."""
    q, k, v, do = _inputs(1, 300, 300, 2, 1, D, HF, 3)
    v = (v.float() * 2e4).clamp(-6e4, 6e4).half()
    do = (do.float() * 1e-4).half()
    got = _run(q, k, v, do, window=100, sinks=2)
    res, tol = _bounds(q, k, v, do, 100, 2, D ** -0.5)
    _check(got, res, _wider(tol, q, k, v, do, 100, 2, D ** -0.5), D)


@gpu
@pytest.mark.parametrize("Tq,Tk,D", [(3, 40000, 64), (130, 20000, 128), (2, 33000, 256)])
def test_long_rows(Tq, Tk, D):
    """P of some 2^-16 each, at the foot of float16's normal numbers."""
    q, k, v, do = _inputs(1, Tq, Tk, 1, 1, D, HF, 4)
    do = (do.float() * 500).half()
    got = _run(q, k, v, do)
    res, tol = _bounds(q, k, v, do, None, 0, D ** -0.5)
    _check(got, res, _wider(tol, q, k, v, do, None, 0, D ** -0.5), Tk)


@gpu
def test_a_token_of_small_cotangent_beside_large_ones():
    q, k, v, do = _inputs(1, 500, 500, 2, 1, 64, HF, 5)
    do = (do.float() * torch.logspace(-4, 2, 500, device=DEV)[None, :, None, None]).half()
    got = _run(q, k, v, do, window=200)
    res, tol = _bounds(q, k, v, do, 200, 0, 0.125)
    _check(got, res, _wider(tol, q, k, v, do, 200, 0, 0.125), "mixed")


@gpu
def test_infinities_do_not_take_the_scale():
    """Packed sequences: one sequence's infinities leave the others' gradients as they are, float16's scale included."""
    cu = torch.tensor([0, 150, 300, 500], dtype=torch.int32)
    q, k, v, do = _inputs(1, 500, 500, 2, 1, 64, HF, 6)
    do[:, 150:300] = 0
    v[:, 150:300] = 0
    want = _run(q, k, v, do, window=90, cu_seqlens=cu)
    for bad in (float("nan"), float("inf")):
        w = [t.clone() for t in (q, k, v, do)]
        for t in w:
            t[:, 150:300] = bad
        got = _run(*w, window=90, cu_seqlens=cu)
        for a, b in ((0, 150), (300, 500)):
            assert all(torch.equal(x[:, a:b], y[:, a:b]) for x, y in zip(want, got)), bad
