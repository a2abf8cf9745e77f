"""Packed rows whose boundaries lie on the device, where the host does not look at them (macai_b200.window_attention): rows
outside every sequence give zeros, in the result and in the gradients; a boundary below an earlier one counts as that one."""
import pytest
import torch

from test_gpu_window_attention import BF, DEV, HF, _bounds, _check, _inputs, _run

gpu = pytest.mark.gpu


def _dirty(like):
    """Memory that the allocator hands out next holds NaN."""
    ts = [torch.full_like(t, float("nan")) for t in like for _ in range(4)]
    ts += [torch.full((like[0].numel(),), float("nan"), device=DEV) for _ in range(2)]
    del ts


def _seqs(cu, T):
    top, out = 0, []
    for a, b in zip(cu, cu[1:]):
        top = max(top, min(max(a, 0), T))
        out.append((top, max(top, min(max(b, 0), T))))
    return out


def _verify(cu, T, H, HK, D, w, s, dt):
    q, k, v, do = _inputs(1, T, T, H, HK, D, dt, T + len(cu))
    _dirty((q, k, v, do))
    got = _run(q, k, v, do, window=w, sinks=s, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    outside = torch.ones(T, dtype=torch.bool, device=DEV)
    for a, b in _seqs(cu, T):
        if b > a:
            outside[a:b] = False
            part = [t[:, a:b] for t in (q, k, v, do)]
            _check([t[:, a:b] for t in got], *_bounds(*part, w, s, D ** -0.5), (a, b))
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        assert (t[:, outside] == 0).all(), (cu, name)


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,cu", [(300, [0, 250]), (300, [20, 300]), (700, [20, 150, 150, 427, 650]), (100, [0, 50]),
                                  (128, [0, 127]), (640, [128, 256]), (513, [0, 0]), (257, [257, 257]), (1, [0, 0]),
                                  (300, [299, 300]), (900, [130, 131, 132, 140])])
def test_rows_outside_every_sequence(T, cu, D, dt):
    _verify(cu, T, 4, 2, D, 90, 3, dt)


@gpu
def test_many_sequences_between_gaps():
    """More sequences than a warp's scan step holds (256), and exactly as many."""
    for n in (256, 257, 700):
        cu = [37]
        for i in range(n):
            cu.append(cu[-1] + (7 * i) % 5)
        _verify(cu, cu[-1] + 200, 2, 1, 64, 3, 0, BF)


@gpu
@pytest.mark.parametrize("cu", [[0, 200, 100, 500], [400, 100, 300, 500], [0, 999, -3, 500], [-7, 100, 100, 90, 480]])
def test_boundaries_that_fall(cu):
    _verify(cu, 500, 4, 2, 128, 60, 1, BF)
