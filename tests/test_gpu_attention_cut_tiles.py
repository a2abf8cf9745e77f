"""The backward of window_attention where the first key tiles are cut into parts with fp32 partial tiles, at head widths
above 128 too (two CTAs a tile, a half of the channels each). Bounds as in the other attention tests: the parts' sums are
fp32."""
import pytest
import torch

from macai_b200 import _lib
from test_gpu_window_attention import BF, HF, _bounds, _check, _inputs, _run

gpu = pytest.mark.gpu
SHAPES = [(1, 900, 900, 8, 1, 256, None, 0), (1, 900, 900, 8, 1, 136, 200, 150), (1, 700, 1000, 4, 1, 248, None, 0),
          (2, 640, 640, 6, 1, 192, 128, 1), (1, 900, 900, 8, 1, 128, None, 0), (1, 900, 900, 8, 1, 72, 200, 150)]


def _is_cut(B, Tq, Tk, H, HK, D, w, s):
    """More workspace than the error word and delta take."""
    delta = (B * H * Tq * 4 + 255) // 256 * 256
    return _lib.load().gd_wattn_workspace_bytes(B, Tq, Tk, H, HK, D, w or 0, s, 0, 1) > 256 + delta


def test_the_shapes_are_cut():
    assert all(_is_cut(*shape) for shape in SHAPES)


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_cut_tiles(shape, dt):
    B, Tq, Tk, H, HK, D, w, s = shape
    q, k, v, do = _inputs(B, Tq, Tk, H, HK, D, dt, D)
    got = _run(q, k, v, do, window=w, sinks=s)
    _check(got, *_bounds(q, k, v, do, w, s, D ** -0.5), shape)
    assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do, window=w, sinks=s)))
