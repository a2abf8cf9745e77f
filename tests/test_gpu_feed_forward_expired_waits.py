"""The feed-forward block where a wait on the device gives up: NaN in all that could not be computed, what is kept for the
backward included, the stage in the error word, and a normal next call."""
import ctypes

import pytest
import torch

from macai_b200 import _lib

pytestmark = pytest.mark.gpu
N, D, F, O = 150, 64, 128, 64   # one tile of every product


def _block(dt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda a, b, s: (torch.randn(a, b, generator=gen) * s).to(dt).cuda()  # noqa: E731
    return r(N, D, 1.0), r(F, D, D ** -0.5), r(F, D, D ** -0.5), r(O, F, F ** -0.5), r(N, O, 0.1)


def _at(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _error(ws):
    where = ctypes.c_int(-1)
    code = _lib.load().gd_read_error(_at(ws), _stream(), ctypes.byref(where))
    return code, where.value


def _forward(x, wg, wu, wd, extra=0):
    lib, half = _lib.load(), x.dtype == torch.float16
    kept = torch.zeros(3, N, F, dtype=torch.int16, device="cuda")
    bounds = torch.zeros(4, dtype=torch.int32, device="cuda") if half else None
    y = torch.zeros(N, O, dtype=x.dtype, device="cuda")
    n = lib.gd_ff_workspace_bytes(N, D, F, O, 0)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    ld = (ctypes.c_longlong * 4)(D, D, D, F)
    _lib.check(lib.gd_ff_fwd(_at(x), _at(wg), _at(wu), _at(wd), _at(kept), _at(bounds), _at(y),
                             (_lib.GD_FLOAT16 if half else _lib.GD_BFLOAT16) | extra, N, D, F, O, ld, _at(ws), n, _stream()), "gd_ff_fwd")
    return y, kept, bounds, _error(ws)


def _backward(x, wg, wu, wd, dy, kept, bounds, extra=0, need=(0, 1, 2, 3)):
    lib, half = _lib.load(), x.dtype == torch.float16
    out = [torch.zeros_like(t) if i in need else None for i, t in enumerate((x, wg, wu, wd))]
    n = lib.gd_ff_workspace_bytes(N, D, F, O, 1)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    ld = (ctypes.c_longlong * 5)(D, D, D, F, O)
    _lib.check(lib.gd_ff_bwd(_at(x), _at(wg), _at(wu), _at(wd), _at(kept), _at(bounds), _at(dy), *(_at(t) for t in out),
                             (_lib.GD_FLOAT16 if half else _lib.GD_BFLOAT16) | extra, N, D, F, O, ld, _at(ws), n, _stream()), "gd_ff_bwd")
    return [t for t in out if t is not None], _error(ws)


def _planes(kept):
    """g and u from what is kept of them."""
    word = lambda t: t.to(torch.int32) & 0xffff  # noqa: E731
    g, u, low = word(kept[0]), word(kept[1]), word(kept[2])
    return ((g << 16) | ((low & 0xff) << 8)).view(torch.float32), ((u << 16) | (low & 0xff00)).view(torch.float32)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_forward(dt):
    """A forward that could not wait for its products keeps no numbers that a backward would take for g and u."""
    x, wg, wu, wd, dy = _block(dt)
    clean = _forward(x, wg, wu, wd)
    assert clean[3][0] == _lib.GD_OK and bool(clean[0].isfinite().all())
    g, u = _planes(clean[1])
    # (what the planes hold: the upper 24 bits, 2^-15 of the value at most below it, the products' own rounding of 64 terms)
    assert float((g - x.float() @ wg.float().T).abs().max()) < 1e-3 and float((u - x.float() @ wu.float().T).abs().max()) < 1e-3
    y, kept, bounds, error = _forward(x, wg, wu, wd, _lib.GD_TEST_WAIT_EXPIRES)
    assert error == (_lib.GD_ERR_TIMEOUT, 85)
    g, u = _planes(kept)
    assert bool(y.isnan().all()) and bool(g.isnan().all()) and bool(u.isnan().all())
    grads, error = _backward(x, wg, wu, wd, dy, kept, bounds)
    assert error[0] == _lib.GD_OK and all(bool(t.isnan().all()) for t in grads)
    again = _forward(x, wg, wu, wd)
    assert again[3][0] == _lib.GD_OK and all(torch.equal(a, b) for a, b in zip(again[:2], clean[:2]))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("need", [(0, 1, 2, 3), (3,), (0,)])
def test_backward(dt, need):
    """A backward that could not wait for what was kept: no gradient is made of numbers that did not arrive."""
    x, wg, wu, wd, dy = _block(dt, seed=1)
    _, kept, bounds, _ = _forward(x, wg, wu, wd)
    clean, error = _backward(x, wg, wu, wd, dy, kept, bounds, need=need)
    assert error[0] == _lib.GD_OK and all(bool(t.isfinite().all()) for t in clean)
    grads, error = _backward(x, wg, wu, wd, dy, kept, bounds, _lib.GD_TEST_WAIT_EXPIRES, need)
    assert error == (_lib.GD_ERR_TIMEOUT, 86) and all(bool(t.isnan().all()) for t in grads)
    again, error = _backward(x, wg, wu, wd, dy, kept, bounds, need=need)
    assert error[0] == _lib.GD_OK and all(torch.equal(a, b) for a, b in zip(again, clean))
