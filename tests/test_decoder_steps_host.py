"""Feed-forward block and cross entropy without a GPU: what they refuse (Python and C ABI), and their float64 definitions
against torch's own operations and against differences."""
import ctypes

import pytest
import torch

from macai_b200 import _lib
from macai_b200.feed_forward import gated_feed_forward
from macai_b200.loss import linear_cross_entropy
from oracle import decoder_steps_f64 as steps

NUL, ONE, ODD = ctypes.c_void_p(0), ctypes.c_void_p(256), ctypes.c_void_p(264)
BF, F16, F32 = _lib.GD_BFLOAT16, _lib.GD_FLOAT16, _lib.GD_FLOAT32


def _ld(*x):
    return (ctypes.c_longlong * len(x))(*x)


def test_feed_forward_abi():
    lib = _lib.load()

    def fwd(x=ONE, y=ONE, kept=ONE, bounds=ONE, dt=BF, rows=10, D=64, F=128, O=64, ld=None, ws=ONE, n=1 << 40):
        return lib.gd_ff_fwd(x, ONE, ONE, ONE, kept, bounds, y, dt, rows, D, F, O, ld or _ld(64, 64, 64, 128), ws, n, NUL)

    def bwd(x=ONE, y=ONE, kept=ONE, bounds=ONE, dt=BF, rows=10, D=64, F=128, O=64, ld=None, ws=ONE, n=1 << 40):
        return lib.gd_ff_bwd(x, ONE, ONE, ONE, kept, bounds, y, ONE, ONE, ONE, ONE, dt, rows, D, F, O,
                             ld or _ld(64, 64, 64, 128, 64), ws, n, NUL)
    for f in (fwd, bwd):
        assert f(dt=F32) == _lib.GD_ERR_ARG and f(x=NUL) == _lib.GD_ERR_ARG and f(y=NUL) == _lib.GD_ERR_ARG
        for kw in ({"D": 60}, {"D": 0}, {"F": 100}, {"F": -8}, {"O": 4}, {"rows": -1}, {"rows": 1 << 31}, {"F": 1 << 25}):
            assert f(**kw) == _lib.GD_ERR_SHAPE, kw
        assert f(ld=_ld(56, 64, 64, 128, 64)) == _lib.GD_ERR_SHAPE and f(ld=_ld(68, 64, 64, 128, 64)) == _lib.GD_ERR_ALIGN
        assert f(ld=_ld(64, 64, 64, 120, 64)) == _lib.GD_ERR_SHAPE and f(x=ODD) == _lib.GD_ERR_ALIGN and f(y=ODD) == _lib.GD_ERR_ALIGN
        assert f(ws=NUL) == _lib.GD_ERR_WORKSPACE and f(ws=ODD) == _lib.GD_ERR_ALIGN
    size = lib.gd_ff_workspace_bytes
    for back, f in ((0, fwd), (1, bwd)):
        need = size(10, 64, 128, 64, back)
        assert need >= 10 * 128 * 2 and f(n=need - 1) == _lib.GD_ERR_WORKSPACE
    assert fwd(dt=F16, bounds=NUL) == _lib.GD_ERR_ARG and bwd(dt=F16, bounds=NUL) == _lib.GD_ERR_ARG
    assert bwd(kept=NUL) == _lib.GD_ERR_ARG
    assert bwd(ld=_ld(64, 64, 64, 128, 60)) == _lib.GD_ERR_SHAPE
    assert fwd(rows=0, x=NUL, y=NUL, ws=NUL) == _lib.GD_OK
    assert size(10, 60, 128, 64, 0) == 0 and size(-1, 64, 128, 64, 0) == 0


def test_cross_entropy_abi():
    lib = _lib.load()

    def fwd(x=ONE, lab=ONE, loss=ONE, red=1, dt=BF, rows=10, D=64, V=100, ldx=64, ldw=64, ws=ONE, n=1 << 40):
        return lib.gd_xent_fwd(x, ONE, lab, 1, loss, ONE, ONE, red, -100, dt, rows, D, V, ldx, ldw, ws, n, NUL)

    def bwd(x=ONE, lab=ONE, loss=ONE, red=1, dt=BF, rows=10, D=64, V=100, ldx=64, ldw=64, ws=ONE, n=1 << 40):
        return lib.gd_xent_bwd(x, ONE, ONE, lab, loss, ONE, ONE, red, dt, rows, D, V, ldx, ldw, ws, n, NUL)
    for back, f in ((0, fwd), (1, bwd)):
        for kw in ({"dt": F32}, {"red": 3}, {"red": -1}, {"x": NUL}, {"lab": NUL}, {"loss": NUL}):
            assert f(**kw) == _lib.GD_ERR_ARG, kw
        for kw in ({"D": 60}, {"D": 0}, {"V": 0}, {"V": 1 << 25}, {"rows": -1}, {"rows": 1 << 25}, {"ldx": 56}, {"ldw": 8}):
            assert f(**kw) == _lib.GD_ERR_SHAPE, kw
        assert f(ldx=68) == _lib.GD_ERR_ALIGN and f(x=ODD) == _lib.GD_ERR_ALIGN and f(ws=ODD) == _lib.GD_ERR_ALIGN
        need = lib.gd_xent_workspace_bytes(10, 64, 100, back)
        assert need > 0 and f(n=need - 1) == _lib.GD_ERR_WORKSPACE and f(ws=NUL) == _lib.GD_ERR_WORKSPACE
    assert fwd(rows=0, x=NUL, lab=NUL, loss=NUL, ws=NUL) == _lib.GD_OK
    assert lib.gd_xent_workspace_bytes(0, 64, 100, 1) == 0 and lib.gd_xent_workspace_bytes(10, 60, 100, 0) == 0
    # the backward never holds more of the logits' gradients than it says
    assert lib.gd_xent_workspace_bytes(1 << 14, 1024, 1 << 17, 1) <= (256 << 20) + (1 << 14) * 1024 * 8 + (1 << 20)


def test_feed_forward_refusals():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    x, w, d = bf(2, 64), bf(128, 64), bf(64, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_feed_forward(x, w, w, d)
    with pytest.raises(TypeError, match="float32"):
        gated_feed_forward(x.float(), w.float(), w.float(), d.float())
    with pytest.raises(ValueError, match="share"):
        gated_feed_forward(x, w, w.half(), d)
    with pytest.raises(ValueError, match="matrix"):
        gated_feed_forward(x, w, w[0], d)
    with pytest.raises(ValueError, match="x must"):
        gated_feed_forward(None, w, w, d)


def test_cross_entropy_refusals():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16)
    lab = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_cross_entropy(x, w, lab)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, lab, reduction="max")
    with pytest.raises(ValueError, match="ignore_index"):
        linear_cross_entropy(x, w, lab, ignore_index=None)
    with pytest.raises(TypeError, match="float32"):
        linear_cross_entropy(x.float(), w.float(), lab)
    with pytest.raises(TypeError, match="labels"):
        linear_cross_entropy(x, w, lab.float())
    with pytest.raises(ValueError, match="share"):
        linear_cross_entropy(x, w.half(), lab)
    with pytest.raises(ValueError, match="weight"):
        linear_cross_entropy(x, w[0], lab)


def test_feed_forward_definition():
    """The formulas' gradients are torch's, and differences'."""
    torch.manual_seed(0)
    ts = [torch.randn(*s).bfloat16() for s in ((5, 16), (24, 16), (24, 16), (8, 24))]
    dy = torch.randn(5, 8).bfloat16()
    got = steps.feed_forward(*ts, dy)
    leaves = [t.double().requires_grad_(True) for t in ts]

    def f(x, wg, wu, wd):
        return (torch.nn.functional.silu(x @ wg.T) * (x @ wu.T)) @ wd.T
    y = f(*leaves)
    want = [y, *torch.autograd.grad(y, leaves, dy.double())]
    for k, v in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), want):
        assert float((got[k][0] - v.detach()).abs().max()) < 1e-12, k
    assert torch.autograd.gradcheck(f, leaves)


def test_cross_entropy_definition():
    torch.manual_seed(0)
    x, w = torch.randn(6, 16).bfloat16(), torch.randn(11, 16).bfloat16()
    lab = torch.tensor([0, 10, -100, 3, 3, -100])
    g = torch.rand(6)
    got = steps.cross_entropy(x, w, lab, g=g)
    leaves = [t.double().requires_grad_(True) for t in (x, w)]

    def f(x, w):
        return torch.nn.functional.cross_entropy(x @ w.T, lab, reduction="none")
    y = f(*leaves)
    want = [y, *torch.autograd.grad(y, leaves, g.double())]
    for k, v in zip(("loss", "dx", "dweight"), want):
        assert float((got[k][0] - v.detach()).abs().max()) < 1e-12, k
    assert torch.autograd.gradcheck(f, leaves)
