"""What the rule's recurrent form refuses, without a GPU; its float64 definition against the reference recurrence."""
import ctypes

import pytest
import torch

from macai_b200 import _lib
from macai_b200.gated_delta import gated_delta_step, recurrent_gated_delta_rule, recurrent_reference
from oracle import decoder_steps_f64 as steps

NUL, ONE, ODD = ctypes.c_void_p(0), ctypes.c_void_p(256), ctypes.c_void_p(264)
BF, F16, F32 = _lib.GD_BFLOAT16, _lib.GD_FLOAT16, _lib.GD_FLOAT32


def test_abi():
    lib = _lib.load()

    def f(q=ONE, o=ONE, s_in=ONE, s_out=ONE, slots=ONE, out=ONE, dt=BF, vdt=BF, B=2, T=1, H=4, HK=2, DK=64, DV=64, S=8,
          flags=0):
        return lib.gd_rule_step(q, ONE, ONE, ONE, ONE, s_in, s_out, slots, out, o, dt, vdt, B, T, H, HK, DK, DV, S, flags, NUL)
    for kw in ({"dt": 7}, {"vdt": F16}, {"dt": F32, "vdt": BF}, {"flags": 4}, {"q": NUL}, {"o": NUL}, {"slots": NUL}, {"out": NUL}):
        assert f(**kw) == _lib.GD_ERR_ARG, kw
    for kw in ({"B": -1}, {"B": 65536}, {"T": -1}, {"H": 3}, {"H": 0}, {"HK": 0}, {"DK": 0}, {"DK": 48}, {"DV": 288}, {"S": -1},
               {"slots": NUL, "out": NUL, "S": 1}):
        assert f(**kw) == _lib.GD_ERR_SHAPE, kw
    assert f(s_in=ODD) == _lib.GD_ERR_ALIGN and f(s_out=ODD) == _lib.GD_ERR_ALIGN
    assert f(B=0, q=NUL, o=NUL, slots=NUL, out=NUL) == _lib.GD_OK


def test_python_refusals():
    q, v, g, s = torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4), torch.zeros(1, 4, 64, 64)
    for f in (gated_delta_step, recurrent_gated_delta_rule):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(q, q, v, g, g, s)
        with pytest.raises(TypeError, match="float"):
            f(q.int(), q, v, g, g, s)
        with pytest.raises(ValueError, match="query"):
            f(q[0], q, v, g, g, s)
    with pytest.raises(NotImplementedError, match="packed"):
        recurrent_gated_delta_rule(q, q, v, g, g, cu_seqlens=torch.tensor([0, 1]))


def test_definition():
    """The oracle's recurrence is the reference's (q already scaled there)."""
    torch.manual_seed(0)
    q, k, v = torch.randn(2, 5, 2, 32).double(), torch.randn(2, 5, 2, 32).double(), torch.randn(2, 5, 4, 64).double()
    g, beta, s0 = -torch.rand(2, 5, 4).double(), torch.rand(2, 5, 4).double(), torch.randn(2, 4, 32, 64).double()
    o, s, eo, es = steps.rule_step(q, k, v, g, beta, s0)
    rep = lambda x: x.repeat_interleave(2, 2)  # noqa: E731
    want, sw = recurrent_reference(rep(q) * 32 ** -0.5, rep(k), v, g, beta, s0)
    assert float((o - want).abs().max()) < 1e-12 and float((s - sw).abs().max()) < 1e-12
    # its bounds hold for the same recurrence in float32
    f = lambda x: x.float()  # noqa: E731
    o32, s32 = recurrent_reference(f(rep(q)) * 32 ** -0.5, f(rep(k)), f(v), f(g), f(beta), f(s0))
    o64, s64, eo, es = steps.rule_step(f(q), f(k), f(v), f(g), f(beta), f(s0))
    assert bool(((o32 - o64).abs() <= eo + 2.0 ** -24 * o64.abs()).all()) and bool(((s32 - s64).abs() <= es).all())
