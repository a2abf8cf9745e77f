"""The C ABI of the softmax-attention layer's steps without a GPU: bad arguments come back as status codes before any
device call."""
import ctypes

from macai_b200 import _lib

NUL, ONE, ODD = ctypes.c_void_p(0), ctypes.c_void_p(256), ctypes.c_void_p(258)
BF, F16, F32 = _lib.GD_BFLOAT16, _lib.GD_FLOAT16, _lib.GD_FLOAT32


def test_rnorm_refusals():
    lib = _lib.load()
    f = lambda x=ONE, w=ONE, s=ONE, y=ONE, dt=BF, wt=BF, rows=10, D=128: lib.gd_rnorm_fwd(  # noqa: E731
        x, ONE, w, s, y, dt, wt, 0, rows, D, 1e-6, NUL)
    assert f(dt=7) == _lib.GD_ERR_ARG and f(wt=F16) == _lib.GD_ERR_ARG
    for D in (0, -1, 16385, 16377):
        assert f(D=D) == _lib.GD_ERR_SHAPE
    assert f(dt=F32, wt=F32, D=8196) == _lib.GD_ERR_SHAPE and f(rows=-1) == _lib.GD_ERR_SHAPE
    assert f(x=NUL) == _lib.GD_ERR_ARG and f(s=NUL) == _lib.GD_ERR_ARG and f(w=NUL) == _lib.GD_ERR_ARG
    assert f(x=ODD) == _lib.GD_ERR_ALIGN and f(y=ODD) == _lib.GD_ERR_ALIGN
    assert f(rows=0, x=NUL, y=NUL, s=NUL, w=NUL) == _lib.GD_OK
    q = lambda group=128, q=ONE, D=128: lib.gd_rnorm_fp8(  # noqa: E731
        ONE, NUL, ONE, NUL, q, ONE, BF, BF, 0, 10, D, group, 1e-6, NUL)
    assert q(group=12) == _lib.GD_ERR_SHAPE and q(group=-8) == _lib.GD_ERR_SHAPE and q(q=NUL) == _lib.GD_ERR_ARG
    assert q(q=ODD) == _lib.GD_ERR_ALIGN and q(D=20000) == _lib.GD_ERR_SHAPE
    assert lib.gd_rnorm_workspace_bytes(100, 128) == 100 * 128 * 4 and lib.gd_rnorm_workspace_bytes(0, 128) == 0
    b = lambda dw=ONE, ws=ONE, n=1 << 30: lib.gd_rnorm_bwd(  # noqa: E731
        NUL, ONE, ONE, ONE, ONE, dw, BF, BF, 0, 10, 128, 1e-6, ws, n, NUL)
    assert b() == _lib.GD_ERR_ARG
    assert lib.gd_rnorm_bwd(ONE, ONE, ONE, ONE, ONE, ONE, BF, BF, 0, 10, 128, 1e-6, ONE, 10 * 128 * 4 - 4,
                            NUL) == _lib.GD_ERR_WORKSPACE


def test_rotary_refusals():
    lib = _lib.load()

    def f(q=ONE, table=ONE, dt=BF, B=2, T=3, H=4, HK=2, D=64, R=32, P=10, k=ONE):
        return lib.gd_rotary(q, k, ONE, ONE, table, NUL, 0, 0, P, dt, B, T, H, HK, D, R, 768, 256, 64, 384, 128, 64, 0,
                             0, NUL)
    assert f(dt=5) == _lib.GD_ERR_ARG
    for kw in ({"R": 31}, {"R": 0}, {"R": 66}, {"D": 0}, {"B": -1}, {"P": 0}, {"H": 1 << 28}):
        assert f(**kw) == _lib.GD_ERR_SHAPE, kw
    assert f(q=NUL) == _lib.GD_ERR_ARG and f(k=NUL) == _lib.GD_ERR_ARG and f(table=NUL) == _lib.GD_ERR_ARG
    assert f(q=ctypes.c_void_p(257)) == _lib.GD_ERR_ALIGN and f(table=ctypes.c_void_p(260)) == _lib.GD_ERR_ALIGN
    assert f(T=0, q=NUL, table=NUL) == _lib.GD_OK
