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


def _strides(T, H, HK, D):
    q, k = [T * H * D, H * D, D], [T * HK * D, HK * D, D]
    return (ctypes.c_longlong * 12)(*q, *k, *k, *q)


def test_window_attention_refusals():
    lib = _lib.load()

    def fwd(q=ONE, o=ONE, low=ONE, lse=ONE, cu=NUL, N=0, dt=BF, B=2, Tq=100, Tk=100, H=4, HK=2, D=64, st=None, w=0, s=0,
            scale=0.125, ws=NUL, n=0):
        return lib.gd_wattn_fwd(q, ONE, ONE, o, low, lse, cu, N, dt, B, Tq, Tk, H, HK, D, st or _strides(Tk, H, HK, D), w,
                                s, scale, ws, n, NUL)

    def bwd(q=ONE, low=ONE, do=ONE, dk=ONE, dt=BF, B=2, Tq=100, Tk=100, H=4, HK=2, D=64, st=None, w=0, s=0, ws=ONE,
            n=1 << 40):
        return lib.gd_wattn_bwd(q, ONE, ONE, ONE, low, ONE, do, ONE, dk, ONE, NUL, 0, dt, B, Tq, Tk, H, HK, D,
                                st or _strides(Tk, H, HK, D), w, s, 0.125, ws, n, NUL)
    for f in (fwd, bwd):
        assert f(dt=F32) == _lib.GD_ERR_ARG and f(q=NUL) == _lib.GD_ERR_ARG
        for kw in ({"D": 0}, {"D": 100}, {"D": 264}, {"H": 5}, {"H": 0}, {"HK": 0}, {"B": -1}, {"B": 65536}, {"Tq": -1},
                   {"Tk": -1}, {"w": -1}, {"s": -1}, {"Tq": 1 << 29}):
            assert f(**kw) == _lib.GD_ERR_SHAPE, kw
        assert f(q=ODD) == _lib.GD_ERR_ALIGN
        for i in range(9):
            st = _strides(100, 4, 2, 64)
            st[i] += 4
            assert f(st=st) == _lib.GD_ERR_ALIGN, i
            st[i] = -64
            assert f(st=st) == _lib.GD_ERR_ALIGN, i
    assert fwd(scale=float("nan")) == _lib.GD_ERR_SHAPE and fwd(scale=float("inf")) == _lib.GD_ERR_SHAPE
    for kw in ({"N": 0}, {"N": 2, "Tk": 90}, {"N": 2}):   # packed rows: a batch of one, as many queries as keys
        assert fwd(cu=ONE, **kw) == _lib.GD_ERR_SHAPE, kw
    assert fwd(o=NUL) == _lib.GD_ERR_ARG and fwd(lse=NUL) == _lib.GD_ERR_ARG
    assert fwd(o=ODD) == _lib.GD_ERR_ALIGN and fwd(low=ODD) == _lib.GD_ERR_ALIGN
    assert fwd(ws=ONE, n=8) == _lib.GD_ERR_WORKSPACE
    assert fwd(B=0, q=NUL, o=NUL) == _lib.GD_OK and fwd(Tq=0, q=NUL, o=NUL) == _lib.GD_OK
    assert bwd(low=NUL) == _lib.GD_ERR_ARG and bwd(do=NUL) == _lib.GD_ERR_ARG and bwd(dk=NUL) == _lib.GD_ERR_ARG
    assert bwd(do=ODD) == _lib.GD_ERR_ALIGN and bwd(dk=ODD) == _lib.GD_ERR_ALIGN
    st = _strides(100, 4, 2, 64)
    st[10] += 4
    assert bwd(st=st) == _lib.GD_ERR_ALIGN
    need = lib.gd_wattn_workspace_bytes(2, 100, 100, 4, 2, 64, 0, 0, 0, 1)
    assert need >= 2 * 4 * 100 * 4 and bwd(n=need - 1) == _lib.GD_ERR_WORKSPACE and bwd(ws=NUL) == _lib.GD_ERR_WORKSPACE
    assert bwd(B=0) == _lib.GD_OK and bwd(Tk=0, dk=NUL, B=0) == _lib.GD_OK
    size = lib.gd_wattn_workspace_bytes
    assert 0 < size(2, 100, 100, 4, 2, 64, 0, 0, 0, 0) <= need
    for bad in ((-1, 100, 100, 4, 2, 64), (2, -1, 100, 4, 2, 64), (2, 100, 100, 5, 2, 64), (2, 100, 100, 4, 0, 64),
                (2, 100, 100, 4, 2, 264)):
        assert size(*bad, 0, 0, 0, 1) == 0, bad


def test_window_attention_step_refusals():
    lib = _lib.load()

    def f(q=ONE, kc=ONE, lengths=ONE, o=ONE, dt=BF, B=3, S=100, H=4, HK=2, D=64, st=None, w=0, s=0, scale=0.125, ws=ONE,
          n=1 << 30):
        st = st or (ctypes.c_longlong * 6)(*([S * HK * D, HK * D, D] * 2))
        return lib.gd_wattn_step(q, ONE, ONE, kc, ONE, lengths, o, dt, B, S, H, HK, D, st, w, s, scale, ws, n, NUL)
    assert f(dt=F32) == _lib.GD_ERR_ARG and f(q=NUL) == _lib.GD_ERR_ARG and f(kc=NUL) == _lib.GD_ERR_ARG
    assert f(lengths=NUL) == _lib.GD_ERR_ARG and f(o=NUL) == _lib.GD_ERR_ARG
    for kw in ({"D": 0}, {"D": 20}, {"D": 264}, {"H": 5}, {"HK": 0}, {"B": -1}, {"B": 65536}, {"S": 0}, {"w": -1},
               {"s": -1}, {"scale": float("nan")}):
        assert f(**kw) == _lib.GD_ERR_SHAPE, kw
    assert f(q=ODD) == _lib.GD_ERR_ALIGN and f(kc=ODD) == _lib.GD_ERR_ALIGN
    assert f(lengths=ctypes.c_void_p(257)) == _lib.GD_ERR_ALIGN
    for i in range(6):
        st = (ctypes.c_longlong * 6)(*([100 * 128, 128, 64] * 2))
        st[i] += 4
        assert f(st=st) == _lib.GD_ERR_ALIGN, i
    assert f(B=0, q=NUL) == _lib.GD_OK
    size = lib.gd_wattn_step_workspace_bytes
    assert size(0, 100, 4, 2, 64, 0, 0) == 0 and size(3, 0, 4, 2, 64, 0, 0) == 0 and size(3, 100, 5, 2, 64, 0, 0) == 0
    need = size(1, 1 << 20, 4, 1, 128, 0, 0)               # one request, one key head: several clusters share its cache
    assert need > 0
    long = dict(B=1, S=1 << 20, H=4, HK=1, D=128)
    assert f(**long, n=need - 1) == _lib.GD_ERR_WORKSPACE and f(**long, ws=NUL) == _lib.GD_ERR_WORKSPACE
