"""What the feed-forward block's entry points refuse beside the test-only flag."""
import ctypes

from macai_b200 import _lib

NUL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(256)


def test_flag():
    lib, flag = _lib.load(), _lib.GD_TEST_WAIT_EXPIRES
    ld = (ctypes.c_longlong * 5)(64, 64, 64, 128, 64)

    def fwd(dt, kept):
        return lib.gd_ff_fwd(ONE, ONE, ONE, ONE, kept, ONE, ONE, dt, 10, 64, 128, 64, ld, ONE, 1, NUL)
    assert fwd(_lib.GD_BFLOAT16 | flag, NUL) == _lib.GD_ERR_ARG      # nothing waits that could be told to give up
    assert fwd(_lib.GD_BFLOAT16 | flag, ONE) == _lib.GD_ERR_WORKSPACE
    assert fwd(_lib.GD_FLOAT32 | flag, ONE) == _lib.GD_ERR_ARG and fwd(_lib.GD_BFLOAT16 | flag | 64, ONE) == _lib.GD_ERR_ARG
    assert lib.gd_ff_bwd(*[ONE] * 11, _lib.GD_FLOAT32 | flag, 10, 64, 128, 64, ld, ONE, 1, NUL) == _lib.GD_ERR_ARG
    assert lib.gd_ff_bwd(*[ONE] * 11, _lib.GD_BFLOAT16 | flag, 10, 64, 128, 64, ld, ONE, 1, NUL) == _lib.GD_ERR_WORKSPACE
