"""Sizes at the limits of the grouped and 4-bit products: refused by the host before it computes or launches anything with them."""
import ctypes

import pytest

from mlx_b200 import _lib

ROWS, WIDTH = 2 ** 30 - 256, 2 ** 31 - 256   # the largest that are taken
P = ctypes.c_void_p(4096)


def mm(T=4, N=8, K=16, transpose=1):
    return _lib.load().b200q_grouped_mm(P, P, P, 8, P, _lib.BF16, T, 2, N, K, transpose, P, 16, None)


def dw(T=4, N=8, K=16):
    return _lib.load().b200q_grouped_mm_dw(P, P, P, 8, P, _lib.BF16, T, 2, N, K, P, 16, None)


def qq(T=4, N=8, K=64, mode=_lib.NVFP4, sizes=P):
    return _lib.load().b200q_grouped_qqmm(P, P, P, sizes, 8, P, _lib.BF16, T, 2 if sizes else 1, N, K, mode, None, None, 0, P, 16, None)


@pytest.mark.parametrize("f", (mm, dw, qq, lambda **kw: qq(sizes=None, **kw), lambda **kw: mm(transpose=0, **kw)))
def test_the_largest_sizes_and_one_more(f):
    """What is taken goes on to the check of the workspace (16 bytes, too few)."""
    assert f() == f(T=ROWS) == f(K=WIDTH) == _lib.ERR_WORKSPACE
    assert f(T=ROWS + 1) == f(T=2 ** 30) == f(K=WIDTH + 32) == _lib.ERR_UNSUPPORTED
    assert f(N=ROWS) == _lib.ERR_WORKSPACE
    if f is dw:
        assert f(N=ROWS + 1) == f(N=WIDTH) == _lib.ERR_UNSUPPORTED
    else:
        assert f(N=WIDTH) == _lib.ERR_WORKSPACE and f(N=WIDTH + 1) == _lib.ERR_UNSUPPORTED
