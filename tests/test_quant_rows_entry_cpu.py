"""Refusals of the native entry points behind norms, activations and rows that end in e4m3 (no launch is reached)."""
import ctypes

import pytest

from gcore_b200.ops import _lib


@pytest.fixture
def lib():
    try:
        return _lib.kernels()
    except RuntimeError as e:
        pytest.skip(str(e))


def test_rows(lib):
    buf = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buf) + 15) // 16 * 16

    def rows(src=at, q=at + 1024, F=256, T=1, act=0, sc32=1, as16=0):
        return lib.gk_rows_quant(src, q, at + 2048, T, F, act, sc32, as16, None)

    assert rows(T=0) == 0 and rows(T=0, act=1, sc32=0, as16=1) == 0
    assert rows(sc32=0) == -1 and rows(as16=1) == -1            # plain rows have one form
    assert rows(F=48) == -1 and rows(F=160, act=1, sc32=0) == -1 and rows(F=0) == -1 and rows(T=-1) == -1
    assert rows(src=at + 8) == -2 and rows(q=at + 8) == -2


def test_norm(lib):
    buf = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buf) + 15) // 16 * 16

    def norm(x=at, H=256, T=1, sc32=1):
        return lib.gk_norm_quant(x, None, at, at, at, None, T, H, 1e-6, sc32, 0, None)

    assert norm(T=0) == 0 and norm(H=16640) == -1 and norm(H=160, sc32=0) == -1 and norm(T=-1) == -1 and norm(x=at + 8) == -2
