"""What `pack8` refuses of its bounds, the same without a GPU."""
import ctypes

import pytest
import torch

from ttt_tk_b200 import saved


@pytest.mark.parametrize("clamp", ["low", ("low",), ("low", "high"), ("low", None, None), (True, None), ([], None), {"low": 1, "both": 2}, 1, (0, 0)])
def test_bounds_that_are_none(clamp):
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="clamp must be"):
        saved.pack8(x, x, clamp=clamp)


def test_bounds_are_taken():
    x = torch.zeros(2, 64)
    for clamp in (None, (None, "low"), ["both", "low"]):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            saved.pack8(x, x, clamp=clamp)


def test_the_c_entry_refuses_a_clamp_that_is_none():
    """Before anything is launched or read."""
    from ttt_tk_b200 import _lib

    class Args(ctypes.Structure):
        _fields_ = [("src", ctypes.c_void_p * 4), ("values", ctypes.c_void_p * 4), ("scales", ctypes.c_void_p * 4), ("dst", ctypes.c_void_p * 4), ("stride", ctypes.c_int64 * 4),
                    ("M", ctypes.c_int64), ("D", ctypes.c_int32), ("dtype", ctypes.c_int32), ("group", ctypes.c_int32), ("count", ctypes.c_int32), ("clamp", ctypes.c_int32 * 4)]

    lib = _lib.lib()
    fn = lib.ttt_b200_pack8
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    for bad in (-1, 3):
        a = Args(M=2, D=64, dtype=0, group=32, count=2)
        a.clamp[1] = bad
        for p in (a.src, a.values, a.scales):
            p[0] = p[1] = 1 << 12
        assert fn(ctypes.byref(a), None) == 1
        assert b"unknown clamp" in lib.ttt_b200_last_error()
