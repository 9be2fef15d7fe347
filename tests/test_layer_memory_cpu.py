"""The memory that the scan's backward asks for is what the header says (no GPU: the scratch depends on sizes and the number of SMs)."""
import ctypes
import struct

import pytest

from ttt_tk_b200 import _lib


def scratch(backward, B, T, D, G, N, dtype=0):
    fn = _lib.lib().ttt_b200_ssm_scan_scratch_bytes
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_int], ctypes.c_uint64
    return fn(struct.pack("=23Q Q 2Q 12q 8i", *[0] * 26, *[0] * 12, B, T, D, G, N, 0, dtype, 1), backward)


# Enough sequences and channels that no sequence is split
@pytest.mark.parametrize("B,T,D,G,N", [(16, 8192, 4096, 1, 64), (64, 512, 2048, 1, 16), (300, 100, 64, 1, 16), (128, 77, 1536, 12, 64), (512, 33, 200, 1, 5)])
def test_scratch_of_the_scans_backward(B, T, D, G, N):
    channels = 128 if N <= 8 else 64 if N <= 16 else 32 if N <= 32 else 16
    tiles = -(-(D // G) // channels)
    up = lambda n: -(-n // 16) * 16  # noqa: E731
    parts = 2 * tiles * B * T * G * N if tiles > 1 else 0
    assert scratch(1, B, T, D, G, N) == 4 * (up(parts) + up(B * D * N) + up(2 * B * D))
    assert scratch(0, B, T, D, G, N) == 0
    if (D, G, N) == (4096, 1, 64):      # the header's example
        assert round(scratch(1, B, T, D, G, N) / 1e9) == 17 and round(B * (T // 16) * D * N * 4 / 1e9, 1) == 8.6
