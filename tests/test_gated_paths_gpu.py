"""The gated recurrence in each of the ways that a call can take through its kernels, for more than one tile of each: sixteen warps, chunks, and the backward of four
fp32 tensors with one tile of rows in shared memory."""
import pytest
import torch

from gated_cases import gated_inputs, hold, run_both

pytestmark = pytest.mark.gpu


def _plan(B, T, D, backward, fp32):
    """(warps, tiles to a chunk, CTAs) that the launcher takes, restated."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n64, columns = -(-T // 64), -(-D // 64) * B

    def rounds(ctas, n):
        return 35 + 15 * n if ctas <= sms else 15 + (24 * n + 20) * -(-ctas // (2 * sms))

    best = (rounds(columns, n64), 8, n64)
    if columns <= sms and T > 64 and not (backward and fp32):
        best = min(best, (35 + 24 * -(-T // 128), 16, -(-T // 128)), key=lambda p: p[0])
    for n in range(2, min(32, n64) + 1):
        chunk = -(-n64 // n)
        chunks = -(-n64 // chunk)
        cost = rounds(columns * chunks, chunk) + rounds(columns * (chunks - 1), chunk) * 6 // 10 + 20
        best = min(best, (cost, 8, chunk), key=lambda p: p[0])
    _, warps, chunk = best
    return warps, chunk, columns * -(-(-(-T // (8 * warps))) // chunk)


# rows on 16-byte boundaries, on boundaries of two values, and on any (an odd D, or an odd distance)
@pytest.mark.parametrize("rows,D", [("whole", 1004), ("wide", 1003), ("odd", 1002), ("wide", 1002)])
@pytest.mark.parametrize("mix,A,igate", [("sqrt", True, True), ("linear", False, False)])
def test_backward_of_fp32_one_tile_deep(rows, D, mix, A, igate):
    """Two CTAs to an SM and several tiles to each."""
    B, T = 3, 700
    warps, chunk, ctas = _plan(B, T, D, True, True)
    assert warps == 8 and chunk >= 2 and ctas > torch.cuda.get_device_properties(0).multi_processor_count
    i = gated_inputs(1, "fp32", B, T, D, "cuda", rows=rows, A=A, igate=igate, lengths=[700, 517, 66])
    hold(i, mix, run_both(i, mix), rows)


@pytest.mark.parametrize("ty", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,D", [("whole", 3000), ("wide", 3002), ("odd", 2999)])
@pytest.mark.parametrize("T,lengths", [(300, None), (300, [300, 133])])
def test_sixteen_warps(ty, rows, D, T, lengths):
    for backward in (False, True):
        warps, chunk, _ = _plan(2, T, D, backward, False)
        assert warps == 16 and chunk >= 2
    i = gated_inputs(2, ty, 2, T, D, "cuda", rows=rows, lengths=lengths)
    hold(i, "sqrt", run_both(i, "sqrt"), f"{ty} {rows}")


@pytest.mark.parametrize("mix,A,igate", [("linear", False, False), (None, True, True)])
def test_sixteen_warps_with_other_parts(mix, A, igate):
    i = gated_inputs(3, "bf16", 2, 300, 3001, "cuda", rows="odd", A=A, igate=igate, lengths=[300, 200])
    hold(i, mix, run_both(i, mix), str(mix))


@pytest.mark.parametrize("ty,rows,D", [("bf16", "whole", 512), ("fp32", "odd", 515), ("fp16", "wide", 514)])
def test_chunks_of_several_tiles(ty, rows, D):
    B, T = 2, 2000
    for backward in (False, True):
        warps, chunk, _ = _plan(B, T, D, backward, ty == "fp32")
        assert warps == 8 and chunk >= 2
    i = gated_inputs(4, ty, B, T, D, "cuda", rows=rows, lengths=[2000, 900])
    hold(i, "sqrt", run_both(i, "sqrt"), f"{ty} {rows}")
