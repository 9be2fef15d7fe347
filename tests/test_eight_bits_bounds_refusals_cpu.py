"""What `pack8` refuses of its bounds, the same without a GPU."""
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
