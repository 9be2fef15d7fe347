"""The gated recurrence with states that are infinite: they stay so, token by token, however the sequence is cut up."""
import pytest
import torch

from gated_cases import ARGS, gated_inputs
from ttt_tk_b200 import ssm

pytestmark = pytest.mark.gpu
INF = float("inf")
# one tile, several of 8 and of 16 warps, chunks
SHAPES = [(1, 40, 64), (2, 300, 66), (2, 300, 3000), (1, 1500, 64), (3, 700, 75)]


def _inputs(ty, B, T, D, A):
    i = gated_inputs(5, ty, B, T, D, "cuda")
    i["A"] = torch.full((D,), A, device="cuda")      # e^A a token at the most: 2^-58 for the farthest, its power over a tile 0 in fp32
    return i


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("A", [-0.5, -8.0, -40.0])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_forward(ty, A, B, T, D):
    i = _inputs(ty, B, T, D, A)
    i["state"][0, 7], i["x"][B - 1, 11, 5], i["x"][0, T // 2, 33] = INF, -INF, INF
    y, end, ck = ssm.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"], return_state=True, return_checkpoints=True)
    want = torch.zeros(B, T, D, device="cuda")
    want[0, :, 7], want[B - 1, 11:, 5], want[0, T // 2:, 33] = INF, -INF, INF
    bad = want != 0
    assert torch.equal(y.float()[bad], want[bad]) and y[~bad].isfinite().all()
    last = bad[:, -1]
    assert torch.equal(end[last], want[:, -1][last]) and end[~last].isfinite().all()
    at = torch.arange(0, T, 64, device="cuda")[1:] - 1      # in front of every 64th token is behind the one before
    assert torch.equal(ck[:, 1:][bad[:, at]], want[:, at][bad[:, at]])


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("A", [-0.5, -8.0, -40.0])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_backward(ty, A, B, T, D):
    """An infinite gradient goes as far back: dx = G b i."""
    i = _inputs(ty, B, T, D, A)
    _, ck = ssm.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"], return_checkpoints=True)
    i["gf"][0, 7], i["gy"][B - 1, T - 2, 5], i["gy"][0, T // 2, 33] = INF, -INF, INF
    g = ssm.gated_scan_backward(i["gy"], i["x"], i["gate"], ck, *[i[k] for k in ARGS], grad_final_state=i["gf"])
    want = torch.zeros(B, T, D, device="cuda")
    want[0, :, 7], want[B - 1, :T - 1, 5], want[0, :T // 2 + 1, 33] = INF, -INF, INF
    bad = want != 0
    assert torch.equal(g[0].float()[bad], want[bad]) and g[0][~bad].isfinite().all()
    first = bad[:, 0]
    assert torch.equal(g[6][first], want[:, 0][first]) and g[6][~first].isfinite().all()
