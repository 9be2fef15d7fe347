"""Activations in 8 bits at the ends of their types: what is finite comes back finite, within half a step of 4 bits."""
import pytest
import torch

from gated_cases import ARGS, GRADS, TYPES, close, gated_inputs
from oracle import gated as og
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import saved, ssm

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _ends(ty, D):
    """Rows whose largest magnitude rounds up to a power of two that the type does not have, and rows just below."""
    fi = torch.finfo(TYPES[ty])
    top = 2.0 ** (16 if ty == "fp16" else 128)
    x = torch.randn(6, D, generator=torch.Generator().manual_seed(D), dtype=torch.float64)
    x[0, 0], x[0, -1] = fi.max, -fi.max
    x[1, ::2] = top * 248.5 / 256
    x[2, D // 2] = -top * 248.5 / 256
    x[3, 0] = top * 247.5 / 256
    x[4] *= top / 16
    x[5, -1] = fi.max / 2
    return x.to(TYPES[ty]).cuda()


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [2, 37, 64, 384, 1003])
@pytest.mark.parametrize("group", [32, 128])
def test_finite_values_come_back_finite(ty, D, group):
    x = _ends(ty, D)
    pack = saved.pack8(x, group=group)
    (y,) = saved.unpack8(*pack, dtype=TYPES[ty])
    assert y.isfinite().all()
    wide = pack[0][1].double().repeat_interleave(group, -1)[:, :D]
    x, y = x.double(), y.double()
    assert ((y - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, wide * 2.0 ** -10)).all()


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [5, 64])
def test_infinities_and_nan_beside_them(ty, D):
    """An infinity becomes 448 times the scale, or the largest value that there is; NaN stays."""
    x = _ends(ty, D)
    x[0, 1], x[1, 1], x[2, 1] = INF, -INF, NAN
    (y,) = saved.unpack8(*saved.pack8(x), dtype=TYPES[ty])
    most = torch.finfo(torch.float16).max if ty == "fp16" else 240.0 * 2.0 ** 120
    assert y[0, 1] == most and y[1, 1] == -most and y[2, 1].isnan() and int(y.isnan().sum()) == 1


def test_one_scale_to_a_row():
    q = torch.tensor([[256.0, -448.0, 240.0, NAN, 1.0]], device="cuda").to(torch.float8_e4m3fn)
    for ty, scale, most in ((torch.float16, 256.0, 65504.0), (torch.bfloat16, 2.0 ** 120, 240.0 * 2.0 ** 120), (torch.float32, 2.0 ** 120, 240.0 * 2.0 ** 120)):
        (y,) = saved.unpack8((q, torch.tensor([scale], device="cuda")), dtype=ty)
        want = [most, -most, 240.0 * scale, scale]
        assert y[0, [0, 1, 2, 4]].tolist() == want and y[0, 3].isnan()


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("T,D,group", [(70, 64, 32), (130, 200, 128), (65, 75, 64), (900, 66, 32)])
def test_gated_backward_from_the_largest_values(ty, T, D, group):
    """The backward's own loads take the values that unpacking gives."""
    i = gated_inputs(2, ty, 2, T, D, "cuda")
    most = torch.finfo(TYPES[ty]).max
    i["x"][0, 10, ::7], i["x"][1, T - 3, 1::5], i["x"][1, 33, D - 1] = most, -most, most
    i["gy"], i["gf"] = i["gy"] * 2.0 ** -100, i["gf"] * 2.0 ** -100
    a = [i[k] for k in ARGS]
    y, ck = ssm.gated_scan(i["x"], i["gate"], *a, state=i["state"], return_checkpoints=True)
    packs = saved.pack8(i["x"], i["gate"], i["input_gate"], group=group)
    got = ssm.gated_scan_backward(i["gy"], packs[0], packs[1], ck, i["A"], packs[2], i["gate_bias"], i["input_bias"], grad_final_state=i["gf"])
    _, _, before = og.gated_scan(i["x"], i["gate"], *a, state=i["state"])
    x8, gate8, input8 = saved.unpack8(*packs, dtype=torch.float32)
    assert x8.isfinite().all()
    ref = og.gated_scan_backward(i["gy"], x8, gate8, before, i["A"], input8, i["gate_bias"], i["input_bias"], grad_final_state=i["gf"])
    # d log a has the factor i x db / d log a = -i x a^2 / b, which is more than fp32 holds for such an x where b is small, whatever x came from: those values of
    # the gate's gradient, and the sums over them, are no numbers to compare
    f = og._Factors(gate8, i["A"], input8, i["gate_bias"], i["input_bias"], "sqrt")
    fits = (f.i * x8.double().cpu() * f.db).abs() < 2.0 ** 127
    assert (x8.abs() > 3e38).cpu()[fits].any()      # (and others as large are compared)
    for k, v in zip(GRADS, got):
        there = fits if k == "gate" else fits.all(1).all(0) if k in ("A", "gate_bias") else torch.ones(v.shape, dtype=torch.bool)
        assert v.cpu()[there].isfinite().all(), k
        close(v.cpu()[there], tuple(t[there] for t in ref[k]), f"grad {k}")


def test_a_large_value_in_a_differentiable_form():
    """65504, the largest fp16, in what the convolution keeps: gradients are those at what was kept, and finite as its forward is."""
    x = torch.randn(2, 40, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    x[0, 5, 7], x[1, 20, 30] = 65504.0, -63520.0
    w = torch.full((64, 4), 2.0 ** -8, device="cuda")
    gy = torch.randn(2, 40, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).half() * 2.0 ** -6
    lv = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    y = ag.short_conv(*lv, saved="e4m3")
    assert y.isfinite().all()
    got = torch.autograd.grad(y, lv, gy)
    x8 = saved.unpack8(*saved.pack8(x), dtype=torch.float16)[0]
    assert all(g.isfinite().all() for g in got)
    for a, b in zip(got, ssm.short_conv_backward(gy, x8, w)):
        assert torch.equal(a, b)
