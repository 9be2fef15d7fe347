"""Masks in what 8 bits keep: a gate of -inf, or of its type's lowest value, is closed in the backward as it was in the forward, and leaves its
neighbours, whose scale it shares, their digits."""
import pytest
import torch

from gated_cases import ARGS, GRADS, TYPES, close, gated_inputs
from oracle import gated as og
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, saved, ssm

pytestmark = pytest.mark.gpu
INF = float("inf")


def _mask(how, ty):
    return {"inf": -INF, "lowest": torch.finfo(TYPES[ty]).min, "far": -1e4}[how]


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [37, 40, 128])
@pytest.mark.parametrize("clamp,lo,hi", [((None,), -INF, INF), (("low",), -448.0, INF), (("both",), -448.0, 448.0)])
def test_pack_with_bounds(ty, D, clamp, lo, hi):
    fi = torch.finfo(TYPES[ty])
    x = torch.randn(50, D, generator=torch.Generator().manual_seed(1)).to(TYPES[ty])
    x[::5, 3], x[1::5, 4], x[2::5, 5], x[3::5, 6], x[4::5, 7] = -INF, fi.min, fi.max, INF, 500.0
    x[7, 9] = float("nan")
    for rows in (x.cuda(), torch.cat([x, x], -1).cuda()[:, :D]):
        ((q, s),) = saved.pack8(rows, group=32, clamp=clamp)
        want, scale = og.e4m3(x.double().clamp(lo, hi), 32)
        assert torch.equal(s.double().cpu(), scale)
        got = q.double().cpu() * scale.repeat_interleave(32, -1)[:, :D]
        assert torch.equal(got.nan_to_num(1e300), want.nan_to_num(1e300))


def test_bounds_of_their_own_for_each_tensor():
    x = torch.full((3, 64), -1e4, device="cuda")
    x[:, 32:] = 1e4
    a, b, c = saved.unpack8(*saved.pack8(x, x, x, clamp=(None, "low", "both")), dtype=torch.float32)
    assert (a[:, :32] == -a[:, 32:]).all() and (a[:, 0] < -9e3).all()
    assert (b[:, :32].abs() <= 448).all() and (b[:, 32:] > 9e3).all()
    assert (c[:, :32] == -448).all() and (c[:, 32:] == 448).all()


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("how", ["inf", "lowest", "far"])
@pytest.mark.parametrize("T,D", [(130, 64), (70, 75), (900, 66)])
def test_closed_gates_of_the_recurrence(ty, how, T, D):
    """Tokens 30 to 49 of every third channel hold their states, and the input gate of others is closed."""
    i = gated_inputs(7, ty, 2, T, D, "cuda")
    shut, none = torch.zeros(2, 2, T, D, dtype=torch.bool, device="cuda")
    shut[:, 30:50, ::3], none[:, 40:45, 1::4] = True, True
    i["gate"][shut], i["input_gate"][none] = _mask(how, ty), _mask(how, ty)
    lv = [i[k].clone().requires_grad_(True) for k in ("x", "gate", *ARGS, "state")]
    y = ag.gated_scan(*lv[:-1], state=lv[-1], saved="e4m3")
    got = dict(zip(("x", "gate", *ARGS, "state"), torch.autograd.grad(y, lv, i["gy"])))
    assert (got["x"][shut] == 0).all() and (got["gate"][shut] == 0).all()
    assert all((got[k][none].float().abs() < 1e-30).all() for k in ("x", "input_gate"))      # (fp32 has a sigmoid of 2^-126)
    held = {k: i[k].double().clamp(-448, 448) for k in ("gate", "input_gate")}
    _, _, before = og.gated_scan(i["x"], held["gate"], i["A"], held["input_gate"], i["gate_bias"], i["input_bias"], state=i["state"])
    kept = {k: og.e4m3(v, 128)[0] for k, v in dict(held, x=i["x"]).items()}
    # a neighbour has lost no more than a scale of 1 takes
    for k, off in (("gate", ~shut), ("input_gate", ~none)):
        v = held[k].cpu()
        assert ((kept[k] - v).abs() <= torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10))[off.cpu()].all()
    ref = og.gated_scan_backward(i["gy"], kept["x"], kept["gate"], before, i["A"], kept["input_gate"], i["gate_bias"], i["input_bias"])
    for k in GRADS:
        close(got[k], ref[k], f"grad {k}")


@pytest.mark.parametrize("how", ["inf", "lowest", "far"])
def test_closed_steps_of_the_state_space_scan(how):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, dt, gy = r(2, 50, 48).bfloat16(), r(2, 50, 48).bfloat16(), r(2, 50, 48).bfloat16()
    A, B, C = -torch.rand(48, 16, generator=g).cuda() - 0.1, r(2, 50, 2, 16).bfloat16(), r(2, 50, 2, 16).bfloat16()
    dt[:, 10:20, ::3], dt[:, 30, 5] = _mask(how, "bf16"), 600.0      # (above there is nothing to bound: delta is dt itself)
    lv = [t.clone().requires_grad_(True) for t in (x, dt, A, B, C)]
    got = torch.autograd.grad(ag.ssm_scan(*lv, saved="e4m3"), lv, gy)
    _, ck = ssm.ssm_scan(x, dt, A, B, C, return_checkpoints=True)
    dt8 = og.e4m3(dt.double().clamp(min=-448), 128)[0].bfloat16().cuda()
    off = dt > -448
    assert ((dt8.float() - dt.float()).abs() <= torch.clamp(dt.float().abs() * 2.0 ** -4, min=2.0 ** -9))[off].all()
    x8 = og.e4m3(x, 128)[0].bfloat16().cuda()
    for a, c in zip(got, ssm.ssm_scan_backward(gy, x8, dt8, A, B, C, ck)):
        assert a.isfinite().all() and torch.equal(a, c)
    assert (got[1][:, 10:20, ::3] == 0).all()


@pytest.mark.parametrize("how", ["lowest", "far"])
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
def test_closed_gates_of_the_block_end(how, activation):
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    o, gate, gx = r(9, 96).bfloat16(), r(9, 96).bfloat16(), r(9, 96).bfloat16()
    gate[2:5, ::2] = _mask(how, "bf16")
    gate[6, 3] = 1e4 if activation == "sigmoid" else 300.0
    lv = [o.clone().requires_grad_(True), gate.clone().requires_grad_(True)]
    x, _ = ag.norm_gate_residual(lv[0], None, lv[1], activation=activation, saved="e4m3")
    got = torch.autograd.grad(x, lv, gx)
    _, _, stats = glue.norm_gate_residual(o, None, gate, activation=activation, return_stats=True)
    gate8 = og.e4m3(gate.double().clamp(-448, 448 if activation == "sigmoid" else INF), 128)[0].bfloat16().cuda()
    off = gate.abs() < 448
    assert ((gate8.float() - gate.float()).abs() <= torch.clamp(gate.float().abs() * 2.0 ** -4, min=2.0 ** -10))[off].all()
    o8 = og.e4m3(o, 128)[0].bfloat16().cuda()
    want = glue.norm_gate_residual_backward(gx, None, o8, stats, None, gate8, activation=activation)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])
    assert (got[0][2:5, ::2] == 0).all() and (got[1][2:5, ::2] == 0).all()
