"""The statement of the gated linear recurrence: its backward by hand against autograd and against differences, and e4m3 against torch's."""
import pytest
import torch

from gated_cases import ARGS, gated_inputs
from oracle import gated as og


def _forward(i, mix, leaves):
    """Token by token with autograd, from the definition."""
    x, gate, A, ig, gb, ib, st = leaves
    B, T, D = x.shape
    v = gate + (gb if gb is not None else 0.0)
    a = torch.exp(A.clamp(max=0.0) * torch.sigmoid(v)) if A is not None else torch.sigmoid(v)
    b = torch.sqrt(1 - a * a) if mix == "sqrt" else 1 - a if mix == "linear" else 1.0
    u = b * x * (torch.sigmoid(ig + (ib if ib is not None else 0.0)) if ig is not None else 1.0)
    h = st if st is not None else torch.zeros(B, D, dtype=torch.float64)
    n, ys = og.lengths_of(i["lengths"], B, T), []
    for t in range(T):
        on = (t < n)[:, None]
        h = torch.where(on, a[:, t] * h + u[:, t], h)
        ys.append(torch.where(on, h, 0.0))
    return torch.stack(ys, 1), h


@pytest.mark.parametrize("mix", ["sqrt", "linear", None])
@pytest.mark.parametrize("A,igate,bias,state,lengths", [(True, True, True, True, [70, 3]), (False, False, False, False, None), (True, False, True, True, [0, 70]),
                                                        (False, True, False, True, None)])
def test_backward_is_the_gradient(mix, A, igate, bias, state, lengths):
    i = gated_inputs(3, "fp32", 2, 70, 5, A=A, igate=igate, bias=bias, state=state, lengths=lengths)
    leaves = [None if i[k] is None else i[k].double().requires_grad_(True) for k in ("x", "gate", *ARGS, "state")]
    y, h = _forward(i, mix, leaves)
    (ya, _), (end, _), before = og.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], mix=mix, state=i["state"], lengths=i["lengths"])
    torch.testing.assert_close(ya, y.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(end, h.detach(), rtol=1e-12, atol=1e-12)
    loss = (y * i["gy"].double()).sum() + ((h * i["gf"].double()).sum() if state else 0.0)
    want = torch.autograd.grad(loss, [v for v in leaves if v is not None])
    got = og.gated_scan_backward(i["gy"], i["x"], i["gate"], before, *[i[k] for k in ARGS], mix=mix, lengths=i["lengths"], grad_final_state=i["gf"])
    names = [k for k, v in zip(("x", "gate", *ARGS, "state"), leaves) if v is not None]
    for k, w in zip(names, want):
        torch.testing.assert_close(got[k][0], w, rtol=1e-9, atol=1e-11, msg=k)


def test_backward_against_differences():
    i = gated_inputs(5, "fp32", 1, 9, 3)
    i = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in i.items()}

    def loss():
        (y, _), (end, _), _ = og.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"])
        return ((y * i["gy"]).sum() + (end * i["gf"]).sum()).item()

    _, _, before = og.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"])
    got = og.gated_scan_backward(i["gy"], i["x"], i["gate"], before, *[i[k] for k in ARGS], grad_final_state=i["gf"])
    for k in ("x", "gate", *ARGS, "state"):
        for j in range(min(4, i[k].numel())):
            flat, d = i[k].view(-1), 1e-6
            keep = flat[j].item()
            flat[j] = keep + d
            up = loss()
            flat[j] = keep - d
            down = loss()
            flat[j] = keep
            assert abs((up - down) / (2 * d) - got[k][0].reshape(-1)[j].item()) < 1e-7, k


@pytest.mark.parametrize("group", [32, 64, 128, 0])
def test_e4m3_is_torchs(group):
    """Of values in the format's range torch rounds the same way."""
    v = torch.randn(7, 131, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.arange(-3.0, 4.0))[:, None]
    q, scale = og.e4m3(v, group)
    g = group or 131
    wide = scale.repeat_interleave(g, -1)[:, :131]
    assert torch.equal((v.double() / wide).float().to(torch.float8_e4m3fn).double() * wide, q)
    top = torch.nn.functional.pad(v.abs(), (0, -131 % g)).unflatten(-1, (-1, g)).amax(-1).double()
    assert (top <= 448 * scale).all() and (top > 224 * scale).all()
