"""The differentiable form of the gated linear recurrence: gradients against the operator's own backward call (bits), and a recurrent block of
convolution, recurrence and block end trained as one and served token by token."""
import pytest
import torch

from gated_cases import ARGS, GRADS, gated_inputs, run_both
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, ssm

pytestmark = pytest.mark.gpu
LEAVES = ("x", "gate", *ARGS, "state")


def test_autograd_is_the_backward_call():
    i = gated_inputs(1, "bf16", 2, 150, 66, "cuda", lengths=[150, 77])
    lv = {k: i[k].clone().requires_grad_(True) for k in LEAVES}
    y, end = ag.gated_scan(lv["x"], lv["gate"], *[lv[k] for k in ARGS], state=lv["state"], lengths=i["lengths"], return_state=True)
    torch.autograd.backward([y, end], [i["gy"], i["gf"]])
    want = run_both(i, "sqrt")
    assert torch.equal(y, want[0]) and torch.equal(end, want[1])
    for k in GRADS:
        assert torch.equal(lv[k].grad, want[2][k]), k


def test_only_some_gradients_arrive():
    i = gated_inputs(2, "fp32", 2, 70, 34, "cuda")
    x = i["x"].clone().requires_grad_(True)
    y, end = ag.gated_scan(x, i["gate"], mix="linear", return_state=True)
    (g,) = torch.autograd.grad(end.sum(), x, retain_graph=True)
    assert torch.isfinite(g).all() and (g[:, -1] > 0).all()
    (g,) = torch.autograd.grad(y.sum(), x)      # an expanded number as upstream gradient
    assert torch.isfinite(g).all() and (g > 0).all()
    assert not ag.gated_scan(i["x"], i["gate"]).requires_grad
    with torch.no_grad():
        assert not ag.gated_scan(x, i["gate"]).requires_grad


def _block(p, h, res):
    """projection -> short convolution -> recurrence -> gate, residual and the next norm."""
    D = p["A"].shape[0]
    q = h @ p["win"].to(h.dtype)
    u = ag.short_conv(q[..., :D], p["conv"], p["conv_b"])
    y = ag.gated_scan(u, q[..., D:2 * D], p["A"], q[..., 2 * D:3 * D], p["gate_b"], p["input_b"])
    return ag.norm_gate_residual(y, res, q[..., 3 * D:], activation="gelu", pre_weight=p["w"])


def _block_plain(p, h, res):
    D = p["A"].shape[0]
    q = h @ p["win"]
    x = torch.nn.functional.pad(q[..., :D], (0, 0, 3, 0))
    u = p["conv_b"] + sum(x[:, k:k + h.shape[1]] * p["conv"][:, k] for k in range(4))
    la = p["A"] * torch.sigmoid(q[..., D:2 * D] + p["gate_b"])
    v = torch.sqrt(1 - torch.exp(2 * la)) * torch.sigmoid(q[..., 2 * D:3 * D] + p["input_b"]) * u
    s, ys = torch.zeros_like(v[:, 0]), []
    for t in range(h.shape[1]):
        s = torch.exp(la[:, t]) * s + v[:, t]
        ys.append(s)
    z = res + torch.stack(ys, 1) * torch.nn.functional.gelu(q[..., 3 * D:], approximate="tanh")
    return z, torch.nn.functional.rms_norm(z, (D,), p["w"], 1e-6)


def _weights(D, device="cuda"):
    g = torch.Generator().manual_seed(5)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(device)  # noqa: E731
    return dict(win=r(D, 4 * D, std=D ** -0.5), conv=r(D, 4, std=0.5), conv_b=r(D, std=0.1), A=-torch.rand(D, generator=g).to(device) - 0.05, gate_b=r(D), input_b=r(D),
                w=1 + r(D, std=0.1)), r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_block_trains_as_in_64_bits(dtype):
    """Tolerance, relative in the 2-norm: a value passes the block's four operators and back, at most 8 roundings to its type with as many again
    for what mixes them, 2^-9 * 8 * 2 in bf16; in fp32 2^-24 * 8 * 64 for sums of 64 terms; twice that for a product with the recurrence's
    states, which sum up to 1 / (1 - a) of them."""
    D, B, T = 64, 2, 130
    p, r = _weights(D)
    h, res = r(B, T, D).to(dtype), r(B, T, D).to(dtype)
    lv = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    x, res1 = h.clone().requires_grad_(True), res.clone().requires_grad_(True)
    z, n = _block(lv, x, res1)
    gz, gn = r(B, T, D).to(dtype), r(B, T, D).to(dtype)
    torch.autograd.backward([z, n], [gz, gn])
    ref = {k: v.double().requires_grad_(True) for k, v in p.items()}
    if dtype is torch.bfloat16:      # the projection is made with rounded weights
        ref["win"] = p["win"].to(dtype).double().requires_grad_(True)
    x2, res2 = h.double().requires_grad_(True), res.double().requires_grad_(True)
    z2, n2 = _block_plain(ref, x2, res2)
    torch.autograd.backward([z2, n2], [gz.double(), gn.double()])
    tol = 2 * (2.0 ** -9 * 16 if dtype is torch.bfloat16 else 2.0 ** -24 * 512)
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    torch.backends.cuda.matmul.allow_tf32 = False
    for what, a, b in [("z", z, z2), ("n", n, n2), ("h", x.grad, x2.grad), ("res", res1.grad, res2.grad)] + [(k, lv[k].grad, ref[k].grad) for k in p]:
        assert rel(a, b) < tol, (what, rel(a, b), tol)


def test_a_block_serves_token_by_token():
    """A prompt, then tokens one at a time from the tables, is the whole sequence."""
    D, T, P = 96, 40, 29
    p, r = _weights(D)
    q = r(1, T, 4 * D)
    kw = dict(activation="gelu", pre_weight=p["w"])

    def after(y, q, res):
        return glue.norm_gate_residual(y, res, q[..., 3 * D:], **kw)[1]

    res = r(1, T, D)
    u = ssm.short_conv(q[..., :D], p["conv"], p["conv_b"])
    a = (p["A"], p["gate_b"], p["input_b"])
    whole = after(ssm.gated_scan(u, q[..., D:2 * D], a[0], q[..., 2 * D:3 * D], *a[1:]), q, res)
    windows, states = torch.randn(4, 3, D, device="cuda"), torch.randn(4, D, device="cuda")
    u, win = ssm.short_conv(q[:, :P, :D], p["conv"], p["conv_b"], return_state=True)
    y, st = ssm.gated_scan(u, q[:, :P, D:2 * D], a[0], q[:, :P, 2 * D:3 * D], *a[1:], return_state=True)
    windows[2], states[2] = win[0], st[0]
    slots = torch.tensor([2], dtype=torch.int32, device="cuda")
    for t in range(P, T):
        row = q[:, t]
        u = ssm.short_conv_step(row[:, :D], windows, p["conv"], p["conv_b"], slots=slots)
        y = ssm.gated_scan_step(u, row[:, D:2 * D], states, a[0], row[:, 2 * D:3 * D], *a[1:], slots=slots)
        torch.testing.assert_close(after(y, row, res[:, t]), whole[:, t], rtol=2e-5, atol=2e-5)


def test_a_training_step_in_a_graph():
    i = gated_inputs(3, "bf16", 2, 200, 64, "cuda")
    lv = {k: i[k].clone().requires_grad_(True) for k in LEAVES}

    def step():
        y, end = ag.gated_scan(lv["x"], lv["gate"], *[lv[k] for k in ARGS], state=lv["state"], return_state=True)
        return torch.autograd.grad([y, end], [lv[k] for k in LEAVES], [i["gy"], i["gf"]])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        lv["gate"].add_(0.25)
    g.replay()
    want = run_both(dict(i, gate=lv["gate"].detach()), "sqrt")[2]
    for k, v in zip(LEAVES, got):
        assert torch.equal(v, want[k]), k
