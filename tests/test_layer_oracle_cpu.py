"""The statements that the layer-side sequence operators are held to (oracle/layer.py), against themselves: the backward formulas against
autograd of other forms of the definitions and against central differences, chunks and lengths against whole sequences."""
import pytest
import torch
import torch.nn.functional as F

from layer_cases import conv_inputs, gen, scan_inputs
from oracle import layer as ol

TIGHT = dict(rtol=1e-9, atol=1e-9)


def _leaves(i, names):
    return {k: i[k].double().requires_grad_(True) for k in names if i[k] is not None}


@pytest.mark.parametrize("K,act,state", [(2, None, True), (3, "silu", False), (4, "silu", True)])
def test_short_conv_formulas(K, act, state):
    B, T, D = 2, 7, 3
    i = conv_inputs(K, "fp32", B, T, D, K, state=state)
    y, end = ol.short_conv(i["x"], i["weight"], i["bias"], act, i["state"])
    lv = _leaves(i, ["x", "weight", "bias", "state"])
    row = torch.cat([lv.get("state", torch.zeros(B, K - 1, D, dtype=torch.float64)), lv["x"]], 1)
    pre = F.conv1d(row.transpose(1, 2), lv["weight"][:, None], lv["bias"], groups=D).transpose(1, 2)
    want, wend = F.silu(pre) if act else pre, row[:, T:]
    torch.testing.assert_close(y, want.detach(), **TIGHT)
    torch.testing.assert_close(end, wend.detach(), **TIGHT)
    ((want * i["gy"]).sum() + (wend * i["gf"]).sum()).backward()
    got = ol.short_conv_backward(i["gy"], i["x"], i["weight"], i["bias"], act, i["state"], None, i["gf"])
    for g, k in zip(got, ["x", "weight", "bias", "state"]):
        if k in lv:
            torch.testing.assert_close(g, lv[k].grad, **TIGHT)


@pytest.mark.parametrize("G,softplus", [(1, True), (2, True), (4, False)])
def test_ssm_scan_formulas(G, softplus):
    B, T, D, N = 2, 6, 4, 3
    i = scan_inputs(G, "fp32", B, T, D, N, G)
    if not softplus:
        i["dt"] = i["dt"].abs() * 0.1
        i["dt_bias"] = i["dt_bias"].abs() * 0.01
    lv = _leaves(i, ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"])
    v = lv["dt"] + lv["dt_bias"]
    delta = F.softplus(v) if softplus else v
    # y as the sum over all earlier tokens, without a recurrence
    S = torch.cumsum(delta, 1)[..., None] * lv["A"]                                   # [B, T, D, N]
    spread = lambda m: m.repeat_interleave(D // G, 2)  # noqa: E731
    u = (delta * lv["x"])[..., None] * spread(lv["B"])
    decay = torch.exp(S[:, :, None] - S[:, None]) * torch.tril(torch.ones(T, T, dtype=torch.float64))[None, :, :, None, None]
    h = (decay * u[:, None]).sum(2) + torch.exp(S) * lv["state"][:, None]
    want = (h * spread(lv["C"])).sum(-1) + lv["D"] * lv["x"]
    kw = dict(D=i["D"], dt_bias=i["dt_bias"], softplus_=softplus, state=i["state"])
    y, end, _ = ol.ssm_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], **kw)
    torch.testing.assert_close(y, want.detach(), rtol=1e-8, atol=1e-8)
    torch.testing.assert_close(end, h[:, -1].detach(), rtol=1e-8, atol=1e-8)
    ((want * i["gy"]).sum() + (h[:, -1] * i["gf"]).sum()).backward()
    got = ol.ssm_scan_backward(i["gy"], i["x"], i["dt"], i["A"], i["B"], i["C"], **kw, grad_final_state=i["gf"])
    for g, k in zip(got, ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"]):
        torch.testing.assert_close(g, lv[k].grad, rtol=1e-7, atol=1e-7, msg=lambda m, k=k: f"{k}: {m}")


@pytest.mark.parametrize("norm,act,post,gate,scale,pre,bias", [
    ("rms", "silu", True, True, True, True, False), ("layer", "gelu", True, True, True, True, True),
    ("layer", "sigmoid", False, True, False, True, True), ("rms", "silu", True, False, True, False, False),
    ("layer", "silu", False, False, False, False, False)])
def test_block_end_formulas(norm, act, post, gate, scale, pre, bias):
    M, D = 3, 10
    g = gen(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = dict(o=r(M, D), residual=r(M, D), gate=r(M, D) if gate else None, post_weight=1 + r(D) if post else None,
             post_bias=r(D) if post and bias else None, scale=r(D) if scale else None, pre_weight=1 + r(D) if pre else None,
             pre_bias=r(D) if pre and bias else None)
    gx, gn = r(M, D), r(M, D)
    lv = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}
    nrm = (lambda v, w, b: F.layer_norm(v, (D,), w, b, 1e-6)) if norm == "layer" else (lambda v, w, b: F.rms_norm(v, (D,), w, 1e-6))
    v = nrm(lv["o"], lv["post_weight"], lv.get("post_bias")) if post else lv["o"]
    if gate:
        v = v * {"silu": F.silu, "gelu": lambda z: F.gelu(z, approximate="tanh"), "sigmoid": torch.sigmoid}[act](lv["gate"])
    x = lv["residual"] + (lv["scale"] * v if scale else v)
    loss = (x * gx).sum()
    kw = dict(norm=norm, activation_=act, **{k: t[k] for k in ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")})
    gx_, gn_ = ol.norm_gate_residual(t["o"], t["residual"], t["gate"], **kw)
    torch.testing.assert_close(gx_, x.detach(), **TIGHT)
    if pre:
        n = nrm(x, lv["pre_weight"], lv.get("pre_bias"))
        torch.testing.assert_close(gn_, n.detach(), **TIGHT)
        loss = loss + (n * gn).sum()
    loss.backward()
    got = ol.norm_gate_residual_backward(gx, gn, t["o"], t["residual"], t["gate"], **kw)
    for a, k in zip(got, ["o", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias"]):
        assert (a is None) == (t[k] is None), k
        if a is not None:
            torch.testing.assert_close(a, lv[k].grad, **TIGHT)


def test_gradients_against_differences():
    """One directional derivative of every input of the three operators."""
    h = 1e-6
    i = conv_inputs(3, "fp32", 2, 5, 4, 3, lengths=[5, 3])
    f = lambda d: (lambda y, e: (torch.nan_to_num(i["gy"].double(), posinf=0.0) * y).sum() + (i["gf"].double() * e).sum())(  # noqa: E731
        *ol.short_conv(d["x"], d["weight"], d["bias"], "silu", d["state"], [5, 3]))
    got = ol.short_conv_backward(i["gy"], i["x"], i["weight"], i["bias"], "silu", i["state"], [5, 3], i["gf"])
    _differences(f, i, ["x", "weight", "bias", "state"], got, h)
    j = scan_inputs(4, "fp32", 2, 5, 4, 3, 2, lengths=[5, 2])
    kw = dict(lengths=[5, 2])
    f = lambda d: (lambda y, e, _: (torch.nan_to_num(j["gy"].double(), posinf=0.0) * y).sum() + (j["gf"].double() * e).sum())(  # noqa: E731
        *ol.ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["dt_bias"], state=d["state"], **kw))
    got = ol.ssm_scan_backward(j["gy"], j["x"], j["dt"], j["A"], j["B"], j["C"], j["D"], j["dt_bias"], state=j["state"],
                               grad_final_state=j["gf"], **kw)
    _differences(f, j, ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"], got, h)


def _differences(f, inputs, names, grads, h):
    for k, g in zip(names, grads):
        v = torch.randn(inputs[k].shape, generator=gen(9), dtype=torch.float64)
        base = inputs[k].double()
        num = (f({**inputs, k: base + h * v}) - f({**inputs, k: base - h * v})) / (2 * h)
        ana = (g * v).sum()
        assert abs(num - ana) <= 1e-6 * max(1.0, float((g.abs() * v.abs()).sum())), (k, float(num), float(ana))


def test_lengths_and_chunks():
    i = scan_inputs(7, "fp32", 2, 9, 3, 2, lengths=[9, 4])
    a = (i["A"],)
    y, end, _ = ol.ssm_scan(i["x"], i["dt"], *a, i["B"], i["C"], i["D"], i["dt_bias"], state=i["state"], lengths=[9, 4])
    assert (y[1, 4:] == 0).all() and torch.isfinite(end).all()
    y0, mid, _ = ol.ssm_scan(i["x"][:1, :5], i["dt"][:1, :5], *a, i["B"][:1, :5], i["C"][:1, :5], i["D"], i["dt_bias"], state=i["state"][:1])
    y1, e1, _ = ol.ssm_scan(i["x"][:1, 5:], i["dt"][:1, 5:], *a, i["B"][:1, 5:], i["C"][:1, 5:], i["D"], i["dt_bias"], state=mid)
    torch.testing.assert_close(torch.cat([y0, y1], 1), y[:1], **TIGHT)
    torch.testing.assert_close(e1, end[:1], **TIGHT)
