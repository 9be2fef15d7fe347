"""The layer-side sequence operators on the GPU against oracle/layer.py; tolerances: tests/layer_cases.py.

Roundings counted (each 2^-24 of the magnitudes added up; exponentials and reciprocals as four): the convolution K products and its
activation (24), its gradients through the slope of silu at a pre-activation of magnitude up to 16 (120), sums over n
tokens n more.  The scan: 16 per token for delta, its exponential and the update, which a state carries along (16 T), N products and sums,
for gradients the same from the other end.  The block end: D for the statistics, 60 for the rest."""
import pytest
import torch

from layer_cases import TYPES, close, conv_inputs, gen, scan_inputs, to, wide
from oracle import layer as ol
from ttt_tk_b200 import glue, ssm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _n(lengths, B):
    return None if lengths is None else list(lengths)


# ---- short convolution ---------------------------------------------------------------------------------------------------
CONV = [
    # type, B, T, D, K, activation, state, lengths, heads, strided
    ("bf16", 1, 1, 8, 4, "silu", True, None, False, False),
    ("bf16", 2, 2, 13, 4, None, True, None, False, False),          # shorter than the window, odd width
    ("fp32", 1, 1, 1, 2, "silu", False, None, False, False),
    ("fp16", 3, 37, 72, 3, "silu", True, (37, 0, 2), False, True),
    ("bf16", 2, 64, 128, 4, None, False, None, True, False),
    ("fp32", 1, 192, 64, 2, "silu", True, (100,), True, True),
    ("bf16", 2, 300, 264, 4, "silu", True, (300, 129), False, True),
    ("fp16", 1, 130, 1003, 2, "silu", False, None, False, False),
    ("fp32", 4, 33, 40, 3, None, True, (-5, 33, 99, 1), False, False),     # lengths are clamped
]


@pytest.mark.parametrize("ty,B,T,D,K,act,state,lengths,heads,strided", CONV)
def test_short_conv(ty, B, T, D, K, act, state, lengths, heads, strided):
    i = conv_inputs(T + D, ty, B, T, D, K, DEV, state, lengths, strided)
    n = None if lengths is None else [min(max(v, 0), T) for v in lengths]
    kw = dict(activation=act, state=i["state"], lengths=i["lengths"], heads=heads)
    y, end = ssm.short_conv(i["x"], i["weight"], i["bias"], return_state=True, **kw)
    heads_of = lambda v: v.reshape(B, T, D // 64, 64).transpose(1, 2).reshape(B, D // 64, T // 64, 64, 64)  # noqa: E731
    turn = heads_of if heads else lambda v: v
    args = (i["x"], i["weight"], i["bias"], act, i["state"], n)
    ref, rend = ol.short_conv(*args)
    amp, _ = ol.short_conv(*args, amp=True)
    close(y, turn(ref), turn(amp), 24, "y")
    assert torch.equal(end.double().cpu(), rend)
    assert torch.equal(y, ssm.short_conv(i["x"], i["weight"], i["bias"], **kw))
    gy = heads_of(i["gy"]).contiguous() if heads else i["gy"]
    got = ssm.short_conv_backward(gy, i["x"], i["weight"], i["bias"], grad_final_state=i["gf"], **kw)
    bargs = (i["gy"], *args, i["gf"])
    want, amps = ol.short_conv_backward(*bargs), ol.short_conv_backward(*bargs, amp=True)
    for k, g, r, a, ops in zip(("x", "weight", "bias", "state"), got, want, amps, (120, 120 + B * T, 120 + B * T, 120)):
        if k == "state" and not state:
            assert g is None
            continue
        close(g, r, a, ops, "grad " + k)
    again = ssm.short_conv_backward(gy, i["x"], i["weight"], i["bias"], grad_final_state=i["gf"], **kw)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


def test_short_conv_without_bias_and_gradient_of_the_state():
    i = conv_inputs(3, "bf16", 2, 20, 24, 4, DEV)
    y = ssm.short_conv(i["x"], i["weight"], state=i["state"])
    close(y, ol.short_conv(i["x"], i["weight"], None, None, i["state"])[0], ol.short_conv(i["x"], i["weight"], None, None, i["state"], amp=True)[0], 24)
    got = ssm.short_conv_backward(i["gy"], i["x"], i["weight"], state=i["state"])
    assert got[2] is None
    want = ol.short_conv_backward(i["gy"], i["x"], i["weight"], None, None, i["state"])
    amp = ol.short_conv_backward(i["gy"], i["x"], i["weight"], None, None, i["state"], amp=True)
    close(got[0], want[0], amp[0], 120)
    close(got[3], want[3], amp[3], 120)


@pytest.mark.parametrize("ty,B,D,K,strided", [("bf16", 3, 64, 4, False), ("fp32", 1, 13, 2, True), ("fp16", 5, 1032, 3, True)])
def test_short_conv_step_is_the_prompt_token_by_token(ty, B, D, K, strided):
    T = 6
    i = conv_inputs(D, ty, B, T, D, K, DEV)
    y, end = ssm.short_conv(i["x"], i["weight"], i["bias"], activation="silu", state=i["state"], return_state=True)
    st = i["state"].clone()
    for t in range(T):
        x = to(wide(i["x"][:, t].cpu(), strided), DEV)
        assert torch.equal(ssm.short_conv_step(x, st, i["weight"], i["bias"], activation="silu"), y[:, t])
    assert torch.equal(st, end)


# ---- scan ----------------------------------------------------------------------------------------------------------------
SCAN = [
    # type, B, T, D, N, G, state, lengths, strided
    ("bf16", 1, 1, 8, 16, 1, True, None, False),
    ("fp32", 1, 1, 1, 1, 1, False, None, False),
    ("bf16", 2, 16, 40, 16, 1, True, None, False),
    ("fp16", 2, 17, 33, 3, 1, False, None, True),
    ("fp32", 3, 35, 66, 5, 2, True, (35, 0, 16), False),
    ("bf16", 2, 50, 96, 32, 3, True, None, True),
    ("fp16", 1, 47, 128, 64, 2, True, None, False),
    ("fp32", 2, 40, 24, 64, 1, False, (40, 33), True),
    ("bf16", 1, 700, 64, 16, 1, True, None, True),              # few channels: chunks
    ("fp32", 2, 333, 20, 8, 1, True, (333, 77), False),         # chunks that lie wholly behind a sequence
    ("bf16", 1, 400, 130, 17, 1, True, (-3,), False),           # no token at all
    ("bf16", 1, 129, 80, 20, 5, False, (999,), False),          # lengths are clamped
]


def _scan_args(i):
    return [i[k] for k in ("x", "dt", "A", "B", "C")]


@pytest.mark.parametrize("ty,B,T,D,N,G,state,lengths,strided", SCAN)
def test_ssm_scan(ty, B, T, D, N, G, state, lengths, strided):
    i = scan_inputs(T + D + N, ty, B, T, D, N, G, DEV, state, lengths, strided)
    n = None if lengths is None else [min(max(v, 0), T) for v in lengths]
    a, extra = _scan_args(i), (i["D"], i["dt_bias"])
    y, end, ck = ssm.ssm_scan(*a, *extra, state=i["state"], lengths=i["lengths"], return_state=True, return_checkpoints=True)
    kw = dict(state=i["state"], lengths=n)
    ref, rend, _ = ol.ssm_scan(*a, *extra, **kw)
    amp, aend, _ = ol.ssm_scan(*a, *extra, amp=True, **kw)
    ops = 16 * T + N + 40
    close(y, ref, amp, ops, "y")
    close(end, rend, aend, ops, "state")
    assert torch.equal(y, ssm.ssm_scan(*a, *extra, state=i["state"], lengths=i["lengths"]))
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, *extra, lengths=i["lengths"], grad_final_state=i["gf"])
    want = ol.ssm_scan_backward(i["gy"], *a, *extra, grad_final_state=i["gf"], **kw)
    amps = ol.ssm_scan_backward(i["gy"], *a, *extra, grad_final_state=i["gf"], amp=True, **kw)
    ops, tok, chn = 32 * T + 2 * N + 80, B * T, D // G
    for k, g, r, m, o in zip(("x", "dt", "A", "B", "C", "D", "dt_bias", "state"), got, want, amps,
                             (ops, ops, ops + tok, ops + chn, ops + chn, tok + 8, ops + tok, ops)):
        close(g, r, m, o, "grad " + k)
    again = ssm.ssm_scan_backward(i["gy"], *a, ck, *extra, lengths=i["lengths"], grad_final_state=i["gf"])
    assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_ssm_scan_without_its_optional_parts():
    i = scan_inputs(5, "fp32", 2, 30, 24, 16, 1, DEV, state=False)
    i["dt"] = i["dt"].abs() * 0.1
    a = _scan_args(i)
    y, ck = ssm.ssm_scan(*a, softplus=False, return_checkpoints=True)
    kw = dict(softplus_=False)
    close(y, ol.ssm_scan(*a, **kw)[0], ol.ssm_scan(*a, amp=True, **kw)[0], 16 * 30 + 56)
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, softplus=False)
    assert got[5] is None and got[6] is None
    want, amps = ol.ssm_scan_backward(i["gy"], *a, **kw), ol.ssm_scan_backward(i["gy"], *a, amp=True, **kw)
    for j in (0, 1, 2, 3, 4, 7):
        close(got[j], want[j], amps[j], 32 * 30 + 112 + 60, str(j))


def test_ssm_scan_of_large_and_small_steps():
    """softplus over its whole range, decays from 1 - 2e-7 to 0, a state that is kept for long."""
    B, T, D, N = 1, 64, 32, 16
    i = scan_inputs(8, "fp32", B, T, D, N, 1, DEV)
    i["dt"] = torch.linspace(-25, 60, T, device=DEV)[None, :, None].expand(B, T, D).contiguous()
    i["dt_bias"] = torch.zeros(D, device=DEV)
    a = _scan_args(i)
    y, end, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], return_state=True, return_checkpoints=True)
    kw = dict(state=i["state"])
    ref, rend, _ = ol.ssm_scan(*a, i["D"], i["dt_bias"], **kw)
    amp, aend, _ = ol.ssm_scan(*a, i["D"], i["dt_bias"], amp=True, **kw)
    close(y, ref, amp, 16 * T + 60)
    close(end, rend, aend, 16 * T + 60)
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], grad_final_state=i["gf"])
    want = ol.ssm_scan_backward(i["gy"], *a, i["D"], i["dt_bias"], grad_final_state=i["gf"], **kw)
    amps = ol.ssm_scan_backward(i["gy"], *a, i["D"], i["dt_bias"], grad_final_state=i["gf"], amp=True, **kw)
    for j in range(8):
        close(got[j], want[j], amps[j], 32 * T + 112 + T + D, str(j))


@pytest.mark.parametrize("ty,B,T,D,N,G,cuts", [("bf16", 1, 600, 64, 16, 1, (1, 16, 17, 300)), ("fp32", 2, 90, 24, 6, 2, (45,))])
def test_ssm_scan_in_chunks(ty, B, T, D, N, G, cuts):
    i = scan_inputs(T, ty, B, T, D, N, G, DEV)
    a, extra = _scan_args(i), (i["D"], i["dt_bias"])
    ref, rend, _ = ol.ssm_scan(*a, *extra, state=i["state"])
    amp, aend, _ = ol.ssm_scan(*a, *extra, state=i["state"], amp=True)
    st, ys, edges = i["state"], [], (0, *cuts, T)
    for p, q in zip(edges, edges[1:]):
        y, st = ssm.ssm_scan(*[t[:, p:q] if t.dim() > 2 else t for t in a], *extra, state=st, return_state=True)
        ys.append(y)
    close(torch.cat(ys, 1), ref, amp, 16 * T + N + 40)
    close(st, rend, aend, 16 * T + N + 40)


@pytest.mark.parametrize("ty,B,D,N,G", [("bf16", 3, 64, 16, 1), ("fp32", 1, 13, 5, 1), ("fp16", 5, 96, 64, 3), ("fp32", 2, 70, 1, 7)])
def test_ssm_scan_step_follows_the_prompt(ty, B, D, N, G):
    T = 5
    i = scan_inputs(D, ty, B, T, D, N, G, DEV)
    a, extra = _scan_args(i), (i["D"], i["dt_bias"])
    ref, rend, _ = ol.ssm_scan(*a, *extra, state=i["state"])
    amp, aend, _ = ol.ssm_scan(*a, *extra, state=i["state"], amp=True)
    st, ys = i["state"].clone(), []
    for t in range(T):
        ys.append(ssm.ssm_scan_step(*[v[:, t] if v.dim() > 2 else v for v in a], st, *extra))
    close(torch.stack(ys, 1), ref, amp, 16 * T + N + 40)
    close(st, rend, aend, 16 * T + N + 40)


def test_steps_with_slots():
    """A table of states, padded rows, and rows that share a slot, which are one after another."""
    B, S, D, N, K = 6, 9, 72, 16, 4
    slots = [4, -1, 0, 4, 12, 4]
    i = scan_inputs(2, "fp32", B, 1, D, N, 1, DEV, state=False)
    c = conv_inputs(3, "fp32", B, 1, D, K, DEV, state=False)
    g = gen(1)
    table, ctable = torch.randn(S, D, N, generator=g).to(DEV), torch.randn(S, K - 1, D, generator=g).to(DEV)
    want, cwant = table.clone(), ctable.clone()
    idx = torch.tensor(slots, dtype=torch.int32, device=DEV)
    a = [v[:, 0] if v.dim() > 2 else v for v in _scan_args(i)]
    y = ssm.ssm_scan_step(*a, table, i["D"], i["dt_bias"], slots=idx)
    cy = ssm.short_conv_step(c["x"][:, 0], ctable, c["weight"], c["bias"], activation="silu", slots=idx)
    for b, s in enumerate(slots):
        if not 0 <= s < S:
            assert (y[b] == 0).all() and (cy[b] == 0).all()
            continue
        one = [v[b:b + 1] if v is not i["A"] else v for v in a]
        st, cst = want[s:s + 1].clone(), cwant[s:s + 1].clone()
        assert torch.equal(ssm.ssm_scan_step(*one, st, i["D"], i["dt_bias"])[0], y[b])
        assert torch.equal(ssm.short_conv_step(c["x"][b:b + 1, 0], cst, c["weight"], c["bias"], activation="silu")[0], cy[b])
        want[s], cwant[s] = st[0], cst[0]
    assert torch.equal(table, want) and torch.equal(ctable, cwant)


# ---- block end -----------------------------------------------------------------------------------------------------------
BLOCK = [
    # type, M, D, norm, activation, residual fp32, residual, gate, post, scale, pre, strided
    ("bf16", 1, 2048, "rms", "silu", False, True, True, True, True, True, False),
    ("fp32", 3, 1, "layer", "gelu", False, True, True, True, True, True, False),
    ("bf16", 5, 13, "rms", "sigmoid", True, True, True, True, True, True, False),
    ("fp16", 37, 1003, "layer", "silu", True, True, True, True, True, True, True),
    ("bf16", 700, 256, "layer", "gelu", False, True, True, True, True, True, True),
    ("fp32", 9, 4096, "rms", "silu", False, True, True, True, True, True, False),
    ("bf16", 7, 4104, "layer", "gelu", True, True, True, True, True, True, False),       # sums over tokens in shared memory
    ("fp32", 6, 8192, "layer", "silu", False, True, True, True, True, True, False),
    ("fp16", 4, 8191, "rms", "silu", False, True, True, True, True, True, False),
    ("bf16", 40, 64, "rms", "silu", False, True, False, False, False, False, False),
    ("bf16", 40, 65, "layer", "silu", False, False, False, False, False, True, False),     # a first block's norm
    ("fp16", 12, 640, "layer", "gelu", False, True, True, False, True, True, False),
    ("fp32", 12, 640, "rms", "sigmoid", False, False, True, True, False, False, False),
    ("bf16", 12, 88, "rms", "silu", True, True, False, True, True, False, False),
    ("bf16", 9, 1036, "layer", "gelu", True, True, True, True, True, True, False),       # runs of four, the last vector has one
    ("fp32", 5, 516, "rms", "sigmoid", False, True, True, True, True, True, False),
    ("fp16", 3, 4100, "layer", "silu", True, True, True, True, True, True, False),
    ("fp16", 6, 300, "rms", "gelu", False, True, True, True, True, True, False),       # a 16-bit stream: one by one
    ("bf16", 7, 512, "layer", "gelu", True, True, True, True, True, True, False),       # rows that fill their threads
    ("fp16", 5, 1024, "rms", "silu", False, True, True, True, True, True, True),
    ("bf16", 5, 384, "layer", "sigmoid", False, True, True, True, True, True, False),
    ("bf16", 150, 512, "rms", "silu", True, True, False, False, False, True, False),       # a residual and the next norm alone
    ("fp16", 40, 203, "layer", "silu", False, True, False, False, False, True, True),
    ("fp32", 3, 4100, "layer", "silu", False, True, False, False, False, True, False),
    ("bf16", 9, 1000, "rms", "silu", False, True, False, False, False, True, False),
]


@pytest.mark.parametrize("ty,M,D,norm,act,res32,res,gate,post,scale,pre,strided", BLOCK)
def test_norm_gate_residual(ty, M, D, norm, act, res32, res, gate, post, scale, pre, strided):
    g = gen(M + D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t, layer = TYPES[ty], norm == "layer"
    rt = torch.float32 if res32 else t
    mk = lambda v: to(wide(v, strided), DEV)  # noqa: E731
    o = mk((r(M, D) * 1.5 + 0.3).to(t))
    x0 = mk((r(M, D) * 2).to(rt)) if res else None
    z = mk((r(M, D) * 2).to(t)) if gate else None
    w = dict(post_weight=1 + 0.1 * r(D) if post else None, post_bias=0.1 * r(D) if post and layer else None,
             scale=0.3 + 0.1 * r(D) if scale else None, pre_weight=1 + 0.1 * r(D) if pre else None,
             pre_bias=0.1 * r(D) if pre and layer else None)
    w = {k: to(v, DEV) for k, v in w.items()}
    kw = dict(norm=norm, activation=act, eps=1e-5, **w)
    okw = {("activation_" if k == "activation" else k): v for k, v in kw.items()}
    x, n, stats = glue.norm_gate_residual(o, x0, z, return_stats=True, **kw)
    ref, rn = ol.norm_gate_residual(o, x0, z, **okw)
    od = o.double().cpu()
    gv = ol.activation(act, z.double().cpu())[0].abs() if gate else 1.0
    sc = w["scale"].double().cpu().abs() if scale else 1.0
    u = od.abs()
    if post:
        b = w["post_bias"].double().cpu().abs() if w["post_bias"] is not None else 0.0
        u = (od.abs() + od.mean(-1, keepdim=True).abs()) * ol._norm(od, layer, 1e-5)[1] * w["post_weight"].double().cpu().abs() + b
    amp = sc * u * gv + (x0.double().cpu().abs() if res else 0.0)
    close(x, ref, amp, D + 60, "x")
    if pre:
        r2 = ol._norm(ref, layer, 1e-5)[1]
        # an error of x enters the statistics too: once more the magnitude, as a mean
        an = (amp + amp.mean(-1, keepdim=True) * (1 + ol._norm(ref, layer, 1e-5)[0].abs())) * r2 * w["pre_weight"].double().cpu().abs()
        close(n, rn, an + (w["pre_bias"].double().cpu().abs() if layer else 0.0), 2 * D + 120, "n")
    else:
        assert n is None
    plain = glue.norm_gate_residual(o, x0, z, **kw)
    assert torch.equal(plain[0], x) and (n is None or torch.equal(plain[1], n))
    gx, gn = mk(r(M, D).to(rt if res else t)), mk(r(M, D).to(t)) if pre else None
    for up in ((gx, gn), (gx, None), (None, gn)):
        if up == (None, None):
            continue
        got = glue.norm_gate_residual_backward(*up, o, stats, x0, z, **kw)
        want = ol.norm_gate_residual_backward(*up, o, x0, z, **okw)
        amps = ol.norm_gate_residual_backward(*up, o, x0, z, amp=True, **okw)
        for k, a, b, m in zip(("o", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias"), got, want, amps):
            assert (a is None) == (b is None), k
            if a is not None:
                # the normalised values that enter every term have the errors of x's magnitude over its deviation: 4 covers these inputs
                close(a, b, m, 4 * (2 * D + 120) + (M if a.dim() == 1 else 0), "grad " + k)
        again = glue.norm_gate_residual_backward(*up, o, stats, x0, z, **kw)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


def test_norm_gate_residual_takes_any_leading_dimensions():
    o = torch.randn(2, 3, 5, 48, device=DEV).bfloat16()
    x, n = glue.norm_gate_residual(o, pre_weight=torch.ones(48, device=DEV))
    assert x.shape == n.shape == o.shape and torch.equal(x, o)
    x1, n1 = glue.norm_gate_residual(o[0, 0, 0], pre_weight=torch.ones(48, device=DEV))
    assert torch.equal(n1, n[0, 0, 0])
