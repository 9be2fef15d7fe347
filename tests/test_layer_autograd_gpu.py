"""The differentiable forms of the layer-side sequence operators, and runs of them together as a layer uses them: gradients against
the operators' own backward calls (bits) and against autograd of plain torch in 64 bits; captured into graphs; on other streams.

Tolerance of the runs: a value that passes through bf16 at k places between the operators carries k roundings of 2^-9 relative to its
own magnitude, and as many again for each operator that mixes it; 2-norm over a tensor of them, at most 8 operators deep: 2^-9 * 8 * 2 = 3.2e-2 in relative
2-norm for bf16, 2^-24 * 8 * 64 (sums over up to 64 terms in a row of 32-bit operations each) = 3.1e-5 for fp32."""
import pytest
import torch
import torch.nn.functional as F

from layer_cases import conv_inputs, gen, scan_inputs
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, layout, ssm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)).item()


def leaves(i, names):
    return {k: i[k].clone().requires_grad_(True) for k in names if i[k] is not None}


def test_short_conv_autograd_is_the_backward_call():
    i = conv_inputs(1, "bf16", 2, 70, 64, 4, DEV, lengths=(70, 31))
    lv = leaves(i, ["weight", "bias", "state"])
    x = torch.nan_to_num(i["x"]).requires_grad_(True)
    gy, gf = torch.nan_to_num(i["gy"], posinf=0.0), i["gf"]
    y, end = ag.short_conv(x, lv["weight"], lv["bias"], activation="silu", state=lv["state"], lengths=i["lengths"], return_state=True)
    torch.autograd.backward([y, end], [gy, gf])
    want = ssm.short_conv_backward(gy, x.detach(), i["weight"], i["bias"], activation="silu", state=i["state"], lengths=i["lengths"],
                                   grad_final_state=gf)
    for a, b in zip((x.grad, lv["weight"].grad, lv["bias"].grad, lv["state"].grad), want):
        assert torch.equal(a, b)
    # the state alone; an expanded upstream gradient
    y, end = ag.short_conv(x, lv["weight"], lv["bias"], state=lv["state"], return_state=True)
    (g,) = torch.autograd.grad(end.float().sum(), x)
    assert (g[:, :67] == 0).all() and (g[:, 67:] == 1).all()
    y = ag.short_conv(x, lv["weight"], heads=False)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, ssm.short_conv_backward(torch.ones_like(y), x.detach(), i["weight"])[0])


def test_ssm_scan_autograd_is_the_backward_call():
    i = scan_inputs(2, "bf16", 2, 50, 48, 16, 2, DEV)
    names = ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"]
    lv = leaves(i, names)
    y, end = ag.ssm_scan(lv["x"], lv["dt"], lv["A"], lv["B"], lv["C"], lv["D"], lv["dt_bias"], state=lv["state"], return_state=True)
    torch.autograd.backward([y, end], [i["gy"], i["gf"]])
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    _, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], return_checkpoints=True)
    want = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], grad_final_state=i["gf"])
    for k, b in zip(names, want):
        assert torch.equal(lv[k].grad, b), k
    # only the state's gradient arrives; no D, no bias; nothing needs a gradient
    y, end = ag.ssm_scan(lv["x"], lv["dt"].detach().abs() * 0.1, lv["A"], i["B"], i["C"], softplus=False, return_state=True)
    (g,) = torch.autograd.grad(end.sum(), lv["x"])
    assert torch.isfinite(g).all() and g.abs().sum() > 0
    y = ag.ssm_scan(*a, i["D"], i["dt_bias"])
    assert not y.requires_grad and torch.equal(y, ssm.ssm_scan(*a, i["D"], i["dt_bias"]))


@pytest.mark.parametrize("res32", [False, True])
def test_norm_gate_residual_autograd_is_the_backward_call(res32):
    g = gen(3)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    o, z = r(2, 9, 96).bfloat16(), r(2, 9, 96).bfloat16()
    x = r(2, 9, 96).to(torch.float32 if res32 else torch.bfloat16)
    w = dict(post_weight=1 + 0.1 * r(96), post_bias=r(96), scale=r(96), pre_weight=1 + 0.1 * r(96), pre_bias=r(96))
    lv = {k: v.clone().requires_grad_(True) for k, v in dict(o=o, residual=x, gate=z, **w).items()}
    kw = dict(norm="layer", activation="gelu")
    y, n = ag.norm_gate_residual(lv["o"], lv["residual"], lv["gate"], **kw, **{k: lv[k] for k in w})
    gx, gn = torch.randn_like(y), torch.randn_like(n)
    torch.autograd.backward([y, n], [gx, gn])
    _, _, stats = glue.norm_gate_residual(o, x, z, return_stats=True, **kw, **w)
    want = glue.norm_gate_residual_backward(gx, gn, o, stats, x, z, **kw, **w)
    for k, b in zip(("o", "residual", "gate", *w), want):
        assert torch.equal(lv[k].grad, b.view_as(lv[k])), k
    y, n = ag.norm_gate_residual(lv["o"], pre_weight=lv["pre_weight"])
    (g1,) = torch.autograd.grad(n.float().sum(), lv["o"])
    assert torch.isfinite(g1.float()).all()


# ---- together ------------------------------------------------------------------------------------------------------------
def _ssm_layer(p, h, res, dtype):
    """norm -> projection -> short convolution -> step sizes, B, C -> scan -> post norm, gate, residual, next norm; `p` of weights."""
    D, N = p["A"].shape
    xz = h @ p["win"].to(dtype)
    u = ag.short_conv(xz[..., :D], p["conv"], p["conv_b"], activation="silu")
    q = u @ p["wq"].to(dtype)
    dt = q[..., :4] @ p["wdt"].to(dtype)
    B, C = q[..., 4:4 + N].unsqueeze(2), q[..., 4 + N:].unsqueeze(2)
    y = ag.ssm_scan(u, dt, p["A"], B, C, p["D"], p["dt_bias"])
    return ag.norm_gate_residual(y, res, xz[..., D:], post_weight=p["w1"], scale=p["scale"], pre_weight=p["w2"])


def _ssm_layer_plain(p, h, res):
    D, N = p["A"].shape
    xz = h @ p["win"]
    x = xz[..., :D]
    K = p["conv"].shape[1]
    pad = F.pad(x, (0, 0, K - 1, 0))
    u = F.silu(p["conv_b"] + sum(pad[:, k:k + x.shape[1]] * p["conv"][:, k] for k in range(K)))
    q = u @ p["wq"]
    delta = F.softplus(q[..., :4] @ p["wdt"] + p["dt_bias"])
    B, C = q[..., 4:4 + N], q[..., 4 + N:]
    s, ys = torch.zeros(x.shape[0], D, N, dtype=x.dtype, device=x.device), []
    for t in range(x.shape[1]):
        s = torch.exp(delta[:, t, :, None] * p["A"]) * s + (delta[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((s * C[:, t, None]).sum(-1))
    y = torch.stack(ys, 1) + p["D"] * u
    z = res + p["scale"] * F.rms_norm(y, (D,), p["w1"], 1e-6) * F.silu(xz[..., D:])
    return z, F.rms_norm(z, (D,), p["w2"], 1e-6)


def _weights(g, D, N, K):
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(DEV)  # noqa: E731
    first = torch.exp(torch.rand(D, generator=g) * 3 - 5)
    return dict(win=r(D, 2 * D, std=D ** -0.5), conv=r(D, K, std=K ** -0.5), conv_b=r(D, std=0.1), wq=r(D, 4 + 2 * N, std=D ** -0.5),
                wdt=r(4, D, std=0.5), A=-(torch.arange(N) + 1.0).repeat(D, 1).to(DEV), D=1 + r(D, std=0.1),
                dt_bias=(first + torch.log(-torch.expm1(-first))).to(DEV), w1=1 + r(D, std=0.1), scale=0.5 + r(D, std=0.1), w2=1 + r(D, std=0.1))


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 3.2e-2), (torch.float32, 3.1e-5)])
def test_a_state_space_layer_runs_and_has_its_gradients(dtype, tol):
    torch.backends.cuda.matmul.allow_tf32 = False
    B, T, D, N, K = 2, 37, 64, 16, 4
    g = gen(11)
    p = _weights(g, D, N, K)
    h, res = (torch.randn(B, T, D, generator=g).to(DEV).to(dtype) for _ in range(2))
    gz, gn = (torch.randn(B, T, D, generator=g).to(DEV).to(dtype) for _ in range(2))
    lv = {k: v.clone().requires_grad_(True) for k, v in dict(p, h=h, res=res).items()}
    z, n = _ssm_layer(lv, lv["h"], lv["res"], dtype)
    torch.autograd.backward([z, n], [gz, gn])
    l64 = {k: v.detach().double().requires_grad_(True) for k, v in lv.items()}
    z64, n64 = _ssm_layer_plain(l64, l64["h"], l64["res"])
    torch.autograd.backward([z64, n64], [gz.double(), gn.double()])
    assert rel(z, z64) <= tol and rel(n, n64) <= tol
    for k in lv:
        assert rel(lv[k].grad, l64[k].grad) <= tol, k


def test_prompt_then_tokens_is_the_whole_sequence():
    """Serving: a right-padded batch of prompts, then single tokens with the states in a table of slots."""
    B, T, D, N, K, S = 3, 40, 96, 16, 4, 7
    lens, more = [40, 11, 23], 5
    i = scan_inputs(5, "fp32", B, T + more, D, N, 1, DEV, state=False)
    c = conv_inputs(6, "fp32", B, T + more, D, K, DEV, state=False)
    slots = torch.tensor([4, 0, 6], dtype=torch.int32, device=DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    args = [i["dt"], i["A"], i["B"], i["C"]]
    full = []      # each sequence by itself, all tokens at once
    for b, m in enumerate(lens):
        u = ssm.short_conv(c["x"][b:b + 1, :m + more], c["weight"], c["bias"], activation="silu")
        full.append(ssm.ssm_scan(u, *[a[b:b + 1, :m + more] if a.dim() > 2 else a for a in args], i["D"], i["dt_bias"])[0])
    u, cst = ssm.short_conv(c["x"][:, :T], c["weight"], c["bias"], activation="silu", lengths=n, return_state=True)
    y, st = ssm.ssm_scan(u, *[a[:, :T] if a.dim() > 2 else a for a in args], i["D"], i["dt_bias"], lengths=n, return_state=True)
    ctable, table = torch.zeros(S, K - 1, D, device=DEV), torch.zeros(S, D, N, device=DEV)
    ctable[slots.long()], table[slots.long()] = cst, st
    rows = torch.arange(B, device=DEV)
    for t in range(more):
        at = n.long() + t
        u1 = ssm.short_conv_step(c["x"][rows, at], ctable, c["weight"], c["bias"], activation="silu", slots=slots)
        y1 = ssm.ssm_scan_step(u1, *[a[rows, at] if a.dim() > 2 else a for a in args], table, i["D"], i["dt_bias"], slots=slots)
        for b, m in enumerate(lens):
            assert rel(y1[b], full[b][m + t]) <= 1e-5
    for b, m in enumerate(lens):
        assert rel(y[b, :m], full[b][:m]) <= 1e-5


def test_short_conv_in_front_of_a_ttt_layer():
    """Queries and keys through the convolution into the operator's tiles, the operator, and the block's end."""
    from ttt_tk_b200.autograd import ttt_linear
    from ttt_tk_b200.glue import unpack_layernorm
    B, T, H = 2, 128, 2
    g = gen(8)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(DEV)  # noqa: E731
    h = r(B, T, H * 64).bfloat16()
    w = r(H * 64, 4, std=0.5).requires_grad_(True)
    q = ag.short_conv(h, w, heads=True)
    assert torch.equal(q, layout.pack_tokens(ag.short_conv(h, w).detach())[0])
    eta = (0.02 * torch.rand(B, H, T // 64, 64, generator=g)).to(DEV).bfloat16()
    gamma, beta = torch.ones(1, H, 1, 64, device=DEV), torch.zeros(1, H, 1, 64, device=DEV)
    W1, b1 = r(B, H, 64, 64, std=0.02), torch.zeros(B, H, 1, 64, device=DEV)
    out, _ = ttt_linear(q, q, q, eta, gamma, beta, W1, b1)
    y = unpack_layernorm(out.detach(), torch.ones(H * 64, device=DEV), torch.zeros(H * 64, device=DEV))
    x, n = glue.norm_gate_residual(y, h, h, scale=torch.full((H * 64,), 0.1, device=DEV), pre_weight=torch.ones(H * 64, device=DEV))
    assert torch.isfinite(x.float()).all() and torch.isfinite(n.float()).all()
    out.float().sum().backward()
    assert w.grad is not None and torch.isfinite(w.grad).all() and w.grad.abs().sum() > 0


# ---- graphs, streams, devices ----------------------------------------------------------------------------------------------
def test_captured_and_replayed():
    """Forward and backward of all three in one graph, twice captured and replayed in turn with new inputs: each has scratch of its own."""
    B, T, D, N = 1, 600, 64, 16      # the scan in chunks
    i = scan_inputs(1, "bf16", B, T, D, N, 1, DEV)
    c = conv_inputs(2, "bf16", B, T, D, 4, DEV)
    w = torch.ones(D, device=DEV)

    def run(x):
        u = ssm.short_conv(x, c["weight"], c["bias"], activation="silu")
        y, st, ck = ssm.ssm_scan(u, i["dt"], i["A"], i["B"], i["C"], i["D"], i["dt_bias"], return_state=True, return_checkpoints=True)
        z, n, stats = glue.norm_gate_residual(y, x, u, return_stats=True, post_weight=w, scale=w, pre_weight=w)
        g = glue.norm_gate_residual_backward(z, n, y, stats, x, u, post_weight=w, scale=w, pre_weight=w)
        s = ssm.ssm_scan_backward(g[0], u, i["dt"], i["A"], i["B"], i["C"], ck, i["D"], i["dt_bias"])
        k = ssm.short_conv_backward(s[0], x, c["weight"], c["bias"], activation="silu")
        return [z, n, st, *[t for t in (*g, *s, *k) if t is not None]]

    xs = [torch.randn(B, T, D, generator=gen(k)).to(DEV).bfloat16() for k in range(3)]
    want = [run(x) for x in xs]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        static = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        graphs.append((static, graph, out))
    for a, b in ((0, 1), (2, 0), (1, 2)):
        graphs[0][0].copy_(xs[a])
        graphs[1][0].copy_(xs[b])
        graphs[0][1].replay()
        graphs[1][1].replay()
        torch.cuda.synchronize()
        for k, (_, _, out) in zip((a, b), graphs):
            assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


def test_autograd_captured_after_an_eager_pass():
    i = scan_inputs(3, "bf16", 1, 40, 64, 16, 1, DEV)
    lv = leaves(i, ["x", "dt", "A", "B", "C", "D", "dt_bias"])

    def step():
        y = ag.ssm_scan(*lv.values())
        return torch.autograd.grad(y.float().sum(), list(lv.values()))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    i = scan_inputs(4, "bf16", 2, 300, 64, 16, 1, DEV)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y0, ck0 = ssm.ssm_scan(*a, i["D"], i["dt_bias"], return_checkpoints=True)
    want = ssm.ssm_scan_backward(i["gy"], *a, ck0, i["D"], i["dt_bias"])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[] for _ in streams]
    for _ in range(5):
        for s, o in zip(streams, out):
            with torch.cuda.stream(s):
                y, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], return_checkpoints=True)
                o.append((y, ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"])))
    torch.cuda.synchronize()
    for o in out:
        for y, g in o:
            assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, want))


def test_empty_batches_and_sequences():
    D, N, K = 16, 4, 3
    for B, T in ((0, 5), (2, 0), (0, 0)):
        i = scan_inputs(1, "bf16", B, T, D, N, 1, DEV)
        c = conv_inputs(1, "bf16", B, T, D, K, DEV)
        a = [i[k] for k in ("x", "dt", "A", "B", "C")]
        y, st, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], return_state=True, return_checkpoints=True)
        assert y.shape == (B, T, D) and ck.shape == (B, 0 if T == 0 else 1, D, N) and torch.equal(st, i["state"])
        g = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], grad_final_state=i["gf"])
        assert torch.equal(g[7], i["gf"]) and (g[2] == 0).all() and (g[5] == 0).all() and (g[6] == 0).all()
        y, end = ssm.short_conv(c["x"], c["weight"], c["bias"], state=c["state"], return_state=True)
        assert y.shape == (B, T, D) and torch.equal(end, c["state"])
        g = ssm.short_conv_backward(c["gy"], c["x"], c["weight"], c["bias"], state=c["state"], grad_final_state=c["gf"])
        assert (g[1] == 0).all() and (g[2] == 0).all() and torch.equal(g[3], c["gf"])
        z, n, s = glue.norm_gate_residual(c["x"], pre_weight=torch.ones(D, device=DEV), return_stats=True)
        assert z.shape == n.shape == (B, T, D) and s.shape == (B * T, 4)
        g = glue.norm_gate_residual_backward(None, n, c["x"], s, pre_weight=torch.ones(D, device=DEV))
        assert g[0].shape == (B, T, D) and (g[6] == 0).all()
    x = torch.zeros(0, D, device=DEV, dtype=torch.bfloat16)
    assert ssm.short_conv_step(x, torch.zeros(0, K - 1, D, device=DEV, dtype=torch.bfloat16), torch.zeros(D, K, device=DEV)).shape == (0, D)


def test_offsets_beyond_32_bits():
    """A sequence whose tensors have more than 2^31 values: the end of it is that of a run that starts there."""
    T, D, K, N, cut = 1_100_000, 2048, 4, 4, 1_099_000
    x = torch.randn(1, T, D, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(D, K, device=DEV)
    y = ssm.short_conv(x, w, activation="silu")
    tail = ssm.short_conv(x[:, cut:], w, activation="silu", state=x[:, cut - K + 1:cut].contiguous())
    assert torch.equal(y[:, cut:], tail)
    gx = ssm.short_conv_backward(y, x, w, activation="silu")[0]
    gt = ssm.short_conv_backward(y[:, cut:], x[:, cut:], w, activation="silu", state=x[:, cut - K + 1:cut].contiguous())[0]
    assert torch.equal(gx[:, cut:], gt)
    del gx, gt, tail
    dt = torch.randn(1, T, 1, device=DEV, dtype=torch.bfloat16).expand(1, T, D).contiguous()
    A = -torch.rand(D, N, device=DEV) - 0.5
    B, C = (torch.randn(1, T, 1, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    y, st = ssm.ssm_scan(x, dt, A, B, C, return_state=True)
    _, mid = ssm.ssm_scan(x[:, :cut], dt[:, :cut], A, B[:, :cut], C[:, :cut], return_state=True)
    yt, end = ssm.ssm_scan(x[:, cut:], dt[:, cut:], A, B[:, cut:], C[:, cut:], state=mid, return_state=True)
    assert rel(st, end) <= 1e-5 and rel(y[:, cut:], yt) <= 2 ** -8
    z, n = glue.norm_gate_residual(x, y, pre_weight=torch.ones(D, device=DEV))
    zt, nt = glue.norm_gate_residual(x[:, cut:], y[:, cut:], pre_weight=torch.ones(D, device=DEV))
    assert torch.equal(z[:, cut:], zt) and torch.equal(n[:, cut:], nt)
