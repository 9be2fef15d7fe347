"""What is measured of the layer-side sequence operators: the short causal convolution, the selective state space
scan, and the end of a block (post norm, gate, scaled residual, the next block's pre norm).

A case is one call pattern at one size.  `op` is "conv", "scan" or "norm"; `mode` is "step" (one token per sequence, the
state updated in place), "fwd" (prompts, evaluation) or "train" (forward and backward).  `type` is the activations'; weights,
scan states and statistics are fp32.

The formulas, with x [B, T, D] and everything in 32 bits between reading and writing:

  conv   y[b,t,d] = act(bias[d] + sum_k w[d,k] x[b,t-K+1+k,d]); inputs in front of the first token come from the state
  scan   delta = softplus(dt + dt_bias);  h[d,n] = exp(delta A[d,n]) h[d,n] + delta x B[g,n];  y = sum_n C[g,n] h[d,n] + D[d] x,
         g = the group of channel d
  norm   u = Norm(o) w1 + b1;  x' = x + scale u act(gate);  n = Norm(x') w2 + b2

Tokens from a sequence's length on give y = 0 and change nothing.
"""
import math

import torch
import torch.nn.functional as F

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------------

def _conv(mode, type, B, T, D, K, act="silu", state=False, ragged=False, heads=False, wide=False, slots=0, name=None):
    c = dict(op="conv", mode=mode, type=type, B=B, T=T, D=D, K=K, act=act, state=state, ragged=ragged, heads=heads, wide=wide,
             slots=slots)
    return dict(c, name=name) if name else c


def _scan(mode, type, B, T, D, N, G=1, state=False, ragged=False, wide=False, slots=0, name=None):
    c = dict(op="scan", mode=mode, type=type, B=B, T=T, D=D, N=N, G=G, state=state, ragged=ragged, wide=wide, slots=slots)
    return dict(c, name=name) if name else c


def _norm(mode, type, M, D, norm="rms", act="silu", res32=False, gate=True, post=True, scale=True, pre=True, wide=False, name=None):
    c = dict(op="norm", mode=mode, type=type, M=M, D=D, norm=norm, act=act, res32=res32, gate=gate, post=post, scale=scale, pre=pre,
             wide=wide)
    return dict(c, name=name) if name else c


def listed():
    return [
        # decoding: one token of each of 8 requests, their states in a table of slots; the smallest call, all latency
        _conv("step", "bf16", 8, 1, 2048, 4, state=True, slots=16, name="conv step 8 x 2048"),
        # queries of a TTT layer of 12 heads, straight into the operator's head-major tiles; no activation
        _conv("fwd", "bf16", 1, 2048, 768, 4, act="none", heads=True, name="conv to heads 2048 x 768"),
        # training at the width of the 32-head workload; x is one half of the input projection's output
        _conv("train", "bf16", 4, 2048, 2048, 4, wide=True, name="conv train 4 x 2048 x 2048"),
        # odd sizes, right-padded batch, chunk with a state and its gradient
        _conv("train", "fp32", 3, 1001, 1003, 3, state=True, ragged=True, name="conv train ragged 3 x 1001 x 1003"),
        # decoding of 64 requests: bound by the scan states
        _scan("step", "bf16", 64, 1, 2048, 16, state=True, slots=100, name="scan step 64 x 2048 x 16"),
        # one long prompt, few channels: parallel work only along the sequence
        _scan("fwd", "bf16", 1, 8192, 1024, 16, state=True, wide=True, name="scan prompt 8192 x 1024 x 16"),
        # training at the width of the 24-head workload
        _scan("train", "bf16", 4, 2048, 1536, 16, wide=True, name="scan train 4 x 2048 x 1536 x 16"),
        # heads with an input and output vector each: 12 groups of 64 channels, wide states
        _scan("train", "fp16", 2, 1000, 768, 64, G=12, name="scan train 2 x 1000 x 768 x 64, 12 groups"),
        # odd sizes, right-padded batch, chunk with a state and its gradient
        _scan("train", "fp32", 3, 777, 203, 5, state=True, ragged=True, name="scan train ragged 3 x 777 x 203 x 5"),
        # decoding: 4 tokens between two blocks
        _norm("fwd", "bf16", 4, 2048, name="norm 4 x 2048"),
        # training, fp32 residual stream, LayerNorm and the layer's GELU gate
        _norm("train", "bf16", 16384, 2048, norm="layer", act="gelu", res32=True, wide=True, name="norm train 16384 x 2048"),
        # odd width, plain residual type
        _norm("train", "fp16", 3001, 1003, name="norm train 3001 x 1003"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["conv", "scan", "norm"])
    mode = rng.choice(["step", "fwd", "train", "train"])
    top = max(work(c)["bytes"] + work(c)["flops"] / 8 for c in listed() if c["op"] == op)
    while True:
        D = _log(rng, 1, 64) * 64 if rng.random() < 0.6 else _log(rng, 8, 4096)
        B, T = (_log(rng, 1, 256), 1) if mode == "step" else (_log(rng, 1, 16), _log(rng, 1, 8192))
        some = [rng.random() < 0.5 for _ in range(6)]
        slots = B + rng.randint(0, B) if mode == "step" else 0
        if op == "conv":
            heads = mode != "step" and D % 64 == 0 and some[2]
            if heads:
                T = -(-T // 64) * 64
            c = _conv(mode, type, B, T, D, rng.choice([2, 3, 4, 4]), rng.choice(["none", "silu"]), mode == "step" or some[0],
                      mode != "step" and some[1], heads, some[3], slots)
        elif op == "scan":
            G = rng.choice([g for g in (1, 1, 2, 3, 4, 8, 12, D // 64) if g and D % g == 0])
            c = _scan(mode, type, B, T, D, rng.choice([16, 16, 16, 4, 8, 32, 64, rng.randint(1, 64)]), G, mode == "step" or some[0],
                      mode != "step" and some[1], some[3], slots)
        else:
            c = _norm("train" if mode == "train" else "fwd", type, _log(rng, 1, 16384), D, rng.choice(["rms", "layer"]),
                      rng.choice(["silu", "gelu", "sigmoid"]), some[0], some[1], some[2], some[3], some[4], some[5])
        if work(c)["bytes"] + work(c)["flops"] / 8 <= top:
            return c


def work(c):
    e = 4 if c["type"] == "fp32" else 2
    train = c["mode"] == "train"
    if c["op"] == "norm":
        r = 4 if c["res32"] or c["type"] == "fp32" else 2
        n = c["M"] * c["D"]
        fwd = n * (e + 2 * r + e * c["gate"] + e * c["pre"])                      # o, x, gate -> x', n
        bwd = n * (2 * e + 3 * r + 2 * e * c["gate"] + e * c["pre"])              # o, x, gate, dx', dn -> do, dx, dgate
        return {"bytes": fwd + train * bwd, "flops": n * (20 + 40 * train)}
    tok = c["B"] * c["T"] * c["D"]
    if c["op"] == "conv":
        K, st = c["K"], c["B"] * (c["K"] - 1) * c["D"] * e * (2 if c["state"] else 0)
        return {"bytes": tok * e * (2 + 3 * train) + st * (1 + train) + c["D"] * (K + 1) * 4 * (1 + train),
                "flops": tok * (2 * K + 4 + (6 * K + 8) * train)}
    N, G = c["N"], c["G"]
    bc = 2 * c["B"] * c["T"] * G * N * e
    st = c["B"] * c["D"] * N * 4 * (2 if c["state"] else 0)
    return {"bytes": tok * e * (3 + 5 * train) + bc * (1 + 2 * train) + st * (1 + train) + c["D"] * N * 4 * (1 + train),
            "flops": tok * N * (7 + 20 * train)}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _rows(g, c, *shape, std=1.0):
    """Activations [..., D]; `wide`: as the first half of a tensor twice as wide, which is how a projection's output is split."""
    *lead, D = shape
    x = torch.randn(*lead, 2 * D if c["wide"] else D, generator=g, device="cuda") * std
    return x.to(TYPES[c["type"]])[..., :D]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda") * std  # noqa: E731
    ty, s = TYPES[c["type"]], dict(c)
    train = c["mode"] == "train"
    if c["op"] == "norm":
        M, D = c["M"], c["D"]
        rt = torch.float32 if c["res32"] else ty
        s["o"] = _rows(g, c, M, D, std=1.5) + 0.25
        s["x"] = rnd(M, D, std=2.0).to(rt)
        s["gate"] = _rows(g, c, M, D) if c["gate"] else None
        layer = c["norm"] == "layer"
        s["w1"] = 1 + rnd(D, std=0.1) if c["post"] else None
        s["b1"] = rnd(D, std=0.1) if c["post"] and layer else None
        s["scale"] = rnd(D, std=0.1) + 0.3 if c["scale"] else None
        s["w2"] = 1 + rnd(D, std=0.1) if c["pre"] else None
        s["b2"] = rnd(D, std=0.1) if c["pre"] and layer else None
        if train:
            s["gx"] = rnd(M, D).to(rt)
            s["gn"] = rnd(M, D).to(ty) if c["pre"] else None
        return s
    B, T, D = c["B"], c["T"], c["D"]
    lead = (B,) if c["mode"] == "step" else (B, T)
    s["lengths"] = None
    if c["ragged"]:      # a right-padded batch: its longest sequence fills it
        n = torch.randint(max(1, T // 3), T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        n[0] = T
        s["lengths"] = n
    s["index"] = None
    if c["slots"]:
        s["index"] = torch.randperm(c["slots"], generator=g, device="cuda")[:B].to(torch.int32)
        if B > 2:
            s["index"][B // 2] = -1          # a padded row of the batch
    rows = c["slots"] or B
    if c["op"] == "conv":
        K = c["K"]
        s["x"] = _rows(g, c, *lead, D)
        s["w"] = rnd(D, K, std=K ** -0.5)
        s["b"] = rnd(D, std=0.1)
        s["st"] = rnd(rows, K - 1, D).to(ty) if c["state"] else None
        if train:
            s["gy"] = rnd(B, D // 64, T // 64, 64, 64).to(ty) if c["heads"] else rnd(B, T, D).to(ty)
            s["gst"] = rnd(B, K - 1, D).to(ty) if c["state"] else None
        return s
    N, G = c["N"], c["G"]
    s["x"] = F.silu(_rows(g, c, *lead, D).float()).to(ty) if not c["wide"] else _rows(g, c, *lead, D, std=0.6)
    # rows of one projection: step sizes' low rank part, then B and C
    low = D // 16 if c["wide"] else 0
    p = rnd(*lead, low + 2 * G * N).to(ty)
    s["Bm"] = p[..., low:low + G * N].unflatten(-1, (G, N))
    s["Cm"] = p[..., low + G * N:].unflatten(-1, (G, N))
    s["dt"] = rnd(*lead, D, std=0.5).to(ty)
    first = torch.exp(torch.rand(D, generator=g, device="cuda") * math.log(100) + math.log(1e-3))     # step sizes 0.001 to 0.1
    s["dtb"] = first + torch.log(-torch.expm1(-first))
    s["A"] = -torch.arange(1, N + 1, device="cuda").float() * (1 + 0.2 * torch.rand(D, N, generator=g, device="cuda"))
    s["Dk"] = 1 + rnd(D, std=0.1)
    s["st"] = rnd(rows, D, N, std=0.5) if c["state"] else None
    if train:
        s["gy"] = rnd(B, T, D).to(ty)
        s["gst"] = rnd(B, D, N, std=0.5) if c["state"] else None
    return s


# ---- plain forms: elementary operations in 32 bits -------------------------------------------------------------------

def _act(x, name):
    """Value and derivative."""
    if name == "none":
        return x, torch.ones_like(x)
    if name == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)
    s = 1 / (1 + torch.exp(-x))
    if name == "sigmoid":
        return s, s * (1 - s)
    return x * s, s * (1 + x * (1 - s))


def _live(s):
    """[B, T, 1]: which tokens are ones of their sequence."""
    n = s["lengths"] if s["lengths"] is not None else torch.full((s["B"],), s["T"], device="cuda")
    return (torch.arange(s["T"], device="cuda") < n[:, None])[..., None], n.long()


def _to_heads(y):
    B, T, D = y.shape
    return y.reshape(B, T, D // 64, 64).transpose(1, 2).reshape(B, D // 64, T // 64, 64, 64)


def _from_heads(y):
    B, H, NC = y.shape[:3]
    return y.reshape(B, H, NC * 64, 64).transpose(1, 2).reshape(B, NC * 64, H * 64)


def _conv_plain(s):
    B, T, D, K, ty = s["B"], s["T"], s["D"], s["K"], TYPES[s["type"]]
    live, n = _live(s)
    x = torch.where(live, s["x"].float(), 0.0)
    w = s["w"]
    head = s["st"].float() if s["st"] is not None else torch.zeros(B, K - 1, D, device="cuda")
    xp = torch.cat([head, x], 1)
    pre = s["b"] + sum(w[:, k] * xp[:, k:k + T] for k in range(K))
    val, slope = _act(pre, s["act"])
    y = torch.where(live, val, 0.0).to(ty)
    out = {"y": _to_heads(y) if s["heads"] else y}
    tail = n[:, None] + torch.arange(K - 1, device="cuda")                       # rows of xp: the last K - 1 inputs
    at = tail[..., None].expand(B, K - 1, D)
    if s["state"]:
        out["state"] = xp.gather(1, at).to(ty)
    if s["mode"] == "train":
        gy = _from_heads(s["gy"]) if s["heads"] else s["gy"]
        g = torch.where(live, gy.float() * slope, 0.0)
        gp = F.pad(g, (0, 0, K - 1, K - 1))
        dxp = sum(w[:, k] * gp[:, K - 1 - k:K - 1 - k + T + K - 1] for k in range(K))
        if s["gst"] is not None:
            dxp = dxp.scatter_add(1, at, s["gst"].float())
            out["grad_state"] = dxp[:, :K - 1].to(ty)
        out["grad_x"] = dxp[:, K - 1:].to(ty)
        out["grad_w"] = torch.stack([(g * xp[:, k:k + T]).sum((0, 1)) for k in range(K)], 1)
        out["grad_b"] = g.sum((0, 1))
    return out


def _slot(s):
    """(rows of the batch that have a state, their slots)."""
    at = s["index"].long()
    live = at >= 0
    return live, at[live]


def _conv_step_plain(s):
    live, at = _slot(s)
    win = torch.cat([s["st"][at], s["x"][live][:, None]], 1)
    y = torch.zeros(s["B"], s["D"], device="cuda", dtype=TYPES[s["type"]])
    y[live] = _act(s["b"] + (win.float() * s["w"].t()).sum(1), s["act"])[0].to(y.dtype)
    s["st"][at] = win[:, 1:]
    return {"y": y, "state": s["st"]}


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, in place in b: runs of twice the length each time."""
    span, T = 1, a.shape[1]
    while span < T:
        b[:, span:] += a[:, span:] * b[:, :-span].clone()
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _spread(v, D):
    """[..., G, N] -> [..., D, N]: a group's vector for each of its channels."""
    return v.float().repeat_interleave(D // v.shape[-2], -2)


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _scan_plain(s):
    T, D, G, ty = s["T"], s["D"], s["G"], TYPES[s["type"]]
    live, _ = _live(s)
    x = torch.where(live, s["x"].float(), 0.0)
    v = s["dt"].float() + s["dtb"]
    delta = torch.where(live, _softplus(v), 0.0)
    Bm = torch.where(live[..., None], s["Bm"].float(), 0.0)
    Cm = torch.where(live[..., None], s["Cm"].float(), 0.0)
    a = torch.exp(delta[..., None] * s["A"])
    b = (delta * x)[..., None] * _spread(Bm, D)
    if s["st"] is not None:
        b[:, 0] += a[:, 0] * s["st"]
    h = _recur(a, b)
    out = {"y": ((h * _spread(Cm, D)).sum(-1) + s["Dk"] * x).to(ty)}
    if s["state"]:
        out["state"] = h[:, -1].clone()
    if s["mode"] == "train":
        gy = torch.where(live, s["gy"].float(), 0.0)
        dh = gy[..., None] * _spread(Cm, D)
        if s["gst"] is not None:
            dh[:, -1] += s["gst"]
        # backwards in time the factor of a step is the next one's
        after = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
        dh = _recur(after, dh.flip(1)).flip(1)
        first = s["st"][:, None] if s["st"] is not None else torch.zeros_like(h[:, :1])
        q = dh * a * torch.cat([first, h[:, :-1]], 1)                            # dh times what was left of the last state
        if s["st"] is not None:
            out["grad_state"] = dh[:, 0] * a[:, 0]
        out["grad_A"] = (q * delta[..., None]).sum((0, 1))
        dB = (dh * _spread(Bm, D)).sum(-1)
        dd = (q * s["A"]).sum(-1) + x * dB
        dv = torch.where(live, dd / (1 + torch.exp(-v)), 0.0)
        out["grad_x"] = torch.where(live, delta * dB + s["Dk"] * gy, 0.0).to(ty)
        out["grad_dt"] = dv.to(ty)
        out["grad_dt_bias"] = dv.sum((0, 1))
        out["grad_D"] = (gy * x).sum((0, 1))
        fold = lambda z: z.unflatten(2, (G, D // G)).sum(3).to(ty)  # noqa: E731
        out["grad_B"] = fold(dh * (delta * x)[..., None])
        out["grad_C"] = fold(h * gy[..., None])
    return out


def _scan_step_plain(s):
    live, at = _slot(s)
    D = s["D"]
    x = s["x"][live].float()
    delta = _softplus(s["dt"][live].float() + s["dtb"])
    h = torch.exp(delta[..., None] * s["A"]) * s["st"][at] + (delta * x)[..., None] * _spread(s["Bm"][live], D)
    y = torch.zeros(s["B"], D, device="cuda", dtype=TYPES[s["type"]])
    y[live] = ((h * _spread(s["Cm"][live], D)).sum(-1) + s["Dk"] * x).to(y.dtype)
    s["st"][at] = h
    return {"y": y, "state": s["st"]}


def _norm_of(x, kind):
    """(normalised, 1 / deviation)."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _norm_back(g, xh, r, kind):
    g0 = g - g.mean(-1, keepdim=True) if kind == "layer" else g
    return r * (g0 - xh * (g * xh).mean(-1, keepdim=True))


def _norm_plain(s):
    ty, kind = TYPES[s["type"]], s["norm"]
    o, x = s["o"].float(), s["x"].float()
    u = o
    if s["post"]:
        oh, r1 = _norm_of(o, kind)
        u = oh * s["w1"] + (s["b1"] if s["b1"] is not None else 0.0)
    gv, gs = _act(s["gate"].float(), s["act"]) if s["gate"] is not None else (1.0, None)
    sc = s["scale"] if s["scale"] is not None else 1.0
    z = x + sc * (u * gv)
    out = {"x": z.to(s["x"].dtype)}
    if s["pre"]:
        zh, r2 = _norm_of(z, kind)
        out["n"] = (zh * s["w2"] + (s["b2"] if s["b2"] is not None else 0.0)).to(ty)
    if s["mode"] == "train":
        d = s["gx"].float()
        if s["pre"]:
            gn = s["gn"].float()
            d = d + _norm_back(gn * s["w2"], zh, r2, kind)
            out["grad_pre_weight"] = (gn * zh).sum(0)
            if s["b2"] is not None:
                out["grad_pre_bias"] = gn.sum(0)
        out["grad_residual"] = d.to(s["x"].dtype)
        if s["scale"] is not None:
            out["grad_scale"] = (d * (u * gv)).sum(0)
        dv = d * sc
        if s["gate"] is not None:
            out["grad_gate"] = (dv * u * gs).to(ty)
        du = dv * gv
        if s["post"]:
            out["grad_post_weight"] = (du * oh).sum(0)
            if s["b1"] is not None:
                out["grad_post_bias"] = du.sum(0)
            du = _norm_back(du * s["w1"], oh, r1, kind)
        out["grad_o"] = du.to(ty)
    return out


def _plain(s):
    if s["op"] == "norm":
        return _norm_plain(s)
    if s["op"] == "conv":
        return _conv_step_plain(s) if s["mode"] == "step" else _conv_plain(s)
    return _scan_step_plain(s) if s["mode"] == "step" else _scan_plain(s)


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _own(s):
    train = s["mode"] == "train"
    if s["op"] == "norm":
        from ttt_tk_b200.glue import norm_gate_residual, norm_gate_residual_backward
        kw = dict(norm=s["norm"], activation=s["act"], post_weight=s["w1"], post_bias=s["b1"], scale=s["scale"], pre_weight=s["w2"],
                  pre_bias=s["b2"], eps=EPS)
        if not train:
            x, n = norm_gate_residual(s["o"], s["x"], s["gate"], **kw)
            return _given(x=x, n=n)
        x, n, stats = norm_gate_residual(s["o"], s["x"], s["gate"], return_stats=True, **kw)
        go, gr, gg, gw1, gb1, gsc, gw2, gb2 = norm_gate_residual_backward(s["gx"], s["gn"], s["o"], stats, s["x"], s["gate"], **kw)
        return _given(x=x, n=n, grad_o=go, grad_residual=gr, grad_gate=gg, grad_post_weight=gw1, grad_post_bias=gb1, grad_scale=gsc,
                      grad_pre_weight=gw2, grad_pre_bias=gb2)
    from ttt_tk_b200 import ssm
    if s["op"] == "conv":
        act = None if s["act"] == "none" else s["act"]
        if s["mode"] == "step":
            y = ssm.short_conv_step(s["x"], s["st"], s["w"], s["b"], activation=act, slots=s["index"])
            return {"y": y, "state": s["st"]}
        kw = dict(activation=act, state=s["st"], lengths=s["lengths"], heads=s["heads"])
        y = ssm.short_conv(s["x"], s["w"], s["b"], return_state=s["state"], **kw)
        y, st = y if s["state"] else (y, None)
        if not train:
            return _given(y=y, state=st)
        gx, gw, gb, gst = ssm.short_conv_backward(s["gy"], s["x"], s["w"], s["b"], grad_final_state=s["gst"], **kw)
        return _given(y=y, state=st, grad_x=gx, grad_w=gw, grad_b=gb, grad_state=gst)
    args = (s["x"], s["dt"], s["A"], s["Bm"], s["Cm"])
    if s["mode"] == "step":
        return {"y": ssm.ssm_scan_step(*args, s["st"], s["Dk"], s["dtb"], slots=s["index"]), "state": s["st"]}
    r = ssm.ssm_scan(*args, s["Dk"], s["dtb"], state=s["st"], lengths=s["lengths"], return_state=s["state"], return_checkpoints=train)
    r = list(r) if isinstance(r, tuple) else [r]
    y, st = r[0], r[1] if s["state"] else None
    if not train:
        return _given(y=y, state=st)
    gx, gdt, gA, gB, gC, gD, gb, gst = ssm.ssm_scan_backward(s["gy"], *args, r[-1], s["Dk"], s["dtb"], lengths=s["lengths"],
                                                             grad_final_state=s["gst"])
    return _given(y=y, state=st, grad_x=gx, grad_dt=gdt, grad_A=gA, grad_B=gB, grad_C=gC, grad_D=gD, grad_dt_bias=gb,
                  grad_state=gst if s["state"] else None)


def _given(**kw):
    return {k: v for k, v in kw.items() if v is not None}


def run(s):
    return _own(s) if own else _plain(s)


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------

_ACT64 = {"none": lambda x: x, "silu": F.silu, "sigmoid": torch.sigmoid, "gelu": lambda x: F.gelu(x, approximate="tanh")}


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _grads(out, pairs, leaves):
    """Gradients of sum(value * upstream) over `pairs` with respect to the leaves, by name."""
    names = [k for k, v in leaves.items() if v is not None]
    got = torch.autograd.grad([v for v, _ in pairs], [leaves[k] for k in names], [g.double() for _, g in pairs])
    out.update({"grad_" + k: v for k, v in zip(names, got)})


def _exact_norm(s):
    lv = dict(o=_leaf(s["o"]), residual=_leaf(s["x"]), gate=_leaf(s["gate"]), post_weight=_leaf(s["w1"]), post_bias=_leaf(s["b1"]),
              scale=_leaf(s["scale"]), pre_weight=_leaf(s["w2"]), pre_bias=_leaf(s["b2"]))
    D = s["D"]

    def norm(x, w, b):
        return F.layer_norm(x, (D,), w, b, EPS) if s["norm"] == "layer" else F.rms_norm(x, (D,), w, EPS)

    v = norm(lv["o"], lv["post_weight"], lv["post_bias"]) if s["post"] else lv["o"]
    if s["gate"] is not None:
        v = v * _ACT64[s["act"]](lv["gate"])
    if s["scale"] is not None:
        v = v * lv["scale"]
    x = lv["residual"] + v
    out, pairs = {"x": x}, [(x, s.get("gx"))]
    if s["pre"]:
        out["n"] = norm(x, lv["pre_weight"], lv["pre_bias"])
        pairs.append((out["n"], s.get("gn")))
    if s["mode"] == "train":
        _grads(out, pairs, lv)
    return out


def _exact_conv(s):
    T, K, D, B = s["T"], s["K"], s["D"], s["B"]
    x, w, b, st = _leaf(s["x"]), _leaf(s["w"]), _leaf(s["b"]), _leaf(s["st"])
    n = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    ys, ends = [], []
    for i in range(B):      # each sequence by itself, at its own length
        head = st[i] if st is not None else torch.zeros(K - 1, D, dtype=torch.float64, device="cuda")
        row = torch.cat([head, x[i, :n[i]]])
        y = _ACT64[s["act"]](F.conv1d(row.t()[None], w[:, None], b, groups=D)[0].t()) if n[i] else row[:0]
        ys.append(torch.cat([y, torch.zeros(T - n[i], D, dtype=torch.float64, device="cuda")]))
        ends.append(row[len(row) - (K - 1):])
    y, end = torch.stack(ys), torch.stack(ends)
    if s["heads"]:
        y = y.view(B, T // 64, 64, D // 64, 64).permute(0, 3, 1, 2, 4)
    out = {"y": y}
    if s["state"]:
        out["state"] = end
    if s["mode"] == "train":
        pairs = [(y, s["gy"])] + ([(end, s["gst"])] if s["gst"] is not None else [])
        _grads(out, pairs, dict(x=x, w=w, b=b, state=st))
    return out


def _exact_scan(s):
    B, T, D, G, N = s["B"], s["T"], s["D"], s["G"], s["N"]
    lv = dict(x=_leaf(s["x"]), dt=_leaf(s["dt"]), A=_leaf(s["A"]), B=_leaf(s["Bm"]), C=_leaf(s["Cm"]), D=_leaf(s["Dk"]),
              dt_bias=_leaf(s["dtb"]), state=_leaf(s["st"]))
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    v = lv["dt"] + lv["dt_bias"]
    delta = torch.where(v > 30, v, torch.log1p(torch.exp(v.clamp(max=30))))
    h = lv["state"] if lv["state"] is not None else torch.zeros(B, D, N, dtype=torch.float64, device="cuda")
    h = h.view(B, G, D // G, N)
    ones, ys = (n.min() == T).item(), []
    A = lv["A"].view(G, D // G, N)
    for t in range(T):      # token by token, as the definition has it
        d = delta[:, t].view(B, G, D // G, 1)
        u = lv["x"][:, t].view(B, G, D // G, 1)
        new = torch.exp(d * A) * h + d * u * lv["B"][:, t, :, None]
        y = (new * lv["C"][:, t, :, None]).sum(-1).reshape(B, D) + lv["D"] * lv["x"][:, t]
        if ones:
            h = new
        else:
            on = (t < n).view(B, 1, 1, 1)
            h, y = torch.where(on, new, h), torch.where(on.view(B, 1), y, 0.0)
        ys.append(y)
    y, h = torch.stack(ys, 1), h.reshape(B, D, N)
    out = {"y": y}
    if s["state"]:
        out["state"] = h
    if s["mode"] == "train":
        _grads(out, [(y, s["gy"])] + ([(h, s["gst"])] if s["gst"] is not None else []), lv)
    return out


def _exact_step(s):
    y = torch.zeros(s["B"], s["D"], dtype=torch.float64, device="cuda")
    st = s["st"].double()
    for i, at in enumerate(s["index"].tolist()):
        if at < 0:
            continue
        x = s["x"][i].double()
        if s["op"] == "conv":
            row = torch.cat([st[at], x[None]])
            y[i] = _ACT64[s["act"]]((row * s["w"].double().t()).sum(0) + s["b"].double())
            st[at] = row[1:]
        else:
            v = s["dt"][i].double() + s["dtb"].double()
            d = torch.log1p(torch.exp(v))[:, None]
            per = s["D"] // s["G"]
            Bm, Cm = (torch.repeat_interleave(s[k][i].double(), per, 0) for k in ("Bm", "Cm"))
            st[at] = torch.exp(d * s["A"].double()) * st[at] + d * x[:, None] * Bm
            y[i] = (st[at] * Cm).sum(1) + s["Dk"].double() * x
    return {"y": y, "state": st}


def exact(c, seed):
    s = prepare(c, seed)
    if c["mode"] == "step":
        return _exact_step(s)
    with torch.enable_grad():
        out = {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[c["op"]](s)
    return {k: v.detach() for k, v in out.items()}
