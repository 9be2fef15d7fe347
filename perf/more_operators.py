"""What is measured of the gated linear recurrence, of activations that are kept in 8 bits for a backward pass, of moving the
rows of state tables, and of the norm with a residual whose output leaves in 8 bits.

A case is one call pattern at one size.  `op` is "gated", "saved", "rows" or "norm8"; `type` is the activations'; weights, states,
checkpoints, scales and statistics are fp32.

The formulas, with x [B, T, D] and everything in 32 bits between reading and writing:

  gated  s = sigmoid(gate + gate_bias);  log a = A[d] s (without A: a = s);  b = sqrt(1 - a^2), 1 - a or 1 (`mix`);
         h = a h + b sigmoid(input_gate + input_bias) x;  y = h.  Tokens from a sequence's length on give y = 0 and change nothing.
  saved  8 bits: of each `group` neighbouring values of a row, scale = the least power of two with max |v| <= 448 scale, and the
         values v / scale in e4m3.  A backward pass from kept values is that of the formula at the values that are kept, with the
         states at every 64th token as the forward pass had them.
  rows   table[target[i]] = table[source[i]], all rows read before one is written; a pair with an index outside the table does nothing.
         Compacting: with n rows in use, the k-th used row from n on moves to the k-th free row in front of n.
  norm8  z = residual + o;  n = Norm(z) weight + bias, in 8 bits as above (group 0: the whole row)
"""
import math

import torch
import torch.nn.functional as F

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
EVERY = 64      # tokens between two states that the backward pass starts from


# ---- cases ----------------------------------------------------------------------------------------------------------

def _gated(mode, type, B, T, D, mix="sqrt", A=True, igate=True, bias=True, state=False, ragged=False, wide=False, slots=0, kept=0, name=None):
    c = dict(op="gated", mode=mode, type=type, B=B, T=T, D=D, mix=mix, A=A, igate=igate, bias=bias, state=state, ragged=ragged, wide=wide,
             slots=slots, kept=kept)
    return dict(c, name=name) if name else c


def _saved(type, M, D, tensors, group, wide=False, name=None):
    c = dict(op="saved", mode="both", type=type, M=M, D=D, tensors=tensors, group=group, wide=wide)
    return dict(c, name=name) if name else c


def _rows_case(mode, type, S, n, D, N, heads=0, name=None):
    c = dict(op="rows", mode=mode, type=type, S=S, n=n, D=D, N=N, heads=heads)
    return dict(c, name=name) if name else c


def _norm8(type, M, D, norm="rms", res=True, res32=False, bias=False, group=128, wide=False, name=None):
    c = dict(op="norm8", mode="fwd", type=type, M=M, D=D, norm=norm, res=res, res32=res32, bias=bias, group=group, wide=wide)
    return dict(c, name=name) if name else c


def listed():
    return [
        # decoding: one token of each of 8 requests, their states in a table of slots; the smallest call, all latency
        _gated("step", "bf16", 8, 1, 2048, state=True, slots=16, name="gated step 8 x 2048"),
        # one long prompt, few channels: parallel work only along the sequence
        _gated("fwd", "bf16", 1, 16384, 1024, state=True, wide=True, name="gated prompt 16384 x 1024"),
        # training at the width of the 32-head workload; x is one half of the input projection's output
        _gated("train", "bf16", 4, 2048, 2048, wide=True, name="gated train 4 x 2048 x 2048"),
        # odd sizes, right-padded batch, chunk with a state and its gradient
        _gated("train", "fp32", 3, 1001, 1003, state=True, ragged=True, name="gated train ragged 3 x 1001 x 1003"),
        # large batch whose backward pass starts from inputs kept in 8 bits: the memory that training is short of
        _gated("train", "bf16", 8, 4096, 2048, kept=128, name="gated train kept 8 x 4096 x 2048"),
        # the plain convex mixture with odd sizes, kept in 8 bits
        _gated("train", "fp16", 2, 777, 1538, mix="linear", A=False, igate=False, state=True, kept=64, name="gated train kept 2 x 777 x 1538"),
        # what a layer's forward pass keeps of a projection's three outputs, and its backward pass takes again
        _saved("bf16", 16384, 2048, 3, 128, wide=True, name="saved 3 x 16384 x 2048"),
        # odd rows, in groups of 32
        _saved("fp16", 3001, 1003, 1, 32, name="saved 3001 x 1003"),
        # a request splits into 8 samples: its convolution window and scan states to 8 other rows
        _rows_case("fork", "bf16", 64, 8, 2048, 16, name="rows fork 8 of 64"),
        # half of 256 sequences have ended: the TTT-MLP weights of 12 heads of the others to the front of their tables
        _rows_case("compact", "fp32", 256, 128, 768, 0, heads=12, name="rows compact 128 of 256"),
        # decoding: 4 tokens in front of an 8-bit projection, a scale to a token
        _norm8("bf16", 4, 2048, group=0, name="norm8 4 x 2048"),
        # a long prompt, fp32 residual stream, scales by 128
        _norm8("bf16", 16384, 2048, res32=True, wide=True, name="norm8 16384 x 2048"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["gated", "gated", "gated", "saved", "rows", "norm8", "norm8"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        D = _log(rng, 1, 64) * 64 if rng.random() < 0.6 else _log(rng, 8, 4096)
        some = [rng.random() < 0.5 for _ in range(6)]
        if op == "gated":
            mode = rng.choice(["step", "fwd", "train", "train"])
            B, T = (_log(rng, 1, 256), 1) if mode == "step" else (_log(rng, 1, 16), _log(rng, 1, 16384))
            c = _gated(mode, type, B, T, D, rng.choice(["sqrt", "sqrt", "linear", "none"]), some[0], some[1], some[2], mode == "step" or some[3],
                       mode != "step" and some[4], some[5], B + rng.randint(0, B) if mode == "step" else 0,
                       rng.choice([0, 0, 32, 64, 128]) if mode == "train" else 0)
        elif op == "saved":
            c = _saved(type, _log(rng, 1, 16384), D, rng.randint(1, 4), rng.choice([32, 64, 128]), some[0])
        elif op == "rows":
            S = _log(rng, 2, 256)
            if some[0]:
                c = _rows_case(rng.choice(["fork", "permute", "clear"]), type, S, rng.randint(1, S), D, rng.choice([4, 8, 16, 64, rng.randint(1, 64)]))
            else:
                heads = rng.choice([1, 4, 12, 24, 32])
                c = _rows_case("compact", "fp32", S, rng.randint(1, S - 1), 64 * heads, 0, heads=heads)
        else:
            c = _norm8(type, _log(rng, 1, 16384), D, rng.choice(["rms", "layer"]), some[0], some[1], some[2], rng.choice([0, 32, 64, 128]), some[3])
        if work(c)["bytes"] <= most:
            return c


def _tables(c):
    """(values of a row, type) of each table: W1, b1, W2, b2 of the heads, or a convolution's last inputs and a scan's states."""
    if c["heads"]:
        return [(c["heads"] * n, torch.float32) for n in (64 * 256, 256, 256 * 64, 64)]
    return [(3 * c["D"], TYPES[c["type"]]), (c["D"] * c["N"], torch.float32)]


def work(c):
    e = 4 if c["type"] == "fp32" else 2
    if c["op"] == "norm8":
        r = 4 if c["res32"] or c["type"] == "fp32" else 2
        # o, x -> z, and the values that the 8 bits stand for in bf16, as `run` gives them back
        return {"bytes": c["M"] * c["D"] * (e + r * (1 + c["res"]) + 2), "flops": 12 * c["M"] * c["D"]}
    if c["op"] == "saved":      # in 8 bits, and back again
        return {"bytes": 2 * c["tensors"] * c["M"] * (c["D"] * (e + 1) + 4 * -(-c["D"] // c["group"])), "flops": 6 * c["tensors"] * c["M"] * c["D"]}
    if c["op"] == "rows":
        width = sum(n * ty.itemsize for n, ty in _tables(c))
        if c["mode"] == "compact":      # of n rows in use the expected n (S - n) / S are behind the n-th place
            return {"bytes": 2 * width * max(1, c["n"] * (c["S"] - c["n"]) // c["S"]), "flops": 0}
        return {"bytes": width * (1 + c["n"] if c["mode"] == "fork" else c["n"] if c["mode"] == "clear" else 2 * c["n"]), "flops": 0}
    n, train = c["B"] * c["T"] * c["D"], c["mode"] == "train"
    ins = 2 + c["igate"]
    state = c["B"] * c["D"] * 4 * (2 if c["state"] else 0)
    back = e * (1 + ins) + (ins if c["kept"] else e * ins)              # dy and the inputs -> the inputs' gradients
    kept = ins if train and c["kept"] else 0                            # written by the forward pass
    return {"bytes": n * (e * (ins + 1) + kept + train * back) + state * (1 + train) + 12 * c["D"] * (1 + train),
            "flops": n * (20 + 40 * train)}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _acts(g, c, *shape, std=1.0):
    """Activations [..., D]; `wide`: as the first half of a tensor twice as wide, which is how a projection's output is split."""
    *lead, D = shape
    x = torch.randn(*lead, 2 * D if c["wide"] else D, generator=g, device="cuda") * std
    return x.to(TYPES[c["type"]])[..., :D]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda") * std  # noqa: E731
    ty, s = TYPES[c["type"]], dict(c)
    if c["op"] == "norm8":
        M, D = c["M"], c["D"]
        s["o"] = _acts(g, c, M, D, std=1.5) + 0.25
        s["x"] = rnd(M, D, std=2.0).to(torch.float32 if c["res32"] else ty) if c["res"] else None
        s["w"] = 1 + rnd(D, std=0.1)
        s["b"] = rnd(D, std=0.1) if c["bias"] else None
        return s
    if c["op"] == "saved":
        # tokens of different size, as activations have them
        s["xs"] = [_acts(g, c, c["M"], c["D"]) * torch.exp(rnd(c["M"], 1)).to(ty) for _ in range(c["tensors"])]
        return s
    if c["op"] == "rows":
        S, n = c["S"], c["n"]
        s["tables"] = [rnd(S, w).to(t) for w, t in _tables(c)]
        order = torch.randperm(S, generator=g, device="cuda")
        if c["mode"] == "compact":
            s["used"] = torch.zeros(S, dtype=torch.bool, device="cuda")
            s["used"][order[:n]] = True
        else:
            s["source"] = order[:1].expand(n).to(torch.int32).contiguous() if c["mode"] == "fork" else order[:n].to(torch.int32)
            s["target"] = torch.roll(order, -1)[:n].to(torch.int32)       # "permute": most targets are other pairs' sources
            if n > 2:
                s["target"][n // 2] = -1                                  # a padded pair
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
    s["x"] = _acts(g, c, *lead, D)
    s["gate"] = _acts(g, c, *lead, D)
    s["igate"] = _acts(g, c, *lead, D) if c["igate"] else None
    # with the gate wide open a step keeps 0.92 to 0.4 ... 0.999 to 0.992 of a state
    s["A"] = 8 * torch.log(0.9 + 0.099 * torch.rand(D, generator=g, device="cuda")) if c["A"] else None
    s["gb"] = rnd(D, std=0.5) + (0.0 if c["A"] else 2.0) if c["bias"] or not c["A"] else None
    s["ib"] = rnd(D, std=0.5) if c["bias"] and c["igate"] else None
    s["st"] = rnd(c["slots"] or B, D) if c["state"] else None
    if c["mode"] == "train":
        s["gy"] = rnd(B, T, D).to(ty)
        s["gst"] = rnd(B, D) if c["state"] else None
    return s


# ---- plain forms: elementary operations in 32 bits -------------------------------------------------------------------

def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1: runs of twice the length each time."""
    span, T = 1, a.shape[1]
    while span < T:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _eight(x, group):
    """The values that 8 bits stand for, [..., D] in fp32."""
    D = x.shape[-1]
    G = group or D
    v = F.pad(x.float(), (0, -D % G)).unflatten(-1, (-1, G))
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))                           # amax = m 2^e, 0.5 <= m < 1
    scale = (torch.clamp(e - 9 + (m > 0.875).int(), min=-126) + 127 << 23).to(torch.int32).view(torch.float32)      # 2^..., by its exponent
    q = (v / scale).to(torch.float8_e4m3fn).float() * scale
    return q.flatten(-2)[..., :D]


def _factors(s, x, gate, igate, live=None):
    """(a, b, i, sigmoid of the gate, d log a / d gate, slope of b by log a) of every token."""
    v = gate.float() + (s["gb"] if s["gb"] is not None else 0.0)
    sg = _sigmoid(v)
    if s["A"] is not None:
        la = sg * s["A"]
        a, m = torch.exp(la), torch.expm1(la)
        dla = la * _sigmoid(-v)
    else:
        a, m = sg, -_sigmoid(-v)
        dla = -m
    if s["mix"] == "sqrt":
        b = torch.sqrt(-m * (2 + m))
        db = -a * a / b
    else:
        b, db = (-m, -a) if s["mix"] == "linear" else (torch.ones_like(a), torch.zeros_like(a))
    i = _sigmoid(igate.float() + (s["ib"] if s["ib"] is not None else 0.0)) if igate is not None else torch.ones_like(a)
    if live is not None:
        a = torch.where(live, a, 1.0)
    return a, b, i, sg, dla, db


def _live(s):
    if s["lengths"] is None:
        return None
    return (torch.arange(s["T"], device="cuda") < s["lengths"][:, None])[..., None]


def _only(live, v):
    return v if live is None else torch.where(live, v, 0.0)


def _gated_plain(s):
    ty, live = TYPES[s["type"]], _live(s)
    x, gate, igate = s["x"].float(), s["gate"], s["igate"]
    a, b, i, sg, dla, db = _factors(s, x, gate, igate, live)
    u = _only(live, b * i * x)
    if s["st"] is not None:
        u[:, 0] += a[:, 0] * s["st"]
    h = _recur(a, u)
    out = {"y": _only(live, h).to(ty)}
    if s["state"]:
        out["state"] = h[:, -1].clone()
    if s["mode"] != "train":
        return out
    first = s["st"][:, None] if s["st"] is not None else torch.zeros_like(h[:, :1])
    before = torch.cat([first, h[:, :-1]], 1)                                    # states in front of the tokens
    if s["kept"]:
        x = _eight(s["x"], s["kept"])
        a, b, i, sg, dla, db = _factors(s, x, _eight(gate, s["kept"]), _eight(igate, s["kept"]) if igate is not None else None, live)
        start = (torch.arange(s["T"], device="cuda") % EVERY == 0)[:, None]
        h = _recur(torch.where(start, 0.0, a), _only(live, b * i * x) + torch.where(start, a * before, 0.0))
        before = torch.where(start, before, torch.cat([first, h[:, :-1]], 1))
    G = _only(live, s["gy"].float())
    if s["gst"] is not None:
        G[:, -1] += s["gst"]
    # backwards in time the factor of a step is the next one's
    after = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    G = _recur(after, G.flip(1)).flip(1)
    dlog = G * (a * before + i * x * db)
    dv = _only(live, dlog * dla)
    out["grad_x"] = _only(live, G * b * i).to(ty)
    out["grad_gate"] = dv.to(ty)
    if s["A"] is not None:
        out["grad_A"] = _only(live, dlog * sg).sum((0, 1))
    if s["gb"] is not None:
        out["grad_gate_bias"] = dv.sum((0, 1))
    if igate is not None:
        di = _only(live, G * b * x * i * (1 - i))
        out["grad_igate"] = di.to(ty)
        if s["ib"] is not None:
            out["grad_input_bias"] = di.sum((0, 1))
    if s["st"] is not None:
        out["grad_state"] = G[:, 0] * a[:, 0]
    return out


def _gated_step_plain(s):
    at = s["index"].long()
    live = at >= 0
    at = at[live]
    x = s["x"][live].float()
    a, b, i, *_ = _factors(s, x, s["gate"][live], s["igate"][live] if s["igate"] is not None else None)
    h = a * s["st"][at] + b * i * x
    y = torch.zeros(s["B"], s["D"], device="cuda", dtype=TYPES[s["type"]])
    y[live] = h.to(y.dtype)
    s["st"][at] = h
    return {"y": y, "state": s["st"]}


def _rows_plain(s):
    if s["mode"] == "compact":
        at = torch.arange(s["S"], device="cuda")
        front = at < s["used"].sum()
        target, source = at[front & ~s["used"]], at[~front & s["used"]]
        place = torch.where(s["used"], at, -1)
        place[source] = target
    else:
        ok = s["target"] >= 0
        source, target = s["source"][ok].long(), s["target"][ok].long()
    for t in s["tables"]:
        if s["mode"] == "clear":
            t[target] = 0.0
        else:
            t[target] = t[source]
    out = {"table%d" % k: t for k, t in enumerate(s["tables"])}
    if s["mode"] == "compact":
        out["place"] = place.to(torch.int32)
    return out


def _norm8_plain(s):
    z = s["o"].float()
    if s["x"] is not None:
        z = z + s["x"].float()
    out = {"x": z.to(s["x"].dtype if s["x"] is not None else s["o"].dtype)}
    if s["norm"] == "layer":
        z = z - z.mean(-1, keepdim=True)
    n = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * s["w"]
    out["n"] = _eight(n + s["b"] if s["b"] is not None else n, s["group"]).bfloat16()
    return out


def _plain(s):
    if s["op"] == "norm8":
        return _norm8_plain(s)
    if s["op"] == "rows":
        return _rows_plain(s)
    if s["op"] == "saved":
        return [_eight(x, s["group"]).to(x.dtype) for x in s["xs"]]
    return _gated_step_plain(s) if s["mode"] == "step" else _gated_plain(s)


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _own(s):
    if s["op"] == "norm8":
        from ttt_tk_b200.glue import norm_residual_8bit
        from ttt_tk_b200.saved import unpack8
        x, q, scales = norm_residual_8bit(s["o"], s["x"], weight=s["w"], bias=s["b"], norm=s["norm"], group=s["group"] or None, eps=EPS)
        return {"x": x, "n": unpack8((q, scales), dtype=torch.bfloat16)[0]}
    if s["op"] == "rows":
        from ttt_tk_b200 import tables
        out = {"table%d" % k: t for k, t in enumerate(s["tables"])}
        if s["mode"] == "compact":
            out["place"] = tables.compact_rows(s["tables"], s["used"])
        elif s["mode"] == "clear":
            tables.clear_rows(s["tables"], s["target"])
        else:
            tables.copy_rows(s["tables"], s["source"], s["target"])
        return out
    if s["op"] == "saved":
        from ttt_tk_b200 import saved
        return saved.unpack8(*saved.pack8(*s["xs"], group=s["group"]), dtype=TYPES[s["type"]])
    from ttt_tk_b200 import ssm
    mix = None if s["mix"] == "none" else s["mix"]
    args = (s["A"], s["igate"], s["gb"], s["ib"])
    if s["mode"] == "step":
        return {"y": ssm.gated_scan_step(s["x"], s["gate"], s["st"], *args, mix=mix, slots=s["index"]), "state": s["st"]}
    train = s["mode"] == "train"
    r = ssm.gated_scan(s["x"], s["gate"], *args, mix=mix, state=s["st"], lengths=s["lengths"], return_state=s["state"], return_checkpoints=train)
    r = list(r) if isinstance(r, tuple) else [r]
    out = {"y": r[0]}
    if s["state"]:
        out["state"] = r[1]
    if not train:
        return out
    x, gate, igate = s["x"], s["gate"], s["igate"]
    if s["kept"]:
        from ttt_tk_b200 import saved
        x, gate, igate = (saved.pack8(*[t for t in (x, gate, igate) if t is not None], group=s["kept"]) + [None])[:3]
    g = ssm.gated_scan_backward(s["gy"], x, gate, r[-1], s["A"], igate, s["gb"], s["ib"], mix=mix, lengths=s["lengths"],
                                grad_final_state=s["gst"])
    names = ("grad_x", "grad_gate", "grad_A", "grad_igate", "grad_gate_bias", "grad_input_bias", "grad_state" if s["state"] else None)
    out.update({k: v for k, v in zip(names, g) if k and v is not None})
    return out


def run(s):
    return _own(s) if own else _plain(s)


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------

def _two(k):
    """2^k, exactly."""
    return (k.long() + 1023 << 52).view(torch.float64)


def _exact_eight(v, group):
    """Group by group, from the definition of the format: 3 bits behind the leading one, the least exponent -6."""
    D = v.shape[-1]
    G = group or D
    out = torch.empty_like(v)
    for d in range(0, D, G):
        p = v[..., d:d + G]
        top = p.abs().amax(-1, keepdim=True)
        k = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448))
        k = torch.where(224 * _two(k) >= top, k - 1, k)      # the logarithm may be off by its last bit
        k = torch.where(448 * _two(k) < top, k + 1, k)
        k = torch.clamp(k, min=-126)
        p = p * _two(-k)
        step = torch.clamp(torch.frexp(p)[1] - 1, min=-6) - 3
        out[..., d:d + G] = torch.round(p * _two(-step)) * _two(step) * _two(k)
    return out


def _exact_gated(s):
    B, T, D = s["B"], s["T"], s["D"]
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    n = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    all_live = min(n) == T
    live = torch.arange(T, device="cuda")[None] < torch.tensor(n, device="cuda")[:, None]

    def leaves(kept):
        """Inputs as doubles that gradients are asked of: the activations as they are or as they were kept."""
        f = (lambda t: _exact_eight(t.double(), s["kept"])) if kept else (lambda t: t.double())
        lv = {k: f(s[k]) for k in ("x", "gate", "igate") if s[k] is not None}
        lv.update({k: s[k].double() for k in ("A", "gb", "ib") if s[k] is not None})
        return {k: v.detach().requires_grad_(True) for k, v in lv.items()}

    def tokens(lv):
        """(a, u) of all tokens."""
        v = lv["gate"] + lv.get("gb", zero)
        if "A" in lv:
            la = lv["A"] * torch.sigmoid(v)
            a = torch.exp(la)
            w = -torch.expm1(2 * la)
            lin = -torch.expm1(la)
        else:
            a = torch.sigmoid(v)
            lin = torch.sigmoid(-v)
            w = lin * (1 + a)
        u = lv["x"] * (torch.sqrt(w) if s["mix"] == "sqrt" else lin if s["mix"] == "linear" else 1.0)
        if "igate" in lv:
            u = u * torch.sigmoid(lv["igate"] + lv.get("ib", zero))
        return a, u

    def walk(a, u, h, starts=None):
        """Token by token; `starts`: the states that every EVERY-th token starts from instead."""
        before, after = torch.empty_like(a), torch.empty_like(a)
        for t in range(T):
            if starts is not None and t % EVERY == 0:
                h = starts[:, t]
            before[:, t] = h
            new = torch.addcmul(u[:, t], a[:, t], h)
            h = new if all_live else torch.where(live[:, t, None], new, h)
            after[:, t] = h
        return before, after, h

    h0 = s["st"].double() if s["st"] is not None else torch.zeros(B, D, dtype=torch.float64, device="cuda")
    with torch.no_grad():
        before, after, end = walk(*tokens(leaves(False)), h0)
    out = {"y": torch.where(live[..., None], after, 0.0)}
    if s["state"]:
        out["state"] = end
    if s["mode"] != "train":
        return out
    del after
    lv = leaves(bool(s["kept"]))
    a, u = tokens(lv)
    if s["kept"]:
        with torch.no_grad():
            before, _, _ = walk(a.detach(), u.detach(), h0, before)
    # L = sum_t G_t (a_t before_t + u_t) has the gradients of the whole sequence with G, before held
    G = torch.zeros_like(before)
    carry = s["gst"].double() if s["gst"] is not None else torch.zeros(B, D, dtype=torch.float64, device="cuda")
    ad = a.detach()
    for t in reversed(range(T)):
        g = s["gy"][:, t].double() + carry
        if all_live:
            G[:, t], carry = g, ad[:, t] * g
        else:
            on = live[:, t, None]
            G[:, t] = torch.where(on, g, 0.0)
            carry = torch.where(on, ad[:, t] * g, carry)
    keys = list(lv)
    for k, v in zip(keys, torch.autograd.grad([a, u], [lv[k] for k in keys], [G * before, G])):
        out[{"x": "grad_x", "gate": "grad_gate", "igate": "grad_igate", "A": "grad_A", "gb": "grad_gate_bias", "ib": "grad_input_bias"}[k]] = v
    if s["st"] is not None:
        out["grad_state"] = carry
    return out


def _exact_step(s):
    y = torch.zeros(s["B"], s["D"], dtype=torch.float64, device="cuda")
    st = s["st"].double()
    for r, at in enumerate(s["index"].tolist()):
        if at < 0:
            continue
        v = s["gate"][r].double() + (s["gb"].double() if s["gb"] is not None else 0.0)
        la = s["A"].double() * torch.sigmoid(v) if s["A"] is not None else F.logsigmoid(v)
        u = s["x"][r].double()
        if s["mix"] != "none":
            u = u * (torch.sqrt(-torch.expm1(2 * la)) if s["mix"] == "sqrt" else -torch.expm1(la))
        if s["igate"] is not None:
            u = u * torch.sigmoid(s["igate"][r].double() + (s["ib"].double() if s["ib"] is not None else 0.0))
        y[r] = st[at] = torch.exp(la) * st[at] + u
    return {"y": y, "state": st}


def _exact_rows(s):
    if s["mode"] == "compact":
        used = s["used"].tolist()
        n = sum(used)
        free = [k for k in range(n) if not used[k]]
        late = [k for k in range(n, s["S"]) if used[k]]
        place = [k if used[k] else -1 for k in range(s["S"])]
        pairs = list(zip(late, free))
        for k, to in pairs:
            place[k] = to
    else:
        pairs = [(a, b) for a, b in zip(s["source"].tolist(), s["target"].tolist()) if b >= 0]
    out = {}
    for k, t in enumerate(s["tables"]):
        d = t.double()
        for a, b in pairs:
            d[b] = 0.0 if s["mode"] == "clear" else t[a].double()
        out["table%d" % k] = d
    if s["mode"] == "compact":
        out["place"] = torch.tensor(place, dtype=torch.int32, device="cuda")
    return out


def _exact_norm8(s):
    z = s["o"].double() + (s["x"].double() if s["x"] is not None else 0.0)
    w, b = s["w"].double(), s["b"].double() if s["b"] is not None else None
    D = (s["D"],)
    n = F.layer_norm(z, D, w, b, EPS) if s["norm"] == "layer" else F.rms_norm(z, D, w, EPS) + (b if b is not None else 0.0)
    return {"x": z, "n": _exact_eight(n, s["group"])}


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "saved":
        return [_exact_eight(x.double(), s["group"]) for x in s["xs"]]
    if c["op"] == "rows":
        return _exact_rows(s)
    if c["op"] == "norm8":
        return _exact_norm8(s)
    if c["mode"] == "step":
        return _exact_step(s)
    with torch.enable_grad():
        out = _exact_gated(s)
    return {k: v.detach() for k, v in out.items()}
