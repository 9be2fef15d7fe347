"""CPU statement (test infrastructure: only tests may import this) of the gated linear recurrence, forward and backward, in 64 bits and
token by token.  The reference contains no code for it; what is stated here is the definition the CUDA kernels are held to.

Every function returns its values and, of each, the error that fp32 arithmetic between reading and writing may leave, in units of 2^-24.  The
errors are carried through the formulas beside the values: a factor with a relative error of k units leaves k times the product's magnitude, a sum
its terms' errors, and each operation half a step, counted as one unit.  What single steps have:

  v = gate + bias       |v| / 2 of the sum and as much of the product with log2 e, whose effect on sigmoid(v) or 1 - sigmoid(v) is at most as large;
  s, 1 - s              2 |v| + 10: exponential and reciprocal four each (2^-22), a sum and a product
  log a = A s           that and 1 more
  a = exp(log a)        |log a| times that, and 4 for the series;  without A as s
  1 - a                 as log a (its relative slope is at most one) and 4
  sqrt(1 - a^2)         1 - a's and 7: half of twice that, of a reciprocal root (4) and two products

What fp32 has no normal number for counts as 0: a below 2^-126 (NONE, in units), and what is said at `least`.
"""
import torch

EVERY = 64
NONE = 2.0 ** -102


def _d(t):
    return None if t is None else t.detach().double().cpu()


def lengths_of(lengths, B, T):
    return torch.full((B,), T) if lengths is None else lengths.detach().cpu().long().clamp(0, T)


def _sigmoid(v):
    """(sigmoid, 1 - sigmoid)"""
    return 1 / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v))


class _Factors:
    def __init__(self, gate, A, input_gate, gate_bias, input_bias, mix):
        v = _d(gate) + (_d(gate_bias) if gate_bias is not None else 0.0)
        self.s, self.other = _sigmoid(v)
        self.ks = 2 * v.abs().clamp(max=130) + 10
        if A is not None:
            self.A = _d(A).clamp(max=0.0)
            la = self.A * self.s
            self.a, m = torch.exp(la), torch.expm1(la)
            kla = self.ks + 1
            self.ka = la.abs().clamp(max=90) * kla + 4
            km = kla + 4
            self.k, self.kk = la * self.other, kla + self.ks + 1       # d log a / d gate
        else:
            self.A = None
            self.a, m = self.s, -self.other
            self.ka, km = self.ks, self.ks
            self.k, self.kk = self.other, self.ks
        if mix == "sqrt":
            w = -m * (2 + m)
            self.b = torch.sqrt(w)
            self.kb = km + 7
            self.db = torch.where(w > 0, -self.a * self.a / torch.where(w > 0, self.b, 1.0), 0.0)
            self.kdb = 2 * self.ka + self.kb + 3
        elif mix == "linear":
            self.b, self.kb, self.db, self.kdb = -m, km, -self.a, self.ka
        else:
            self.b, self.kb = torch.ones_like(m), torch.zeros_like(m)
            self.db, self.kdb = torch.zeros_like(m), torch.zeros_like(m)
        if input_gate is not None:
            vi = _d(input_gate) + (_d(input_bias) if input_bias is not None else 0.0)
            self.i, self.rest = _sigmoid(vi)
            self.ki = 2 * vi.abs().clamp(max=130) + 10
        else:
            self.i, self.rest, self.ki = torch.ones_like(m), torch.zeros_like(m), torch.zeros_like(m)
        self.w, self.kw = self.b * self.i, self.kb + self.ki + 1
        # below 2^-126 fp32 has no 1 - a^2 (and no sigmoid below 2^-127, which A enlarges): b is 0 where it is less than this
        self.least = 2.0 ** -62 / 2.0 ** -24 * (1 if self.A is None else (1 - self.A) ** 0.5) if mix == "sqrt" else 2.0 ** -120


def states(x, f, state, n, starts=None):
    """(states in front of each token, behind each token, last state), each with its error; a token joins a few steps of a tree more."""
    x = _d(x)
    B, T, D = x.shape
    h = _d(state) if state is not None else torch.zeros(B, D, dtype=torch.float64)
    e = torch.zeros_like(h)
    before, after, eb, ea = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    for t in range(T):
        if starts is not None and t % EVERY == 0:
            h, e = starts[0][:, t], starts[1][:, t]
        on = (t < n)[:, None]
        before[:, t], eb[:, t] = h, e
        xt = torch.where(on, x[:, t], 0.0)
        u = f.w[:, t] * xt
        new = f.a[:, t] * h + u
        # 4 more to a factor a: products of factors over tokens, and the joins
        enew = f.a[:, t] * e + (f.a[:, t] * h).abs() * (f.ka[:, t] + 4) + u.abs() * (f.kw[:, t] + 2) + (f.i[:, t] * xt).abs() * f.least + h.abs() * NONE + new.abs()
        h, e = torch.where(on, new, h), torch.where(on, enew, e)
        after[:, t], ea[:, t] = torch.where(on, h, 0.0), torch.where(on, e, 0.0)
    return (before, eb), (after, ea), (h, e)


def gated_scan(x, gate, A=None, input_gate=None, gate_bias=None, input_bias=None, mix="sqrt", state=None, lengths=None):
    """(y, its error), (final state, its error), (states in front of each token, their error)"""
    f = _Factors(gate, A, input_gate, gate_bias, input_bias, mix)
    before, after, end = states(x, f, state, lengths_of(lengths, *x.shape[:2]))
    return after, end, before


def gated_scan_backward(grad_y, x, gate, before, A=None, input_gate=None, gate_bias=None, input_bias=None, mix="sqrt", lengths=None,
                        grad_final_state=None):
    """{name: (gradient, its error)}; `before`: the states in front of the tokens, of which every 64th counts (the others are computed
    again, from the inputs given here)."""
    f = _Factors(gate, A, input_gate, gate_bias, input_bias, mix)
    x, gy = _d(x), _d(grad_y)
    B, T, D = x.shape
    n = lengths_of(lengths, B, T)
    live = (torch.arange(T)[None] < n[:, None])[..., None]
    x, gy = torch.where(live, x, 0.0), torch.where(live, gy, 0.0)
    (h, eh), _, _ = states(x, f, None, n, before)
    c = _d(grad_final_state) if grad_final_state is not None else torch.zeros(B, D, dtype=torch.float64)
    ec = torch.zeros_like(c)
    G, eG = torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(range(T)):
        on = (t < n)[:, None]
        g = gy[:, t] + c
        eg = ec + g.abs()
        G[:, t], eG[:, t] = torch.where(on, g, 0.0), torch.where(on, eg, 0.0)
        c, ec = torch.where(on, f.a[:, t] * g, c), torch.where(on, f.a[:, t] * eg + (f.a[:, t] * g).abs() * (f.ka[:, t] + 5), ec)
    ah, ix = f.a * h, f.i * x * f.db
    q = ah + ix
    eq = f.a * eh + ah.abs() * (f.ka + 2) + ix.abs() * (f.kdb + f.ki + 3) + (h.abs() + (f.i * x).abs()) * NONE
    dl = torch.where(live, G * q, 0.0)
    el = eG * q.abs() + G.abs() * eq + dl.abs()
    # the slope's term where b is 0 in fp32: k db and s db are below this times G i x
    el_floor = (G * f.i * x).abs() * f.least
    out = {"x": (G * f.w, eG * f.w.abs() + (G * f.w).abs() * (f.kw + 1) + G.abs() * f.i * f.least)}
    dg = dl * f.k
    out["gate"] = (dg, el * f.k.abs() + dg.abs() * (f.kk + 1) + el_floor)
    xr = f.w * x * f.rest
    di = G * xr
    if input_gate is not None:
        out["input_gate"] = (di, eG * xr.abs() + di.abs() * (f.kw + f.ki + 4) + el_floor)
    adds = T / 4 + 64 + B      # of a sum in a row, at most

    def total(v, e):
        v, e = torch.where(live, v, 0.0), torch.where(live, e, 0.0)
        return v.sum((0, 1)), e.sum((0, 1)) + adds * v.abs().sum((0, 1))

    if A is not None:
        v, e = total(dl * f.s, el * f.s + (dl * f.s).abs() * (f.ks + 1) + el_floor)
        up = _d(A) > 0
        out["A"] = (torch.where(up, 0.0, v), e)
    if gate_bias is not None:
        out["gate_bias"] = total(*out["gate"])
    if input_bias is not None:
        out["input_bias"] = total(*out["input_gate"])
    out = {k: (torch.where(live, v, 0.0), torch.where(live, e, 0.0)) if v.dim() == 3 else (v, e) for k, (v, e) in out.items()}
    out["state"] = (c, ec)
    return out


def e4m3(v, group):
    """The values that 8 bits stand for: of each `group` neighbours of a row, the least power of two `scale` with max |v| <= 448 scale, and v / scale
    rounded to 4 significant bits (below 2^-6 to multiples of 2^-9), ties to even.  [..., D] -> (values, scales [..., ceil(D / group)]).
    Infinities are out of the maximum and become 448 scale; NaN stays."""
    v = _d(v)
    D = v.shape[-1]
    group = group or D
    pad = torch.nn.functional.pad(v, (0, -D % group)).unflatten(-1, (-1, group))
    top = torch.where(pad.isfinite(), pad.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    k = torch.where(top > 0, e - 9 + (m > 0.875).int(), -126).clamp(min=-126)
    scale = torch.exp2(k.double())
    p = pad / scale
    step = torch.exp2((torch.frexp(p)[1] - 1).clamp(min=-6, max=8).double() - 3)
    q = (torch.round(p / step) * step).clamp(-448, 448) * scale
    return q.flatten(-2)[..., :D], scale.squeeze(-1)
