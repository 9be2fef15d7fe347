"""CPU statements (test infrastructure: only tests may import this) of the layer-side sequence operators: the short causal
convolution, the selective state space scan and the block end, forward and backward, in 64 bits and token by token.  The
reference contains no code for them; what is stated here is the definition the CUDA kernels are held to.

Each function takes `amp`: with it every term enters with its absolute value, so that the result is the sum of the magnitudes whose
rounding errors an fp32 computation can carry: what an absolute tolerance is proportional to.

The backward functions are the formulas by hand; tests hold them to autograd and to differences of the forward ones.
"""
import math

import torch


def _d(t, amp=False):
    if t is None:
        return None
    t = t.detach().double().cpu()
    return t.abs() if amp else t


def sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def activation(name, v):
    """(value, slope)"""
    if name is None:
        return v, torch.ones_like(v)
    s = sigmoid(v)
    if name == "sigmoid":
        return s, s * (1 - s)
    if name == "silu":
        return v * s, s * (1 + v * (1 - s))
    k, c = math.sqrt(2 / math.pi), 0.044715
    # (1 + tanh(u)) / 2 as sigmoid(2 u): far on the left 1 + tanh(u) is 0 even in 64 bits
    s, o = sigmoid(2 * k * (v + c * v ** 3)), sigmoid(-2 * k * (v + c * v ** 3))
    return v * s, s + v * s * o * 2 * k * (1 + 3 * c * v * v)


def softplus(v):
    return torch.where(v > 0, v, 0.0) + torch.log1p(torch.exp(-v.abs()))


def _lengths(lengths, B, T):
    return [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]


# ---- short convolution: x [B, T, D], weight [D, K], state [B, K - 1, D] --------------------------------------------------
def short_conv(x, weight, bias=None, activation_=None, state=None, lengths=None, amp=False):
    """(y, final state)"""
    x, w, bias, state = (_d(t, amp) for t in (x, weight, bias, state))
    B, T, D = x.shape
    K = w.shape[1]
    y, end = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, K - 1, D, dtype=torch.float64)
    for b, n in enumerate(_lengths(lengths, B, T)):
        row = torch.cat([state[b] if state is not None else torch.zeros(K - 1, D, dtype=torch.float64), x[b, :n]])
        for t in range(n):
            pre = (row[t:t + K] * w.t()).sum(0) + (bias if bias is not None else 0.0)
            y[b, t] = pre if amp else activation(activation_, pre)[0]
        end[b] = row[n:n + K - 1]
    return y, end


def short_conv_backward(grad_y, x, weight, bias=None, activation_=None, state=None, lengths=None, grad_final_state=None, amp=False):
    """(grad_x, grad_weight, grad_bias, grad_state); with `amp` the slope of silu counts as 1.1, its largest value"""
    gy, gf = _d(grad_y, amp), _d(grad_final_state, amp)
    xr, wr, br, sr = (_d(t) for t in (x, weight, bias, state))
    x, w, state = (_d(t, amp) for t in (x, weight, state))
    B, T, D = x.shape
    K = w.shape[1]
    gx, gs = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, K - 1, D, dtype=torch.float64)
    gw, gb = torch.zeros(D, K, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    for b, n in enumerate(_lengths(lengths, B, T)):
        none = torch.zeros(K - 1, D, dtype=torch.float64)
        real = torch.cat([sr[b] if sr is not None else none, xr[b, :n]])
        row = torch.cat([state[b] if state is not None else none, x[b, :n]])
        grow = torch.zeros_like(row)
        for t in range(n):
            pre = (real[t:t + K] * wr.t()).sum(0) + (br if br is not None else 0.0)
            g = gy[b, t] * (1.1 if amp and activation_ else activation(activation_, pre)[1])
            grow[t:t + K] += g * w.t()
            gw += (g * row[t:t + K]).t()
            gb += g
        if gf is not None:
            grow[n:] += gf[b]
        gx[b, :n], gs[b] = grow[K - 1:], grow[:K - 1]
    return gx, gw, gb, gs


# ---- state space scan: x, dt [B, T, D], A [D, N], B, C [B, T, G, N] -------------------------------------------------------
def _scan_terms(x, dt, A, Bm, Cm, Dk, dt_bias, softplus_, amp):
    x, Bm, Cm, Dk = (_d(t, amp) for t in (x, Bm, Cm, Dk))
    A, v = _d(A), _d(dt)
    D = x.shape[-1]
    v = v + (_d(dt_bias) if dt_bias is not None else 0.0)
    delta = softplus(v) if softplus_ else v
    slope = sigmoid(v) if softplus_ else torch.ones_like(v)
    spread = lambda m: m.repeat_interleave(D // m.shape[-2], -2)  # noqa: E731
    return x, delta, slope, A, spread(Bm), spread(Cm), Dk if Dk is not None else torch.zeros(D, dtype=torch.float64)


def ssm_scan(x, dt, A, Bm, Cm, D=None, dt_bias=None, softplus_=True, state=None, lengths=None, amp=False):
    """(y, final state, states [B, T + 1, D, N] before each token and behind the last)"""
    x, delta, _, A, Bm, Cm, Dk = _scan_terms(x, dt, A, Bm, Cm, D, dt_bias, softplus_, amp)
    B, T, Dn = x.shape
    N = A.shape[1]
    dabs = delta.abs() if amp else delta
    h = _d(state, amp) if state is not None else torch.zeros(B, Dn, N, dtype=torch.float64)
    n = torch.tensor(_lengths(lengths, B, T))
    y, hs = torch.zeros(B, T, Dn, dtype=torch.float64), [h]
    for t in range(T):
        on = (t < n)[:, None]
        new = torch.exp(delta[:, t, :, None] * A) * h + (dabs[:, t] * x[:, t])[..., None] * Bm[:, t]
        new, xt = torch.where(on[..., None], new, h), torch.where(on, x[:, t], 0.0)
        y[:, t] = torch.where(on, (torch.where(on[..., None], new * Cm[:, t], 0.0)).sum(-1) + Dk * xt, 0.0)
        h = new
        hs.append(h)
    return y, h, torch.stack(hs, 1)


def ssm_scan_backward(grad_y, x, dt, A, Bm, Cm, D=None, dt_bias=None, softplus_=True, state=None, lengths=None,
                      grad_final_state=None, amp=False):
    """(grad_x, grad_dt, grad_A, grad_B, grad_C, grad_D, grad_dt_bias, grad_state)"""
    G = Bm.shape[-2]
    _, _, hs = ssm_scan(x, dt, A, Bm, Cm, D, dt_bias, softplus_, state, lengths, amp)
    x, delta, slope, A, Bm, Cm, Dk = _scan_terms(x, dt, A, Bm, Cm, D, dt_bias, softplus_, amp)
    gy = _d(grad_y, amp)
    B, T, Dn = x.shape
    N = A.shape[1]
    Aa, dabs = (A.abs(), delta.abs()) if amp else (A, delta)
    n = torch.tensor(_lengths(lengths, B, T))
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    gx, gdt, gB, gC = z(B, T, Dn), z(B, T, Dn), z(B, T, Dn, N), z(B, T, Dn, N)
    gA, gD, gb = z(Dn, N), z(Dn), z(Dn)
    carry = _d(grad_final_state, amp) if grad_final_state is not None else z(B, Dn, N)
    on = torch.arange(T) < n[:, None]                  # behind a sequence everything is zero: exp(0) = 1, and no terms
    keep = lambda v: torch.where(on[(...,) + (None,) * (v.dim() - 2)], v, 0.0)  # noqa: E731
    x, delta, dabs, slope, gy, Bm, Cm = (keep(v) for v in (x, delta, dabs, slope, gy, Bm, Cm))
    for t in reversed(range(T)):
        a = torch.exp(delta[:, t, :, None] * A)
        g = gy[:, t, :, None] * Cm[:, t] + carry
        gC[:, t] = gy[:, t, :, None] * hs[:, t + 1]
        gB[:, t] = g * (dabs[:, t] * x[:, t])[..., None]
        dB = (g * Bm[:, t]).sum(-1)
        q = g * a * hs[:, t]
        gA += (q * dabs[:, t, :, None]).sum(0)
        gx[:, t] = dabs[:, t] * dB + Dk * gy[:, t]
        gdt[:, t] = ((q * Aa).sum(-1) + x[:, t] * dB) * slope[:, t]
        gb += gdt[:, t].sum(0)
        gD += (gy[:, t] * x[:, t]).sum(0)
        carry = a * g
    fold = lambda v: v.unflatten(2, (G, Dn // G)).sum(3)  # noqa: E731
    return gx, gdt, gA, fold(gB), fold(gC), gD, gb, carry


# ---- block end: o, residual, gate [M, D] -------------------------------------------------------------------------------------
def _norm(v, layer, eps):
    if layer:
        v = v - v.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    return v * r, r


def norm_gate_residual(o, residual=None, gate=None, norm="rms", activation_="silu", post_weight=None, post_bias=None, scale=None,
                       pre_weight=None, pre_bias=None, eps=1e-6):
    """(x, n or None)"""
    o, residual, gate, w1, b1, sc, w2, b2 = (_d(t) for t in (o, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias))
    layer = norm == "layer"
    v = o
    if w1 is not None:
        v = _norm(o, layer, eps)[0] * w1 + (b1 if b1 is not None else 0.0)
    if gate is not None:
        v = v * activation(activation_, gate)[0]
    x = (v if sc is None else sc * v) + (residual if residual is not None else 0.0)
    return x, None if w2 is None else _norm(x, layer, eps)[0] * w2 + (b2 if b2 is not None else 0.0)


def norm_gate_residual_backward(grad_x, grad_n, o, residual=None, gate=None, norm="rms", activation_="silu", post_weight=None,
                                post_bias=None, scale=None, pre_weight=None, pre_bias=None, eps=1e-6, amp=False):
    """(grad_o, grad_residual, grad_gate, grad_post_weight, grad_post_bias, grad_scale, grad_pre_weight, grad_pre_bias)"""
    grad_x, grad_n, o, residual, gate, w1, b1, sc, w2, b2 = (
        _d(t) for t in (grad_x, grad_n, o, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias))
    layer = norm == "layer"
    m = (lambda t: t.abs()) if amp else (lambda t: t)
    sign = 1.0 if amp else -1.0
    zero = torch.zeros_like(o)
    oh, r1 = _norm(o, layer, eps) if w1 is not None else (o, None)
    u = oh * w1 + (b1 if b1 is not None else 0.0) if w1 is not None else o
    gv, gs = activation(activation_, gate) if gate is not None else (torch.ones_like(o), zero)
    s = sc if sc is not None else torch.ones(o.shape[-1], dtype=torch.float64)
    z = s * u * gv + (residual if residual is not None else 0.0)

    def back(g, h, r):
        out = g + sign * m(h) * (g * m(h)).mean(-1, keepdim=True)
        return r * (out + sign * g.mean(-1, keepdim=True) if layer else out)

    d = m(grad_x) if grad_x is not None else zero
    g2 = gb2 = None
    if w2 is not None:
        zh, r2 = _norm(z, layer, eps)
        gn = m(grad_n) if grad_n is not None else zero
        d = d + back(gn * m(w2), zh, r2)
        g2, gb2 = (gn * m(zh)).sum(0), gn.sum(0)
    # u is a sum itself: worked out with an error of half a step of |oh w1| + |b1|, however near to zero it comes, so these are its
    # magnitudes (u = 9.7e-7 of two terms of 0.08 is off by up to 2^-24 0.16 / 9.7e-7 = 1 %)
    ua = (m(oh) * m(w1) + (m(b1) if b1 is not None else 0.0) if w1 is not None else m(o)) if amp else u
    gsc = (d * m(ua * gv)).sum(0)
    dv = d * m(s)
    gg = dv * m(ua * gs)
    du = dv * m(gv)
    g1 = gb1 = None
    go = du
    if w1 is not None:
        g1, gb1 = (du * m(oh)).sum(0), du.sum(0)
        go = back(du * m(w1), oh, r1)
    return (go, d if residual is not None else None, gg if gate is not None else None, g1, gb1 if b1 is not None else None,
            gsc if sc is not None else None, g2, gb2 if b2 is not None else None)
