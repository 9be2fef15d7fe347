"""`torch.autograd.Function` around the operator pair, with the buffer handling the raw API leaves
to its callers (the reference ships only the two functions, README.md:22-96): checkpoints and
scratch are allocated once per shape and reused, the per-batch norm-gradient rows are summed, and
the state after the last mini-batch is returned so that sequences can be processed in chunks.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from .buffers import GRAD_NAMES, alloc_backward_buffers, alloc_checkpoints
from .ops import ttt_backward, ttt_forward

# One scratch set per (shape, device, CUDA stream): backward passes on the same stream are ordered and may
# share it (its contents mean nothing between calls); passes on different streams could overlap on the
# GPU and get their own.
_scratch_cache = {}


def _scratch(B, H, NC, cgs, device):
    key = (B, H, cgs, device.index, torch._C._cuda_getCurrentRawStream(device.index))
    if key not in _scratch_cache:
        _scratch_cache[key] = alloc_backward_buffers(B, H, 1, cgs, device)[0]
    return _scratch_cache[key]


class TTTMLPFunction(torch.autograd.Function):
    """(XQW, W1_last, b1_last, W2_last, b2_last) = f(XQ, XK, XV, last_eta, norm_weight, norm_bias,
    W1, b1, W2, b2, checkpoint_group_size).  Tensors as in `ttt_forward`."""

    @staticmethod
    def forward(ctx, XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, W2, b2, checkpoint_group_size):
        B, H, NC = XQ.shape[:3]
        cgs = int(checkpoint_group_size)
        dev = XQ.device
        args = [t.contiguous() for t in (XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, W2, b2)]
        ck = alloc_checkpoints(B, H, NC, cgs, dev)
        out = torch.empty_like(args[0])
        final = tuple(torch.empty_like(t) for t in args[6:10])
        ttt_forward(*args, *ck, out, cgs, final_state=final)
        ctx.save_for_backward(*args[:6], *ck, out)
        ctx.cgs = cgs
        ctx.eta_shape = last_eta.shape
        return (out,) + final

    @staticmethod
    def backward(ctx, g_out, g_W1, g_b1, g_W2, g_b2):
        saved = ctx.saved_tensors
        XQ, XK, XV, last_eta, gamma, beta = saved[:6]
        ck, out = saved[6:10], saved[10]
        B, H, NC = XQ.shape[:3]
        cgs, dev = ctx.cgs, XQ.device
        zeros = lambda ref, g: torch.zeros_like(ref) if g is None else g.contiguous().to(torch.float32)
        g_W1 = zeros(ck[0][:, :, 0], g_W1)
        g_b1 = zeros(ck[1][:, :, 0], g_b1)
        g_W2 = zeros(ck[2][:, :, 0], g_W2)
        g_b2 = zeros(ck[3][:, :, 0], g_b2)
        g_out = torch.zeros_like(XQ) if g_out is None else g_out.contiguous().to(torch.bfloat16)
        scratch = _scratch(B, H, NC, cgs, dev)
        bf, f32 = torch.bfloat16, torch.float32
        o = {
            "grad_L_ttt_norm_weight": torch.empty(B, H, 1, 64, dtype=f32, device=dev),
            "grad_L_ttt_norm_bias": torch.empty(B, H, 1, 64, dtype=f32, device=dev),
            "grad_L_W1_init": torch.empty(B, H, 64, 256, dtype=f32, device=dev),
            "grad_L_b1_init": torch.empty(B, H, 1, 256, dtype=f32, device=dev),
            "grad_L_W2_init": torch.empty(B, H, 256, 64, dtype=f32, device=dev),
            "grad_L_b2_init": torch.empty(B, H, 1, 64, dtype=f32, device=dev),
            "grad_L_last_eta": torch.empty(B, H, NC, 64, 1, dtype=bf, device=dev),
            "grad_L_XQ": torch.empty_like(XQ), "grad_L_XK": torch.empty_like(XQ), "grad_L_XV": torch.empty_like(XQ),
        }
        eta5 = last_eta if last_eta.dim() == 5 else last_eta.unsqueeze(-1)
        ttt_backward(XQ, XK, XV, eta5.contiguous(), gamma, beta, *ck, out, *scratch,
                     g_W1, g_b1, g_W2, g_b2, g_out, *[o[k] for k in GRAD_NAMES], cgs)
        d_gamma = o["grad_L_ttt_norm_weight"].sum(dim=0, keepdim=True)
        d_beta = o["grad_L_ttt_norm_bias"].sum(dim=0, keepdim=True)
        d_eta = o["grad_L_last_eta"].reshape(ctx.eta_shape)
        return (o["grad_L_XQ"], o["grad_L_XK"], o["grad_L_XV"], d_eta, d_gamma, d_beta,
                o["grad_L_W1_init"], o["grad_L_b1_init"], o["grad_L_W2_init"], o["grad_L_b2_init"], None)


def ttt_mlp(XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, W2, b2, checkpoint_group_size=None):
    """Differentiable TTT-MLP layer core.  Returns (XQW, (W1, b1, W2, b2) after the last mini-batch)."""
    NC = XQ.shape[2]
    if checkpoint_group_size is None:
        checkpoint_group_size = max(1, int(math.sqrt(NC)))
    r = TTTMLPFunction.apply(XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, W2, b2,
                             checkpoint_group_size)
    return r[0], tuple(r[1:])


_linear_scratch_cache = {}


def _linear_scratch(B, H, cgs, device):
    from .ops import linear_backward_scratch_bytes
    key = (B, H, cgs, device.index, torch._C._cuda_getCurrentRawStream(device.index))
    if key not in _linear_scratch_cache:
        _linear_scratch_cache[key] = torch.empty(linear_backward_scratch_bytes(B, H, cgs), dtype=torch.uint8,
                                                 device=device)
    return _linear_scratch_cache[key]


class TTTLinearFunction(torch.autograd.Function):
    """(XQW, W1_last, b1_last) = f(XQ, XK, XV, last_eta, norm_weight, norm_bias, W1, b1, checkpoint_group_size):
    the TTT-Linear operator pair (`ttt_linear_forward` / `ttt_linear_backward`)."""

    @staticmethod
    def forward(ctx, XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, checkpoint_group_size):
        from .ops import ttt_linear_forward
        B, H, NC = XQ.shape[:3]
        cgs = int(checkpoint_group_size)
        dev = XQ.device
        args = [t.contiguous() for t in (XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1)]
        n = math.ceil(NC / cgs)
        ck = (torch.empty(B, H, n, 64, 64, dtype=torch.float32, device=dev),
              torch.empty(B, H, n, 1, 64, dtype=torch.float32, device=dev))
        out = torch.empty_like(args[0])
        final = (torch.empty_like(args[6]), torch.empty_like(args[7]))
        ttt_linear_forward(*args, *ck, out, cgs, final_state=final)
        ctx.save_for_backward(*args[:6], *ck)
        ctx.cgs = cgs
        ctx.eta_shape = last_eta.shape
        return (out,) + final

    @staticmethod
    def backward(ctx, g_out, g_W1, g_b1):
        from .ops import ttt_linear_backward
        XQ, XK, XV, last_eta, gamma, beta, Wc, bc = ctx.saved_tensors
        B, H, NC = XQ.shape[:3]
        cgs, dev = ctx.cgs, XQ.device
        f32 = torch.float32
        g_W1 = torch.zeros(B, H, 64, 64, dtype=f32, device=dev) if g_W1 is None else g_W1.contiguous().to(f32)
        g_b1 = torch.zeros(B, H, 1, 64, dtype=f32, device=dev) if g_b1 is None else g_b1.contiguous().to(f32)
        g_out = torch.zeros_like(XQ) if g_out is None else g_out.contiguous().to(torch.bfloat16)
        d_gamma = torch.empty(B, H, 1, 64, dtype=f32, device=dev)
        d_beta = torch.empty(B, H, 1, 64, dtype=f32, device=dev)
        d_W1 = torch.empty(B, H, 64, 64, dtype=f32, device=dev)
        d_b1 = torch.empty(B, H, 1, 64, dtype=f32, device=dev)
        d_eta = torch.empty(B, H, NC, 64, dtype=torch.bfloat16, device=dev)
        dq, dk, dv = torch.empty_like(XQ), torch.empty_like(XQ), torch.empty_like(XQ)
        eta4 = last_eta.reshape(B, H, NC, 64)
        ttt_linear_backward(XQ, XK, XV, eta4, gamma, beta, Wc, bc, g_W1, g_b1, g_out, d_gamma, d_beta, d_W1, d_b1, d_eta,
                            dq, dk, dv, cgs, scratch=_linear_scratch(B, H, cgs, dev))
        return (dq, dk, dv, d_eta.reshape(ctx.eta_shape), d_gamma.sum(dim=0, keepdim=True),
                d_beta.sum(dim=0, keepdim=True), d_W1, d_b1, None)


def ttt_linear(XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, checkpoint_group_size=None):
    """Differentiable TTT-Linear layer core.  Returns (XQW, (W1, b1) after the last mini-batch)."""
    NC = XQ.shape[2]
    if checkpoint_group_size is None:
        checkpoint_group_size = max(1, int(math.sqrt(NC)))
    r = TTTLinearFunction.apply(XQ, XK, XV, last_eta, ttt_norm_weight, ttt_norm_bias, W1, b1, checkpoint_group_size)
    return r[0], tuple(r[1:])


# ---- layer-side sequence operators (`ttt_tk_b200.ssm`, the block end of `ttt_tk_b200.glue`) ------------------------------------
# What is no tensor (None among it) passes, for the operator to take or to refuse.
def _rows(t):
    """With a contiguous last dimension (an upstream gradient can be an expanded number; of no elements that counts as contiguous as it is)."""
    if not isinstance(t, torch.Tensor) or t.dim() == 0 or t.stride(-1) == 1 or t.size(-1) == 1:
        return t
    return t.contiguous() if t.numel() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _whole(t):
    return t.contiguous() if isinstance(t, torch.Tensor) else t


def _tokens(t):
    """[..., D] as [tokens, D]."""
    if not isinstance(t, torch.Tensor) or t.dim() in (0, 2):
        return t
    return t.unsqueeze(0) if t.dim() == 1 else t.flatten(0, -2)


# `saved`: what a forward keeps of its activations for the backward, None for themselves or "e4m3" for 8 bits (`ttt_tk_b200.saved`).
def _saved(name):
    if not (name is None or isinstance(name, str)) or name not in (None, "e4m3"):
        raise ValueError(f"saved must be None or 'e4m3', got {name!r}")
    return name is not None and torch.is_grad_enabled()


def _even(t):
    """With rows at a fixed distance."""
    at_all = t.dim() < 3 or t.size(0) <= 1 or t.size(1) <= 1 or t.stride(0) == t.stride(1) * t.size(1)
    return t if at_all else t.contiguous()


def _pack(*ts, clamp=None):
    """Tensors of one shape (None among them) in 8 bits, flat: values, scales, values, ...; those of one type in one launch.  `clamp` as `pack8`'s."""
    from .saved import pack8
    flat, clamp = [None] * (2 * len(ts)), clamp or (None,) * len(ts)
    for ty in {t.dtype for t in ts if t is not None}:
        at = [k for k, t in enumerate(ts) if t is not None and t.dtype == ty]
        for k, p in zip(at, pack8(*[_even(ts[k]) for k in at], clamp=[clamp[k] for k in at])):
            flat[2 * k], flat[2 * k + 1] = p
    return flat


def _unpack(flat, types):
    """And back, in their types."""
    from .saved import unpack8
    ts = [None] * len(types)
    for ty in set(types) - {None}:
        at = [k for k, t in enumerate(types) if t == ty]
        for k, t in zip(at, unpack8(*[(flat[2 * k], flat[2 * k + 1]) for k in at], dtype=ty)):
            ts[k] = t
    return ts


class ShortConvFunction(torch.autograd.Function):
    """(y, final state or None) = f(x, weight, bias, state, activation, lengths, heads, return_state, packed)."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, activation, lengths, heads, return_state, packed=False):
        from . import ssm
        x, weight, bias, state = _rows(x), _whole(weight), _whole(bias), _whole(state)
        r = ssm.short_conv(x, weight, bias, activation=activation, state=state, lengths=lengths, heads=heads, return_state=return_state)
        ctx.packed = x.dtype if packed and any(ctx.needs_input_grad) else None
        ctx.save_for_backward(weight, bias, state, lengths, *([x] if ctx.packed is None else _pack(x)))
        ctx.kw = dict(activation=activation, heads=heads)
        ctx.set_materialize_grads(False)
        return r if return_state else (r, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gf):
        from . import ssm
        weight, bias, state, lengths, *kept = ctx.saved_tensors
        (x,) = kept if ctx.packed is None else _unpack(kept, [ctx.packed])
        if gy is None:
            B, T, D = x.shape
            gy = x.new_zeros((B, D // 64, T // 64, 64, 64) if ctx.kw["heads"] else (B, T, D))
        gy = _whole(gy) if ctx.kw["heads"] else _rows(gy)
        g = ssm.short_conv_backward(gy, x, weight, bias, state=state, lengths=lengths, grad_final_state=_whole(gf), **ctx.kw)
        return g + (None,) * 5


def short_conv(x, weight, bias=None, *, activation=None, state=None, lengths=None, heads=False, return_state=False, saved=None):
    """Differentiable `ttt_tk_b200.ssm.short_conv`.  `saved` "e4m3": x is kept in 8 bits, and the gradients are those at what was kept."""
    y, end = ShortConvFunction.apply(x, weight, bias, state, activation, lengths, heads, return_state, _saved(saved))
    return (y, end) if return_state else y


class SSMScanFunction(torch.autograd.Function):
    """(y, final state or None) = f(x, dt, A, B, C, D, dt_bias, state, softplus, lengths, return_state, recorded, packed).

    `recorded`: whether gradients are recorded where it is called, which is not to be seen inside `forward` (and `needs_input_grad` says
    what the inputs ask for, recorded or not): the checkpoints, fp32 [batch, T / 16, D, N], are written for a backward that can come."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, dt_bias, state, softplus, lengths, return_state, recorded=True, packed=False):
        from . import ssm
        x, dt, B, C = (_rows(t) for t in (x, dt, B, C))
        A, D, dt_bias, state = (_whole(t) for t in (A, D, dt_bias, state))
        keep = recorded and any(ctx.needs_input_grad)
        r = ssm.ssm_scan(x, dt, A, B, C, D, dt_bias, softplus=softplus, state=state, lengths=lengths, return_state=return_state,
                         return_checkpoints=keep)
        r = r if isinstance(r, tuple) else (r,)
        ctx.packed = x.dtype if packed else None
        if keep:
            ctx.save_for_backward(A, B, C, D, dt_bias, lengths, r[-1], *(_pack(x, dt, clamp=(None, "low" if softplus else None)) if packed else (x, dt)))
        ctx.softplus, ctx.has_state = softplus, state is not None
        ctx.set_materialize_grads(False)
        return r[0], r[1] if return_state else None

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gf):
        from . import ssm
        A, B, C, D, dt_bias, lengths, ck, *kept = ctx.saved_tensors
        x, dt = kept if ctx.packed is None else _unpack(kept, [ctx.packed] * 2)
        gy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if gy is None else _rows(gy)
        g = ssm.ssm_scan_backward(gy, x, dt, A, B, C, ck, D, dt_bias, softplus=ctx.softplus, lengths=lengths,
                                  grad_final_state=_whole(gf))
        return g[:7] + (g[7] if ctx.has_state else None,) + (None,) * 5


def ssm_scan(x, dt, A, B, C, D=None, dt_bias=None, *, softplus=True, state=None, lengths=None, return_state=False, saved=None):
    """Differentiable `ttt_tk_b200.ssm.ssm_scan`; where gradients are recorded, the checkpoints are kept for the backward.  `saved` "e4m3": x and dt are
    kept in 8 bits, and the gradients are those at what was kept, with the checkpoints as the forward has them; a dt below -448 (a mask's -inf) is kept as
    -448, which softplus takes to 0 as well as it (with a dt_bias of less than 300)."""
    y, end = SSMScanFunction.apply(x, dt, A, B, C, D, dt_bias, state, softplus, lengths, return_state, torch.is_grad_enabled(), _saved(saved))
    return (y, end) if return_state else y


class GatedScanFunction(torch.autograd.Function):
    """(y, final state or None) = f(x, gate, A, input_gate, gate_bias, input_bias, state, mix, lengths, return_state, recorded, packed);
    `recorded` as in `SSMScanFunction`."""

    @staticmethod
    def forward(ctx, x, gate, A, input_gate, gate_bias, input_bias, state, mix, lengths, return_state, recorded=True, packed=False):
        from . import ssm
        x, gate, input_gate = (_rows(t) for t in (x, gate, input_gate))
        A, gate_bias, input_bias, state = (_whole(t) for t in (A, gate_bias, input_bias, state))
        keep = recorded and any(ctx.needs_input_grad)
        r = ssm.gated_scan(x, gate, A, input_gate, gate_bias, input_bias, mix=mix, state=state, lengths=lengths, return_state=return_state,
                           return_checkpoints=keep)
        r = r if isinstance(r, tuple) else (r,)
        if keep:
            kept = (x, gate, input_gate)
            ctx.save_for_backward(A, gate_bias, input_bias, lengths, r[-1], *(_pack(*kept, clamp=(None, "both", "both")) if packed else kept))
        ctx.mix, ctx.has_state, ctx.like = mix, state is not None, (x.shape, x.dtype, x.device)
        ctx.set_materialize_grads(False)
        return r[0], r[1] if return_state else None

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gf):
        from . import ssm
        A, gate_bias, input_bias, lengths, ck, *kept = ctx.saved_tensors
        if len(kept) == 6:      # in 8 bits, which the backward takes as they are
            kept = [(kept[k], kept[k + 1]) if kept[k] is not None else None for k in (0, 2, 4)]
        x, gate, input_gate = kept
        shape, dtype, device = ctx.like
        gy = torch.zeros(shape, dtype=dtype, device=device) if gy is None else _rows(gy)
        g = ssm.gated_scan_backward(gy, x, gate, ck, A, input_gate, gate_bias, input_bias, mix=ctx.mix, lengths=lengths,
                                    grad_final_state=_whole(gf))
        return g[:6] + (g[6] if ctx.has_state else None,) + (None,) * 5


def gated_scan(x, gate, A=None, input_gate=None, gate_bias=None, input_bias=None, *, mix="sqrt", state=None, lengths=None, return_state=False,
               saved=None):
    """Differentiable `ttt_tk_b200.ssm.gated_scan`; where gradients are recorded, the checkpoints are kept for the backward.  `saved` "e4m3": x and the
    gates are kept in 8 bits, and the gradients are those at what was kept, with the checkpoints as the forward has them.  Gates beyond 448 on either side,
    infinities among them, are kept as -448 and 448: a closed gate stays closed (with biases of less than 300)."""
    y, end = GatedScanFunction.apply(x, gate, A, input_gate, gate_bias, input_bias, state, mix, lengths, return_state, torch.is_grad_enabled(),
                                     _saved(saved))
    return (y, end) if return_state else y


class NormGateResidualFunction(torch.autograd.Function):
    """(x, n or None) = f(o, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, activation, eps, packed); o,
    residual and gate [tokens, D]."""

    @staticmethod
    def forward(ctx, o, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, activation, eps, packed=False):
        from .glue import norm_gate_residual as run
        o, residual, gate = (_rows(t) for t in (o, residual, gate))
        weights = [_whole(t) for t in (post_weight, post_bias, scale, pre_weight, pre_bias)]
        ctx.kw = dict(norm=norm, activation=activation, eps=eps)
        x, n, stats = run(o, residual, gate, **dict(zip(_BLOCK_WEIGHTS, weights)), return_stats=True, **ctx.kw)
        kept = [o, residual, gate]
        ctx.packed = [None if t is None else t.dtype for t in kept] if packed and any(ctx.needs_input_grad) else None
        ctx.save_for_backward(stats, *weights, *(kept if ctx.packed is None else _pack(*kept, clamp=(None, None, "both" if activation == "sigmoid" else "low"))))
        ctx.set_materialize_grads(False)
        return x, n

    @staticmethod
    @once_differentiable
    def backward(ctx, gx, gn):
        from .glue import norm_gate_residual_backward as run
        if gx is None and gn is None:
            return (None,) * 12
        stats, *kept = ctx.saved_tensors
        weights, kept = kept[:5], kept[5:]
        o, residual, gate = kept if ctx.packed is None else _unpack(kept, ctx.packed)
        return run(_rows(gx), _rows(gn), o, stats, residual, gate, **dict(zip(_BLOCK_WEIGHTS, weights)), **ctx.kw) + (None,) * 4


_BLOCK_WEIGHTS = ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")


def norm_gate_residual(o, residual=None, gate=None, *, norm="rms", activation="silu", post_weight=None, post_bias=None, scale=None,
                       pre_weight=None, pre_bias=None, eps=1e-6, saved=None):
    """Differentiable `ttt_tk_b200.glue.norm_gate_residual`, with rows at any distances.  `saved` "e4m3": o, residual and gate are kept in 8 bits, and the
    gradients are those at what was kept, with the statistics as the forward has them; a gate below -448 (a mask) is kept as -448."""
    for name, t in (("residual", residual), ("gate", gate)):
        if isinstance(o, torch.Tensor) and isinstance(t, torch.Tensor) and t.shape != o.shape:
            raise ValueError(f"norm_gate_residual: {name} must have the shape of o, {list(o.shape)}, got {list(t.shape)}")
    x, n = NormGateResidualFunction.apply(*[_tokens(t) for t in (o, residual, gate)], post_weight, post_bias, scale, pre_weight, pre_bias, norm, activation, eps,
                                          _saved(saved))
    return x.view(o.shape), None if n is None else n.view(o.shape)
