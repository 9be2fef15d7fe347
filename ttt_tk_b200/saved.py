"""Activations that a forward pass keeps for its backward pass in 8 bits (CUDA, `csrc/ttt_eight_bits.cu`), at half the memory of 16 bits.

    (qx, sx), (qg, sg) = pack8(x, gate)                  # values float8_e4m3fn, scales fp32 [..., ceil(D / 128)]
    x, gate = unpack8((qx, sx), (qg, sg))                # bf16

Of each `group` neighbouring values of a row the scale is the least power of two with max |v| <= 448 scale, and v / scale is kept in e4m3: a
value is off by at most 2^-4 of itself, and where it is below 2^-6 of the scale by at most 2^-10 of that.  A power of two divides exactly, so the
format's rounding is the only one.  What is finite comes back finite: a value that rounds up to 2^16 in fp16 or 2^128 in bf16 and fp32 is the type's
largest, of the last two 240 2^120.  Infinities are left out of the maximum and become 448 scale, or that largest value; NaN stays NaN.

`ttt_tk_b200.ssm.gated_scan_backward` takes packed inputs as they are; the differentiable operators of `ttt_tk_b200.autograd` with `saved="e4m3"` keep
theirs this way, gates with `clamp`.  Calls are stream-ordered and do not synchronise.  A bad argument raises ValueError.
"""
import torch

from . import ssm

_CLAMPS = {None: 0, "low": 1, "both": 2}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def pack8(*xs, group=128, clamp=None):
    """One to four tensors [..., D] of the same shape and type (bf16, fp16 or fp32, rows at a fixed distance) -> a list of (values, scales), one
    launch.  `group`: 32, 64 or 128.

    `clamp`: for gates, one of None, "low" and "both" for each tensor: values below -448 count as -448, with "both" those above 448 as 448 too, infinities
    among them.  To a sigmoid, SiLU, GELU or softplus that is all the same, and a mask (-inf, or its type's lowest value) stays one, where it would
    otherwise set its neighbours' scale, or as an infinity become 448 times theirs."""
    return ssm._host().pack8(xs, _group(group, "32, 64 or 128"), _clamp(clamp, len(xs)))


def unpack8(*packs, dtype=torch.bfloat16):
    """The values that (values, scales) stand for, in `dtype` (bf16, fp16 or fp32), for one to four of the same shape, one launch.  The group is
    that of the scales' shape; [...] is one scale to a row (`glue.norm_residual_8bit` with group None)."""
    if not isinstance(dtype, torch.dtype) or dtype not in _TYPES:
        raise ValueError(f"dtype must be torch.bfloat16, torch.float16 or torch.float32, got {dtype!r}")
    return ssm._host().unpack8(packs, _TYPES[dtype])


def _clamp(clamp, n):
    if clamp is None:
        return None
    if not isinstance(clamp, (tuple, list)) or len(clamp) != n or any(not (c is None or isinstance(c, str)) or c not in _CLAMPS for c in clamp):
        raise ValueError(f"clamp must be None, or one of None, 'low' and 'both' for each tensor, got {clamp!r}")
    return tuple(_CLAMPS[c] for c in clamp)


def _group(group, what):
    if not isinstance(group, int) or isinstance(group, bool) or group < 1 or group > 128:
        raise ValueError(f"group must be {what}, got {group!r}")
    return group
