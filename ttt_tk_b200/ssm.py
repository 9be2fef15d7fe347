"""Layer-side sequence operators with a state of their own (CUDA, `csrc/ttt_short_conv.cu`, `csrc/ttt_ssm_scan_sm100.cu`): the short
causal convolution in front of a TTT layer's queries and keys or of a state space layer, and the selective state space scan that
models mix with TTT layers.  Each for prompts, for training and for single tokens.

    y, state = short_conv(x, weight, bias, activation="silu", return_state=True)       # [B, T, D]
    y, state, ck = ssm_scan(x, dt, A, B, C, D, dt_bias, return_state=True, return_checkpoints=True)
    y = short_conv_step(x, state, weight, bias, activation="silu", slots=slots)        # [B, D], one token; `state` in place
    y = ssm_scan_step(x, dt, A, B, C, state, D, dt_bias, slots=slots)

Activations are bf16, fp16 or fp32 (all of a call the same), with any strides but the innermost, so that a slice of a projection's
output can be passed as it is; weights, biases, A, D, scan states and checkpoints are contiguous fp32.  Everything between reading and
writing is fp32, and sums have a fixed order: the same call gives the same bits.  Calls are stream-ordered and do not synchronise.
A bad argument raises ValueError.  Differentiable forms: `ttt_tk_b200.autograd.short_conv` and `ssm_scan`.

`lengths` (int32 [B], on the GPU): a right-padded batch.  Tokens from a sequence's length on are not read, whatever they hold; their
outputs and gradients are zero and they change no state.

A step's `slots` (int32 [B], on the GPU) name the rows of the table `state` that the rows of the batch have; a row whose slot is not
one of the table is padding (y = 0, no state touched), and rows that name the same slot are taken in their order, like tokens after one
another.  The statements the operators match are in `oracle/layer.py`.
"""
from .build import load_layer_host

_HOST = None
_ACTIVATIONS = {None: 0, "silu": 1}


def _host():
    global _HOST
    if _HOST is None:
        host = load_layer_host()      # may build: before the library is loaded
        from . import _lib
        _lib.lib()
        _HOST = host
    return _HOST


def _activation(name):
    if not (name is None or isinstance(name, str)) or name not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'silu', got {name!r}")
    return _ACTIVATIONS[name]


def short_conv(x, weight, bias=None, *, activation=None, state=None, lengths=None, heads=False, return_state=False):
    """y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - K + 1 + k, d]): a depthwise causal convolution of width K = 2, 3 or 4.

    `x` [B, T, D]; `weight` fp32 [D, K]; `bias` fp32 [D]; `activation` None or "silu".  `state` [B, K - 1, D], of x's type: the
    inputs in front of the first token (zeros without it).  `heads`: y leaves as the TTT operator's [B, D / 64, T / 64, 64, 64]
    instead of [B, T, D] (`layout.pack_tokens` in the same pass; multiples of 64 tokens and channels).  Returns y, or with
    `return_state` (y, state): the last K - 1 inputs of each sequence, the next chunk's or step's state."""
    y, end = _host().conv(x, weight, bias, _activation(activation), state, lengths, heads, return_state)
    return (y, end) if return_state else y


def short_conv_backward(grad_y, x, weight, bias=None, *, activation=None, state=None, lengths=None, heads=False,
                        grad_final_state=None):
    """Gradients of `short_conv` from its inputs: (grad_x, grad_weight, grad_bias, grad_state), the last two None where there
    is no bias or state.  `grad_y` as y; `grad_final_state` [B, K - 1, D], of x's type, is added where the final state came from."""
    return _host().conv_backward(grad_y, x, weight, bias, _activation(activation), state, lengths, heads, grad_final_state)


def short_conv_step(x, state, weight, bias=None, *, activation=None, slots=None):
    """`short_conv` of one token per row: `x` [B, D]; `state` [B, K - 1, D], or with `slots` a table [S, K - 1, D], is updated in
    place.  Returns y [B, D]."""
    return _host().conv_step(x, state, weight, bias, _activation(activation), slots)


def ssm_scan(x, dt, A, B, C, D=None, dt_bias=None, *, softplus=True, state=None, lengths=None, return_state=False,
             return_checkpoints=False):
    """Selective state space scan:

        delta = softplus(dt + dt_bias)                              (softplus=False: dt + dt_bias)
        h[d, n] = exp(delta[d] A[d, n]) h[d, n] + delta[d] x[d] B[g, n]
        y[d]    = sum_n C[g, n] h[d, n] + D[d] x[d]                 g = d // (D / G), the group of channel d

    `x`, `dt` [batch, T, D]; `A` fp32 [D, N], finite, 1 to 64 states; `B`, `C` [batch, T, G, N], G dividing the channels; `D`,
    `dt_bias` fp32 [D]; `state` fp32 [batch, D, N] in front of the first token (zeros without it).  Returns y [batch, T, D], followed
    by the state behind each sequence's last token where `return_state` asks for it, and by the states before every 16th
    token, fp32 [batch, ceil(T / 16), D, N], that `ssm_scan_backward` starts from, where `return_checkpoints` does (those behind a
    sequence's end hold nothing)."""
    y, end, ck = _host().scan(x, dt, A, B, C, D, dt_bias, softplus, state, lengths, return_state, return_checkpoints)
    if not (return_state or return_checkpoints):
        return y
    return (y,) + ((end,) if return_state else ()) + ((ck,) if return_checkpoints else ())


def ssm_scan_backward(grad_y, x, dt, A, B, C, checkpoints, D=None, dt_bias=None, *, softplus=True, lengths=None,
                      grad_final_state=None):
    """Gradients of `ssm_scan` from its inputs and checkpoints: (grad_x, grad_dt, grad_A, grad_B, grad_C, grad_D, grad_dt_bias,
    grad_state); grad_D and grad_dt_bias None where there is none.  Those of the activations have their type, the others are fp32;
    grad_state fp32 [batch, D, N] is that of the state in front of the first token.

    Memory: the checkpoints are N / 4 bytes per token and channel, and its scratch, for grad_B and grad_C, 1/2, 2, 8 or 32 bytes per token and
    channel at 8, 16, 32 or 64 states, where a group has more than 128, 64, 32 or 16 channels."""
    return _host().scan_backward(grad_y, x, dt, A, B, C, D, dt_bias, softplus, checkpoints, lengths, grad_final_state)


def ssm_scan_step(x, dt, A, B, C, state, D=None, dt_bias=None, *, softplus=True, slots=None):
    """`ssm_scan` of one token per row: `x`, `dt` [batch, D]; `B`, `C` [batch, G, N]; `state` fp32 [batch, D, N], or with `slots` a
    table [S, D, N], is updated in place.  Returns y [batch, D]."""
    return _host().scan_step(x, dt, A, B, C, D, dt_bias, softplus, state, slots)
