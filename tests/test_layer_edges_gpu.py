"""The layer-side sequence operators at the ends of their ranges and where calls meet.
Statements: oracle/layer.py; tolerances: tests/layer_cases.py."""
import ctypes
import os
import struct
import subprocess
import sys
import threading

import pytest
import torch

from layer_cases import TYPES, close, conv_inputs, gen, scan_inputs
from oracle import layer as ol
from ttt_tk_b200 import _lib, glue, ssm

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---- block end: gates of any size -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("parts", ["all", "gate"])
def test_gradients_at_gates_of_any_size(ty, act, parts):
    """A closed gate (the type's lowest value, as a mask leaves it) passes no gradient, an open one passes it whole.  The sizes lie away
    from -87, where 1 / (1 + exp(-v)) leaves fp32: what is below is 0."""
    t, M, D = TYPES[ty], 6, 64
    top = torch.finfo(t).max
    g = gen(4)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    sizes = [-top, -min(top, 1e30), -min(top, 1e25), -min(top, 1e19), -min(top, 1e13), -1e3, -100.0, 0.0, 100.0, 1e3]
    if parts == "gate":      # (a gate that is open that wide leaves no room for the rest of a row's arithmetic)
        sizes += [min(top, 1e13), min(top, 1e19), min(top, 1e25), min(top, 1e30), top]
    gate = torch.tensor(sizes).repeat(M * D // len(sizes) + 1)[:M * D].view(M, D).to(t)
    small = 2.0 ** -6 if parts == "gate" else 1.0      # products with the widest gate have to be numbers of the type
    o, res, gx = (r(M, D).clamp(-4, 4) * s for s in (small, 1.0, small))
    o, res, gx = o.to(t), res.to(t), gx.to(t)
    w = {} if parts == "gate" else dict(post_weight=1 + 0.1 * r(D), scale=0.3 + 0.1 * r(D), pre_weight=1 + 0.1 * r(D))
    gn = None if parts == "gate" else r(M, D).to(t)
    dev = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    o, res, gate, gx, gn = (dev(v) for v in (o, res, gate, gx, gn))
    kw = dict(activation=act, **{k: dev(v) for k, v in w.items()})
    x, n, stats = glue.norm_gate_residual(o, res, gate, return_stats=True, **kw)
    assert torch.isfinite(x).all() and (n is None or torch.isfinite(n).all())
    got = glue.norm_gate_residual_backward(gx, gn, o, stats, res, gate, **kw)
    okw = {("activation_" if k == "activation" else k): v for k, v in kw.items()}
    want = ol.norm_gate_residual_backward(gx, gn, o, res, gate, **okw)
    amps = ol.norm_gate_residual_backward(gx, gn, o, res, gate, amp=True, **okw)
    for k, a, b, m in zip(("o", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight"), got, want, amps):
        assert (a is None) == (b is None), k
        if a is not None:
            assert torch.isfinite(a).all(), k
            # (the statistics' sums have up to 28 roundings in a row at this width, and M tokens follow one another in a weight's)
            close(a, b, m, 4 * (2 * 28 + 120) + M, "grad " + k)


# ---- convolution: what lies behind a sequence is zero ---------------------------------------------------------------------
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("ty,D,K,T,n", [("bf16", 64, 4, 40, 21), ("fp32", 13, 3, 19, 8), ("fp32", 64, 2, 64, 63), ("fp16", 72, 4, 300, 130)])
def test_gradients_behind_a_sequence_that_ends_with_infinities(act, ty, D, K, T, n):
    i = conv_inputs(7, ty, 1, T, D, K, DEV)
    i["x"][0, n - 1, ::2] = float("inf")
    i["x"][0, n - 2, 1::4] = float("nan")
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = ssm.short_conv_backward(i["gy"], i["x"], i["weight"], i["bias"], activation=act, state=i["state"], lengths=lengths,
                                  grad_final_state=i["gf"])
    want = ol.short_conv_backward(i["gy"], i["x"], i["weight"], i["bias"], act, i["state"], [n], i["gf"])
    assert (got[0][0, n:] == 0).all()
    for k, a, b in zip(("x", "weight", "bias", "state"), got, want):
        fine = torch.isfinite(b)
        assert torch.isfinite(a.cpu())[fine].all(), k      # a number wherever the formula has one
    if act is None:      # nothing but the weights' gradients sees x
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all() and torch.isfinite(got[3]).all()


# ---- scan: states that grow ----------------------------------------------------------------------------
def test_chunks_over_which_a_state_grows_beyond_fp32():
    """Factors of exp(8) a token: over a chunk of 16 more than fp32 holds, while the states themselves are zero or small there."""
    B, T, D, N = 1, 600, 64, 16      # (one CTA's worth of channels: every tile of 16 tokens is a chunk)
    i = scan_inputs(9, "fp32", B, T, D, N, 1, DEV, state=False)
    i["A"] = torch.full((D, N), 2.0, device=DEV)
    i["dt"] = torch.full((B, T, D), 4.0, device=DEV)
    i["x"][:, :T - 3] = 0
    i["gy"][:, 3:] = 0
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y, end, ck = ssm.ssm_scan(*a, softplus=False, return_state=True, return_checkpoints=True)
    ref, rend, _ = ol.ssm_scan(*a, softplus_=False)
    amp, aend, _ = ol.ssm_scan(*a, softplus_=False, amp=True)
    close(y, ref, amp, 16 * 8 + N + 40, "y")      # (nothing is there before the last three tokens)
    close(end, rend, aend, 16 * 8, "state")
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, softplus=False)
    want = ol.ssm_scan_backward(i["gy"], *a, softplus_=False)
    amps = ol.ssm_scan_backward(i["gy"], *a, softplus_=False, amp=True)
    for k, g, r, m in zip(("x", "dt", "A", "B", "C", "", "", "state"), got, want, amps):
        if k:
            close(g, r, m, 32 * 8 + 2 * N + 80 + D, "grad " + k)


def test_a_small_state_that_grows_over_a_chunk():
    B, T, D, N = 1, 18, 64, 16      # two chunks
    i = scan_inputs(10, "fp32", B, T, D, N, 1, DEV)
    i["A"] = torch.full((D, N), 2.0, device=DEV)
    i["dt"] = torch.full((B, T, D), 4.0, device=DEV)
    i["x"][:] = 0
    i["state"] = i["state"] * 1e-30
    i["gy"][:] = 0
    i["gf"] = i["gf"] * 1e-30
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y, end, ck = ssm.ssm_scan(*a, softplus=False, state=i["state"], return_state=True, return_checkpoints=True)
    ref, rend, _ = ol.ssm_scan(*a, softplus_=False, state=i["state"])
    amp, aend, _ = ol.ssm_scan(*a, softplus_=False, state=i["state"], amp=True)
    # a factor's exponent of 8 log2(e) = 11.5 is rounded twice: 12 + 12 roundings of the factor, and 16 as elsewhere
    close(y, ref, amp, 40 * T + N + 40, "y")
    close(end, rend, aend, 40 * T, "state")
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, softplus=False, grad_final_state=i["gf"])
    want = ol.ssm_scan_backward(i["gy"], *a, softplus_=False, state=i["state"], grad_final_state=i["gf"])
    amps = ol.ssm_scan_backward(i["gy"], *a, softplus_=False, state=i["state"], grad_final_state=i["gf"], amp=True)
    for j, k in ((0, "x"), (1, "dt"), (2, "A"), (7, "state")):
        close(got[j], want[j], amps[j], 80 * T + 2 * N + 80, "grad " + k)


# ---- decays: of the lowest value
@pytest.mark.parametrize("T", [13, 600])
def test_decays_of_the_lowest_value(T):
    """A = the lowest fp32 forgets a state wherever delta is not zero, and keeps it where it is: steps of zero and tokens behind a sequence."""
    B, D, N = 2, 64, 16
    low = torch.finfo(torch.float32).min
    i = scan_inputs(11, "fp32", B, T, D, N, 1, DEV)
    i["A"][:, ::3] = low
    n = [T - 4, 0]
    i["dt"] = i["dt"].abs() * 0.1 + 0.01
    i["dt"][:, T // 3:T // 2] = 0
    lengths = torch.tensor(n, dtype=torch.int32, device=DEV)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y, end = ssm.ssm_scan(*a, i["D"], softplus=False, state=i["state"], lengths=lengths, return_state=True)
    ref, rend, _ = ol.ssm_scan(*a, i["D"], softplus_=False, state=i["state"], lengths=n)
    amp, aend, _ = ol.ssm_scan(*a, i["D"], softplus_=False, state=i["state"], lengths=n, amp=True)
    close(y, ref, amp, 16 * T + N + 40, "y")
    close(end, rend, aend, 16 * T + N + 40, "state")
    st = i["state"].clone()
    one = [t[:, 0] if t.dim() > 2 else t for t in a]
    one[1] = torch.zeros_like(one[1])
    ssm.ssm_scan_step(*one, st, softplus=False)
    assert torch.equal(st, i["state"])


# ---- threads: two of the host -----------------------------------------------------------------------------------------------------
def test_two_threads_with_different_amounts_of_shared_memory():
    """The same kernel with 160 KB and 80 KB of shared memory, called through the C entry from two threads."""
    lib = _lib.lib()
    fn = lib.ttt_b200_norm_gate_residual_backward
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.ttt_b200_norm_gate_residual_scratch_bytes.argtypes = [ctypes.c_void_p]
    lib.ttt_b200_norm_gate_residual_scratch_bytes.restype = ctypes.c_uint64

    def call(D):
        M = 2
        o, gx, go = (torch.ones(M, D, device=DEV) for _ in range(3))
        w, gw = (torch.ones(D, device=DEV) for _ in range(2))
        _, _, stats = glue.norm_gate_residual(o, post_weight=w, return_stats=True)
        # o, residual, gate, weights x 5, x, n, stats, grad_x, grad_n, grad_o, grad_residual, grad_gate, sums x 5, scratch
        p = [0] * 22
        p[0], p[3], p[10], p[11], p[13], p[16] = (t.data_ptr() for t in (o, w, stats, gx, go, gw))
        tail = (D, D, D, D, D, M, D, 2, 0, 0, 1, 1e-6)
        size = lib.ttt_b200_norm_gate_residual_scratch_bytes(struct.pack("=22Q Q 6q 5i f", *p, 0, *tail))
        scratch = torch.empty(size, dtype=torch.uint8, device=DEV)
        p[21] = scratch.data_ptr()
        stream = torch.cuda.Stream()
        return struct.pack("=22Q Q 6q 5i f", *p, size, *tail), stream, (o, gx, go, w, gw, stats, scratch)

    calls = [call(8188), call(4100)]      # (8192 fills its threads, which is another kernel)
    torch.cuda.synchronize()
    codes = [[], []]
    start = threading.Barrier(2)

    def work(k):
        args, stream, _ = calls[k]
        start.wait()
        for _ in range(3000):
            codes[k].append(fn(args, stream.cuda_stream))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(codes[0]) == len(codes[1]) == 3000
    assert not any(codes[0]) and not any(codes[1]), [sum(map(bool, c)) for c in codes]


# ---- bits: tokens behind a sequence
@pytest.mark.parametrize("ty,B,T,D,N", [("bf16", 2, 16, 64, 16), ("fp32", 2, 333, 20, 8), ("bf16", 3, 700, 64, 16), ("fp16", 1, 400, 130, 64)])
def test_no_token_changes_no_bit_of_a_state(ty, B, T, D, N):
    """Sequences without tokens, in one chunk and in several: their states and the gradients of these pass through as they are."""
    i = scan_inputs(T, ty, B, T, D, N, 1, DEV)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y, end, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], lengths=zero, return_state=True, return_checkpoints=True)
    assert torch.equal(end, i["state"]) and (y == 0).all()
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], lengths=zero, grad_final_state=i["gf"])
    assert torch.equal(got[7], i["gf"])
    assert all((g == 0).all() for g in got[:7])


@pytest.mark.parametrize("T,n", [(16, 9), (16, 15), (32, 17), (700, 689)])
def test_tokens_behind_a_sequence_change_no_bit_of_its_state(T, n):
    """As many tiles with and without the tokens behind: the same chunks, the same states."""
    i = scan_inputs(n, "bf16", 2, T, 64, 16, 1, DEV)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    cut = [t[:, :n] if t.dim() > 2 else t for t in a]
    lengths = torch.full((2,), n, dtype=torch.int32, device=DEV)
    y, end, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], lengths=lengths, return_state=True, return_checkpoints=True)
    y1, end1, ck1 = ssm.ssm_scan(*cut, i["D"], i["dt_bias"], state=i["state"], return_state=True, return_checkpoints=True)
    assert (T + 15) // 16 == (n + 15) // 16 and torch.equal(end, end1) and torch.equal(y[:, :n], y1) and torch.equal(ck, ck1)
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], lengths=lengths, grad_final_state=i["gf"])
    want = ssm.ssm_scan_backward(i["gy"][:, :n], *cut, ck1, i["D"], i["dt_bias"], grad_final_state=i["gf"])
    for k in (0, 1, 3, 4):
        assert torch.equal(got[k][:, :n], want[k]) and (got[k][:, n:] == 0).all()
    for k in (2, 5, 6, 7):
        assert torch.equal(got[k], want[k])

# ---- sums that have few roundings in a row -----------------------------------------------------------------------------------
BLOCK = [
    # type, M, D, norm, residual fp32, all parts
    ("fp32", 5, 64, "layer", False, True), ("fp32", 3, 1003, "layer", False, True), ("fp32", 4, 1024, "rms", False, True),
    ("bf16", 4, 2048, "layer", True, True), ("fp32", 3, 4096, "layer", False, False), ("fp32", 4, 4100, "layer", False, True),
    ("bf16", 3, 4104, "layer", True, True), ("fp32", 4, 8192, "layer", False, True), ("fp16", 4, 8191, "layer", True, True),
    ("fp32", 2, 8190, "rms", False, True), ("fp32", 3, 8192, "layer", False, False),
]


def _block_magnitudes(gx, gn, o, res, gate, layer, eps, post_weight=None, scale=None, pre_weight=None):
    """What the roundings of the block end's gradients are relative to: (o, residual, gate, post_weight, None, scale, pre_weight).  A normalised
    value (v - mean) r is off by 2^-24 of (|v| + |mean|) r however near to zero it comes (v = 0.3 + 1e-6 about a mean of 0.3: half a step of
    0.3, 1.5e-8, is 1.5 % of it), so these stand for it in every term; of z = residual + scale u act(gate), |z| is the sum of its terms'."""
    gx, gn, o, res, gate, w1, sc, w2 = (ol._d(t) for t in (gx, gn, o, res, gate, post_weight, scale, pre_weight))
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    r1, big = 1.0, o.abs()
    if w1 is not None:
        r1 = ol._norm(o, layer, eps)[1]
        big = (o.abs() + (mean(o).abs() if layer else 0.0)) * r1
    u = big * (w1.abs() if w1 is not None else 1.0)
    gv, gs = ol.activation("sigmoid", gate) if gate is not None else (torch.ones_like(o), None)
    s = sc.abs() if sc is not None else 1.0
    z = s * u * gv + res.abs()
    r2 = ol._norm(ol.norm_gate_residual(o, res, gate, "layer" if layer else "rms", "sigmoid", w1, None, sc, w2, None, eps)[0], layer, eps)[1]
    zn = (z + (mean(z) if layer else 0.0)) * r2
    back = lambda g, h, r: r * (g + h * mean(g * h) + (mean(g) if layer else 0.0))  # noqa: E731
    d = gx.abs() + back(gn.abs() * w2.abs(), zn, r2)
    du = d * s * gv
    return (back(du * w1.abs(), big, r1) if w1 is not None else du, d, d * s * u * gs if gate is not None else None,
            (du * big).sum(0) if w1 is not None else None, None, (d * u * gv).sum(0) if sc is not None else None, (gn.abs() * zn).sum(0))


@pytest.mark.parametrize("ty,M,D,norm,res32,full", BLOCK)
def test_the_means_of_the_norms_backward(ty, M, D, norm, res32, full):
    """Upstream gradients of one sign, so that the means that a norm's backward takes off are as large as what they are taken off, and
    tolerances that count the roundings in a row of these sums, not their terms: at most eight pairs, their halves, five shuffles, a warp's
    count and reciprocal (5), four more shuffles and 1 / D: 28, once for the statistics and once for the means."""
    t, rt, g = TYPES[ty], torch.float32 if res32 else TYPES[ty], gen(D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    o, res, gate = (r(M, D) * 1.5 + 0.3).to(t).to(DEV), (r(M, D) * 2).to(rt).to(DEV), (1 + r(M, D)).to(t).to(DEV)
    w = dict(post_weight=1 + 0.1 * r(D), scale=0.5 + 0.1 * r(D), pre_weight=1 + 0.1 * r(D)) if full else dict(pre_weight=1 + 0.1 * r(D))
    w = {k: v.to(DEV) for k, v in w.items()}
    gate = gate if full else None
    kw = dict(norm=norm, activation="sigmoid", eps=1e-5, **w)
    okw = {("activation_" if k == "activation" else k): v for k, v in kw.items()}
    x, n, stats = glue.norm_gate_residual(o, res, gate, return_stats=True, **kw)
    ref, _ = ol.norm_gate_residual(o, res, gate, **okw)
    zh = ol._norm(ref, norm == "layer", 1e-5)[0]
    gx = (0.5 + 0.05 * r(M, D)).to(x.dtype).to(DEV)
    gn = (1 + 0.1 * r(M, D) + 0.5 * zh.float()).to(t).to(DEV)      # (its mean and its mean with the normalised values)
    got = glue.norm_gate_residual_backward(gx, gn, o, stats, res, gate, **kw)
    want = ol.norm_gate_residual_backward(gx, gn, o, res, gate, **okw)
    amps = _block_magnitudes(gx, gn, o, res, gate, norm == "layer", 1e-5, **w)
    for k, a, b, m in zip(("o", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight"), got, want, amps):
        if a is not None:
            # (4: z's errors once more in its statistics, as for all of these inputs)
            close(a, b, m, 4 * (2 * 28 + 120) + (M if a.dim() == 1 else 0), "grad " + k)


def _bounded(got, ref, bound, what):
    """`bound`: in roundings of 2^-24"""
    d = (got.double().cpu() - ref).abs()
    tol = bound * (1 + 2.0 ** -10) * 2.0 ** -24 + 2.0 ** -24 * ref.abs() + 2.0 ** -126
    assert (d <= tol).all(), (what, (d / tol).max().item())


@pytest.mark.parametrize("B,T,D,N,G", [(1, 700, 64, 16, 1), (4, 64, 2560, 16, 1), (2, 333, 20, 5, 1), (1, 500, 48, 64, 3)])
def test_errors_of_a_state_decay_with_it(B, T, D, N, G):
    """The state's error is a recursion of its own: what a token adds decays with the state.  Per token, in roundings of 2^-24: delta
    2 (|dt| + |bias|) + 16 of itself (its sum; the exponential, two reciprocals and the series); the factor exp(delta A) |delta A| times those of
    delta, of A log2(e), of the product and of the sum of up to 16 deltas where chunks are joined (16 + 2), and 4 of the exponential;
    delta x B three products and a sum.  y: 12 for its products, N / 4 lanes' and D x's sums."""
    i = scan_inputs(T + N, "fp32", B, T, D, N, G, DEV)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    y, end, ck = ssm.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"], return_state=True, return_checkpoints=True)
    ref, rend, _ = ol.ssm_scan(*a, i["D"], i["dt_bias"], state=i["state"])
    x, dt, A, Bm, Cm = (t.double().cpu() for t in a)
    bias, st, gy, gf = (i[k].double().cpu() for k in ("dt_bias", "state", "gy", "gf"))
    spread = lambda m: m.repeat_interleave(D // G, -2)  # noqa: E731
    Bm, Cm = spread(Bm).abs(), spread(Cm).abs()
    delta = ol.softplus(dt + bias)
    steps = 2 * (dt.abs() + bias.abs()) + 16
    h, e, by = st.abs(), torch.zeros_like(st), torch.zeros_like(x)
    for t in range(T):
        z = delta[:, t, :, None] * A
        f, u = torch.exp(z), (delta[:, t] * x[:, t].abs())[..., None] * Bm[:, t]
        e = f * e + f * h * (z.abs() * (steps[:, t, :, None] + 18) + 4) + u * (steps[:, t, :, None] + 4) + (f * h + u)
        h = f * h + u
        m = (h * Cm[:, t]).sum(-1) + (i["D"].double().cpu() * x[:, t]).abs()
        by[:, t] = (e * Cm[:, t]).sum(-1) + 12 * m
    _bounded(end, rend, e, "state")
    _bounded(y, ref, by, "y")
    # the gradient of the first state, the same from the other end
    got = ssm.ssm_scan_backward(i["gy"], *a, ck, i["D"], i["dt_bias"], grad_final_state=i["gf"])[7]
    want = ol.ssm_scan_backward(i["gy"], *a, i["D"], i["dt_bias"], state=i["state"], grad_final_state=i["gf"])[7]
    c, e = gf.abs(), torch.zeros_like(gf)
    for t in reversed(range(T)):
        z = delta[:, t, :, None] * A
        f, u = torch.exp(z), gy[:, t, :, None].abs() * Cm[:, t]
        e = f * (e + u + (c + u) * (z.abs() * (steps[:, t, :, None] + 18) + 4 + 2))
        c = f * (c + u)
    _bounded(got, want, e, "grad state")


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------
def test_backward_of_more_than_two_to_the_31_values():
    """Activations, checkpoints and gradients of more than 2^31 values: the gradients at the end are those of a run that starts there."""
    T, D, N, cut = 1_100_000, 2048, 16, 1_099_008
    r = lambda *s: torch.randn(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
    x, gy = r(1, T, D), r(1, T, D)
    dt = r(1, T, 1).expand(1, T, D).contiguous()
    A = -torch.rand(D, N, device=DEV) - 0.5
    B, C = r(1, T, 1, N), r(1, T, 1, N)
    y, ck = ssm.ssm_scan(x, dt, A, B, C, return_checkpoints=True)
    assert min(t.numel() for t in (x, y, ck)) > 2 ** 31
    del y
    got = ssm.ssm_scan_backward(gy, x, dt, A, B, C, ck)
    tail = (x[:, cut:], dt[:, cut:], A, B[:, cut:], C[:, cut:])
    _, ct = ssm.ssm_scan(*tail, state=ck[:, cut // 16].contiguous(), return_checkpoints=True)
    want = ssm.ssm_scan_backward(gy[:, cut:], *tail, ct)
    for k in (0, 1, 3, 4):      # two roundings to bf16 of the same sums
        assert rel(got[k][:, cut:], want[k]) <= 2 ** -8, k
    assert all(torch.isfinite(got[k]).all() for k in (2, 7))
    del got, want, ck, ct, dt, B, C
    res, gate, gn = r(1, T, D), r(1, T, D), r(1, T, D)
    w = torch.ones(D, device=DEV)
    kw = dict(post_weight=w, scale=w, pre_weight=w)
    _, _, stats = glue.norm_gate_residual(x, res, gate, return_stats=True, **kw)
    got = glue.norm_gate_residual_backward(gy, gn, x, stats, res, gate, **kw)
    want = glue.norm_gate_residual_backward(gy[:, cut:], gn[:, cut:], x[:, cut:], stats[cut:], res[:, cut:], gate[:, cut:], **kw)
    for k in range(3):
        assert torch.equal(got[k][:, cut:], want[k]), k


# ---- captured steps, first calls in a capture, other streams ----------------------------------------------------------------
def test_captured_steps_follow_their_slots():
    """Steps captured once and replayed with other tokens and slots, among them padding and a slot that is named twice."""
    B, S, D, N, K = 5, 8, 72, 16, 4
    g = gen(21)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    A, w, b, skip, bias, one = -r(D, N).abs(), r(D, K), r(D), r(D), r(D) - 3, torch.ones(D, device=DEV)
    static = dict(x=r(B, D), dt=r(B, D), B=r(B, 1, N), C=r(B, 1, N), slots=torch.zeros(B, dtype=torch.int32, device=DEV))
    start = (r(S, K - 1, D), r(S, D, N))

    def run(i, ctable, table):
        u = ssm.short_conv_step(i["x"], ctable, w, b, activation="silu", slots=i["slots"])
        y = ssm.ssm_scan_step(u, i["dt"], A, i["B"], i["C"], table, skip, bias, slots=i["slots"])
        return (y, *glue.norm_gate_residual(y, i["x"], u, post_weight=one, scale=one, pre_weight=one))

    steps = [{**{k: r(*v.shape) for k, v in static.items() if k != "slots"}, "slots": torch.tensor(s, dtype=torch.int32, device=DEV)}
             for s in ([0, 1, 2, 3, 4], [7, -1, 3, 3, 0], [S, 5, 3, 0, 5], [-2, S + 1, -1, 99, -1])]
    tables = [t.clone() for t in start]
    run(static, *tables)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static, *tables)
    for t, s in zip(tables, start):
        t.copy_(s)
    eager = [t.clone() for t in start]
    for i in steps:
        for k, v in i.items():
            static[k].copy_(v)
        graph.replay()
        want = run(i, *eager)
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        assert all(torch.equal(p, q) for p, q in zip(tables, eager))


def test_first_calls_of_a_process_in_a_capture():
    """Nothing has been loaded or allowed yet when the capture begins; the rows need more than 48 KB of shared memory."""
    code = """
import torch
from ttt_tk_b200 import glue, ssm
o, gx = (torch.randn(3, 8188, device="cuda") for _ in range(2))
w = torch.rand(8188, device="cuda") + 0.5
x = torch.randn(2, 300, 64, device="cuda"); c = torch.randn(64, 4, device="cuda")
A = -torch.rand(64, 16, device="cuda"); B = torch.randn(2, 300, 1, 16, device="cuda")
def run():
    z, n, st = glue.norm_gate_residual(o, o, o, post_weight=w, scale=w, pre_weight=w, return_stats=True)
    g = glue.norm_gate_residual_backward(gx, n, o, st, o, o, post_weight=w, scale=w, pre_weight=w)
    y, ck = ssm.ssm_scan(ssm.short_conv(x, c), x, A, B, B, return_checkpoints=True)
    s = ssm.ssm_scan_backward(y, x, x, A, B, B, ck)
    return [t for t in (z, n, *g, y, *s, *ssm.short_conv_backward(y, x, c)) if t is not None]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(got, want))
print("as eager")
"""
    root = os.path.join(os.path.dirname(__file__), "..")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as eager" in r.stdout, r.stderr[-2000:]


def test_conv_and_block_end_on_streams_of_their_own():
    i = conv_inputs(5, "bf16", 2, 700, 512, 4, DEV)
    w = torch.ones(512, device=DEV)

    def run():
        u = ssm.short_conv(i["x"], i["weight"], i["bias"], activation="silu", state=i["state"])
        z, n, st = glue.norm_gate_residual(u, i["x"], i["gy"], return_stats=True, post_weight=w, scale=w, pre_weight=w)
        g = glue.norm_gate_residual_backward(z, n, u, st, i["x"], i["gy"], post_weight=w, scale=w, pre_weight=w)
        return [u, z, n, *[t for t in g if t is not None],
                *ssm.short_conv_backward(g[0], i["x"], i["weight"], i["bias"], activation="silu", state=i["state"])]

    want = run()
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want))
