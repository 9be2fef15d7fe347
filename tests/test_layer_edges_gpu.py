"""The layer-side sequence operators at the ends of their ranges and where calls meet.
Statements: oracle/layer.py; tolerances: tests/layer_cases.py."""
import ctypes
import struct
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
