"""The gated recurrence, activations in 8 bits, the norm into 8 bits and rows of tables where calls meet: captured steps whose slots change, first calls of a
process inside a capture, several streams and host threads at once, states that no token may change, tensors beyond 2^31 values."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from gated_cases import ARGS, GRADS, gated_inputs, run_both
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, saved, ssm, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("ty,B,T,D", [("bf16", 2, 16, 64), ("fp32", 2, 333, 20), ("bf16", 3, 1500, 64), ("fp16", 1, 400, 130)])
def test_no_token_changes_no_bit_of_a_state(ty, B, T, D):
    i = gated_inputs(T, ty, B, T, D, DEV, lengths=[0] * B)
    y, end, g = run_both(i, "sqrt")
    assert torch.equal(end, i["state"]) and (y == 0).all()
    assert torch.equal(g.pop("state"), i["gf"]) and all((v == 0).all() for v in g.values())


@pytest.mark.parametrize("T,n", [(64, 9), (128, 120), (300, 290), (1500, 1490)])
def test_tokens_behind_a_sequence_change_no_bit(T, n):
    """As many tiles with and without the tokens behind: the same chunks, the same bits."""
    i = gated_inputs(n, "bf16", 2, T, 66, DEV, lengths=[n, n])
    y, end, g = run_both(i, "sqrt")
    j = dict(i, lengths=None, **{k: i[k][:, :n] for k in ("x", "gate", "input_gate", "gy")})
    y1, end1, g1 = run_both(j, "sqrt")
    assert torch.equal(end, end1) and torch.equal(y[:, :n], y1) and (y[:, n:] == 0).all()
    for k in GRADS:
        v = g[k][:, :n] if g[k].dim() == 3 else g[k]
        assert torch.equal(v, g1[k]), k


def test_captured_steps_follow_their_slots():
    B, S, D = 5, 8, 72
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    A, w = -r(D).abs(), r(D, 4)
    static = dict(x=r(B, D), gate=r(B, D), ig=r(B, D), slots=torch.zeros(B, dtype=torch.int32, device=DEV),
                  source=torch.zeros(2, dtype=torch.int32, device=DEV), target=torch.zeros(2, dtype=torch.int32, device=DEV))
    start = (r(S, 3, D), r(S, D))

    def run(i, windows, states):
        tables.copy_rows((windows, states), i["source"], i["target"])
        u = ssm.short_conv_step(i["x"], windows, w, slots=i["slots"])
        y = ssm.gated_scan_step(u, i["gate"], states, A, i["ig"], slots=i["slots"])
        return (y, *glue.norm_residual_8bit(y, i["x"], weight=A, group=32)[::2])

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    steps = [dict({k: r(B, D) for k in ("x", "gate", "ig")}, slots=i32(s), source=i32(a), target=i32(b))
             for s, a, b in (([0, 1, 2, 3, 4], [0, 0], [5, 6]), ([7, -1, 3, 3, 0], [1, 2], [2, 1]), ([S, 5, 3, 0, 5], [-1, 4], [3, 9]))]
    both = [t.clone() for t in start]
    run(static, *both)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static, *both)
    for t, s in zip(both, start):
        t.copy_(s)
    eager = [t.clone() for t in start]
    for i in steps:
        for k, v in i.items():
            static[k].copy_(v)
        graph.replay()
        want = run(i, *eager)
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(out, want))
        assert all(torch.equal(p, q) for p, q in zip(both, eager))


def test_first_calls_of_a_process_in_a_capture():
    """Nothing has been loaded or allowed yet when the capture begins; the kernels need more than 48 KB of shared memory, and a long sequence scratch."""
    code = """
import torch
from ttt_tk_b200 import glue, saved, ssm, tables
x, g, i, gy = (torch.randn(1, 1200, 64, device="cuda") for _ in range(4))
A = -torch.rand(64, device="cuda")
t = torch.randn(3000, 40, device="cuda"); s = torch.arange(2000, dtype=torch.int32, device="cuda"); d = torch.flip(s, (0,)).contiguous()
used = torch.rand(3000, device="cuda") < 0.5
def run(t):
    y, ck = ssm.gated_scan(x, g, A, i, return_checkpoints=True)
    p = saved.pack8(x, g, i)
    out = [y, *ssm.gated_scan_backward(gy, x, g, ck, A, i), *ssm.gated_scan_backward(gy, p[0], p[1], ck, A, p[2]), *saved.unpack8(*p)]
    z, q, sc = glue.norm_residual_8bit(y, x, weight=A)
    tables.copy_rows(t, s, d)
    return [v for v in (*out, z, q.float(), sc, tables.compact_rows(t, used)) if v is not None]
t1 = t.clone()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run(t1)
graph.replay()
want = run(t)
torch.cuda.synchronize()
assert torch.equal(t, t1) and all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(got, want))
print("as eager")
"""
    root = os.path.join(os.path.dirname(__file__), "..")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as eager" in r.stdout, r.stderr[-2000:]


def _all_of(i):
    y, end, g = run_both(i, "sqrt")
    p = saved.pack8(i["x"], i["gate"])
    return [y, end, *[g[k] for k in GRADS], *saved.unpack8(*p), *glue.norm_residual_8bit(y, i["x"], weight=i["A"])[::2]]


def test_several_streams_at_once():
    cases = [gated_inputs(k, "bf16", 2, T, 64, DEV) for k, T in enumerate((300, 1500, 77))]
    want = [_all_of(i) for i in cases]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(5):
        for s, i in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append(_all_of(i))
    torch.cuda.synchronize()
    for n, o in enumerate(outs):
        assert all(torch.equal(p, q) for p, q in zip(o, want[n % 3]))


def test_several_threads_at_once():
    """Host threads whose calls need different amounts of shared memory."""
    cases = [gated_inputs(k, ty, 2, T, D, DEV) for k, (ty, T, D) in enumerate((("fp32", 700, 130), ("bf16", 200, 64), ("fp16", 90, 33)))]
    want = [_all_of(i) for i in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got = _all_of(cases[k])
                s.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[k])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_autograd_captured_after_an_eager_pass():
    i = gated_inputs(3, "bf16", 1, 140, 64, DEV)
    lv = [i[k].clone().requires_grad_(True) for k in ("x", "gate", *ARGS)]

    def step():
        y = ag.gated_scan(*lv, saved="e4m3")
        return torch.autograd.grad(y.float().sum(), lv)

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


def test_norm_of_more_than_two_to_the_31_values():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    M, D = (1 << 18) + 40, 8192
    o = torch.randn(64, D, device=DEV, dtype=torch.bfloat16).repeat(M // 64 + 1, 1)[:M]
    w = torch.rand(D, device=DEV) + 0.5
    x, q, s = glue.norm_residual_8bit(o, o, weight=w, group=128)
    at = M // 64 * 64
    x2, q2, s2 = glue.norm_residual_8bit(o[at:], o[at:], weight=w, group=128)
    assert torch.equal(x[at:], x2) and torch.equal(q[at:].float(), q2.float()) and torch.equal(s[at:], s2)
    assert torch.equal(saved.unpack8((q, s))[0][at:], saved.unpack8((q2, s2))[0])
