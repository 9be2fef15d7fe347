"""The gated linear recurrence on the GPU against its statement in 64 bits."""
import itertools

import pytest
import torch

from gated_cases import ARGS, GRADS, close, gated_inputs, hold, run_both
from oracle import gated as og

pytestmark = pytest.mark.gpu


def _run(seed, ty, B, T, D, mix="sqrt", **kw):
    i = gated_inputs(seed, ty, B, T, D, "cuda", **kw)
    hold(i, mix, run_both(i, mix), f"{ty} {B} x {T} x {D}")


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 7, 2), (1, 8, 63), (2, 9, 64), (3, 63, 65), (1, 64, 130), (2, 65, 6), (1, 200, 96), (2, 513, 33)])
def test_sizes(ty, B, T, D):
    _run(T, ty, B, T, D)


@pytest.mark.parametrize("mix", ["sqrt", "linear", None])
@pytest.mark.parametrize("A,igate,bias,state", list(itertools.product([True, False], repeat=4)))
def test_parts(mix, A, igate, bias, state):
    _run(1, "fp32", 2, 80, 34, mix, A=A, igate=igate, bias=bias, state=state)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", ["wide", "odd", "time"])
@pytest.mark.parametrize("D", [64, 72, 75])
def test_strides(ty, rows, D):
    _run(2, ty, 3, 70, D, rows=rows)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("lengths", [[0, 1, 150], [64, 65, 63], [0, 0, 0], [150, 128, 129], [-5, 1000, 8]])
def test_ragged(ty, lengths):
    """Tokens behind a sequence are not read: they hold NaN and infinities here, those of the gradient too."""
    i = gated_inputs(4, ty, 3, 150, 70, "cuda", lengths=lengths)
    n = og.lengths_of(i["lengths"], 3, 150)
    for k in ("x", "gate", "input_gate", "gy"):
        for b in range(3):
            i[k][b, n[b]:] = float("nan")
            i[k][b, n[b] + 1:] = float("inf")
    got = run_both(i, "sqrt")
    for b in range(3):
        for v in (got[0], *[got[2][k] for k in ("x", "gate", "input_gate")]):
            assert (v[b, n[b]:] == 0).all()
    clean = {k: torch.nan_to_num(v, 0.0, 0.0, 0.0) if k in ("x", "gate", "input_gate", "gy") else v for k, v in i.items()}
    hold(clean, "sqrt", got, str(lengths))


def test_far_gates():
    """Gates far from zero on both sides, infinities among them: a state is held, or let go of."""
    i = gated_inputs(6, "fp32", 1, 40, 64, "cuda", bias=False)
    far = torch.tensor([-1e30, -300.0, -88.0, -40.0, -12.0, 12.0, 40.0, 88.0, 300.0, 1e30], device="cuda")
    i["gate"][0, 5:15] = far[:, None]
    i["input_gate"][0, 10:20] = far[:, None]
    for mix in ("sqrt", "linear", None):
        hold(i, mix, run_both(i, mix), f"far {mix}")
    j = dict(i, A=None)
    for mix in ("sqrt", "linear", None):
        hold(j, mix, run_both(j, mix), f"far without A {mix}")


def test_a_gate_of_minus_infinity_holds_the_state():
    i = gated_inputs(7, "bf16", 2, 130, 64, "cuda")
    i["gate"][:, 30:] = float("-inf")
    y, end, g = run_both(i, "sqrt")
    assert (y[:, 30:] == y[:, 29:30]).all() and torch.equal(end.bfloat16(), y[:, -1])
    assert all(v.isfinite().all() for v in g.values())
    assert (g["x"][:, 30:] == 0).all() and (g["gate"][:, 30:] == 0).all() and (g["input_gate"][:, 30:] == 0).all()


def test_a_of_zero_above_and_far_below():
    i = gated_inputs(8, "fp32", 2, 70, 64, "cuda")
    i["A"][:4] = torch.tensor([0.0, 1.5, -100.0, -1e4])
    hold(i, "linear", run_both(i, "linear"), "A")
    y, _, g = run_both(i, "sqrt")
    assert y.isfinite().all() and all(v.isfinite().all() for v in g.values()) and g["A"][1] == 0
    assert torch.equal(y[:, :, 0], i["state"][:, None, 0].expand(2, 70))      # a = 1: nothing comes in, nothing goes


def test_nan_reaches_what_follows_and_nothing_else():
    for k in ("x", "gate", "input_gate"):
        i = gated_inputs(9, "bf16", 2, 200, 70, "cuda")
        i[k][1, 90, 33] = float("nan")
        y, end, _ = run_both(i, "sqrt")
        bad = y.isnan()
        assert bad[1, 90:, 33].all() and int(bad.sum()) == 110 and end[1, 33].isnan() and int(end.isnan().sum()) == 1


@pytest.mark.parametrize("B,T,D", [(1, 3000, 64), (1, 1100, 200), (2, 700, 64)])
def test_few_channels_and_long_sequences(B, T, D):
    """Tiles behind one another in the CTAs of a cluster, the last round of them not full."""
    _run(10, "bf16", B, T, D, lengths=[T - 37] * B)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
def test_chunks_without_tokens(ty):
    """Long sequences in chunks beside short and empty ones, whose later chunks have nothing."""
    _run(19, ty, 4, 1500, 70, lengths=[1500, 700, 1, 0])
    _run(20, ty, 3, 900, 128, "linear", A=False, lengths=[130, 900, 64], rows="wide")


def test_expanded_inputs():
    """One gate for all tokens, one sequence for the batch."""
    i = gated_inputs(21, "bf16", 3, 300, 66, "cuda")
    i["gate"] = i["gate"][:, :1].expand(3, 300, 66)
    i["x"] = i["x"][:1].expand(3, 300, 66)
    hold(i, "sqrt", run_both(i, "sqrt"), "expanded")


def test_a_long_sequence_keeps_its_precision():
    i = gated_inputs(11, "fp32", 1, 5000, 64, "cuda")
    i["A"][:] = -1e-3
    hold(i, "sqrt", run_both(i, "sqrt"), "long")


def test_pieces_are_the_whole():
    """A sequence in pieces, the state handed on, is the whole sequence, gradients too."""
    i = gated_inputs(12, "fp32", 2, 300, 66, "cuda")
    whole = run_both(i, "sqrt")
    parts, cut, st = [], [0, 1, 65, 200, 300], i["state"]
    for a, b in zip(cut, cut[1:]):
        p = dict(i, state=st, **{k: i[k][:, a:b] for k in ("x", "gate", "input_gate", "gy")})
        parts.append(p)
        st = run_both(dict(p, gf=None), "sqrt")[1]
    gf, gx = i["gf"], []
    for p in reversed(parts):
        _, _, g = run_both(dict(p, gf=gf), "sqrt")
        gf = g["state"]
        gx.insert(0, g["x"])
    torch.testing.assert_close(st, whole[1], rtol=2e-5, atol=2e-5)
    torch.testing.assert_close(torch.cat(gx, 1), whole[2]["x"], rtol=2e-5, atol=2e-5)
    torch.testing.assert_close(gf, whole[2]["state"], rtol=2e-5, atol=2e-5)


def test_the_same_call_gives_the_same_bits():
    for shape in ((2, 900, 70), (1, 2000, 64)):
        i = gated_inputs(13, "bf16", *shape, "cuda")
        first = run_both(i, "sqrt")
        for _ in range(3):
            again = run_both(i, "sqrt")
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
            assert all(torch.equal(first[2][k], again[2][k]) for k in GRADS)


def test_no_tokens_and_no_sequences():
    from ttt_tk_b200 import ssm
    for B, T in ((0, 5), (2, 0)):
        i = gated_inputs(14, "bf16", B, T, 64, "cuda")
        y, end, g = run_both(i, "sqrt")
        assert y.shape == (B, T, 64) and torch.equal(end, i["state"]) and torch.equal(g["state"], i["gf"])
        assert (g["A"] == 0).all() and (g["gate_bias"] == 0).all()
        assert ssm.gated_scan(i["x"], i["gate"]).shape == (B, T, 64)


def _step_inputs(ty, B, S, D, **kw):
    i = gated_inputs(15, ty, B, 1, D, "cuda", **kw)
    i = {k: v[:, 0] if isinstance(v, torch.Tensor) and v.dim() == 3 else v for k, v in i.items()}
    i["state"] = torch.randn(S, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    return i


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,D,rows", [(1, 1, "whole"), (8, 2048, "wide"), (5, 77, "odd"), (3, 258, "whole")])
@pytest.mark.parametrize("mix,A", [("sqrt", True), ("linear", False), (None, True)])
def test_step(ty, B, D, rows, mix, A):
    from ttt_tk_b200 import ssm
    i = _step_inputs(ty, B, B + 4, D, A=A, rows=rows)
    slots = torch.randperm(B + 4, generator=torch.Generator().manual_seed(2))[:B].to(torch.int32).cuda()
    table = i["state"].clone()
    y = ssm.gated_scan_step(i["x"], i["gate"], table, *[i[k] for k in ARGS], mix=mix, slots=slots)
    one = lambda k: None if i[k] is None else i[k][:, None]  # noqa: E731
    ya, end, _ = og.gated_scan(one("x"), one("gate"), i["A"], one("input_gate"), i["gate_bias"], i["input_bias"], mix, i["state"][slots.long()])
    close(y[:, None], ya, "y")
    close(table[slots.long()], end, "state")
    rest = torch.ones(B + 4, dtype=torch.bool)
    rest[slots.long().cpu()] = False
    assert torch.equal(table[rest.cuda()], i["state"][rest.cuda()])


def test_step_without_slots_and_with_padding_and_repeats():
    from ttt_tk_b200 import ssm
    i = _step_inputs("bf16", 6, 6, 130)
    a = [i[k] for k in ARGS]
    table = i["state"].clone()
    plain = ssm.gated_scan_step(i["x"], i["gate"], table, *a)
    by_slot = i["state"].clone()
    assert torch.equal(ssm.gated_scan_step(i["x"], i["gate"], by_slot, *a, slots=torch.arange(6, dtype=torch.int32, device="cuda")), plain)
    assert torch.equal(by_slot, table)
    # rows 0, 2 and 5 are tokens after one another of slot 3; rows 1 and 4 are padding
    slots = torch.tensor([3, -1, 3, 0, 6, 3], dtype=torch.int32, device="cuda")
    table = i["state"].clone()
    y = ssm.gated_scan_step(i["x"], i["gate"], table, *a, slots=slots)
    assert (y[1] == 0).all() and (y[4] == 0).all()
    pick = [0, 2, 5]
    seq = lambda k: i[k][pick][None]  # noqa: E731
    ya, end, _ = og.gated_scan(seq("x"), seq("gate"), i["A"], seq("input_gate"), i["gate_bias"], i["input_bias"], "sqrt", i["state"][3:4])
    close(y[pick][None], ya, "y")
    close(table[3:4], end, "state")
    assert torch.equal(table[[1, 2, 4, 5]], i["state"][[1, 2, 4, 5]])


def test_steps_are_the_scan():
    from ttt_tk_b200 import ssm
    i = gated_inputs(16, "bf16", 2, 40, 96, "cuda")
    a = [i[k] for k in ARGS]
    y, end = ssm.gated_scan(i["x"], i["gate"], *a, state=i["state"], return_state=True)
    st = i["state"].clone()
    for t in range(40):
        z = ssm.gated_scan_step(i["x"][:, t], i["gate"][:, t], st, i["A"], i["input_gate"][:, t], i["gate_bias"], i["input_bias"])
        torch.testing.assert_close(z.float(), y[:, t].float(), rtol=1e-2, atol=1e-2)
    torch.testing.assert_close(st, end, rtol=2e-5, atol=2e-5)


def test_another_stream_and_a_graph():
    i = gated_inputs(17, "bf16", 2, 300, 64, "cuda")
    want = run_both(i, "sqrt")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_both(i, "sqrt")
    s.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[2][k], want[2][k]) for k in GRADS)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run_both(i, "sqrt")
    j = gated_inputs(18, "bf16", 2, 300, 64, "cuda")
    for k in ("x", "gate", "input_gate", "gy", "state", "gf", "A", "gate_bias", "input_bias"):
        i[k].copy_(j[k])
    g.replay()
    want = run_both(j, "sqrt")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and all(torch.equal(got[2][k], want[2][k]) for k in GRADS)


def test_more_values_than_31_bits_count():
    """One sequence of 2^31 + values; its end is that of its last piece by itself, from the state in front of it."""
    from ttt_tk_b200 import ssm
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    D, T = 65536, 32768 + 70
    x = torch.randn(1, 64, D, device="cuda", dtype=torch.bfloat16).repeat(1, T // 64 + 1, 1)[:, :T]
    g = torch.full((1, 1, D), 0.5, device="cuda", dtype=torch.bfloat16).expand(1, T, D)
    A = -torch.rand(D, device="cuda")
    y, end, ck = ssm.gated_scan(x, g, A, return_state=True, return_checkpoints=True)
    at = T // 64 * 64 - 64
    y2, end2 = ssm.gated_scan(x[:, at:], g[:, at:], A, state=ck[:, at // 64], return_state=True)
    assert torch.equal(y[:, at:], y2) and torch.equal(end, end2)
    gy = torch.randn(1, 64, D, device="cuda", dtype=torch.bfloat16).repeat(1, T // 64 + 1, 1)[:, :T]
    gx = ssm.gated_scan_backward(gy, x, g, ck, A)[0]
    gx2 = ssm.gated_scan_backward(gy[:, at:], x[:, at:], g[:, at:], ck[:, at // 64:], A)[0]
    assert torch.equal(gx[:, at:], gx2)

