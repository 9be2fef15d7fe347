"""What the gated linear recurrence refuses, before anything is launched; a call that is right in all else ends with the device's message."""
import ctypes

import pytest
import torch

from gated_cases import gated_inputs
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import ssm

BF = torch.bfloat16


def _args(**kw):
    i = gated_inputs(1, "bf16", 2, 70, 8)
    return {**{k: i[k] for k in ("x", "gate", "A", "input_gate", "gate_bias", "input_bias", "state")}, **kw}


BAD = [
    ({}, "CUDA"),
    ({"x": torch.zeros(2, 8, dtype=BF)}, "B, T, D"),
    ({"x": torch.zeros(2, 70, 8, dtype=torch.float64)}, "bfloat16"),
    ({"x": torch.zeros(2, 70, 16, dtype=BF)[..., ::2]}, "contiguous"),
    ({"gate": torch.zeros(2, 70, 7, dtype=BF)}, "gate must be"),
    ({"gate": torch.zeros(2, 70, 8)}, "gate must have type"),
    ({"gate": None}, "gate must be a tensor"),
    ({"input_gate": torch.zeros(1, 70, 8, dtype=BF)}, "input_gate must be"),
    ({"input_gate": None}, "input_bias needs input_gate"),
    ({"A": torch.zeros(7)}, "A must be"),
    ({"A": torch.zeros(8, dtype=BF)}, "A must have"),
    ({"A": torch.zeros(16)[::2]}, "contiguous"),
    ({"gate_bias": torch.zeros(8, 1)}, "gate_bias"),
    ({"input_bias": torch.zeros(9)}, "input_bias"),
    ({"state": torch.zeros(2, 8, dtype=BF)}, "state"),
    ({"state": torch.zeros(1, 8)}, "state"),
    ({"lengths": torch.zeros(2, dtype=torch.int64)}, "lengths"),
    ({"mix": "mean"}, "mix must be"),
    ({"mix": ["sqrt"]}, "mix must be"),
    ({"mix": 1}, "mix must be"),
]


@pytest.mark.parametrize("kw,msg", BAD)
def test_gated_scan(kw, msg):
    with pytest.raises(ValueError, match=msg):
        ssm.gated_scan(**_args(**kw))


@pytest.mark.parametrize("name", ["x", "gate", "A", "input_gate", "gate_bias", "input_bias", "state", "lengths"])
@pytest.mark.parametrize("kind", [3, [1.0], "x", torch.zeros(())])
def test_differentiable_form_takes_no_other_kinds(name, kind):
    with pytest.raises(ValueError):
        ag.gated_scan(**_args(**{name: kind}))


def test_backward():
    i = gated_inputs(1, "bf16", 2, 70, 8)
    a = [i[k] for k in ("A", "input_gate", "gate_bias", "input_bias")]
    ck = torch.zeros(2, 2, 8)
    for gy, c, msg in ((i["gy"].float(), ck, "grad_y"), (i["gy"][:, :5], ck, "grad_y"), (i["gy"], ck[:, :1], "checkpoints"), (i["gy"], None, "checkpoints"),
                       (i["gy"], ck.bfloat16(), "checkpoints"), (i["gy"], ck, "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ssm.gated_scan_backward(gy, i["x"], i["gate"], c, *a)
    with pytest.raises(ValueError, match="grad_final_state"):
        ssm.gated_scan_backward(i["gy"], i["x"], i["gate"], ck, *a, grad_final_state=torch.zeros(2, 7))


def test_backward_from_8_bits():
    i = gated_inputs(1, "bf16", 2, 70, 130)
    q = torch.zeros(2, 70, 130, dtype=torch.float8_e4m3fn)
    ck = torch.zeros(2, 2, 130)
    s128, s64 = torch.ones(2, 70, 2), torch.ones(2, 70, 3)
    call = lambda x, g, ig=None: ssm.gated_scan_backward(i["gy"], x, g, ck, i["A"], ig)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        call((q, s128), (q, s128), (q, s128))
    for x, g, ig, msg in (((q, s128), (q, s64), None, "same for all"), ((q, s128), i["gate"], None, "as the other inputs"), ((q,), (q, s128), None, "as the other inputs"),
                          ((q[:, :5], s128), (q, s128), None, "x must be"), ((q.view(torch.uint8), s128), (q, s128), None, "x must have type"),
                          ((q, s128.bfloat16()), (q, s128), None, "float32"), ((q, torch.ones(2, 70, 4)), (q, s128), None, "scales"),
                          ((q, s128), (q, s128), i["input_gate"], "input_gate must be \\(values"), ((q, 1.0), (q, s128), None, "tensor")):
        with pytest.raises(ValueError, match=msg):
            call(x, g, ig)
    with pytest.raises(ValueError):
        call(i["x"], (q, s128))


def test_step():
    i = gated_inputs(1, "bf16", 2, 1, 8)
    x, g = i["x"][:, 0], i["gate"][:, 0]
    for st, kw, msg in ((torch.zeros(3, 8), {}, "row for each"), (torch.zeros(2, 7), {}, "state must be"), (torch.zeros(2, 8, 1), {}, "dimensions"),
                        (torch.zeros(2, 8, dtype=BF), {}, "state must have"), (torch.zeros(0, 8), {"slots": torch.zeros(2, dtype=torch.int32)}, "no rows"),
                        (torch.zeros(8, 2).t(), {}, "contiguous"), (torch.zeros(3, 8), {"slots": torch.zeros(2)}, "slots"), (torch.zeros(2, 8), {}, "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ssm.gated_scan_step(x, g, st, i["A"], **kw)
    with pytest.raises(ValueError, match="B, D"):
        ssm.gated_scan_step(i["x"], i["gate"], torch.zeros(2, 8))


def test_sizes_that_indices_could_not_hold():
    x = torch.zeros(1, 1, 1, dtype=BF).expand(1, (1 << 30) + 1, 1)
    with pytest.raises(ValueError, match="too large"):
        ssm.gated_scan(x, x)


def test_the_c_abi_refuses_null_and_bad_sizes():
    from ttt_tk_b200 import _lib
    lib = _lib.lib()
    for name in ("gated_scan", "gated_scan_backward", "gated_scan_step"):
        fn = getattr(lib, "ttt_b200_" + name)
        fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        assert fn(None, None) == 1
        assert b"NULL" in lib.ttt_b200_last_error()
        assert fn(ctypes.byref(ctypes.create_string_buffer(1024)), None) == 1      # a struct of zeros
