"""What the layer-side sequence operators refuse, before anything is launched.  Shapes and types are checked before devices, so these
run without a GPU; a call that is right in all else ends with the device's message.  (No compute calls here.)"""
import pytest
import torch

from layer_cases import conv_inputs, scan_inputs
from ttt_tk_b200 import glue, ssm

BF, F32 = torch.bfloat16, torch.float32


def _conv(**kw):
    i = conv_inputs(1, "bf16", 2, 64, 64, 4)
    a = dict(x=i["x"], weight=i["weight"], bias=i["bias"], state=i["state"])
    a.update(kw)
    return ssm.short_conv(a.pop("x"), a.pop("weight"), a.pop("bias"), **a)


@pytest.mark.parametrize("kw,msg", [
    ({}, "CUDA"),
    ({"x": torch.zeros(2, 64, dtype=BF)}, "B, T, D"),
    ({"x": torch.zeros(2, 64, 64, dtype=torch.float64)}, "bfloat16"),
    ({"x": torch.zeros(2, 64, 64, dtype=torch.int32)}, "bfloat16"),
    ({"x": torch.zeros(2, 64, 64, dtype=BF).transpose(1, 2)}, "contiguous"),
    ({"x": None}, "tensor"),
    ({"weight": torch.zeros(64, 5)}, "K = 2, 3 or 4"),
    ({"weight": torch.zeros(64, 1)}, "K = 2, 3 or 4"),
    ({"weight": torch.zeros(63, 4)}, "weight"),
    ({"weight": torch.zeros(64, 4, dtype=BF)}, "weight"),
    ({"weight": torch.zeros(4, 64).t()}, "contiguous"),
    ({"weight": None}, "weight"),
    ({"bias": torch.zeros(63)}, "bias"),
    ({"state": torch.zeros(2, 4, 64, dtype=BF)}, "state"),
    ({"state": torch.zeros(2, 3, 64)}, "state"),
    ({"lengths": torch.zeros(2, dtype=torch.int64)}, "lengths"),
    ({"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
    ({"activation": "gelu"}, "activation"),
    ({"x": torch.zeros(2, 63, 64, dtype=BF), "heads": True}, "multiples of 64"),
    ({"x": torch.zeros(2, 64, 64, dtype=BF)[..., :32], "weight": torch.zeros(32, 4), "bias": None, "state": None, "heads": True}, "multiples of 64"),
])
def test_short_conv(kw, msg):
    with pytest.raises(ValueError, match=msg):
        _conv(**kw)


def test_short_conv_backward_and_step():
    i = conv_inputs(1, "bf16", 2, 64, 64, 4)
    with pytest.raises(ValueError, match="grad_y"):
        ssm.short_conv_backward(i["gy"][:, :3], i["x"], i["weight"])
    with pytest.raises(ValueError, match="grad_y"):
        ssm.short_conv_backward(i["gy"], i["x"], i["weight"], heads=True)
    with pytest.raises(ValueError, match="grad_final_state"):
        ssm.short_conv_backward(i["gy"], i["x"], i["weight"], grad_final_state=i["gf"].float())
    st, x = torch.zeros(5, 3, 64, dtype=BF), i["x"][:, 0]
    with pytest.raises(ValueError, match="row for each"):
        ssm.short_conv_step(x, st, i["weight"])
    with pytest.raises(ValueError, match="slots"):
        ssm.short_conv_step(x, st, i["weight"], slots=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="slots"):
        ssm.short_conv_step(x, st, i["weight"], slots=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="state"):
        ssm.short_conv_step(x, st[:, :2], i["weight"], slots=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="contiguous"):
        ssm.short_conv_step(x, torch.zeros(5, 64, 3, dtype=BF).transpose(1, 2), i["weight"], slots=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="no rows"):
        ssm.short_conv_step(x, st[:0], i["weight"], slots=torch.zeros(2, dtype=torch.int32))


def _scan(**kw):
    i = scan_inputs(1, "bf16", 2, 5, 8, 4, 2)
    a = {k: i[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "state")}
    a.update(kw)
    return ssm.ssm_scan(*[a.pop(k) for k in ("x", "dt", "A", "B", "C", "D", "dt_bias")], **a)


@pytest.mark.parametrize("kw,msg", [
    ({}, "CUDA"),
    ({"x": torch.zeros(2, 5, 8, dtype=torch.float64)}, "bfloat16"),
    ({"dt": torch.zeros(2, 5, 8)}, "dt"),
    ({"dt": torch.zeros(2, 5, 7, dtype=BF)}, "dt"),
    ({"A": torch.zeros(8, 65)}, "1 to 64"),
    ({"A": torch.zeros(8, 0)}, "1 to 64"),
    ({"A": torch.zeros(8, 4, dtype=BF)}, "A"),
    ({"A": torch.zeros(7, 4)}, "A"),
    ({"B": torch.zeros(2, 5, 3, 4, dtype=BF), "C": torch.zeros(2, 5, 3, 4, dtype=BF)}, "groups"),
    ({"B": torch.zeros(2, 5, 4, dtype=BF)}, "B must be"),
    ({"C": torch.zeros(2, 5, 1, 4, dtype=BF)}, "C must be"),
    ({"C": torch.zeros(2, 5, 4, 2, dtype=BF).transpose(2, 3)}, "contiguous"),
    ({"D": torch.zeros(7)}, "D must be"),
    ({"dt_bias": torch.zeros(8, dtype=BF)}, "dt_bias"),
    ({"state": torch.zeros(2, 8, 3)}, "state"),
    ({"lengths": torch.zeros(2)}, "lengths"),
])
def test_ssm_scan(kw, msg):
    with pytest.raises(ValueError, match=msg):
        _scan(**kw)


def test_ssm_scan_backward_and_step():
    i = scan_inputs(1, "bf16", 2, 17, 8, 4)
    a = [i[k] for k in ("x", "dt", "A", "B", "C")]
    with pytest.raises(ValueError, match="checkpoints"):
        ssm.ssm_scan_backward(i["gy"], *a, torch.zeros(2, 1, 8, 4))
    with pytest.raises(ValueError, match="checkpoints"):
        ssm.ssm_scan_backward(i["gy"], *a, None)
    with pytest.raises(ValueError, match="grad_y"):
        ssm.ssm_scan_backward(i["gy"].float(), *a, torch.zeros(2, 2, 8, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ssm.ssm_scan_backward(i["gy"], *a, torch.zeros(2, 2, 8, 4))
    s = [t[:, 0] if t.dim() > 2 else t for t in a]
    with pytest.raises(ValueError, match="row for each"):
        ssm.ssm_scan_step(*s, torch.zeros(3, 8, 4))
    with pytest.raises(ValueError, match="state"):
        ssm.ssm_scan_step(*s, torch.zeros(2, 8, 4, dtype=BF))
    with pytest.raises(ValueError, match="B must be"):
        ssm.ssm_scan_step(*s[:3], a[3], s[4], torch.zeros(2, 8, 4))


@pytest.mark.parametrize("o,kw,msg", [
    (torch.zeros(3, 8, dtype=BF), {}, "CUDA"),
    (torch.zeros(3, 8193, dtype=BF), {}, "8192"),
    (torch.zeros(3, 8, dtype=torch.float64), {}, "bfloat16"),
    (torch.zeros((), dtype=BF), {}, "o must be"),
    (torch.zeros(8, 3, dtype=BF).t(), {}, "contiguous"),
    (torch.zeros(2, 4, 6, 8, dtype=BF)[:, :3], {}, "fixed distance"),
    (torch.zeros(3, 8, dtype=BF), {"residual": torch.zeros(3, 8, dtype=torch.float16)}, "residual"),
    (torch.zeros(3, 8, dtype=BF), {"residual": torch.zeros(1, 8, dtype=BF)}, "residual"),
    (torch.zeros(3, 8, dtype=BF), {"gate": torch.zeros(3, 8)}, "gate"),
    (torch.zeros(3, 8, dtype=BF), {"post_weight": torch.zeros(7)}, "post_weight"),
    (torch.zeros(3, 8, dtype=BF), {"post_bias": torch.zeros(8)}, "post_bias"),
    (torch.zeros(3, 8, dtype=BF), {"pre_bias": torch.zeros(8)}, "pre_bias"),
    (torch.zeros(3, 8, dtype=BF), {"scale": torch.zeros(8, dtype=BF)}, "scale"),
    (torch.zeros(3, 8, dtype=BF), {"eps": -1.0}, "eps"),
    (torch.zeros(3, 8, dtype=BF), {"eps": float("nan")}, "eps"),
    (torch.zeros(3, 8, dtype=BF), {"norm": "batch"}, "norm"),
    (torch.zeros(3, 8, dtype=BF), {"activation": "relu"}, "activation"),
])
def test_norm_gate_residual(o, kw, msg):
    with pytest.raises(ValueError, match=msg):
        glue.norm_gate_residual(o, **kw)


def test_norm_gate_residual_backward():
    o, st = torch.zeros(3, 8, dtype=BF), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="grad_x or grad_n"):
        glue.norm_gate_residual_backward(None, None, o, st)
    with pytest.raises(ValueError, match="pre_weight"):
        glue.norm_gate_residual_backward(None, o, o, st)
    with pytest.raises(ValueError, match="stats"):
        glue.norm_gate_residual_backward(o, None, o, st[:2])
    with pytest.raises(ValueError, match="grad_x"):
        glue.norm_gate_residual_backward(o.float(), None, o, st)
    with pytest.raises(ValueError, match="grad_x"):
        glue.norm_gate_residual_backward(o, None, o, st, torch.zeros(3, 8))


def test_the_c_abi_refuses_null_and_bad_sizes():
    import ctypes
    from ttt_tk_b200 import _lib
    lib = _lib.lib()
    for name in ("short_conv", "short_conv_backward", "short_conv_step", "ssm_scan", "ssm_scan_backward", "ssm_scan_step",
                 "norm_gate_residual", "norm_gate_residual_backward"):
        fn = getattr(lib, "ttt_b200_" + name)
        fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        assert fn(None, None) == 1
        assert b"NULL" in lib.ttt_b200_last_error()
        assert fn(ctypes.byref(ctypes.create_string_buffer(1024)), None) == 1      # a struct of zeros


def test_sizes_that_indices_could_not_hold():
    """Expanded tensors hold nothing of their own; their sizes are refused before anything is read."""
    one = torch.zeros(1, 1, 1, dtype=BF)
    with pytest.raises(ValueError, match="too large"):
        ssm.short_conv(one.expand(1, (1 << 30) + 1, 1), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="too large"):
        x = one.expand(1, (1 << 30) + 1, 1)
        ssm.ssm_scan(x, x, torch.zeros(1, 1), x.unsqueeze(-1), x.unsqueeze(-1))


def test_a_flag_that_is_neither_true_nor_false():
    with pytest.raises(RuntimeError, match="ambiguous"):
        _conv(heads=torch.ones(2))
    i = scan_inputs(1, "bf16", 2, 8, 16, 4, 1)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ssm.ssm_scan(*[i[k] for k in ("x", "dt", "A", "B", "C")], softplus=torch.ones(2))


@pytest.mark.parametrize("missing", ["residual", "gate"])
def test_c_block_backward_without_a_place_for_a_gradient(missing):
    """An input whose gradient has no place: refused before the scratch is looked at, so nothing is launched."""
    import ctypes
    import struct

    from ttt_tk_b200 import _lib
    lib = _lib.lib()
    word = ctypes.create_string_buffer(64)
    at = ctypes.addressof(word) + 15 & ~15      # (never read)
    p = [0] * 22      # o, residual, gate, weights x 5, x, n, stats, grad_x, grad_n, grad_o, grad_residual, grad_gate, sums x 5, scratch
    for k in (0, 10, 11, 13, {"residual": 1, "gate": 2}[missing]):
        p[k] = at
    args = struct.pack("=22Q Q 6q 5i f", *p, 0, 8, 8, 8, 8, 8, 1, 8, 0, 0, 0, 1, 1e-6)
    fn = lib.ttt_b200_norm_gate_residual_backward
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.ttt_b200_last_error.restype = ctypes.c_char_p
    assert fn(args, None) == 1 and b"null tensor pointer" in lib.ttt_b200_last_error()
    p[{"residual": 14, "gate": 15}[missing]] = at
    args = struct.pack("=22Q Q 6q 5i f", *p, 0, 8, 8, 8, 8, 8, 1, 8, 0, 0, 0, 1, 1e-6)
    assert fn(args, None) == 1 and b"scratch" in lib.ttt_b200_last_error()
