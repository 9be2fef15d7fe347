"""What activations in 8 bits, the norm into them and the rows of tables refuse, before anything is launched."""
import ctypes

import pytest
import torch

from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, saved, tables

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("xs,kw,msg", [
    ((torch.zeros(3, 8),), {}, "CUDA"),
    ((), {}, "one to four"),
    ((torch.zeros(3, 8),) * 5, {}, "one to four"),
    ((torch.zeros(3, 8), torch.zeros(3, 9)), {}, "share shape"),
    ((torch.zeros(3, 8), torch.zeros(3, 8, dtype=BF)), {}, "share shape"),
    ((torch.zeros(3, 8, dtype=torch.float64),), {}, "bfloat16"),
    ((torch.zeros(()),), {}, "D"),
    ((torch.zeros(3, 0),), {}, "no values"),
    ((torch.zeros(8, 3).t(),), {}, "contiguous"),
    ((torch.zeros(2, 4, 6, 8)[:, :3],), {}, "fixed distance"),
    ((3,), {}, "tensor"),
    ((None,), {}, "tensor"),
    ((torch.zeros(3, 8),), {"group": 16}, "group"),
    ((torch.zeros(3, 8),), {"group": 0}, "group"),
    ((torch.zeros(3, 8),), {"group": None}, "group"),
    ((torch.zeros(3, 8),), {"group": 64.0}, "group"),
    ((torch.zeros(3, 8),), {"group": True}, "group"),
])
def test_pack8(xs, kw, msg):
    with pytest.raises(ValueError, match=msg):
        saved.pack8(*xs, **kw)


def _pack(*shape, groups=1):
    return torch.zeros(*shape, dtype=F8), torch.ones(*shape[:-1], groups)


@pytest.mark.parametrize("packs,kw,msg", [
    ((_pack(3, 8),), {}, "CUDA"),
    ((), {}, "one to four"),
    ((torch.zeros(3, 8),), {}, "values, scales"),
    (((torch.zeros(3, 8, dtype=F8),),), {}, "values, scales"),
    (((torch.zeros(3, 8, dtype=BF), torch.ones(3, 1)),), {}, "float8"),
    (((torch.zeros(8, 3, dtype=F8).t(), torch.ones(3, 1)),), {}, "contiguous"),
    ((_pack(3, 200, groups=3),), {}, "scales"),
    (((torch.zeros(3, 8, dtype=F8), torch.ones(3, 1, dtype=BF)),), {}, "scales"),
    ((_pack(3, 256, groups=2), _pack(3, 256, groups=4)), {}, "same for all"),
    ((_pack(3, 8), _pack(4, 8)), {}, "share"),
    ((_pack(3, 8),), {"dtype": torch.float64}, "dtype"),
    ((_pack(3, 8),), {"dtype": "bf16"}, "dtype"),
    ((_pack(3, 8),), {"dtype": "torch.float16"}, "dtype"),
])
def test_unpack8(packs, kw, msg):
    with pytest.raises(ValueError, match=msg):
        saved.unpack8(*packs, **kw)


@pytest.mark.parametrize("o,kw,msg", [
    (torch.zeros(3, 8, dtype=BF), {}, "CUDA"),
    (torch.zeros(3, 8193, dtype=BF), {"weight": torch.ones(8193)}, "8192"),
    (torch.zeros(3, 8, dtype=torch.float64), {}, "bfloat16"),
    (torch.zeros((), dtype=BF), {}, "o must be"),
    (torch.zeros(8, 3, dtype=BF).t(), {}, "contiguous"),
    (torch.zeros(2, 4, 6, 8, dtype=BF)[:, :3], {}, "fixed distance"),
    (torch.zeros(3, 8, dtype=BF), {"residual": torch.zeros(3, 8, dtype=torch.float16)}, "residual"),
    (torch.zeros(3, 8, dtype=BF), {"residual": torch.zeros(1, 8, dtype=BF)}, "residual"),
    (torch.zeros(3, 8, dtype=BF), {"weight": torch.ones(7)}, "weight"),
    (torch.zeros(3, 8, dtype=BF), {"weight": None}, "weight"),
    (torch.zeros(3, 8, dtype=BF), {"bias": torch.ones(8, dtype=BF)}, "bias"),
    (torch.zeros(3, 8, dtype=BF), {"norm": "batch"}, "norm"),
    (torch.zeros(3, 8, dtype=BF), {"group": 16}, "group"),
    (torch.zeros(3, 8, dtype=BF), {"group": 0}, "group"),
    (torch.zeros(3, 8, dtype=BF), {"group": "row"}, "group"),
    (torch.zeros(3, 8, dtype=BF), {"eps": -1.0}, "eps"),
    (torch.zeros(3, 8, dtype=BF), {"eps": None}, "eps"),
    (torch.zeros(3, 8, dtype=BF), {"eps": float("nan")}, "eps"),
])
def test_norm_residual_8bit(o, kw, msg):
    with pytest.raises(ValueError, match=msg):
        glue.norm_residual_8bit(o, **{"weight": torch.ones(8), **kw})


I = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731, E741


@pytest.mark.parametrize("ts,source,target,msg", [
    ([torch.zeros(4, 3)], I(2), I(2), "CUDA"),
    ([], I(2), I(2), "1 to 16"),
    ([torch.zeros(4, 3)] * 17, I(2), I(2), "1 to 16"),
    (None, I(2), I(2), "tables must be"),
    ([3], I(2), I(2), "tensor"),
    ([torch.zeros(())], I(2), I(2), "rows"),
    ([torch.zeros(3, 4).t()], I(2), I(2), "contiguous"),
    ([torch.zeros(4, 3), torch.zeros(5, 3)], I(2), I(2), "as many rows"),
    ([torch.zeros(4, 3)], I(2), I(3), "as many rows"),
    ([torch.zeros(4, 3)], torch.zeros(2), I(2), "source"),
    ([torch.zeros(4, 3)], I(2), torch.zeros(2, dtype=torch.int64), "target"),
    ([torch.zeros(4, 3)], torch.zeros(2, 1, dtype=torch.int32), I(2), "source"),
    ([torch.zeros(4, 3)], I(4)[::2], I(2), "source"),
    ([torch.zeros(4, 3)], I(4097), I(4097), "4096"),
    ([torch.zeros(4, 3)], None, I(2), "tensor"),
])
def test_copy_rows(ts, source, target, msg):
    with pytest.raises(ValueError, match=msg):
        tables.copy_rows(ts, source, target)


def test_tables_that_overlap():
    t = torch.zeros(4, 3)
    for ts in ([t, t], [t, t.view(torch.int32)], [t[:3], t[1:]]):
        with pytest.raises(ValueError, match="overlap"):
            tables.copy_rows(ts, I(1), I(1))


def test_rows_named_from_within_a_table():
    """One block of the GPU would read them while another writes that table."""
    at, used = torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.bool)
    states = torch.zeros(4, 3)
    for call in (lambda: tables.copy_rows([states, at], at, I(4)), lambda: tables.copy_rows([states, at], I(4), at), lambda: tables.copy_rows([at], at[1:3], I(2)),
                 lambda: tables.clear_rows([at], at), lambda: tables.compact_rows([states, used], used), lambda: tables.compact_rows(used.view(torch.uint8), used)):
        with pytest.raises(ValueError, match="overlap a table"):
            call()
    with pytest.raises(ValueError, match="CUDA"):      # next to one another
        tables.copy_rows([states[:2], at[:2]], at[2:], I(2))


def test_clear_and_compact():
    t = torch.zeros(4, 3)
    for rows, msg in ((torch.zeros(2), "rows"), (I(4097), "4096"), (None, "tensor"), (I(2), "CUDA")):
        with pytest.raises(ValueError, match=msg):
            tables.clear_rows(t, rows)
    for ts, used, msg in ((t, torch.zeros(4, dtype=torch.uint8), "used"), (t, torch.zeros(3, dtype=torch.bool), "used"), (t, torch.zeros(8, dtype=torch.bool)[::2], "contiguous"),
                          (torch.zeros(8193, 1), torch.zeros(8193, dtype=torch.bool), "8192"), (t, None, "tensor"), (t, torch.zeros(4, dtype=torch.bool), "CUDA")):
        with pytest.raises(ValueError, match=msg):
            tables.compact_rows(ts, used)


@pytest.mark.parametrize("name", ["e5m2", 8, True, ["e4m3"], torch.zeros(2)])
def test_what_is_no_way_to_keep(name):
    x = torch.zeros(2, 3, 8)
    for call in (lambda: ag.short_conv(x, torch.zeros(8, 4), saved=name), lambda: ag.gated_scan(x, x, saved=name), lambda: ag.norm_gate_residual(x, saved=name),
                 lambda: ag.ssm_scan(x, x, torch.zeros(8, 4), torch.zeros(2, 3, 1, 4), torch.zeros(2, 3, 1, 4), saved=name)):
        with pytest.raises(ValueError, match="saved must be"):
            call()


def test_the_c_abi_refuses_null_and_bad_sizes():
    from ttt_tk_b200 import _lib
    lib = _lib.lib()
    for name in ("pack8", "unpack8", "norm_residual_8bit", "copy_rows", "clear_rows", "compact_rows"):
        fn = getattr(lib, "ttt_b200_" + name)
        fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        assert fn(None, None) == 1
        assert b"NULL" in lib.ttt_b200_last_error()
        assert fn(ctypes.byref(ctypes.create_string_buffer(2048)), None) == 1      # a struct of zeros
