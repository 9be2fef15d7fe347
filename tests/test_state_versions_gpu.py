"""What changes a table or a state in place says so to autograd: a backward that kept it refuses instead of taking what is there now."""
import pytest
import torch

from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import ssm, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _calls(windows, states, wide):
    """Each call and the tensors it changes."""
    B, D = 3, 64
    x, A, w = torch.randn(B, D, device=DEV), -torch.rand(D, device=DEV), torch.randn(D, 4, device=DEV)
    N = wide.shape[-1]
    bc, An = torch.randn(B, 1, N, device=DEV), -torch.rand(D, N, device=DEV)
    slots = _i32([4, 0, 2])
    yield lambda: tables.copy_rows((windows, states), _i32([0]), _i32([1])), (windows, states)
    yield lambda: tables.clear_rows([windows, states], _i32([2])), (windows, states)
    yield lambda: tables.compact_rows((windows, states), torch.tensor([False, True, False, True, True, False], device=DEV)), (windows, states)
    yield lambda: tables.copy_rows(states, _i32([0]), _i32([1])), (states,)
    yield lambda: ssm.gated_scan_step(x, x, states, A, slots=slots), (states,)
    yield lambda: ssm.gated_scan_step(x, x, states[:B], A), (states,)
    yield lambda: ssm.short_conv_step(x, windows, w, slots=slots), (windows,)
    yield lambda: ssm.ssm_scan_step(x, x, An, bc, bc, wide, slots=slots), (wide,)


def _tables():
    return torch.randn(6, 3, 64, device=DEV), torch.randn(6, 64, device=DEV), torch.randn(6, 64, 16, device=DEV)


def test_versions_go_up():
    ts = _tables()
    for n, (call, changed) in enumerate(_calls(*ts)):
        before = [t._version for t in ts]
        call()
        for t, v in zip(ts, before):
            assert (t._version > v) == any(t is c for c in changed), n


def test_a_backward_refuses_a_state_that_has_moved():
    windows, states, _ = _tables()
    x, w = torch.randn(2, 5, 64, device=DEV), torch.randn(64, 4, device=DEV, requires_grad=True)
    y = ag.short_conv(x, w, state=windows[:2])
    tables.copy_rows((windows, states), _i32([4]), _i32([0]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = ag.short_conv(x, w, state=windows[:2].clone())
    tables.clear_rows((windows, states), _i32([0]))
    y.sum().backward()
    assert w.grad.isfinite().all()


def test_tensors_without_versions():
    """Those of inference mode have none."""
    with torch.inference_mode():
        ts = _tables()
        for call, changed in _calls(*ts):
            before = [t.clone() for t in changed]
            call()
            assert any(not torch.equal(a, b) for a, b in zip(before, changed))
    for call, _ in _calls(*ts):      # and outside of it
        call()
