"""What the differentiable forms of the layer-side sequence operators refuse and ask of the operators, without a GPU: shapes and types are
checked before devices, and what is asked is read from the call that arrives."""
import pytest
import torch

from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, ssm

BF = torch.bfloat16


# ---- block end -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["residual", "gate"])
@pytest.mark.parametrize("shape", [(3, 2, 8), (6, 8), (1, 6, 8), (2, 3, 4), (8,), (1, 1, 8)])
def test_block_end_takes_no_other_shape_of_as_many_tokens(name, shape):
    """Tokens in flat order are not the tokens of another shape."""
    o = torch.zeros(2, 3, 8, dtype=BF)
    with pytest.raises(ValueError, match=f"{name} must have the shape of o"):
        ag.norm_gate_residual(o, **{name: torch.zeros(shape, dtype=BF)})


def test_block_end_of_equal_shapes_reaches_the_device_check():
    o = torch.zeros(2, 3, 8, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        ag.norm_gate_residual(o, o, o, pre_weight=torch.ones(8))
    with pytest.raises(ValueError, match="CUDA"):      # a size of one in front, rows that do not follow one another
        ag.norm_gate_residual(torch.zeros(2, 4, 6, 8, dtype=BF)[:, :3])


@pytest.mark.parametrize("o,msg", [(torch.zeros((), dtype=BF), "o must be"), (torch.zeros(3, 0, dtype=BF), "1 to 8192"),
                                   (torch.zeros(0, 8193, dtype=BF), "1 to 8192")])
def test_block_end_without_values_to_a_token(o, msg):
    with pytest.raises(ValueError, match=msg):
        ag.norm_gate_residual(o)


# ---- scan ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode, torch.enable_grad])
@pytest.mark.parametrize("leaf", [True, False])
@pytest.mark.parametrize("state", [True, False])
def test_checkpoints_are_kept_only_for_a_backward_that_can_come(monkeypatch, mode, leaf, state):
    """Weights that are parameters ask for a gradient even where none is recorded."""
    asked = []

    def scan(x, dt, A, B, C, D, dt_bias, softplus, state, lengths, return_state, return_checkpoints):
        asked.append((return_state, return_checkpoints))
        return (torch.zeros_like(x), torch.zeros(2, 8, 4) if return_state else None, torch.zeros(2, 1, 8, 4) if return_checkpoints else None)

    monkeypatch.setattr(ssm, "_host", lambda: type("Host", (), {"scan": staticmethod(scan)}))
    x, B = torch.zeros(2, 5, 8), torch.zeros(2, 5, 1, 4)
    A, D = (torch.nn.Parameter(torch.zeros(s), requires_grad=leaf) for s in ((8, 4), (8,)))
    with mode():
        r = ag.ssm_scan(x, x, A, B, B, D, return_state=state)
    wanted = leaf and mode is torch.enable_grad
    assert asked == [(state, wanted)]
    y = r[0] if state else r
    assert y.requires_grad == wanted and y.shape == x.shape


# ---- arguments of another kind --------------------------------------------------------------------------------------------
def _scan_args(**kw):
    a = dict(x=torch.zeros(2, 5, 8), dt=torch.zeros(2, 5, 8), A=torch.zeros(8, 4), B=torch.zeros(2, 5, 1, 4), C=torch.zeros(2, 5, 1, 4))
    return {**a, **kw}


@pytest.mark.parametrize("kind", [3, [1.0], "x"])
def test_what_is_not_a_tensor(kind):
    o = torch.zeros(2, 3, 8)
    for call in (lambda: ag.short_conv(kind, torch.zeros(8, 4)), lambda: ag.short_conv(o, kind), lambda: ag.short_conv(o, torch.zeros(8, 4), kind),
                 lambda: ag.short_conv(o, torch.zeros(8, 4), state=kind), lambda: ag.short_conv(o, torch.zeros(8, 4), lengths=kind),
                 *[lambda k=k: ag.ssm_scan(**_scan_args(**{k: kind})) for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "state", "lengths")],
                 lambda: ag.norm_gate_residual(kind), lambda: ag.norm_gate_residual(o, kind), lambda: ag.norm_gate_residual(o, gate=kind),
                 lambda: ag.norm_gate_residual(o, pre_weight=kind)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("zero", ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"])
def test_tensors_without_dimensions(zero):
    with pytest.raises(ValueError, match="must be"):
        ag.ssm_scan(**_scan_args(**{zero: torch.zeros(())}))


@pytest.mark.parametrize("name", [["silu"], {}, 1, "SILU", torch.zeros(2)])
def test_names_of_no_activation_or_norm(name):
    o = torch.zeros(2, 3, 8)
    for call in (lambda: ssm.short_conv(o, torch.zeros(8, 4), activation=name), lambda: ag.short_conv(o, torch.zeros(8, 4), activation=name),
                 lambda: ssm.short_conv_step(o[0], torch.zeros(3, 3, 8), torch.zeros(8, 4), activation=name),
                 lambda: glue.norm_gate_residual(o, activation=name), lambda: ag.norm_gate_residual(o, norm=name)):
        with pytest.raises(ValueError, match="activation|norm must be"):
            call()


@pytest.mark.parametrize("eps", ["1e-5", None, [1.0], -1e-30])
def test_an_epsilon_that_is_no_number(eps):
    with pytest.raises(ValueError, match="eps"):
        glue.norm_gate_residual(torch.zeros(2, 8), eps=eps)
