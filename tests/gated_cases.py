"""Inputs and tolerances of the tests of the gated linear recurrence and of what 8 bits keep.  A value may be off by half a step of its type and by the
error that `oracle/gated.py` carries beside it, which may have been rounded as well."""
import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def close(got, want, what=""):
    ref, err = want
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + (1 + fi.eps) * err * 2.0 ** -24 + fi.smallest_normal * fi.eps / 2 + 2.0 ** -120
    got = got.detach().double().cpu()
    assert got.isfinite().all() or not ref.isfinite().all(), f"{what}: not finite"
    bad = ~((got - ref).abs() <= tol) & ~(got.isnan() & ref.isnan()) & ~(got == ref)
    if bad.any():
        i = int(((got - ref).abs() / tol).nan_to_num(1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; the worst, at {i}: got {got.flatten()[i].item():.9g}, "
                             f"want {ref.flatten()[i].item():.9g}, allowed {tol.flatten()[i].item():.3g}")


def apart(t, how):
    """The same values in rows at other distances: "whole" as they are, "wide" the second half of rows twice as wide, "odd" rows that start on
    any boundary, "time" with the tokens' dimension outermost; what lies between is NaN."""
    if t is None or how == "whole":
        return t
    if how == "time":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    D = t.shape[-1]
    w = torch.full((*t.shape[:-1], 2 * D if how == "wide" else D + 3), float("nan"), dtype=t.dtype, device=t.device)
    at = D if how == "wide" else 1
    w[..., at:at + D] = t
    return w[..., at:at + D]


def gated_inputs(seed, ty, B, T, D, device="cpu", A=True, igate=True, bias=True, state=True, lengths=None, rows="whole"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ty = TYPES[ty]
    i = dict(x=r(B, T, D).to(ty), gate=(2 * r(B, T, D)).to(ty), input_gate=r(B, T, D).to(ty) if igate else None,
             A=8 * torch.log(0.9 + 0.0999 * torch.rand(D, generator=g)) if A else None, gate_bias=r(D) + (0 if A else 2) if bias else None,
             input_bias=r(D) if bias and igate else None, state=r(B, D) if state else None,
             lengths=torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None, gy=r(B, T, D).to(ty), gf=r(B, D) if state else None)
    i = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in i.items()}
    for k in ("x", "gate", "input_gate", "gy"):
        i[k] = apart(i[k], rows)
    return i


ARGS = ("A", "input_gate", "gate_bias", "input_bias")
GRADS = ("x", "gate", "A", "input_gate", "gate_bias", "input_bias", "state")


def run_both(i, mix, step=False):
    """(y, final state, gradients by name) of the kernels."""
    from ttt_tk_b200 import ssm
    kw = dict(mix=mix, lengths=i["lengths"])
    y, end, ck = ssm.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"], return_state=True, return_checkpoints=True, **kw)
    g = ssm.gated_scan_backward(i["gy"], i["x"], i["gate"], ck, *[i[k] for k in ARGS], grad_final_state=i["gf"], **kw)
    return y, end, dict(zip(GRADS, g))


def hold(i, mix, got, what=""):
    from oracle import gated as og
    y, end, grads = got
    ya, enda, before = og.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], mix=mix, state=i["state"], lengths=i["lengths"])
    close(y, ya, what + " y")
    close(end, enda, what + " state")
    ref = og.gated_scan_backward(i["gy"], i["x"], i["gate"], before, *[i[k] for k in ARGS], mix=mix, lengths=i["lengths"], grad_final_state=i["gf"])
    for k in GRADS:
        if k in ref:
            close(grads[k], ref[k], f"{what} grad {k}")
        else:
            assert grads[k] is None, k
