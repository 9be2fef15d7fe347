"""Inputs and tolerances of the tests of the layer-side sequence operators.

Tolerance of a value v of type t: half a step of t, relative to v (bf16 2^-8, fp16 2^-11, fp32 2^-24), plus `ops` roundings of 2^-24
relative to the magnitudes that were added up (the oracle's `amp`), plus half of the type's smallest step.  `ops` counts the fp32
operations in a row that a value has gone through, an exponential or reciprocal (2^-22) as four of them."""
import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def close(got, ref, amp, ops, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + (1 + fi.eps) * ops * 2.0 ** -24 * amp + fi.smallest_normal * fi.eps / 2 + 2.0 ** -126
    d = (got.detach().double().cpu() - ref).abs()
    bad = ~(d <= tol)
    if bad.any():
        i = int((d / tol).nan_to_num(1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; the worst, at {i}: got {got.flatten()[i].item():.9g}, "
                             f"want {ref.flatten()[i].item():.9g}, off {d.flatten()[i].item():.3g}, allowed {tol.flatten()[i].item():.3g}")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def wide(t, on):
    """The same values as the second half of a tensor twice as wide (rows that are further apart)."""
    if not on:
        return t
    w = torch.full((*t.shape[:-1], 2 * t.shape[-1]), float("nan"), dtype=t.dtype, device=t.device)
    w[..., t.shape[-1]:] = t
    return w[..., t.shape[-1]:]


def conv_inputs(seed, ty, B, T, D, K, device="cpu", state=True, lengths=None, strided=False):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ty = TYPES[ty]
    i = dict(x=wide(r(B, T, D).to(ty), strided), weight=r(D, K) * 0.6, bias=r(D) * 0.2, state=r(B, K - 1, D).to(ty) if state else None,
             lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32), gy=wide(r(B, T, D).to(ty), strided),
             gf=r(B, K - 1, D).to(ty))
    if lengths is not None:      # what lies behind a sequence's end is never looked at
        for b, n in enumerate(lengths):
            i["x"][b, max(0, n):] = float("nan")
            i["gy"][b, max(0, n):] = float("inf")
    return {k: to(v, device) for k, v in i.items()}


def to(t, device):
    """To the device with the strides it has."""
    if t is None or device == "cpu":
        return t
    if t.is_contiguous():
        return t.to(device)
    base = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).to(device)
    return torch.as_strided(base, t.shape, t.stride(), t.storage_offset())


def scan_inputs(seed, ty, B, T, D, N, G=1, device="cpu", state=True, lengths=None, strided=False):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ty = TYPES[ty]
    first = torch.exp(torch.rand(D, generator=g) * 4.6 - 6.9)
    p = r(B, T, (3 if strided else 0) + 2 * G * N).to(ty)      # one projection's rows, B and C two slices of them
    low = 3 if strided else 0
    i = dict(x=wide(r(B, T, D).to(ty), strided), dt=wide((r(B, T, D) * 0.7).to(ty), strided),
             A=-(torch.arange(N) + 1.0) * (1 + 0.3 * torch.rand(D, N, generator=g)), B=p[..., low:low + G * N].unflatten(-1, (G, N)),
             C=p[..., low + G * N:].unflatten(-1, (G, N)), D=1 + 0.2 * r(D), dt_bias=first + torch.log(-torch.expm1(-first)),
             state=r(B, D, N) * 0.5 if state else None, lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32),
             gy=wide(r(B, T, D).to(ty), strided), gf=r(B, D, N) * 0.5)
    if lengths is not None:
        for b, n in enumerate(lengths):
            for k in ("x", "dt", "gy"):
                i[k][b, max(0, n):] = float("nan")
            for k in ("B", "C"):
                i[k][b, max(0, n):] = float("inf")
    out = {k: to(v, device) for k, v in i.items() if k not in "BC"}
    p = p.to(device)
    out["B"], out["C"] = p[..., low:low + G * N].unflatten(-1, (G, N)), p[..., low + G * N:].unflatten(-1, (G, N))
    return out
