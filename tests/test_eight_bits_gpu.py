"""Activations in 8 bits against their statement in 64 bits (bit by bit: a power of two divides exactly, so the format's rounding is the only
one), the norm whose output leaves in 8 bits, and backward passes from what was kept."""
import pytest
import torch

from gated_cases import ARGS, GRADS, TYPES, apart, close, gated_inputs
from oracle import gated as og
from ttt_tk_b200 import autograd as ag
from ttt_tk_b200 import glue, saved, ssm

pytestmark = pytest.mark.gpu


def _rows(seed, ty, *shape):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(TYPES[ty]).cuda()


def _same(pack, x, group):
    q, s = pack
    want, scale = og.e4m3(x, group)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.dtype == torch.float32 and s.shape == scale.shape
    wide = scale.repeat_interleave(group or x.shape[-1], -1)[..., :x.shape[-1]]
    assert torch.equal(s.double().cpu(), scale)
    got = q.double().cpu() * wide
    assert torch.equal(got.nan_to_num(1e300), want.nan_to_num(1e300))


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 128), (4, 33, 1003), (1, 4096), (700, 64), (2, 3, 2, 136)])
def test_there_and_back(ty, group, shape):
    x = _rows(1, ty, *shape)
    pack = saved.pack8(x, group=group)
    _same(pack[0], x, group)
    (y,) = saved.unpack8(*pack, dtype=TYPES[ty])
    assert y.dtype == TYPES[ty] and torch.equal(y.double().cpu(), og.e4m3(x, group)[0].to(TYPES[ty]).double())


@pytest.mark.parametrize("how", ["wide", "odd"])
def test_several_tensors_in_rows_at_other_distances(how):
    xs = [apart(_rows(k, "bf16", 3, 40, 200), how) for k in range(4)]
    for p, x in zip(saved.pack8(*xs, group=64), xs):
        _same(p, x, 64)
    packs = saved.pack8(*xs)
    for y, x in zip(saved.unpack8(*packs), xs):
        assert torch.equal(y.double().cpu(), og.e4m3(x, 128)[0])      # 4 bits are less than bf16 has


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("how", ["whole", "wide"])
def test_rows_of_whole_groups(ty, group, how):
    """Values and scales that follow one another, sources that do or not, the last block in part."""
    xs = [_rows(k, ty, 7, 123, 256) for k in range(3)]
    given = [xs[0], xs[1] if how == "whole" else apart(xs[1], "wide"), xs[2]]
    packs = saved.pack8(*given, group=group)
    for p, x in zip(packs, xs):
        _same(p, x, group)
    for y, x in zip(saved.unpack8(*packs, dtype=TYPES[ty]), xs):
        assert torch.equal(y.double().cpu(), og.e4m3(x, group)[0].to(TYPES[ty]).double())


def test_values_at_the_edges():
    """Zeros, the largest and least values of each type, infinities, NaN, and maxima on both sides of 448 times a power of two."""
    inf, nan = float("inf"), float("nan")
    for ty in (torch.float32, torch.bfloat16, torch.float16):
        fi = torch.finfo(ty)
        rows = [[0.0] * 4, [fi.max, -fi.max, 1.0, fi.tiny], [fi.smallest_normal * fi.eps, 0.0, 0.0, 0.0], [inf, 1.0, -inf, 0.5], [nan, 3.0, -2.0, 0.0], [inf, inf, nan, -inf],
                [448.0, 1.0, 0.0, 0.001], [450.0, 1.0, 17.5, -18.5], [1.75, 1.0, 0.0, 2.0 ** -9], [1.7578125, 232.0, 248.0, 0.5], [fi.tiny, -fi.tiny, 0.0, fi.tiny / 2],
                [1.75, 1.75 * 2.0 ** -15, 1.75 * 2.0 ** -17, 1.75 * 2.0 ** -14]]
        x = torch.tensor(rows, dtype=torch.float64).to(ty)
        _same(saved.pack8(x.cuda(), group=32)[0], x, 32)
    x = torch.full((2, 300), nan, device="cuda")
    (y,) = saved.unpack8(*saved.pack8(x), dtype=torch.float32)
    assert y.isnan().all()


def test_a_row_alone():
    x = _rows(3, "bf16", 1, 300)[0]
    _same(saved.pack8(x, group=64)[0], x, 64)
    (p,) = saved.pack8(x)
    assert torch.equal(saved.unpack8((p[0], torch.ones((), device="cuda")))[0], p[0].bfloat16())      # one scale to a row


def test_no_rows():
    (p,) = saved.pack8(torch.zeros(0, 5, 40, device="cuda"))
    assert p[0].shape == (0, 5, 40) and p[1].shape == (0, 5, 1)
    assert saved.unpack8(p)[0].shape == (0, 5, 40)


def test_more_values_than_32_bits_count():
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    x = torch.randn(64, 4096, device="cuda", dtype=torch.bfloat16).repeat(16400, 1)      # 2^32 + values
    (p,) = saved.pack8(x)
    (few,) = saved.pack8(x[:64])
    for a, b in zip(p, few):
        a = a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a
        b = b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b
        assert torch.equal(a[:64], b) and torch.equal(a[-64:], b)
    y = saved.unpack8(p)[0]
    assert torch.equal(y[:64], y[-64:]) and torch.equal(y[-64:], saved.unpack8(few)[0])


def test_more_lanes_than_32_bits_count():
    """Rows of one value: sixteen lanes to each."""
    M = (1 << 28) + 5
    x = torch.randn(1 << 10, 1, device="cuda", dtype=torch.bfloat16).repeat((1 << 18) + 1, 1)[:M]
    (p,) = saved.pack8(x)
    (few,) = saved.pack8(x[:1 << 10])
    assert torch.equal(p[1][:1 << 10], few[1]) and torch.equal(p[1][1 << 28:], few[1][:5])
    assert torch.equal(p[0][1 << 28:].float(), few[0][:5].float())
    assert torch.equal(saved.unpack8(p)[0][1 << 28:], saved.unpack8(few)[0][:5])


# ---- norm -------------------------------------------------------------------------------------------------------------------
def _norm64(z, w, b, layer, eps):
    """(n, what fp32 may be off by in units of 2^-24): the sums' D / 32 + 16 additions of magnitudes in a row and as many for squares, halved by the root;
    some eight operations."""
    D = z.shape[-1]
    mean = z.mean(-1, keepdim=True) if layer else torch.zeros_like(z[..., :1])
    c = z - mean
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * r * w + b
    adds = D / 32 + 16
    emean = (adds * z.abs().mean(-1, keepdim=True) if layer else 0.0) + z.abs()
    return n, (emean * r * w.abs()) + (c * r * w).abs() * (adds + 8 + 2 * (emean * r).mean(-1, keepdim=True)) + n.abs() + b.abs()


def _norm_case(ty, shape, norm="rms", res=True, res32=False, bias=False, group=128, rows="whole", eps=1e-6):
    D = shape[-1]
    g = torch.Generator().manual_seed(D)
    o = apart(_rows(1, ty, *shape), rows)
    residual = apart(_rows(2, "fp32" if res32 else ty, *shape), rows) if res else None
    w, b = (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (0.3 * torch.randn(D, generator=g)).cuda() if bias else None
    x, q, s, stats = glue.norm_residual_8bit(o, residual, weight=w, bias=b, norm=norm, group=group, eps=eps, return_stats=True)
    z = o.double().cpu() + (residual.double().cpu() if res else 0.0)
    if res:
        close(x, (z, z.abs()), "x")
        assert x.dtype == residual.dtype and x.is_contiguous()
    else:
        assert x is o or x.data_ptr() == o.data_ptr()
    n, err = _norm64(z, w.double().cpu(), b.double().cpu() if bias else torch.zeros(D, dtype=torch.float64), norm == "layer", eps)
    # the scale is that of a maximum that fp32 may have off by `err`
    G = group or D
    pad = lambda t: torch.nn.functional.pad(t, (0, -D % G)).unflatten(-1, (-1, G))  # noqa: E731
    off = pad(err * 2.0 ** -24)
    lo = og.e4m3((pad(n).abs() - off).clamp(min=0).flatten(-2), G)[1]
    hi = og.e4m3((pad(n).abs() + off).flatten(-2), G)[1]
    sc = s.double().cpu() if group else s.double().cpu()[..., None]
    assert ((sc >= lo) & (sc <= hi)).all()
    wide = sc.repeat_interleave(G, -1)[..., :D]
    got = q.double().cpu() * wide
    # half a step of 4 bits, or of the least step 2^-9, of the scale, of a value that is off by err
    tol = (n.abs() + err * 2.0 ** -24) * 2.0 ** -4 + wide * 2.0 ** -10 + err * 2.0 ** -24
    assert ((got - n).abs() <= tol).all()
    # and nothing but that: where the borders of a rounding are further away than err, the value is the one
    steps = torch.exp2((torch.frexp(n / wide)[1] - 1).clamp(min=-6, max=8).double() - 3) * wide
    at = n / steps
    sure = ((at - torch.floor(at) - 0.5).abs() * steps > 2 * err * 2.0 ** -24) & (sc.repeat_interleave(G, -1)[..., :D] == lo.repeat_interleave(G, -1)[..., :D])
    assert sure.double().mean() > 0.9 or n.numel() < 50
    assert torch.equal(got[sure], (torch.round(at) * steps)[sure])
    return o, residual, w, b, stats


@pytest.mark.parametrize("ty", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [1, 31, 64, 200, 1003, 2048, 4100, 8192])
@pytest.mark.parametrize("group", [32, 128, None])
def test_norm(ty, D, group):
    _norm_case(ty, (5, D), group=group)


@pytest.mark.parametrize("norm,res,res32,bias", [("layer", True, True, True), ("rms", False, False, True), ("layer", False, False, False), ("rms", True, True, False)])
@pytest.mark.parametrize("rows", ["whole", "wide", "odd"])
def test_norm_parts(norm, res, res32, bias, rows):
    for D in (96, 520):
        _norm_case("bf16", (2, 70, D), norm, res, res32, bias, 64, rows)


def test_norm_of_many_tokens_and_none():
    _norm_case("bf16", (20000, 72))
    x, q, s = glue.norm_residual_8bit(torch.zeros(0, 72, device="cuda"), weight=torch.ones(72, device="cuda"), group=None)
    assert q.shape == (0, 72) and s.shape == (0,)


def test_norm_of_zeros():
    x, q, s = glue.norm_residual_8bit(torch.zeros(3, 72, device="cuda"), weight=torch.ones(72, device="cuda"))
    assert (q.float() == 0).all() and s.isfinite().all()


@pytest.mark.parametrize("norm,bias", [("rms", False), ("layer", True)])
def test_norm_backward_from_its_statistics(norm, bias):
    """The block end's backward takes the statistics of this forward: it is the same norm."""
    o, residual, w, b, stats = _norm_case("bf16", (40, 264), norm, True, False, bias)
    kw = dict(norm=norm, pre_weight=w, pre_bias=b)
    _, _, want = glue.norm_gate_residual(o, residual, return_stats=True, **kw)
    torch.testing.assert_close(stats, want, rtol=2e-6, atol=2e-6)
    gx, gn = torch.randn_like(o), torch.randn_like(o)
    for a, c in zip(glue.norm_gate_residual_backward(gx, gn, o, stats, residual, **kw), glue.norm_gate_residual_backward(gx, gn, o, want, residual, **kw)):
        assert (a is None) == (c is None)
        if a is not None:
            torch.testing.assert_close(a.float(), c.float(), rtol=1e-2, atol=1e-2)


# ---- backward passes from what was kept -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,D", [(70, 64), (130, 200), (9, 75), (65, 130), (200, 1040), (900, 66)])
def test_gated_backward_from_8_bits(ty, group, T, D):
    for igate, lengths in ((True, None), (False, [T, T // 2])):
        i = gated_inputs(1, ty, 2, T, D, "cuda", igate=igate, lengths=lengths)
        a = [i[k] for k in ARGS]
        y, ck = ssm.gated_scan(i["x"], i["gate"], *a, state=i["state"], lengths=i["lengths"], return_checkpoints=True)
        packs = saved.pack8(*[i[k] for k in ("x", "gate", "input_gate") if i[k] is not None], group=group) + [None]
        got = ssm.gated_scan_backward(i["gy"], packs[0], packs[1], ck, i["A"], packs[2] if igate else None, i["gate_bias"], i["input_bias"], lengths=i["lengths"],
                                      grad_final_state=i["gf"])
        _, _, before = og.gated_scan(i["x"], i["gate"], *a, state=i["state"], lengths=i["lengths"])
        kept = {k: og.e4m3(i[k], group)[0] if i[k] is not None else None for k in ("x", "gate", "input_gate")}
        ref = og.gated_scan_backward(i["gy"], kept["x"], kept["gate"], before, i["A"], kept["input_gate"], i["gate_bias"], i["input_bias"], lengths=i["lengths"],
                                     grad_final_state=i["gf"])
        for k, v in zip(GRADS, got):
            if k in ref:
                close(v, ref[k], f"grad {k}")
            else:
                assert v is None


def _leaves(**kw):
    return {k: v.clone().requires_grad_(True) for k, v in kw.items() if v is not None}


@pytest.mark.parametrize("rows", ["whole", "time"])
def test_differentiable_forms_keep_8_bits(rows):
    """Each takes its gradients at the values that 8 bits stand for: those of its backward call with the unpacked ones, bit by bit; and what it keeps is
    half as much."""
    i = gated_inputs(2, "bf16", 2, 130, 128, "cuda", rows=rows)
    lv = _leaves(**{k: i[k] for k in ("x", "gate", *ARGS, "state")})
    y = ag.gated_scan(lv["x"], lv["gate"], *[lv[k] for k in ARGS], state=lv["state"], saved="e4m3")
    got = torch.autograd.grad(y, list(lv.values()), i["gy"])
    packs = saved.pack8(*[i[k].contiguous() for k in ("x", "gate", "input_gate")])
    y0, ck = ssm.gated_scan(i["x"], i["gate"], *[i[k] for k in ARGS], state=i["state"], return_checkpoints=True)
    assert torch.equal(y, y0)
    want = ssm.gated_scan_backward(i["gy"], packs[0], packs[1], ck, i["A"], packs[2], i["gate_bias"], i["input_bias"])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    w, b = torch.randn(128, 4, device="cuda"), torch.randn(128, device="cuda")
    lv = _leaves(x=i["x"], w=w, b=b)
    y = ag.short_conv(lv["x"], lv["w"], lv["b"], activation="silu", saved="e4m3")
    assert torch.equal(y, ssm.short_conv(i["x"], w, b, activation="silu"))
    got = torch.autograd.grad(y, list(lv.values()), i["gy"])
    x8 = saved.unpack8(packs[0])[0]
    for a, c in zip(got, ssm.short_conv_backward(i["gy"], x8, w, b, activation="silu")):
        assert torch.equal(a, c)


def test_the_scan_and_the_block_end_keep_8_bits():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, dt, gy = r(2, 50, 48).bfloat16(), r(2, 50, 48).bfloat16(), r(2, 50, 48).bfloat16()
    A, B, C = -torch.rand(48, 16, generator=g).cuda() - 0.1, r(2, 50, 2, 16).bfloat16(), r(2, 50, 2, 16).bfloat16()
    lv = _leaves(x=x, dt=dt, A=A, B=B, C=C)
    y = ag.ssm_scan(*lv.values(), saved="e4m3")
    got = torch.autograd.grad(y, list(lv.values()), gy)
    _, ck = ssm.ssm_scan(x, dt, A, B, C, return_checkpoints=True)
    x8, dt8 = saved.unpack8(*saved.pack8(x, dt))
    for a, c in zip(got, ssm.ssm_scan_backward(gy, x8, dt8, A, B, C, ck)):
        assert torch.equal(a, c)
    o, gate, res = r(2, 9, 96).bfloat16(), r(2, 9, 96).bfloat16(), r(2, 9, 96)
    w = dict(post_weight=1 + 0.1 * r(96), scale=r(96), pre_weight=1 + 0.1 * r(96))
    lv = _leaves(o=o, residual=res, gate=gate, **w)
    z, n = ag.norm_gate_residual(lv["o"], lv["residual"], lv["gate"], **{k: lv[k] for k in w}, saved="e4m3")
    gz, gn = torch.randn_like(z), torch.randn_like(n)
    got = torch.autograd.grad([z, n], list(lv.values()), [gz, gn])
    _, _, stats = glue.norm_gate_residual(o, res, gate, return_stats=True, **w)
    o8, gate8 = saved.unpack8(*saved.pack8(o, gate))
    (res8,) = saved.unpack8(*saved.pack8(res), dtype=torch.float32)
    want = [v for v in glue.norm_gate_residual_backward(gz, gn, o8, stats, res8, gate8, **w) if v is not None]
    want = [want[0], want[1], want[2], *want[3:]]
    for a, c in zip(got, want):
        assert torch.equal(a, c.view_as(a))


def test_nothing_to_keep():
    """No sequences, no tokens: there are 8 bits of nothing, and gradients of nothing."""
    A = -torch.rand(40, device="cuda")
    for B, T in ((0, 5), (2, 0)):
        x = torch.zeros(B, T, 40, device="cuda", requires_grad=True)
        w = torch.zeros(40, 4, device="cuda", requires_grad=True)
        for y in (ag.gated_scan(x, x, A, saved="e4m3"), ag.short_conv(x, w, saved="e4m3"), ag.norm_gate_residual(x, pre_weight=A, saved="e4m3")[1]):
            (g,) = torch.autograd.grad(y.sum(), x)
            assert g.shape == x.shape


def test_backward_twice_and_without_gradients():
    i = gated_inputs(5, "bf16", 2, 70, 64, "cuda")
    x = i["x"].clone().requires_grad_(True)
    y = ag.gated_scan(x, i["gate"], i["A"], saved="e4m3")
    (a,) = torch.autograd.grad(y, x, i["gy"], retain_graph=True)
    (b,) = torch.autograd.grad(y, x, i["gy"])
    assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(ag.gated_scan(x, i["gate"], i["A"], saved="e4m3"), y)


def test_what_is_kept_is_half():
    x = torch.randn(4, 512, 1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(1024, 4, device="cuda")
    kept = {}
    for how in (None, "e4m3"):
        start = torch.cuda.memory_allocated()
        y = ag.short_conv(x * 1, w, saved=how)      # the input is of this call alone
        kept[how] = torch.cuda.memory_allocated() - start - y.numel() * 2
        del y
    assert kept["e4m3"] < 0.55 * kept[None]


def test_another_stream_and_a_graph():
    x = [_rows(k, "bf16", 300, 512) for k in range(2)]
    w = torch.ones(512, device="cuda")

    def both():
        p = saved.pack8(*x)
        return [t for pair in p for t in pair] + list(glue.norm_residual_8bit(x[0], x[1], weight=w)) + saved.unpack8(*p)

    bits = lambda ts: [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in ts]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bits(got), bits(both())))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = both()
    for k in range(2):
        x[k].copy_(_rows(k + 5, "bf16", 300, 512))
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(bits(got), bits(both())))
