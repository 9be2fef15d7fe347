"""The norm into 8 bits where its value lies on the border of two roundings: rows of +-k, whose norm is +-1 exactly, with weights half way between two
values of 4 bits.  In 64 bits they go to the even one; a norm that is off by one unit of fp32 sends half of them the other way."""
import pytest
import torch

from oracle import gated as og
from ttt_tk_b200 import glue

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("ty,D,most", [(torch.float32, 64, 512), (torch.float32, 96, 512), (torch.bfloat16, 96, 256), (torch.float32, 520, 64), (torch.float32, 1002, 64),
                                       (torch.bfloat16, 2048, 32), (torch.float32, 2600, 32), (torch.float32, 7000, 16)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("group", [32, None])
def test_ties(norm, ty, D, most, residual, group):
    """Sums of k^2 have at most 24 bits, so that they, the mean of the squares and the mean, 0, are exact; the root's reciprocal is right to more than 2^-40 as the sum
    it is kept as, and so c / deviation is 1 when it is rounded once."""
    assert most * most * D // (8 if D % 8 == 0 else 1) < 1 << 24      # (a thread's part is eight times k^2)
    k = torch.arange(1, most + 1, dtype=torch.float64)
    z = k[:, None] * torch.tensor([1.0, -1.0], dtype=torch.float64).repeat(D // 2)
    w = torch.tensor([1.0625, 1.0625, 1.1875, 1.1875], dtype=torch.float64).repeat(D // 4 + 1)[:D]
    zero = torch.zeros_like(z).to(ty).cuda()
    o, r = (zero, z.to(ty).cuda()) if residual else (z.to(ty).cuda(), None)
    _, q, s, stats = glue.norm_residual_8bit(o, r, weight=w.float().cuda(), norm=norm, group=group, eps=0.0, return_stats=True)
    n = torch.sign(z) * w
    want, scale = og.e4m3(n, group)
    assert torch.equal(s.double().cpu().view(scale.shape if group else (-1, 1)), scale)
    got = q.double().cpu() * (scale.repeat_interleave(32, -1)[:, :D] if group else scale)
    off = got != want
    assert not off.any(), f"{int(off.sum())} of {off.numel()} values, {int(off.any(-1).sum())} of {most} rows"
    # the statistic is 1 / k rounded once
    assert torch.equal(stats[:, 3].cpu(), (1 / k).float())


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("D", [64, 96, 1002, 4096])
def test_a_row_with_an_infinity(norm, D):
    """Its deviation is infinite: the others become 0 or, beside an infinite mean, no numbers, as in 64 bits; the rows around it are as they would be."""
    z = torch.randn(3, D, generator=torch.Generator().manual_seed(D))
    w = torch.ones(D)
    want = glue.norm_residual_8bit(z.cuda(), weight=w.cuda(), norm=norm, group=32)[1].float()
    z[1, 5] = float("inf")
    got = glue.norm_residual_8bit(z.cuda(), weight=w.cuda(), norm=norm, group=32)[1].float()
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    d = z.double()
    c = d - d.mean(-1, keepdim=True) if norm == "layer" else d
    n = c / (c * c).mean(-1, keepdim=True).sqrt()
    assert torch.equal(got[1].isnan().cpu(), n[1].isnan()) and (got[1].cpu()[~n[1].isnan()] == 0).all()
