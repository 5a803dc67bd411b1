"""Group norm of many pixels of which the first ones are far from the others: the variance keeps its digits."""
import pytest
import torch

from eagersgd_b200.ops import functional as ops

EPS = 1e-5
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("outliers", ["first", "first few", "first half", "last"])
@pytest.mark.parametrize("c,groups,side", [(32, 4, 512), (30, 6, 300), (64, 64, 256)])
def test_variance_of_groups_with_outliers(c, groups, side, outliers, dtype):
    """What z says of 1 / deviation, by least squares in 64 bits, against that of the formula."""
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(2, c, side, side, device="cuda", generator=g).to(dtype).contiguous(memory_format=torch.channels_last)
    pixels = x.permute(0, 2, 3, 1).view(2, side * side, c)                     # the memory as it lies
    where = {"first": slice(0, 1), "first few": slice(0, 100), "first half": slice(0, side * side // 2), "last": slice(side * side - 1, None)}
    pixels[:, where[outliers]] += 1000.0
    z = ops.group_norm_act(x, groups, torch.ones(c, device="cuda"), torch.zeros(c, device="cuda"), eps=EPS)
    v, got = (t.double().permute(0, 2, 3, 1).reshape(2, -1, groups, c // groups).permute(0, 2, 1, 3).reshape(2, groups, -1) for t in (x, z))
    d = v - v.mean(2, keepdim=True)
    want = (d.square().mean(2) + EPS).rsqrt()
    slope = (got * d).sum(2) / d.square().sum(2)
    # a sum of n terms, twice what is left of them, is off by 2 n roundings of it at most, and its root by half of that; a thread has
    # side^2 / 32 rows or fewer (fewer channels have more threads a row).  z's own roundings even out but for half a step of the largest.
    rounding = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
    assert ((slope / want - 1).abs() < (side * side / 32 + 64) * 2.0 ** -24 + rounding).all()
