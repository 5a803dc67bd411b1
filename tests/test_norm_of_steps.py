"""Group norm where every step of every sequence is a sample of one pixel, as the scan layers call it."""
import pytest
import torch

from near import near
from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops
from test_group_norm import EPS

BF16, F32 = torch.bfloat16, torch.float32
gpu = pytest.mark.gpu


def _refusal(x, groups):
    c = x.shape[1]
    with pytest.raises(RuntimeError) as e:
        _build.load_torch().group_norm_act(x, groups, torch.ones(c), torch.zeros(c), 0, None, EPS)
    return str(e.value)


@pytest.mark.parametrize("steps,hidden,groups", [(16 * 4099, 2048, 1), (128 * 1024, 1024, 1), (64 * 4099, 1024, 1), (1 << 21, 2048, 32), (1 << 29, 24, 3)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_as_many_steps_as_a_grid_holds(steps, hidden, groups, dtype):
    assert "not on a GPU" in _refusal(torch.zeros(1, hidden, 1, 1, dtype=dtype).expand(steps, -1, -1, -1), groups)


@pytest.mark.parametrize("steps,hidden,groups", [(1 << 31, 8, 1), (1 << 29, 4099, 4099), (1 << 62, 1, 1)])
def test_more_are_refused(steps, hidden, groups):
    assert "too large" in _refusal(torch.zeros(1, hidden, 1, 1).expand(steps, -1, -1, -1), groups)


def _steps(n, c, dtype, shift=0.0):
    """Inputs that cost no host time: [n, c, 1, 1] on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(n + c)
    return [(torch.randn(n, c, 1, 1, device="cuda", generator=g) * 1.5 + s).to(dtype) for s in (shift, 0.0)]


def _against_the_formula(n, c, groups, dtype):
    x, dz = _steps(n, c, dtype, 0.5)
    gamma = (1 + 0.2 * torch.randn(c, device="cuda")).requires_grad_()
    beta = (0.2 * torch.randn(c, device="cuda")).requires_grad_()
    leaf = x.requires_grad_()
    z = ops.group_norm_act(leaf, groups, gamma, beta)
    dx, dgamma, dbeta = torch.autograd.grad(z, [leaf, gamma, beta], dz)
    per = c // groups
    wide_g, sums = gamma.detach().double().view(groups, per), torch.zeros(4, c, dtype=torch.float64, device="cuda")
    for i in range(0, n, 1 << 14):                                             # a portion at a time: 64 bits of all would not be small
        v, d = (t.detach()[i:i + (1 << 14)].double().view(-1, groups, per) for t in (x, dz))
        rstd = (v.var(2, unbiased=False, keepdim=True) + EPS).rsqrt()
        h = (v - v.mean(2, keepdim=True)) * rstd
        want = (h * wide_g + beta.detach().double().view(groups, per)).view(-1, c)
        e = d * wide_g
        want_dx = ((e - e.mean(2, keepdim=True) - h * (e * h).mean(2, keepdim=True)) * rstd).view(-1, c)
        # means and variances of one row, some 40 roundings of the largest value
        spread = 8 * (v.abs().amax() * rstd.amax()).item() + 64
        near(z[i:i + (1 << 14)].view(-1, c), want, want.abs().max().item(), spread, "z")
        term = (rstd.amax() * e.abs().amax() * (1 + h.abs().amax() ** 2)).item()
        near(dx[i:i + (1 << 14)].view(-1, c), want_dx, term, 4 * spread, "dx")
        for j, t in enumerate((d * h, d, (d * h).abs() + d.abs(), d.abs())):
            sums[j] += t.reshape(-1, c).sum(0)
    # sums over the samples: no more roundings than eight lanes have terms each, and those of a term
    near(dgamma, sums[0], sums[2], n / 8 + 16 + spread, "dgamma")
    near(dbeta, sums[1], sums[3], n / 8 + 16, "dbeta")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,c,groups", [(1, 96, 1), (165, 96, 1), (5296, 1024, 1), (9000, 1024, 4), (20000, 1000, 8), (3000, 4100, 4), (40000, 72, 9)])
def test_norms_of_steps(n, c, groups, dtype):
    _against_the_formula(n, c, groups, dtype)


@gpu
def test_more_than_two_to_the_27_channels_in_all():
    _against_the_formula(16 * 4099, 2048, 1, BF16)


@gpu
@pytest.mark.parametrize("n,c,dtype", [(64000, 1024, BF16), (20000, 2048, F32)])
def test_the_backward_pass_takes_no_more_room_than_it_leaves(n, c, dtype):
    """... and 64 MB: a sample's share of dgamma and dbeta is four times a bf16 sample of one pixel."""
    x, dz = _steps(n, c, dtype)
    p = [torch.ones(c, device="cuda", requires_grad=True) for _ in range(2)]
    z = ops.group_norm_act(x.requires_grad_(), 1, *p)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(z, [x, *p], dz)
    torch.cuda.synchronize()
    left = torch.cuda.memory_allocated() - before
    assert left < x.numel() * x.element_size() + (1 << 21)
    assert torch.cuda.max_memory_allocated() - before < left + (64 << 20) + (1 << 21)
    del grads


@gpu
def test_a_portion_more_goes_where_the_first_one_went():
    """Into an accumulator of a training step, and beside samples of an odd number and a shortcut with an activation."""
    n, c = 9001, 2048                                                          # portions of 4096
    x, dz = _steps(n, c, BF16)
    gamma, beta = (torch.nn.Parameter(torch.randn(c, device="cuda")) for _ in range(2))
    leaves = [x.requires_grad_(), gamma, beta, dz.clone().requires_grad_()]
    f = lambda v, r: ops.group_norm_act(v, 4, gamma, beta, "silu", r)  # noqa: E731
    dx, dgamma, dbeta, dres = torch.autograd.grad(f(x, leaves[3]), leaves, dz)
    want = [torch.zeros(c, device="cuda") for _ in range(2)]
    for i in range(0, n, 4096):
        v, r, d = (t.detach()[i:i + 4096] for t in (x, leaves[3], dz))
        part = torch.autograd.grad(f(v.requires_grad_(), r.requires_grad_()), [v, gamma, beta, r], d)
        assert torch.equal(part[0], dx[i:i + 4096]) and torch.equal(part[3], dres[i:i + 4096])
        want[0] += part[1]
        want[1] += part[2]
    assert torch.equal(dgamma, want[0]) and torch.equal(dbeta, want[1])
    sinks = _build.load_torch().GradSinks([2], lambda bucket: None)
    acc = [torch.full((c,), 0.5, device="cuda") for _ in range(2)]
    for p, a in zip((gamma, beta), acc):
        sinks.add(p, a, 0)
    sinks.begin_step()
    sinks.set_active(True)
    f(x, leaves[3]).backward(dz)
    sinks.set_active(False)
    sinks.close()
    for a, w in zip(acc, want):
        near(a, w.double() + 0.5, w.double().abs() + 0.5, 8, "accumulator")
