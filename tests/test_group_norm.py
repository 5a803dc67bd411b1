"""Group norm with shortcut and activation: against the formula in 64 bits, and what it refuses."""
import pytest
import torch

from near import near
from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops

BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
gpu = pytest.mark.gpu


def _image(g, *shape, dtype=BF16, device="cuda", scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(device).contiguous(memory_format=torch.channels_last)


def _formula(x, groups, gamma, beta, activation, residual):
    """(z, pre) in 64 bits."""
    n, c = x.shape[:2]
    v = x.reshape(n, groups, -1)
    mean = v.mean(2, keepdim=True)
    var = ((v - mean) ** 2).mean(2, keepdim=True)
    pre = ((v - mean) / (var + EPS).sqrt()).reshape(x.shape) * gamma.view(1, c, 1, 1) + beta.view(1, c, 1, 1)
    pre = pre if residual is None else pre + residual
    z = pre.clamp(min=0) if activation == "relu" else pre * torch.sigmoid(pre) if activation == "silu" else pre
    return z, pre


def _check(x, groups, gamma, beta, activation, residual, dz, dev=None):
    """Forward and backward on x's device against the formula, whose gradients come from differentiating it."""
    wide = [t.detach().double().cpu().contiguous().requires_grad_() for t in (x, gamma, beta)]
    wr = residual.detach().double().cpu().contiguous().requires_grad_() if residual is not None else None
    want, pre = _formula(wide[0], groups, wide[1], wide[2], activation, wr)
    if activation == "relu":            # next to its border either slope is right
        dz = torch.where(pre.detach().abs().to(dz.device) < 1e-3, 0.0, dz.double()).to(dz.dtype).contiguous(memory_format=torch.channels_last)
    wants = torch.autograd.grad(want, wide + ([wr] if wr is not None else []), dz.double().cpu())
    leaves = [t.detach().requires_grad_() for t in (x, gamma, beta)] + ([residual.detach().requires_grad_()] if wr is not None else [])
    z = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation, leaves[3] if wr is not None else None)
    assert z.dtype == x.dtype and z.is_contiguous(memory_format=torch.channels_last)
    gots = torch.autograd.grad(z, leaves, dz)
    per = x[0].numel() // groups
    v = wide[0].detach().reshape(x.shape[0], groups, per)
    rstd = 1.0 / (v.var(2, unbiased=False) + EPS).sqrt()
    # The mean of values up to m is off by some 8 roundings of m, and n with it by that times rstd; the sums of squares about a value of
    # the data lose as much as a thread's rows (up to 64 here) of them.
    spread = 8 * (v.abs().amax(2) * rstd).max().item() + 64
    top = (pre.detach().abs().max() + gamma.abs().max().cpu()).item()
    near(z, want.detach(), top, spread, "z")
    a = dz.double().cpu().abs() * (1.2 if activation == "silu" else 1.0)
    n = ((v - v.mean(2, keepdim=True)) * rstd.unsqueeze(2)).reshape(x.shape)
    wg = gamma.double().cpu().abs().view(1, -1, 1, 1)
    # dx: every term is at most that large, and slope' <= 1 carries the error of pre on
    term = (rstd.amax() * (a * wg * (1 + top)).amax() * (1 + n.abs().amax() ** 2)).item()
    near(gots[0], wants[0], term, 4 * spread, "dx")
    for k, name, amp in ((1, "dgamma", (a * (1 + top) * (n.abs() + 1)).sum((0, 2, 3))), (2, "dbeta", (a * (1 + top)).sum((0, 2, 3)))):
        near(gots[k], wants[k], amp, 2 * spread, name)
    if wr is not None:
        near(gots[3], wants[3], (a * (1 + top)).amax().item(), 2 * spread, "dresidual")


SHAPES = [
    # n, c, h, w, groups
    (1, 8, 1, 1, 1), (2, 6, 3, 5, 3), (3, 5, 1, 1, 1), (2, 24, 7, 7, 8), (1, 48, 15, 15, 6), (2, 64, 9, 11, 32), (4, 16, 32, 32, 4),
    (1, 2048, 7, 7, 32), (2, 264, 5, 3, 3), (1, 64, 112, 112, 32), (3, 4096, 1, 2, 1), (2, 1032, 2, 2, 43), (1, 4095, 2, 1, 1), (17, 32, 1, 3, 8),
]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,c,h,w,groups", SHAPES)
def test_sizes(n, c, h, w, groups, dtype):
    g = torch.Generator().manual_seed(n * c + h)
    x, dz, res = (_image(g, n, c, h, w, dtype=dtype, scale=s, shift=t) for s, t in ((2, 0.5), (1, 0), (1, 0)))
    gamma, beta = (torch.randn(c, generator=g) * 0.3 + 1).cuda(), (torch.randn(c, generator=g) * 0.3).cuda()
    _check(x, groups, gamma, beta, "silu", res if (n + c) % 2 else None, dz)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("activation", [None, "relu", "silu"])
@pytest.mark.parametrize("residual", [False, True])
def test_activations_and_shortcut(dtype, activation, residual):
    g = torch.Generator().manual_seed(3)
    x, dz, res = (_image(g, 3, 40, 6, 7, dtype=dtype) for _ in range(3))
    gamma, beta = torch.randn(40, generator=g).cuda(), torch.randn(40, generator=g).cuda()
    _check(x, 5, gamma, beta, activation, res if residual else None, dz)


@gpu
@pytest.mark.parametrize("shift", [100.0, -3000.0])
def test_a_mean_far_from_zero_costs_no_digits_of_the_variance(shift):
    g = torch.Generator().manual_seed(4)
    x, dz = _image(g, 2, 32, 28, 28, dtype=F32, shift=shift), _image(g, 2, 32, 28, 28, dtype=F32)
    _check(x, 4, torch.ones(32).cuda(), torch.zeros(32).cuda(), "silu", None, dz)


@gpu
def test_first_pixel_of_a_group_far_from_the_others():
    g = torch.Generator().manual_seed(5)
    x, dz = _image(g, 1, 32, 56, 56, dtype=F32), _image(g, 1, 32, 56, 56, dtype=F32)
    x[0, :, 0, 0] = 1000.0
    _check(x, 4, torch.ones(32).cuda(), torch.zeros(32).cuda(), None, None, dz)


@gpu
def test_constant_groups_and_values_that_are_no_numbers():
    x = torch.full((2, 16, 4, 4), 3.0, device="cuda").contiguous(memory_format=torch.channels_last)
    gamma, beta = torch.ones(16).cuda(), torch.arange(16.0).cuda()
    z = ops.group_norm_act(x, 4, gamma, beta)
    assert torch.equal(z, beta.view(1, 16, 1, 1).expand_as(z))
    x[1, 5, 2, 2] = float("nan")            # stays in its sample's group
    z = ops.group_norm_act(x, 4, gamma, beta, "relu")
    bad = torch.zeros(2, 16, dtype=torch.bool)
    bad[1, 4:8] = True
    assert torch.equal(torch.isnan(z).all((2, 3)).cpu(), bad) and torch.equal(torch.isnan(z).any(3).any(2).cpu(), bad)


@gpu
def test_other_layouts_and_beginnings():
    """NCHW, slices of something wider, and a tensor that does not begin on 16 bytes give what the dense tensor gives."""
    g = torch.Generator().manual_seed(6)
    x = _image(g, 2, 32, 6, 6)
    gamma, beta = torch.randn(32, generator=g).cuda(), torch.randn(32, generator=g).cuda()
    want = ops.group_norm_act(x, 4, gamma, beta, "silu", residual=x)
    wide = torch.cat([x, x], 1).contiguous(memory_format=torch.channels_last)[:, 32:]
    odd = torch.empty(x.numel() + 1, dtype=BF16, device="cuda")[1:].view(2, 6, 6, 32).permute(0, 3, 1, 2)
    odd.copy_(x)
    for v in (x.contiguous(), wide, odd):
        assert torch.equal(ops.group_norm_act(v, 4, gamma, beta, "silu", residual=v), want)
        assert torch.equal(ops.group_norm_act(v.detach().requires_grad_(), 4, gamma, beta, "silu", residual=v), want)


@gpu
def test_nothing_in_nothing_out():
    gamma = torch.ones(8, device="cuda", requires_grad=True)
    beta = torch.zeros(8, device="cuda", requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        z = ops.group_norm_act(x, 2, gamma, beta, "silu")
        dx, dg, db = torch.autograd.grad(z.sum(), [x, gamma, beta])
        assert z.shape == dx.shape == shape and not dg.any() and not db.any()


@gpu
def test_some_gradients_only():
    g = torch.Generator().manual_seed(7)
    x, dz, res = (_image(g, 2, 16, 5, 5) for _ in range(3))
    p = [torch.randn(16, generator=g).cuda() for _ in range(2)]
    leaves = [t.detach().requires_grad_() for t in (x, p[0], p[1], res)]
    all_ = torch.autograd.grad(ops.group_norm_act(leaves[0], 4, leaves[1], leaves[2], "silu", leaves[3]), leaves, dz)
    for k in range(4):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, p[0], p[1], res))]
        got, = torch.autograd.grad(ops.group_norm_act(some[0], 4, some[1], some[2], "silu", some[3]), some[k], dz)
        assert torch.equal(got, all_[k])


@gpu
def test_the_same_input_twice_and_a_kept_graph():
    g = torch.Generator().manual_seed(8)
    x, dz = _image(g, 2, 16, 5, 5, dtype=F32).requires_grad_(), _image(g, 2, 16, 5, 5, dtype=F32)
    gamma, beta = torch.ones(16).cuda(), torch.zeros(16).cuda()
    z = ops.group_norm_act(x, 4, gamma, beta, None, x)
    first, = torch.autograd.grad(z, x, dz, retain_graph=True)
    again, = torch.autograd.grad(z, x, dz)
    assert torch.equal(first, again)
    wide = x.detach().double().cpu().contiguous().requires_grad_()
    want, = torch.autograd.grad(_formula(wide, 4, gamma.double().cpu(), beta.double().cpu(), None, wide)[0], wide, dz.double().cpu())
    near(first, want, 30.0, 200, "dx")


@gpu
def test_captured_on_its_own_stream_and_replayed():
    g = torch.Generator().manual_seed(9)
    x, gamma, beta = _image(g, 2, 64, 14, 14), torch.ones(64).cuda(), torch.zeros(64).cuda()
    xs = [_image(g, 2, 64, 14, 14) for _ in range(2)]
    with torch.no_grad():
        wants = [ops.group_norm_act(v, 8, gamma, beta, "relu") for v in xs]
        graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
        for graph in graphs:
            with torch.cuda.graph(graph):
                outs.append(ops.group_norm_act(x, 8, gamma, beta, "relu"))
        for v, want, graph, out in zip(xs, wants, graphs, outs):
            x.copy_(v)
            graph.replay()
            assert torch.equal(out, want)


@gpu
def test_images_past_32_bits():
    x = torch.zeros(1100, 256, 128, 64, dtype=BF16, device="cuda").permute(0, 3, 1, 2)         # 2.3e9 values, channels last
    g = torch.Generator().manual_seed(1)
    x[-1:].copy_(_image(g, 1, 64, 256, 128))
    gamma, beta = torch.randn(64, generator=g).cuda(), torch.randn(64, generator=g).cuda()
    z = ops.group_norm_act(x, 4, gamma, beta, "silu")
    want = ops.group_norm_act(x[-1:], 4, gamma, beta, "silu").double().cpu()
    near(z[-1:], want, want.abs().max().item(), 4096, "z", roundings=2)      # split otherwise: sums in another order
    del z
    leaf = x.requires_grad_()
    z = ops.group_norm_act(leaf, 4, gamma, beta, "silu")
    dx, = torch.autograd.grad(z, leaf, x.detach())
    one = x[-1:].detach().requires_grad_()
    want, = torch.autograd.grad(ops.group_norm_act(one, 4, gamma, beta, "silu"), one, one.detach())
    near(dx[-1:], want.double().cpu(), want.double().abs().max().item(), 4096, "dx", roundings=2)


@gpu
def test_gradient_against_differences():
    g = torch.Generator().manual_seed(10)
    x, dz, res = (_image(g, 1, 8, 3, 3, dtype=F32) for _ in range(3))
    gamma, beta = torch.randn(8, generator=g).cuda(), torch.randn(8, generator=g).cuda()
    leaves = [t.detach().requires_grad_() for t in (x, gamma, beta, res)]
    grads = torch.autograd.grad(ops.group_norm_act(leaves[0], 2, leaves[1], leaves[2], "silu", leaves[3]), leaves, dz)
    d = [torch.randn(t.shape, generator=g).cuda().contiguous(memory_format=torch.channels_last if t.dim() == 4 else torch.contiguous_format)
         for t in leaves]

    def at(e):
        a = [t.detach() + e * v for t, v in zip(leaves, d)]
        return (ops.group_norm_act(a[0], 2, a[1], a[2], "silu", a[3]).double() * dz.double()).sum().item()
    e = 2.0 ** -7
    slope = sum((u.double() * v.double()).sum().item() for u, v in zip(grads, d))
    # the difference: third derivatives times e^2 (6e-5), and roundings of z (2^-22 of some 70 values of size one) over 2 e
    assert abs((at(e) - at(-e)) / (2 * e) - slope) < 1e-2 * max(1.0, abs(slope))


# ------------------------------------------------------------------------------------------------ without a GPU
def test_the_restatement_is_the_formula():
    g = torch.Generator().manual_seed(11)
    for dtype in (BF16, F32, torch.float64):
        x, res = (_image(g, 2, 12, 3, 4, dtype=dtype, device="cpu") for _ in range(2))
        gamma, beta = torch.randn(12, generator=g), torch.randn(12, generator=g)
        z = ops.group_norm_act(x, 3, gamma, beta, "silu", res)
        want = _formula(x.double(), 3, gamma.double(), beta.double(), "silu", res.double())[0]
        assert z.dtype == x.dtype and (z.double() - want).abs().max() < (2e-2 if dtype == BF16 else 1e-5)


def _fits():
    x = torch.zeros(2, 16, 4, 4, dtype=BF16).contiguous(memory_format=torch.channels_last)
    return dict(x=x, groups=4, gamma=torch.ones(16), beta=torch.zeros(16), act=1, residual=x.clone(), eps=1e-5)


@pytest.mark.parametrize("name,value,message", [
    ("x", torch.zeros(2, 16, 4, dtype=BF16), "4-D"),
    ("x", torch.zeros(2, 16, 4, 4, dtype=torch.float16), "neither"),
    ("x", torch.zeros(2, 12, 4, 4, dtype=BF16), "gamma"),
    ("groups", 3, "groups"), ("groups", 0, "groups"), ("groups", -4, "groups"),
    ("gamma", torch.ones(15), "gamma"), ("gamma", torch.ones(16, dtype=BF16), "gamma"), ("beta", torch.ones(32)[::2], "beta"),
    ("residual", torch.zeros(2, 16, 4, 5, dtype=BF16), "residual"), ("residual", torch.zeros(2, 16, 4, 4), "residual"),
    ("act", 3, "activation"), ("eps", -1.0, "eps"), ("x", None, "not on a GPU"),
])
def test_refusals(name, value, message):
    a = _fits()
    if value is not None:
        a[name] = value
    with pytest.raises(RuntimeError, match=message):
        _build.load_torch().group_norm_act(*a.values())


def test_too_many_channels_a_group_and_unknown_activations_are_refused():
    x = torch.zeros(1, 4097, 1, 1)
    with pytest.raises(RuntimeError, match="channels a group"):
        _build.load_torch().group_norm_act(x, 1, torch.ones(4097), torch.ones(4097), 0, None, 1e-5)
    with pytest.raises(ValueError, match="gelu"):
        ops.group_norm_act(x, 1, torch.ones(4097), torch.ones(4097), "gelu")
