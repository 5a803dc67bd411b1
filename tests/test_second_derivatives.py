"""Group norm, scans and distillation have first derivatives alone: asked for a second one they refuse, and do not give zero."""
import pytest
import torch

from eagersgd_b200.ops import functional as ops
from eagersgd_b200.ops import scan

gpu = pytest.mark.gpu


def _calls(dev="cuda", dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=dtype).to(dev)  # noqa: E731
    image, p, seq, narrow, taps = r(2, 8, 3, 3), r(8), r(2, 7, 6), r(2, 7, 4), r(6, 3)
    values, named = r(2, 3), torch.tensor([[1, 2, 3], [4, 5, 6]], device=dev)
    return {"group_norm_act": (image, lambda x: ops.group_norm_act(x, 2, p, p, "silu")),
            "group_norm_act, shortcut": (image, lambda x: ops.group_norm_act(image.detach(), 2, p, p, "silu", x)),
            "distillation_loss": (r(2, 9), lambda x: ops.distillation_loss(x, values, named)),
            "causal_conv": (seq, lambda x: scan.causal_conv(x, taps)),
            "selective_scan": (seq, lambda x: scan.selective_scan(x, seq, -torch.ones(6, 4, dtype=dtype, device=dev), narrow, narrow))}


@gpu
@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_refused_once_it_is_asked_for(name):
    x, f = _calls()[name]
    x.requires_grad_()
    y = f(x).square().sum()
    plain, = torch.autograd.grad(y, x, retain_graph=True)
    first, = torch.autograd.grad(y, x, create_graph=True)
    assert torch.equal(first, plain)
    with pytest.raises(RuntimeError, match="no second derivative"):
        # beside another path from the gradient to x: without the refusal that path alone would count
        torch.autograd.grad((first * x).sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (first * x).sum().backward()


@gpu
def test_a_shortcut_without_activation_has_them_all():
    """Its gradient is the one that arrives."""
    x, p = torch.randn(2, 8, 3, 3, device="cuda", requires_grad=True), torch.ones(8, device="cuda")
    image = torch.randn(2, 8, 3, 3, device="cuda")
    z = ops.group_norm_act(image, 2, p, p, None, x)
    first, = torch.autograd.grad((z ** 3).sum(), x, create_graph=True)
    second, = torch.autograd.grad((first * image).sum(), x)
    assert torch.allclose(second, 6 * z.detach() * image, rtol=1e-5, atol=1e-5)


@gpu
def test_the_gradient_that_arrives():
    """A backward pass is linear in it, but that derivative is not made either."""
    x, f = _calls()["group_norm_act"]
    x.requires_grad_()
    dz = torch.randn_like(x).requires_grad_()
    dx, = torch.autograd.grad(f(x), x, dz, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(dx.sum(), dz)


@gpu
def test_a_graph_that_is_created_and_not_used():
    x, f = _calls()["selective_scan"]
    x.requires_grad_()
    f(x).sum().backward(create_graph=True)
    got, x.grad = x.grad.detach(), None
    f(x).sum().backward()
    assert torch.equal(got, x.grad)


@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_the_restatements_have_one(name):
    x, f = _calls("cpu", torch.float64)[name]
    x.requires_grad_()
    first, = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
    assert torch.autograd.grad((first * x).sum(), x)[0].any()
