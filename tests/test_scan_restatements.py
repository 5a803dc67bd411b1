"""The plain forms of the causal convolution and the selective scan (CPU, fp64) keep the kernels' promises."""
import pytest
import torch

from eagersgd_b200.ops import scan
from test_scan import _conv_case, _scan_case

F32, F64 = torch.float32, torch.float64
LENGTHS = torch.tensor([0, 1, 3, 5, 9, 99])


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("spoil", [float("nan"), float("inf"), 1e38])
@pytest.mark.parametrize("softplus", [True, False])
def test_what_lies_behind_a_sequence_is_nobodys(dtype, spoil, softplus):
    c, dy, state = _scan_case(6, 9, 5, 4, dtype, "cpu")
    if not softplus:
        c["delta"], c["delta_bias"] = c["delta"].abs() * 0.1, c["delta_bias"].abs() * 0.01
    results = []
    for value in (0.0, spoil):
        leaves = {k: v.clone() for k, v in c.items()}
        for k in ("u", "delta", "B", "C", "z"):
            for i, n in enumerate(LENGTHS):
                leaves[k][i, n:] = value
        leaves = {k: v.requires_grad_() for k, v in leaves.items()}
        y, h = scan.selective_scan(**leaves, softplus=softplus, state=state, lengths=LENGTHS, return_state=True)
        results.append((y.detach(), h, *torch.autograd.grad(y, list(leaves.values()), dy)))
    for a, b in zip(*results):
        assert torch.isfinite(b).all() and torch.equal(a, b)
    x, w, bias, dy = _conv_case(6, 9, 5, 3, dtype, "cpu")
    results = []
    for value in (0.0, spoil):
        leaf = x.clone()
        for i, n in enumerate(LENGTHS):
            leaf[i, n:] = value
        leaves = [v.detach().requires_grad_() for v in (leaf, w, bias)]
        y, last = scan.causal_conv(*leaves, lengths=LENGTHS, return_state=True)
        results.append((y.detach(), last, *torch.autograd.grad(y, leaves, dy)))
    for a, b in zip(*results):
        assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("b,t", [(0, 5), (3, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_empty_sequences_and_batches(b, t, dtype):
    c, dy, state = _scan_case(b, t, 6, 4, dtype, "cpu")
    leaves = {k: v.detach().requires_grad_() for k, v in c.items()}
    y, h = scan.selective_scan(**leaves, state=state, return_state=True)
    assert y.shape == (b, t, 6) and y.dtype == dtype and torch.equal(h, state.to(h.dtype))
    for g, k in zip(torch.autograd.grad(y, list(leaves.values()), dy), leaves):
        assert g.shape == leaves[k].shape and not g.any()
    assert scan.selective_scan(**dict(c, D=None, z=None, delta_bias=None)).shape == (b, t, 6)
    for k in (2, 4):
        x, w, bias, dy = _conv_case(b, t, 6, k, dtype, "cpu")
        leaves = [v.requires_grad_() for v in (x, w, bias)]
        ahead = torch.randn(b, k - 1, 6, dtype=dtype)
        y, last = scan.causal_conv(*leaves, state=ahead, return_state=True)
        assert y.shape == (b, t, 6) and torch.equal(last, ahead)
        for g, v in zip(torch.autograd.grad(y, leaves, dy), leaves):
            assert g.shape == v.shape and not g.any()
        assert scan.causal_conv(x, w).shape == (b, t, 6)
