"""Gradients of the selective scan where rounding or a value that is no number would show: against the recurrence in 64 bits."""
import pytest
import torch

from near import near
from test_scan import _amplitudes, _scan_case, _scan_formula
from eagersgd_b200.ops import scan

BF16, F32 = torch.bfloat16, torch.float32
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [5, 16, 31, 64])
def test_channels_that_nearly_cancel_leave_their_difference(n, dtype):
    """Pairs of channels with opposite gradients and time steps one bf16 step apart: dB and dC are 2^-7 of their terms, which a sum of
    factors of eleven bits (off by up to 2^-11 of the terms) would not show to the eight bits that the result has."""
    c, dy, _ = _scan_case(4, 9, 6, n, dtype)
    c.update(D=None, z=None, delta_bias=None)
    c["delta"] = (0.5 + 0.4 * c["delta"].float().abs().clamp(max=1.0)).to(dtype)
    for k in ("u", "delta"):
        c[k][..., 1::2] = c[k][..., ::2]
    c["delta"][..., 1::2] *= 1 + 2.0 ** -7
    c["A"][1::2] = c["A"][::2]
    dy[..., 1::2] = -dy[..., ::2]
    wide = {k: None if v is None else v.double().cpu().requires_grad_() for k, v in c.items()}
    want, _ = _scan_formula(*[wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")], False, None, None)
    wants = torch.autograd.grad(want, [wide["B"], wide["C"]], dy.double().cpu())
    _, _, amp = _amplitudes(c, dy, False, None, None)
    leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in c.items()}
    gots = torch.autograd.grad(scan.selective_scan(**leaves, softplus=False), [leaves["B"], leaves["C"]], dy)
    for k, got, wanted in zip("BC", gots, wants):
        # twelve roundings a step of the state or of its gradient, as much for the other factor, and the sum over the channels
        near(got, wanted, amp[k], 2 * (12 * 9 + 2 * 6 + 32), "d" + k)
