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


def _holes(got, want, name, four):
    """What is no number in the formula is none; nothing else is, but for the other steps of its four where ``four`` is set."""
    got, want = torch.isnan(got).cpu(), torch.isnan(want)
    assert (got | ~want).all(), (name, "a NaN is lost")
    if four:
        t = want.shape[1]
        want = torch.nn.functional.pad(want, (0, 0, 0, -t % 4)).unflatten(1, (-1, 4)).any(2, keepdim=True).expand(-1, -1, 4, -1).flatten(1, 2)[:, :t]
    assert (want | ~got).all(), (name, "a NaN where there is none")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("where", ["u", "dy", "state", "delta", "B", "C"])
@pytest.mark.parametrize("b,t,d,n", [(2, 37, 24, 16), (1, 200, 40, 5), (2, 13, 9, 33)])
def test_what_is_no_number_reaches_what_it_should(b, t, d, n, where, gated, dtype):
    c, dy, state = _scan_case(b, t, d, n, dtype)
    if not gated:
        c["z"] = None
    hole = {"state": state, "dy": dy}.get(where, c.get(where))
    at = (b - 1, t // 2, 3) if where != "state" else (b - 1, d - 1, n - 1)
    # as arithmetic makes them, as they are written down, and with every bit or hardly a bit set
    patterns = [0x7fffffff, 0x7fc00000, -1, 0x7f800001] if hole.dtype == F32 else [0x7fff, 0x7fc0, -1, 0x7f81]
    names = [k for k, v in c.items() if v is not None]
    for bits in patterns:
        hole.view(torch.int32 if hole.dtype == F32 else torch.int16)[at] = bits
        wide = {k: None if v is None else v.double().cpu().requires_grad_() for k, v in c.items()}
        want, want_h = _scan_formula(*[wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")], True, state.double().cpu(), None)
        wants = torch.autograd.grad(want, [wide[k] for k in names], dy.double().cpu())
        leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in c.items()}
        y, h = scan.selective_scan(**leaves, state=state, return_state=True)
        gots = torch.autograd.grad(y, [leaves[k] for k in names], dy)
        _holes(y, want, "y", False)
        _holes(h, want_h, "state", False)
        for k, got, wanted in zip(names, gots, wants):
            _holes(got, wanted, "d" + k, k in ("B", "C"))
        assert torch.isnan(wants[names.index("B")]).any() or torch.isnan(wants[names.index("C")]).any()
