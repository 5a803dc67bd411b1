"""Few sequences are scanned in chunks of steps: what goes from chunk to chunk, and sequences that end inside one."""
import pytest
import torch

from near import near
from eagersgd_b200.ops import scan
from test_scan import _amplitudes, _scan_case, _scan_check, _scan_formula

BF16, F32 = torch.bfloat16, torch.float32
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
gpu = pytest.mark.gpu


def _against(c, dy, state, softplus):
    """Element by element: the sizes of these run over tens of decades."""
    wide = {k: v.double().cpu().requires_grad_() for k, v in c.items()}
    h0 = None if state is None else state.double().cpu()
    want, want_h = _scan_formula(*[wide[k] for k in NAMES], softplus, h0, None)
    wants = torch.autograd.grad(want, [wide[k] for k in NAMES], dy.double().cpu())
    leaves = {k: v.detach().requires_grad_() for k, v in c.items()}
    y, h = scan.selective_scan(**leaves, softplus=softplus, state=state, return_state=True)
    gots = torch.autograd.grad(y, [leaves[k] for k in NAMES], dy)
    return (y, want.detach()), (h, want_h.detach()), dict(zip(NAMES, zip(gots, wants)))


@gpu
@pytest.mark.parametrize("n", [4, 16, 40])
def test_states_of_zero_pass_chunks_that_would_overflow(n):
    """Rates above zero, inputs in the last steps alone and gradients in the first ones alone: e^(dt A) of a chunk is infinite, the
    state and its gradient that pass it are zero."""
    c, dy, _ = _scan_case(1, 330, 16, n, F32)
    c["A"] = c["A"].abs().clamp(max=2.0)
    c["delta"], c["delta_bias"] = 3 + 0.1 * c["delta"], torch.zeros_like(c["delta_bias"])
    c["u"][:, :-8] = 0
    dy[:, 8:] = 0
    (y, want), (h, want_h), grads = _against(c, dy, None, True)
    amp_y, amp_h, amp = _amplitudes(c, torch.ones_like(dy), True, None, None)
    # a rate of 2 and steps of 3 multiply by e^6 each: eight roundings of its argument and twelve others, of the last eight steps
    near(y, want, amp_y, 2000, "y")
    near(h, want_h, amp_h, 2000, "state")
    for k in ("u", "z", "B", "C", "D", "delta"):
        got, wanted = grads[k]
        assert torch.isfinite(got).all(), k
        assert ((got.double().cpu() - wanted).abs() <= 2000 * 2.0 ** -24 * wanted.abs().max()).all(), k
    assert torch.isfinite(grads["A"][0]).all() and grads["u"][1].any()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_states_fade_over_a_chunk(dtype):
    """e^(dt A) of a chunk is below what fp32 has, times the state it is not."""
    c, dy, state = _scan_case(1, 200, 16, 16, dtype)
    c["A"] = -torch.full_like(c["A"], 1.0)
    c["delta"] = torch.full_like(c["delta"], 6.0)
    state = state * 1e30
    (y, want), (h, want_h), _ = _against(c, dy, state, False)
    amp_y, amp_h, _ = _amplitudes(c, dy, False, state, None)
    # A channel whose bias makes its steps negative grows by e^(200 |dt|), e^22 or more here: times 1e30 that is beyond fp32.
    held = (6 + c["delta_bias"] > -0.01).cpu()
    assert held.sum() >= 8
    # an argument of 6 is off by four roundings of it and the exponential by four more, a step; the sums as ever
    near(y[..., held.cuda()], want[..., held], amp_y[..., held], 40 * 200, "y")
    near(h[:, held.cuda()], want_h[:, held], amp_h[:, held], 40 * 200, "state")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,t,d,n", [(1, 330, 40, 16), (3, 500, 24, 5), (6, 260, 16, 33)])
def test_chunks_of_sequences_that_end(b, t, d, n, dtype):
    c, dy, state = _scan_case(b, t, d, n, dtype)
    for lengths in (torch.linspace(0, t, b).long(), torch.tensor([1, 16, 17, t - 1, t + 5, 127])[:b], torch.full((b,), t // 2)):
        _scan_check(c, dy, state=state, lengths=lengths.cuda())
