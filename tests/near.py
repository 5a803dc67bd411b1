"""How far a kernel's result may be from the same formula in 64 bits."""
import torch

# a rounding to the type is off by half a step at most, relative to the value
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ULP = 2.0 ** -24            # ... and one in the fp32 arithmetic ahead of it


def near(got, want, amp, steps, what="", roundings=1):
    """``got`` is ``want`` but for ``roundings`` to its type and ``steps`` roundings in fp32 of terms that add up to ``amp``."""
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    got, half = got.detach(), HALF[got.dtype] * roundings
    got = got.double().to(want.device)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    if not isinstance(amp, torch.Tensor):
        amp = torch.tensor(float(amp))
    amp = amp.double().to(want.device).expand_as(want)
    bound = half * want.abs() + steps * ULP * (1 + half) * amp + 1e-37
    off = (got - want).abs()[fine] - bound[fine]
    assert off.numel() == 0 or off.max() <= 0, "%s: off by %.3g, allowed %.3g" % (
        what, (got - want).abs()[fine][off.argmax()], bound[fine][off.argmax()])
