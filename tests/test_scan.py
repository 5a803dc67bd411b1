"""The short causal convolution and the selective scan: whole sequences, single steps and gradients against the recurrences in 64 bits."""
import pytest
import torch

from near import near
from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops
from eagersgd_b200.ops import scan

BF16, F32 = torch.bfloat16, torch.float32
gpu = pytest.mark.gpu


def _wide(*ts):
    return [None if t is None else t.detach().double().cpu() for t in ts]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ causal convolution
def _conv_formula(x, w, bias, activation, state, lengths):
    """(y, the last K - 1 inputs), step by step."""
    b, t, d = x.shape
    k = w.shape[1]
    ys, last = [], []
    for i in range(b):
        n = t if lengths is None else max(0, min(t, int(lengths[i])))
        ahead = x.new_zeros(k - 1, d) if state is None else state[i]
        seq = torch.cat([ahead, x[i, :n]])
        rows = []
        for s in range(n):
            pre = sum(w[:, j] * seq[s + j] for j in range(k))
            pre = pre if bias is None else pre + bias
            rows.append(pre * torch.sigmoid(pre) if activation == "silu" else pre)
        rows += [x.new_zeros(d)] * (t - n)
        ys.append(torch.stack(rows) if rows else x.new_zeros(0, d))
        last.append(seq[n:n + k - 1])
    return torch.stack(ys), torch.stack(last)


CONV = [(1, 1, 1, 2), (2, 3, 8, 4), (1, 5, 7, 3), (3, 17, 24, 4), (2, 70, 264, 4), (1, 300, 40, 2), (5, 33, 129, 3), (1, 2, 2048, 4), (2, 1030, 16, 4)]


def _conv_case(b, t, d, k, dtype, device="cuda"):
    g = _gen(b * t + d)
    x, dy = (torch.randn(b, t, d, generator=g).to(dtype).to(device) for _ in range(2))
    return x, torch.randn(d, k, generator=g).to(device), torch.randn(d, generator=g).to(device), dy


def _conv_check(x, w, bias, activation, state, lengths, dy):
    leaves = [v.detach().requires_grad_() for v in (x, w, bias) if v is not None]
    wide = [v.requires_grad_() for v in _wide(x, w, bias) if v is not None]
    ws, = _wide(state)
    wb = wide[2] if bias is not None else None
    want, want_last = _conv_formula(wide[0], wide[1], wb, activation, ws, lengths)
    wants = torch.autograd.grad(want, wide, _wide(dy)[0], allow_unused=True)
    wants = [torch.zeros_like(v) if g is None else g for v, g in zip(wide, wants)]
    y, last = scan.causal_conv(*leaves, *([None] if bias is None else []), activation, state, lengths, True)
    gots = torch.autograd.grad(y, leaves, dy)
    assert not last.requires_grad and torch.equal(last.double().cpu(), want_last.detach())     # inputs, as they are
    amax = lambda v: v.detach().abs().max().item() if v is not None and v.numel() else 0.0  # noqa: E731
    pre = w.shape[1] * amax(w) * max(amax(x), amax(state)) + amax(bias)          # no sum of products is larger
    # K products and sums, and an activation of a dozen operations whose slope is below 1.1
    near(y, want.detach(), 2 * pre + 1, 32, "y")
    near(gots[0], wants[0], w.shape[1] * amax(w) * amax(dy) * (2 + pre), 64, "dx")
    n = x.shape[0] * x.shape[1]
    # a sum of n terms, each with the slope's error (up to pre roundings), in partial sums of fewer than 64 + n / 64
    terms = 1.1 * n * amax(dy) * (1 + pre)
    near(gots[1], wants[1], terms * max(amax(x), amax(state)), 96, "dweight")
    if bias is not None:
        near(gots[2], wants[2], terms, 96, "dbias")
    with torch.no_grad():
        assert torch.equal(scan.causal_conv(x, w, bias, activation, state, lengths), y)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,t,d,k", CONV)
def test_conv_sizes(b, t, d, k, dtype):
    x, w, bias, dy = _conv_case(b, t, d, k, dtype)
    _conv_check(x, w, bias if t % 2 else None, "silu" if d % 2 == 0 or t == 1 else None, None, None, dy)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [2, 3, 4])
def test_conv_lengths_and_states(dtype, k):
    """Sequences of every length from none on, with a state ahead; what lies behind them is not read."""
    x, w, bias, dy = _conv_case(8, 37, 40, k, dtype)
    lengths = torch.tensor([0, 1, 2, 3, 5, 36, 37, 99])
    state = torch.randn(8, k - 1, 40, generator=_gen(2)).to(dtype).cuda()
    _conv_check(x, w, bias, "silu", state, lengths.cuda(), dy)
    spoilt = x.clone()
    for i, n in enumerate(lengths):
        spoilt[i, n:] = float("nan")
    leaf = spoilt.requires_grad_()
    y = scan.causal_conv(leaf, w, bias, "silu", state, lengths.cuda())
    assert torch.equal(y, scan.causal_conv(x, w, bias, "silu", state, lengths.cuda()))
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.isfinite(dx).all() and all(not dx[i, n:].any() for i, n in enumerate(lengths))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_conv_layouts(dtype):
    """Slices of a projection, time-first and transposed inputs, and ones that begin anywhere."""
    x, w, bias, dy = _conv_case(2, 19, 32, 4, dtype)
    want = scan.causal_conv(x, w, bias)
    wide = torch.randn(2, 19, 96, device="cuda").to(dtype)
    wide[:, :, 32:64] = x
    odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x)
    for v in (wide[:, :, 32:64], x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2), odd, x.flip(1).flip(1)):
        assert torch.equal(scan.causal_conv(v, w, bias), want)
        leaf = v.detach().requires_grad_()
        got, = torch.autograd.grad(scan.causal_conv(leaf, w, bias), leaf, dy)
        ref = x.detach().requires_grad_()
        assert torch.equal(got, torch.autograd.grad(scan.causal_conv(ref, w, bias), ref, dy)[0])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,d,k", [(1, 1, 2), (3, 40, 4), (16, 2048, 4), (5, 129, 3)])
def test_conv_steps_continue_a_sequence(b, d, k, dtype):
    x, w, bias, _ = _conv_case(b, 9, d, k, dtype)
    want, want_state = scan.causal_conv(x, w, bias, return_state=True)
    y, state = scan.causal_conv(x[:, :5], w, bias, return_state=True)
    assert torch.equal(y, want[:, :5])
    for t in range(5, 9):
        before = state.clone()
        out = None if t == 5 else state if t == 6 else torch.empty_like(state)      # its own, in place, the caller's
        y, new = scan.causal_conv_step(x[:, t], state, w, bias, out=out)
        assert out is None or new.data_ptr() == out.data_ptr()
        assert out is state or torch.equal(state, before)
        assert torch.equal(y, want[:, t])
        state = new
    assert torch.equal(state, want_state)


# ------------------------------------------------------------------------------------------------ selective scan
def _scan_formula(u, delta, A, B, C, D, z, bias, softplus, state, lengths):
    """(y, last state, the same recurrence over absolute values as an amplitude)."""
    raw = delta if bias is None else delta + bias
    dt = torch.nn.functional.softplus(raw, threshold=50.0) if softplus else raw
    b, t, d = u.shape
    n = torch.full((b,), t) if lengths is None else lengths.clamp(0, t)
    h = u.new_zeros(b, d, A.shape[1]) if state is None else state
    ys = []
    for i in range(t):
        live = (i < n).view(b, 1, 1)
        new = torch.exp(dt[:, i, :, None] * A) * h + dt[:, i, :, None] * u[:, i, :, None] * B[:, i, None, :]
        h = torch.where(live, new, h)
        y = (h * C[:, i, None, :]).sum(2)
        y = y if D is None else y + D * u[:, i]
        y = y if z is None else y * z[:, i] * torch.sigmoid(z[:, i])
        ys.append(torch.where(live[:, :, 0], y, torch.zeros_like(y)))
    return torch.stack(ys, 1) if ys else u.new_zeros(b, 0, d), h


def _scan_case(b, t, d, n, dtype, device="cuda", seed=0):
    g = _gen(seed + b * t + d + n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rate = torch.exp(torch.rand(d, generator=g) * 4.6 - 6.9)
    c = dict(u=r(b, t, d).to(dtype), delta=(0.5 * r(b, t, d)).to(dtype), A=-torch.arange(1, n + 1).float().repeat(d, 1) * torch.exp(0.1 * r(d, n)),
             B=r(b, t, n).to(dtype), C=r(b, t, n).to(dtype), D=1 + 0.1 * r(d), z=r(b, t, d).to(dtype), delta_bias=rate + torch.log(-torch.expm1(-rate)))
    return {k: v.to(device) for k, v in c.items()}, r(b, t, d).to(dtype).to(device), r(b, d, n).to(device)


def _amplitudes(c, dy, softplus, state, lengths):
    """The results of the same formulas with every term's absolute value: what the roundings of the terms are relative to."""
    w = {k: None if v is None else v.detach().double().cpu() for k, v in c.items()}
    raw = w["delta"] if w["delta_bias"] is None else w["delta"] + w["delta_bias"]
    dt = (torch.nn.functional.softplus(raw, threshold=50.0) if softplus else raw).abs().detach().requires_grad_()
    a = dict(u=w["u"].abs(), A=w["A"], B=w["B"].abs(), C=w["C"].abs(), D=None if w["D"] is None else w["D"].abs(),
             z=None if w["z"] is None else w["z"].abs() + 1)
    for k in a:
        if a[k] is not None:
            a[k] = a[k].detach().requires_grad_()
    y, h = _scan_formula(a["u"], dt, a["A"], a["B"], a["C"], a["D"], a["z"], None, False, None if state is None else _wide(state)[0].abs(), lengths)
    leaves = {k: v for k, v in a.items() if v is not None}
    leaves["dt"] = dt
    grads = torch.autograd.grad(y, list(leaves.values()), dy.double().cpu().abs() + 1e-3, allow_unused=True)
    return y.detach(), h.detach(), {k: torch.zeros_like(v) if g is None else g.abs() for (k, v), g in zip(leaves.items(), grads)}


def _scan_check(c, dy, softplus=True, state=None, lengths=None):
    names = [k for k, v in c.items() if v is not None]
    wide = {k: (v.detach().double().cpu().requires_grad_() if v is not None else None) for k, v in c.items()}
    args = [wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    lens = None if lengths is None else lengths.cpu()
    want, want_h = _scan_formula(*args, softplus, _wide(state)[0], lens)
    wants = torch.autograd.grad(want, [wide[k] for k in names], dy.double().cpu(), allow_unused=True)
    wants = [torch.zeros_like(wide[k]) if g is None else g for k, g in zip(names, wants)]
    leaves = {k: (v.detach().requires_grad_() if v is not None else None) for k, v in c.items()}
    y, h = scan.selective_scan(**leaves, softplus=softplus, state=state, lengths=lengths, return_state=True)
    assert y.dtype == c["u"].dtype and h.dtype == F32 and not h.requires_grad
    gots = torch.autograd.grad(y, [leaves[k] for k in names], dy)
    amp_y, amp_h, amp = _amplitudes(c, dy, softplus, state, lens)
    t, n = c["u"].shape[1], c["A"].shape[1]
    # every step multiplies the state by an exponential (of an argument of a few units: 8 roundings) and adds a product; the sums
    # over the states and the gate add 2 n + 32
    steps = 12 * max(t, 1) + 2 * n + 32
    near(y, want.detach(), amp_y, steps, "y")
    near(h, want_h.detach(), amp_h, steps, "state")
    big = lambda v: v.max().item() if v.numel() else 0.0  # noqa: E731
    for k, got, wanted in zip(names, gots, wants):
        if k in ("B", "C"):
            # sums over the channels of products of a state: with bf16 sequences the two factors have eleven bits, each off by half a step
            bits = 2.0 ** 14 if c["u"].dtype == BF16 else 0.0
            near(got, wanted, big(amp[k]), 2 * steps + bits, "d" + k)
        elif k in ("delta", "delta_bias"):
            near(got, wanted, big(amp["dt"]) if k == "delta" else amp["dt"].sum((0, 1)).max().item(), 4 * steps, "d" + k)
        elif k == "z":
            near(got, wanted, 2 * big(amp_y) * (dy.double().abs().max().item() + 1e-3), 2 * steps, "dz")
        else:
            near(got, wanted, big(amp[k]), 4 * steps, "d" + k)
    with torch.no_grad():
        assert torch.equal(scan.selective_scan(**c, softplus=softplus, state=state, lengths=lengths), y)


SCAN = [(1, 1, 1, 1), (2, 3, 5, 4), (1, 8, 33, 16), (3, 9, 64, 16), (2, 33, 40, 5), (1, 70, 129, 8), (2, 65, 31, 32), (1, 40, 24, 64), (4, 17, 100, 3),
        (1, 130, 260, 16), (2, 31, 17, 17)]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,t,d,n", SCAN)
def test_scan_sizes(b, t, d, n, dtype):
    c, dy, _ = _scan_case(b, t, d, n, dtype)
    _scan_check(c, dy)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("without", [("z",), ("D",), ("delta_bias",), ("z", "D", "delta_bias")])
def test_scan_without_some_operands(without, dtype):
    c, dy, _ = _scan_case(2, 21, 24, 16, dtype)
    _scan_check({k: None if k in without else v for k, v in c.items()}, dy)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_time_steps_as_they_are(dtype):
    c, dy, _ = _scan_case(2, 21, 24, 16, dtype)
    c["delta"], c["delta_bias"] = (c["delta"].float().abs() * 0.1).to(dtype), c["delta_bias"].abs() * 0.01
    c["delta"][:, 3] = 0                # the state waits for a step
    _scan_check(c, dy, softplus=False)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_lengths_and_states(dtype):
    c, dy, state = _scan_case(9, 37, 40, 16, dtype)
    lengths = torch.tensor([0, 1, 7, 8, 9, 32, 33, 37, 99])
    _scan_check(c, dy, state=state, lengths=lengths.cuda())
    y, h = scan.selective_scan(**c, state=state, lengths=lengths.cuda(), return_state=True)
    assert torch.equal(h[0], state[0])
    spoilt = {k: v.clone() for k, v in c.items()}
    for k in ("u", "delta", "B", "C", "z"):
        for i, n in enumerate(lengths):
            spoilt[k][i, n:] = float("nan")
        spoilt[k].requires_grad_()
    y2 = scan.selective_scan(**spoilt, state=state, lengths=lengths.cuda())
    assert torch.equal(y, y2)
    for g in torch.autograd.grad(y2, [spoilt[k] for k in ("u", "delta", "B", "C", "z")], dy):
        assert torch.isfinite(g).all() and all(not g[i, n:].any() for i, n in enumerate(lengths))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_layouts(dtype):
    """Operands that are slices of projections, time-first, or begin anywhere."""
    c, dy, _ = _scan_case(2, 19, 32, 16, dtype)
    want = scan.selective_scan(**c)
    grads = lambda v: torch.autograd.grad(scan.selective_scan(**v), [v[k] for k in v], dy)  # noqa: E731
    ref = grads({k: v.detach().requires_grad_() for k, v in c.items()})
    wide = torch.cat([c["z"], c["u"], c["delta"]], 2)
    bc = torch.cat([c["B"], c["C"], c["u"][:, :, :5]], 2)
    sliced = dict(c, z=wide[:, :, :32], u=wide[:, :, 32:64], delta=wide[:, :, 64:], B=bc[:, :, :16], C=bc[:, :, 16:32])
    first = dict(c, **{k: c[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("u", "z", "B")})
    odd = dict(c, **{k: torch.empty(c[k].numel() + 1, dtype=dtype, device="cuda")[1:].view(c[k].shape).copy_(c[k]) for k in ("u", "delta", "z", "B", "C")})
    across = dict(c, **{k: c[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("u", "C")})
    for v in (sliced, first, odd, across):
        assert torch.equal(scan.selective_scan(**v), want)
        for got, wanted in zip(grads({k: t.detach().requires_grad_() for k, t in v.items()}), ref):
            assert torch.equal(got, wanted)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,d,n", [(1, 1, 1), (3, 40, 16), (2, 129, 5), (4, 24, 64), (70, 33, 8), (250, 260, 16)])
def test_scan_steps_continue_a_sequence(b, d, n, dtype):
    c, _, state = _scan_case(b, 9, d, n, dtype)
    wide = {k: v.double().cpu() for k, v in c.items()}
    want, want_h = _scan_formula(*[wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")], True, _wide(state)[0], None)
    amp_y, amp_h, _ = _amplitudes(c, torch.zeros_like(c["u"]), True, state, None)
    part = {k: v if k in ("A", "D", "delta_bias") else v[:, :5] for k, v in c.items()}
    y, h = scan.selective_scan(**part, state=state, return_state=True)
    near(y, want[:, :5], amp_y[:, :5], 200, "y")
    for t in range(5, 9):
        before, out = h.clone(), None if t == 5 else h if t == 6 else torch.empty_like(h)
        now = {k: v if k in ("A", "D", "delta_bias") else v[:, t] for k, v in c.items()}
        y, new = scan.selective_scan_step(**now, state=h, out=out)
        assert out is None or new.data_ptr() == out.data_ptr()
        assert out is h or torch.equal(h, before)
        near(y, want[:, t], amp_y[:, t], 200, "y")
        h = new
    near(h, want_h, amp_h, 200, "state")


@gpu
def test_scan_a_long_sequence_in_parts():
    """Eight thousand steps at once, and in four parts with the state handed on."""
    c, _, _ = _scan_case(1, 8200, 16, 16, F32)
    want, want_h = scan.selective_scan(**c, return_state=True)
    h, ys = None, []
    for a, b in ((0, 1), (1, 4097), (4097, 8199), (8199, 8200)):
        part = {k: v if k in ("A", "D", "delta_bias") else v[:, a:b] for k, v in c.items()}
        y, h = scan.selective_scan(**part, state=h, return_state=True)
        ys.append(y)
    wide = {k: v.double().cpu() for k, v in c.items()}
    exact, exact_h = _scan_formula(*[wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")], True, None, None)
    amp_y, amp_h, _ = _amplitudes(c, torch.zeros_like(c["u"]), True, None, None)
    # the slowest state forgets over some 2000 steps (a time step of 0.0005): 12 roundings for each of these
    for y, s in ((want, want_h), (torch.cat(ys, 1), h)):
        near(y, exact, amp_y, 24000, "y")
        near(s, exact_h, amp_h, 24000, "state")


@gpu
def test_scan_extreme_time_steps():
    """Steps so long that a state forgets everything, and so short that nothing happens."""
    c, dy, state = _scan_case(2, 20, 24, 16, F32)
    c["delta"][:, 5] = 200.0
    c["delta"][:, 9] = -100.0
    c["delta"][:, 11] = 20.001
    c["z"][:, 3], c["z"][:, 4] = 90.0, -90.0
    _scan_check(c, dy, state=state)


@gpu
def test_scan_gradient_against_differences():
    c, dy, _ = _scan_case(1, 12, 8, 4, F32)
    leaves = {k: v.detach().requires_grad_() for k, v in c.items()}
    grads = torch.autograd.grad(scan.selective_scan(**leaves), list(leaves.values()), dy)
    g, e = _gen(3), 2.0 ** -8
    d = {k: torch.randn(v.shape, generator=g).cuda() for k, v in c.items()}
    ends = [(scan.selective_scan(**{k: v + s * e * d[k] for k, v in c.items()}).double() * dy.double()).sum().item() for s in (1, -1)]
    slope = sum((a.double() * d[k].double()).sum().item() for k, a in zip(c, grads))
    # e^2 times third derivatives, and roundings of 96 values of order one over 2 e
    assert abs((ends[0] - ends[1]) / (2 * e) - slope) < 1e-2 * max(1.0, abs(slope))


@gpu
def test_scan_repeats_itself_and_captures():
    """No sum depends on the order in which blocks finish; two captured graphs and an eager call do not share anything."""
    c, dy, _ = _scan_case(4, 50, 72, 16, BF16)
    leaves = {k: v.detach().requires_grad_() for k, v in c.items()}

    def step():
        y = scan.selective_scan(**leaves)
        return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))
    want = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for graph in graphs:
        graph.replay()
    step()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
def test_on_another_stream():
    c, dy, _ = _scan_case(2, 40, 32, 16, BF16)
    want = scan.selective_scan(**c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = dict(c, u=c["u"].detach().requires_grad_())
        y = scan.selective_scan(**leaf)
        du, = torch.autograd.grad(y, leaf["u"], dy)
    torch.cuda.current_stream().wait_stream(side)
    ref = dict(c, u=c["u"].detach().requires_grad_())
    assert torch.equal(y, want) and torch.equal(du, torch.autograd.grad(scan.selective_scan(**ref), ref["u"], dy)[0])


@gpu
def test_empty_sequences_and_batches():
    for b, t in ((0, 5), (3, 0)):
        c, dy, state = _scan_case(b, t, 24, 16, F32)
        leaves = {k: v.detach().requires_grad_() for k, v in c.items()}
        y, h = scan.selective_scan(**leaves, state=state, return_state=True)
        assert y.shape == (b, t, 24) and torch.equal(h, state)
        for g, k in zip(torch.autograd.grad(y, list(leaves.values()), dy), leaves):
            assert g.shape == leaves[k].shape and not g.any()
        x, w, bias, dy = _conv_case(b, t, 24, 4, F32)
        leaves = [v.requires_grad_() for v in (x, w, bias)]
        y, last = scan.causal_conv(*leaves, return_state=True)
        assert y.shape == (b, t, 24) and last.shape == (b, 3, 24) and not last.any()
        for g, v in zip(torch.autograd.grad(y, leaves, dy), leaves):
            assert g.shape == v.shape and not g.any()


@gpu
def test_rows_further_apart_than_32_bits():
    """Slices of sequences whose rows and whose batch entries lie gigabytes apart."""
    big = torch.empty(2, 3, 1 << 30, dtype=BF16, device="cuda")                # 12 GB: strides of 2^30 and 3 * 2^30
    c, dy, _ = _scan_case(2, 3, 64, 16, BF16)
    far = dict(c)
    for i, k in enumerate(("u", "delta", "z", "B", "C")):
        far[k] = big[:, :, (1 << 29) + 128 * i:(1 << 29) + 128 * i + c[k].shape[2]].copy_(c[k])
    w, bias = torch.randn(64, 4, device="cuda"), torch.randn(64, device="cuda")
    for f, names in ((lambda v: scan.selective_scan(**v), ("u", "delta", "z", "B", "C")), (lambda v: scan.causal_conv(v["u"], w, bias), ("u",))):
        grads = []
        for v in (c, far):
            v = {k: t.detach().requires_grad_(k in names) for k, t in v.items()}
            y = f(v)
            grads.append((y.detach(), *torch.autograd.grad(y, [v[k] for k in names], dy)))
        assert all(torch.equal(a, b) for a, b in zip(*grads))


@gpu
def test_expanded_operands():
    """One sequence's steps for all, one step's operands for every step, and a gradient that is one number."""
    c, _, _ = _scan_case(3, 11, 40, 16, F32)
    shared = dict(c, B=c["B"][:1].expand(3, -1, -1), C=c["C"][:, :1].expand(-1, 11, -1), delta=c["delta"][:1, :1, :1].expand(3, 11, 40))
    dense = {k: v.contiguous() for k, v in shared.items()}
    got, want = ([], [])
    for v, out in ((shared, got), (dense, want)):
        leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
        y = scan.selective_scan(**leaves)
        out += [y.detach(), *torch.autograd.grad(y.sum(), list(leaves.values()))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_steps_in_inference_mode():
    c, _, state = _scan_case(2, 3, 24, 16, BF16)
    x, w, bias, _ = _conv_case(2, 5, 24, 4, BF16)
    with torch.inference_mode():
        last = torch.zeros(2, 3, 24, dtype=BF16, device="cuda")
        ys = [scan.causal_conv_step(x[:, t], last, w, bias, out=last)[0] for t in range(5)]
        h = state.clone()
        for t in range(3):
            now = {k: v if k in ("A", "D", "delta_bias") else v[:, t] for k, v in c.items()}
            y, h = scan.selective_scan_step(**now, state=h, out=h)
        want, want_h = scan.selective_scan(**c, state=state, return_state=True)
    assert torch.equal(torch.stack(ys, 1), scan.causal_conv(x, w, bias))
    assert torch.allclose(y.float(), want[:, 2].float(), rtol=2.0 ** -7, atol=1e-3) and torch.allclose(h, want_h, rtol=1e-5, atol=1e-5)


@gpu
def test_many_sequences_of_many_lengths():
    """More sequences than a block has threads, and fewer: the order in which they are worked on is nobody's business."""
    for b in (100, 200):
        c, dy, _ = _scan_case(b, 24, 16, 4, F32)
        lengths = torch.randint(0, 25, (b,), generator=_gen(b)).cuda()
        got = scan.selective_scan(**c, lengths=lengths)
        for i in (0, 1, b // 2, b - 1):
            one = {k: v if k in ("A", "D", "delta_bias") else v[i:i + 1] for k, v in c.items()}
            assert torch.equal(scan.selective_scan(**one, lengths=lengths[i:i + 1])[0], got[i])


# ------------------------------------------------------------------------------------------------ without a GPU
@pytest.mark.parametrize("dtype", [F32, torch.float64])
def test_the_restatements_are_the_formulas(dtype):
    x, w, bias, _ = _conv_case(4, 9, 6, 3, dtype, "cpu")
    lengths = torch.tensor([0, 1, 5, 9])
    state = torch.randn(4, 2, 6, generator=_gen(1), dtype=torch.float64).to(dtype)
    y, last = scan.causal_conv(x, w, bias, "silu", state, lengths, True)
    want, want_last = _conv_formula(x.double(), w.double(), bias.double(), "silu", state.double(), lengths)
    assert (y.double() - want).abs().max() < 1e-5 and torch.equal(last.double(), want_last)
    y1, s1 = scan.causal_conv_step(x[:, 0], state, w, bias)
    assert torch.equal(y1[1], y[1, 0]) and torch.equal(s1[1], last[1])
    c, _, h0 = _scan_case(4, 9, 6, 5, dtype, "cpu")
    y, h = scan.selective_scan(**c, state=h0, lengths=lengths, return_state=True)
    wide = [v.double() for v in (c["u"], c["delta"], c["A"], c["B"], c["C"], c["D"], c["z"], c["delta_bias"])]
    want, want_h = _scan_formula(*wide, True, h0.double(), lengths)
    assert (y.double() - want).abs().max() < 1e-4 and (h.double() - want_h).abs().max() < 1e-4
    now = {k: v if k in ("A", "D", "delta_bias") else v[:, 0] for k, v in c.items()}
    y1, h1 = scan.selective_scan_step(**now, state=h0.to(dtype))
    assert torch.allclose(y1[1], y[1, 0], rtol=1e-5, atol=1e-5) and torch.allclose(h1[1].double(), h[1].double(), rtol=1e-5, atol=1e-5)


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


CONV_FITS = dict(x=_t(2, 5, 8), weight=_t(8, 4, dtype=F32), bias=_t(8, dtype=F32), act=2, state=_t(2, 3, 8), lengths=torch.zeros(2, dtype=torch.int64),
                 want=True)
CONV_STEP_FITS = dict(x=_t(2, 8), state=_t(2, 3, 8), weight=_t(8, 4, dtype=F32), bias=_t(8, dtype=F32), act=2, out=None)
SCAN_FITS = dict(u=_t(2, 5, 8), delta=_t(2, 5, 8), A=_t(8, 4, dtype=F32), B=_t(2, 5, 4), C=_t(2, 5, 4), D=_t(8, dtype=F32), z=_t(2, 5, 8),
                 bias=_t(8, dtype=F32), softplus=True, state=_t(2, 8, 4, dtype=F32), lengths=torch.zeros(2, dtype=torch.int64), want=True)
STEP_FITS = dict(u=_t(2, 8), delta=_t(2, 8), A=_t(8, 4, dtype=F32), B=_t(2, 4), C=_t(2, 4), state=_t(2, 8, 4, dtype=F32), D=_t(8, dtype=F32), z=_t(2, 8),
                 bias=_t(8, dtype=F32), softplus=True, out=None)
ROOM = torch.zeros(2 * 8 * 4 + 8)


@pytest.mark.parametrize("op,fits,change,message", [
    ("causal_conv", CONV_FITS, dict(x=_t(2, 8)), "3-D"), ("causal_conv", CONV_FITS, dict(x=_t(2, 5, 8, dtype=torch.float16)), "neither"),
    ("causal_conv", CONV_FITS, dict(weight=_t(8, 4)), "weight"), ("causal_conv", CONV_FITS, dict(weight=_t(7, 4, dtype=F32)), "weight"),
    ("causal_conv", CONV_FITS, dict(weight=_t(8, 5, dtype=F32)), "taps"), ("causal_conv", CONV_FITS, dict(weight=_t(8, 1, dtype=F32)), "taps"),
    ("causal_conv", CONV_FITS, dict(weight=_t(4, 8, dtype=F32).t()), "in a row"), ("causal_conv", CONV_FITS, dict(bias=_t(7, dtype=F32)), "bias"),
    ("causal_conv", CONV_FITS, dict(act=1), "activation"), ("causal_conv", CONV_FITS, dict(state=_t(2, 4, 8)), "state"),
    ("causal_conv", CONV_FITS, dict(state=_t(2, 3, 8, dtype=F32)), "state"), ("causal_conv", CONV_FITS, dict(state=_t(2, 3, 8).requires_grad_()), "detach"),
    ("causal_conv", CONV_FITS, dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths"),
    ("causal_conv", CONV_FITS, dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths"), ("causal_conv", CONV_FITS, {}, "not on a GPU"),
    ("causal_conv_step", CONV_STEP_FITS, dict(x=_t(2, 1, 8)), "2-D"), ("causal_conv_step", CONV_STEP_FITS, dict(out=_t(2, 3, 7)), "room"),
    ("causal_conv_step", CONV_STEP_FITS, dict(x=_t(2, 8).requires_grad_()), "no_grad"), ("causal_conv_step", CONV_STEP_FITS, dict(state=_t(3, 3, 8)), "state"),
    ("causal_conv_step", CONV_STEP_FITS, {}, "not on a GPU"),
    ("selective_scan", SCAN_FITS, dict(u=_t(2, 8)), "3-D"), ("selective_scan", SCAN_FITS, dict(delta=_t(2, 4, 8)), "delta"),
    ("selective_scan", SCAN_FITS, dict(delta=_t(2, 5, 8, dtype=F32)), "delta"), ("selective_scan", SCAN_FITS, dict(A=_t(8, 65, dtype=F32)), "states"),
    ("selective_scan", SCAN_FITS, dict(A=_t(8, 4)), "A is"), ("selective_scan", SCAN_FITS, dict(A=_t(8, 0, dtype=F32)), "states"),
    ("selective_scan", SCAN_FITS, dict(B=_t(2, 5, 5)), "B"), ("selective_scan", SCAN_FITS, dict(C=_t(2, 5, 4, dtype=F32)), "C"),
    ("selective_scan", SCAN_FITS, dict(D=_t(7, dtype=F32)), "D"), ("selective_scan", SCAN_FITS, dict(z=_t(2, 5, 9)), "z"),
    ("selective_scan", SCAN_FITS, dict(bias=_t(8)), "delta_bias"), ("selective_scan", SCAN_FITS, dict(state=_t(2, 8, 4)), "state"),
    ("selective_scan", SCAN_FITS, dict(state=_t(2, 4, 8, dtype=F32).transpose(1, 2)), "in a row"),
    ("selective_scan", SCAN_FITS, dict(state=_t(2, 8, 4, dtype=F32).requires_grad_()), "detach"),
    ("selective_scan", SCAN_FITS, dict(lengths=torch.zeros(1, dtype=torch.int64)), "lengths"), ("selective_scan", SCAN_FITS, {}, "not on a GPU"),
    ("selective_scan_step", STEP_FITS, dict(u=_t(2, 1, 8)), "2-D"), ("selective_scan_step", STEP_FITS, dict(state=_t(2, 8, 5, dtype=F32)), "state"),
    ("selective_scan_step", STEP_FITS, dict(z=_t(2, 8).requires_grad_()), "no_grad"), ("selective_scan_step", STEP_FITS, dict(out=_t(2, 8, 4)), "out"),
    ("selective_scan_step", STEP_FITS, {}, "not on a GPU"),
])
def test_refusals(op, fits, change, message):
    with pytest.raises(RuntimeError, match=message):
        getattr(_build.load_torch(), op)(*dict(fits, **change).values())


def test_activations_that_there_are_not():
    for f in (lambda: scan.causal_conv(_t(1, 2, 3), _t(3, 2, dtype=F32), activation="relu"),
              lambda: scan.causal_conv_step(_t(1, 3), _t(1, 1, 3), _t(3, 2, dtype=F32), activation="relu")):
        with pytest.raises(ValueError, match="relu"):
            f()


@gpu
def test_a_state_that_overlaps_the_new_one_is_refused():
    c, _, _ = _scan_case(2, 1, 8, 4, F32)
    now = {k: v if k in ("A", "D", "delta_bias") else v[:, 0] for k, v in c.items()}
    room = torch.zeros(72, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        scan.selective_scan_step(**now, state=room[:64].view(2, 8, 4), out=room[8:].view(2, 8, 4))


@gpu
def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """The eager graph's gradient node waits on its own stream, which a capture cannot; without that graph the capture goes through."""
    c, dy, _ = _scan_case(1, 8, 8, 4, F32)
    leaves = {k: v.requires_grad_() for k, v in c.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = scan.selective_scan(**leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go of it"):
        with torch.cuda.graph(graph):
            scan.selective_scan(**leaves)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = scan.selective_scan(**leaves)
        du, = torch.autograd.grad(y, leaves["u"], dy)
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(y, scan.selective_scan(**leaves))
