"""The operators around a sequence or image classifier that learns from a teacher, as cases that can be timed.

* ``norm``     group normalisation of channels-last activations with shortcut and activation (``ops.group_norm_act``)
* ``conv``     the short causal convolution ahead of a scan, for whole sequences and for one step (``causal_conv``, ``causal_conv_step``)
* ``scan``     the selective state-space scan, in training, over a prompt and for one step (``selective_scan``, ``selective_scan_step``)
* ``distill``  the loss against a teacher's top logits with its gradient (``ops.distillation_loss``)

``run`` computes them in elementary torch operations in 32 bits, or, where ``own`` is set, by the framework's kernels; ``exact`` in
64 bits, by loops over time and the formulas as they are written down.
"""
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # the last stage of a ResNet-50 for a single image: a request that waits for its answer
        _norm("norm 1x2048x7x7", "bfloat16", 1, 2048, 7, 7, 32, "relu", True, False),
        # the first stage of ResNet-50 at a large batch, forward and backward, with the shortcut of a residual block
        _norm("norm train 128x256x56x56", "bfloat16", 128, 256, 56, 56, 32, "silu", True, True),
        # an fp32 network on small images with a batch and a width that are no powers of two
        _norm("norm train fp32 100x48x15x15", "float32", 100, 48, 15, 15, 6, "silu", False, True),
        # ahead of the scan over the frame features of a batch of clips
        _conv("conv train 16x331x2048", "bfloat16", 16, 331, 2048, 4, False, True),
        # the next frame of sixteen streams
        _conv("conv step 16x2048", "bfloat16", 16, 1, 2048, 4, True, False),
        # a training batch of clips of different lengths
        _scan("scan train 16x331x2048", "bfloat16", 16, 331, 2048, 16, "train", True),
        # a small fp32 model with a few states, odd sizes
        _scan("scan train fp32 3x77x500", "float32", 3, 77, 500, 8, "train", False),
        # one long sequence whose state is kept for the steps that follow
        _scan("scan prompt 1x4099x2048", "bfloat16", 1, 4099, 2048, 16, "prompt", False),
        # the next step of one stream, and of many
        _scan("scan step 1x2048", "bfloat16", 1, 1, 2048, 16, "step", False),
        _scan("scan step 250x2048", "bfloat16", 250, 1, 2048, 16, "step", False),
        # an image classifier's training batch (fp32 logits) with labels beside the teacher
        _distill("distill 256x1000", "float32", 256, 1000, 50, 2.0, 0.3),
        # every position of a batch of sequences over a large set of classes
        _distill("distill 4096x32000", "bfloat16", 4096, 32000, 64, 1.0, 0.0),
    ]


def _norm(name, dtype, batch, channels, height, width, groups, activation, residual, train):
    return {"name": name, "kind": "norm", "dtype": dtype, "batch": batch, "channels": channels, "height": height, "width": width,
            "groups": groups, "activation": activation, "residual": residual, "train": train}


def _conv(name, dtype, batch, length, channels, taps, step, train):
    return {"name": name, "kind": "conv", "dtype": dtype, "batch": batch, "length": length, "channels": channels, "taps": taps,
            "step": step, "train": train}


def _scan(name, dtype, batch, length, channels, states, form, ragged):
    return {"name": name, "kind": "scan", "dtype": dtype, "batch": batch, "length": length, "channels": channels, "states": states,
            "form": form, "ragged": ragged}


def _distill(name, dtype, rows, classes, top, temperature, hard_weight):
    return {"name": name, "kind": "distill", "dtype": dtype, "rows": rows, "classes": classes, "top": top, "temperature": temperature,
            "hard_weight": hard_weight}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "conv", "conv", "scan", "scan", "scan", "distill", "distill"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "norm":
        groups = rng.choice([1, 4, 6, 8, 16, 32])
        channels = groups * _log_int(rng, 1, 2048 // groups)
        height, width = _log_int(rng, 1, 112), _log_int(rng, 1, 112)
        if channels // groups * height * width < 32:      # a group of a few values has next to no gradient
            height, width = 7, 7
        most = (128 * 256 * 56 * 56) // (channels * height * width * (2 if dtype == "float32" else 1))
        train = rng.random() < 0.7
        # the slope of a ReLU jumps: next to its border two right gradients differ, so it is measured in inference
        case = _norm("", dtype, _log_int(rng, 1, max(1, min(256, most))), channels, height, width, groups,
                     rng.choice(["silu", "none"] if train else ["relu", "silu", "none"]), rng.random() < 0.5, train)
    elif kind == "conv":
        step = rng.random() < 0.3
        channels, batch = _log_int(rng, 24, 4096), _log_int(rng, 1, 256 if step else 32)
        length = 1 if step else _log_int(rng, 1, max(1, min(4099, 16 * 331 * 1024 // (channels * batch))))
        case = _conv("", dtype, batch, length, channels, rng.choice([2, 3, 4]), step, not step and rng.random() < 0.7)
    elif kind == "scan":
        form = rng.choice(["train", "train", "prompt", "step"])
        channels, states = _log_int(rng, 24, 4096), rng.choice([4, 8, 16, 16, 16, 5, 32])
        batch = _log_int(rng, 1, 250 if form == "step" else 24)
        most = 16 * 331 * 1024 * 16 // (channels * states * batch)
        length = 1 if form == "step" else _log_int(rng, 1, max(1, min(4099, most)))
        case = _scan("", dtype, batch, length, channels, states, form, form != "step" and rng.random() < 0.5)
    else:
        classes = _log_int(rng, 10, 100000)
        rows = _log_int(rng, 1, min(8192, 4096 * 16000 // classes))
        case = _distill("", dtype, rows, classes, min(classes, _log_int(rng, 1, 128)), rng.choice([1.0, 2.0, 4.0, 2.5]),
                        rng.choice([0.0, 0.0, 0.3, 0.5]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- preparation
class _Inputs:
    """Numbers on the GPU from the seed alone."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda").manual_seed(seed % (1 << 62))

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=self.generator).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.generator)

    def whole(self, low, high, *shape):
        return torch.randint(low, high, shape, device="cuda", generator=self.generator)


def prepare(case, seed):
    return {"norm": _prepare_norm, "conv": _prepare_conv, "scan": _prepare_scan, "distill": _prepare_distill}[case["kind"]](
        case, _Inputs(seed))


def _prepare_norm(case, made):
    dtype, shape = TYPES[case["dtype"]], (case["batch"], case["channels"], case["height"], case["width"])

    def image(scale=1.0, shift=0.0):
        return (made.normal(*shape) * scale + shift).to(dtype).contiguous(memory_format=torch.channels_last)

    # what a convolution hands on: channels with a mean of their own
    x = image(1.5, made.normal(1, case["channels"], 1, 1))
    s = {"case": case, "x": x, "gamma": 1.0 + 0.2 * made.normal(case["channels"]), "beta": 0.2 * made.normal(case["channels"]),
         "residual": image() if case["residual"] else None}
    if case["train"]:
        s["dz"] = image()
        for k in ("x", "gamma", "beta", "residual"):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


def _prepare_conv(case, made):
    dtype, b, t, d, k = TYPES[case["dtype"]], case["batch"], case["length"], case["channels"], case["taps"]
    s = {"case": case, "weight": made.normal(d, k) / math.sqrt(k), "bias": 0.2 * made.normal(d)}
    if case["step"]:
        s["x"] = made.normal(b, d, dtype=dtype)
        s["state"] = made.normal(b, k - 1, d, dtype=dtype)
        s["next"] = torch.empty_like(s["state"])        # two buffers in turn, as a loop over steps would use them
        return s
    s["x"] = made.normal(b, t, d, dtype=dtype)
    if case["train"]:
        s["dy"] = made.normal(b, t, d, dtype=dtype)
        for name in ("x", "weight", "bias"):
            s[name].requires_grad_()
    return s


def _prepare_scan(case, made):
    dtype, b, t, d, n = TYPES[case["dtype"]], case["batch"], case["length"], case["channels"], case["states"]
    lead = (b,) if case["form"] == "step" else (b, t)
    x = made.normal(*lead, d)
    rate = torch.exp(made.uniform(d) * math.log(100.0) + math.log(0.001))            # time steps between 0.001 and 0.1
    s = {"case": case, "u": (x * torch.sigmoid(x)).to(dtype), "delta": (0.5 * made.normal(*lead, d)).to(dtype),
         "A": -torch.arange(1, n + 1, device="cuda").float().repeat(d, 1) * torch.exp(0.1 * made.normal(d, n)),
         "B": made.normal(*lead, n, dtype=dtype), "C": made.normal(*lead, n, dtype=dtype), "D": 1.0 + 0.1 * made.normal(d),
         "z": made.normal(*lead, d, dtype=dtype), "bias": rate + torch.log(-torch.expm1(-rate)), "lengths": None}
    if case["form"] == "step":
        s["state"] = made.normal(b, d, n)
        s["next"] = torch.empty_like(s["state"])
    if case["ragged"]:                                   # clips of different lengths, the first the longest
        s["lengths"] = made.whole(max(1, t // 3), t + 1, b)
        s["lengths"][0] = t
    if case["form"] == "train":
        s["dy"] = made.normal(b, t, d, dtype=dtype)
        for name in ("u", "delta", "A", "B", "C", "D", "z", "bias"):
            s[name].requires_grad_()
    return s


def _prepare_distill(case, made):
    dtype, rows, v, k = TYPES[case["dtype"]], case["rows"], case["classes"], case["top"]
    logits = (2.0 * made.normal(rows, v)).to(dtype)
    # a teacher that mostly agrees, sure of a few classes; its classes are different ones
    first = made.whole(0, v, rows, 1)
    classes = (first + torch.arange(k, device="cuda") * max(1, v // k)) % v
    values = (8.0 * made.uniform(rows, k).sort(dim=1, descending=True)[0] + logits.float().gather(1, classes)).to(dtype)
    return {"case": case, "logits": logits.requires_grad_(), "values": values, "classes": classes,
            "labels": classes[:, 0].contiguous() if case["hard_weight"] > 0 else None}


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan, "distill": _own_distill}[case["kind"]](case, state)
    with torch.no_grad():
        return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan, "distill": _plain_distill}[case["kind"]](case, state)


def _named(names, values):
    return dict(zip(names, values))


def _own_norm(case, s):
    from eagersgd_b200.ops import functional as ops
    activation = None if case["activation"] == "none" else case["activation"]
    z = ops.group_norm_act(s["x"], case["groups"], s["gamma"], s["beta"], activation=activation, residual=s["residual"], eps=EPS)
    if not case["train"]:
        return {"z": z}
    names = ["x", "gamma", "beta"] + (["residual"] if case["residual"] else [])
    return {"z": z.detach(), **_named(names, torch.autograd.grad(z, [s[k] for k in names], s["dz"]))}


def _own_conv(case, s):
    from eagersgd_b200.ops import scan
    if case["step"]:
        y, state = scan.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], out=s["next"])
        return {"y": y, "state": state}
    if not case["train"]:
        y, state = scan.causal_conv(s["x"], s["weight"], s["bias"], return_state=True)
        return {"y": y, "state": state}
    y = scan.causal_conv(s["x"], s["weight"], s["bias"])
    names = ["x", "weight", "bias"]
    return {"y": y.detach(), **_named(names, torch.autograd.grad(y, [s[k] for k in names], s["dy"]))}


def _own_scan(case, s):
    from eagersgd_b200.ops import scan
    if case["form"] == "step":
        y, state = scan.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                            delta_bias=s["bias"], out=s["next"])
        return {"y": y, "state": state}
    if case["form"] == "prompt":
        y, state = scan.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["bias"],
                                       lengths=s["lengths"], return_state=True)
        return {"y": y, "state": state}
    y = scan.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["bias"], lengths=s["lengths"])
    names = ["u", "delta", "A", "B", "C", "D", "z", "bias"]
    return {"y": y.detach(), **_named(names, torch.autograd.grad(y, [s[k] for k in names], s["dy"]))}


def _own_distill(case, s):
    from eagersgd_b200.ops import functional as ops
    loss = ops.distillation_loss(s["logits"], s["values"], s["classes"], temperature=case["temperature"], labels=s["labels"],
                                 hard_weight=case["hard_weight"])
    return {"loss": loss.detach(), "logits": torch.autograd.grad(loss, s["logits"])[0]}


# ---------------------------------------------------------------------------------------------------- plain forms, 32 bits
def _plain_norm(case, s):
    b, c, h, w, g = case["batch"], case["channels"], case["height"], case["width"], case["groups"]
    dtype = s["x"].dtype
    x = s["x"].float().reshape(b, g, -1)
    mean = x.mean(2, keepdim=True)
    centred = x - mean
    rstd = 1.0 / (centred.square().mean(2, keepdim=True) + EPS).sqrt()
    normal = (centred * rstd).reshape(b, c, h, w)
    gamma, beta = s["gamma"].reshape(1, c, 1, 1), s["beta"].reshape(1, c, 1, 1)
    pre = normal * gamma + beta
    if case["residual"]:
        pre = pre + s["residual"].float()
    if case["activation"] == "relu":
        z, slope = pre.clamp(min=0), (pre > 0).float()
    elif case["activation"] == "silu":
        gate = 1.0 / (1.0 + torch.exp(-pre))
        z, slope = pre * gate, gate * (1.0 + pre * (1.0 - gate))
    else:
        z, slope = pre, torch.ones_like(pre)
    out = {"z": _image(z, dtype)}
    if not case["train"]:
        return out
    d = s["dz"].float() * slope
    dn = (d * gamma).reshape(b, g, -1)
    flat = normal.reshape(b, g, -1)
    dx = (dn - dn.mean(2, keepdim=True) - flat * (dn * flat).mean(2, keepdim=True)) * rstd
    out.update(x=_image(dx.reshape(b, c, h, w), dtype), gamma=(d * normal).sum((0, 2, 3)), beta=d.sum((0, 2, 3)))
    if case["residual"]:
        out["residual"] = _image(d, dtype)
    return out


def _image(v, dtype):
    return v.to(dtype).contiguous(memory_format=torch.channels_last)


def _plain_conv(case, s):
    b, t, d, k = case["batch"], case["length"], case["channels"], case["taps"]
    x, w, dtype = s["x"].float(), s["weight"], s["x"].dtype
    if case["step"]:
        window = torch.cat([s["state"].float(), x.unsqueeze(1)], 1)                     # [b, k, d]
        pre = (window * w.t()).sum(1) + s["bias"]
        return {"y": (pre / (1.0 + torch.exp(-pre))).to(dtype), "state": window[:, 1:].to(dtype)}
    padded = torch.cat([x.new_zeros(b, k - 1, d), x], 1)
    windows = padded.unfold(1, k, 1)                                                    # [b, t, d, k]
    pre = (windows * w).sum(3) + s["bias"]
    gate = 1.0 / (1.0 + torch.exp(-pre))
    y = (pre * gate).to(dtype)
    if not case["train"]:
        return {"y": y, "state": padded[:, t:].to(dtype)}
    dpre = s["dy"].float() * gate * (1.0 + pre * (1.0 - gate))
    ahead = torch.cat([dpre, dpre.new_zeros(b, k - 1, d)], 1).unfold(1, k, 1)           # dpre[t .. t + k - 1]
    return {"y": y, "x": (ahead * w.flip(1)).sum(3).to(dtype), "weight": (windows * dpre.unsqueeze(3)).sum((0, 1)),
            "bias": dpre.sum((0, 1))}


def _recurrence(a, b):
    """h[t] = a[t] * h[t - 1] + b[t] along dimension 1, by doubling the span that a pair (a, b) covers."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_scan(case, s):
    dtype, b, t, d, n = s["u"].dtype, case["batch"], case["length"], case["channels"], case["states"]
    u, z, A = s["u"].float(), s["z"].float(), s["A"]
    raw = s["delta"].float() + s["bias"]
    dt = torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0))))
    gate = 1.0 / (1.0 + torch.exp(-z))
    if case["form"] == "step":
        a = torch.exp(dt.unsqueeze(2) * A)
        h = a * s["state"] + (dt * u).unsqueeze(2) * s["B"].float().unsqueeze(1)
        y = (h * s["C"].float().unsqueeze(1)).sum(2) + s["D"] * u
        return {"y": (y * z * gate).to(dtype), "state": h}
    if s["lengths"] is not None:                         # a step of length zero leaves the state as it is
        inside = (torch.arange(t, device=u.device) < s["lengths"].unsqueeze(1)).unsqueeze(2)
        dt = dt * inside
    B, C = s["B"].float().unsqueeze(2), s["C"].float().unsqueeze(2)                     # [b, t, 1, n]
    a = torch.exp(dt.unsqueeze(3) * A)
    h = _recurrence(a, (dt * u).unsqueeze(3) * B)
    y = (h * C).sum(3) + s["D"] * u
    out = y * z * gate
    if s["lengths"] is not None:
        out = out * inside
    if case["form"] == "prompt":
        return {"y": out.to(dtype), "state": h[:, -1].contiguous()}
    dout = s["dy"].float()
    if s["lengths"] is not None:
        dout = dout * inside
    dy = dout * z * gate
    dz = dout * y * gate * (1.0 + z * (1.0 - gate))
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _recurrence(later.flip(1), (dy.unsqueeze(3) * C).flip(1)).flip(1)
    dC = (dy.unsqueeze(3) * h).sum(2)
    decay = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * a * dh              # dh[t] * a[t] * h[t - 1]
    along = (dh * B).sum(3)
    dB = (dh * (dt * u).unsqueeze(3)).sum(2)
    ddt = (decay * A).sum(3) + along * u
    ddelta = ddt / (1.0 + torch.exp(-raw))
    if s["lengths"] is not None:
        ddelta = ddelta * inside
    return {"y": out.to(dtype), "u": (along * dt + s["D"] * dy).to(dtype), "delta": ddelta.to(dtype),
            "A": (decay * dt.unsqueeze(3)).sum((0, 1)), "B": dB.to(dtype), "C": dC.to(dtype), "D": (dy * u).sum((0, 1)),
            "z": dz.to(dtype), "bias": ddelta.sum((0, 1))}


def _plain_distill(case, s):
    temperature, hard, rows = case["temperature"], case["hard_weight"], case["rows"]
    logits, classes = s["logits"].float(), s["classes"]
    soft = logits / temperature
    peak = soft.max(1, keepdim=True)[0]
    e = torch.exp(soft - peak)
    total = e.sum(1, keepdim=True)
    lse = peak + torch.log(total)
    v = s["values"].float() / temperature
    v = v - v.max(1, keepdim=True)[0]
    ev = torch.exp(v)
    tv = ev.sum(1, keepdim=True)
    p = ev / tv
    log_p = v - torch.log(tv)
    kl = (p * (log_p - (soft.gather(1, classes) - lse))).sum(1)
    loss = (1.0 - hard) * temperature * temperature * kl.sum() / rows
    scale = (1.0 - hard) * temperature / rows
    d = (e / total * scale).scatter_add(1, classes, -p * scale)
    if hard > 0:
        peak = logits.max(1, keepdim=True)[0]
        e = torch.exp(logits - peak)
        total = e.sum(1, keepdim=True)
        own_label = s["labels"].unsqueeze(1)
        loss = loss + hard * (peak + torch.log(total) - logits.gather(1, own_label)).sum() / rows
        d = (d + e / total * (hard / rows)).scatter_add(1, own_label, torch.full_like(peak, -hard / rows))
    return {"loss": loss, "logits": d.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "distill": _exact_distill}[case["kind"]](
            case, prepare(case, seed))


def _wide(s, *names):
    return [None if s[k] is None else s[k].detach().double() for k in names]


def _exact_norm(case, s):
    x, gamma, beta, residual = _wide(s, "x", "gamma", "beta", "residual")
    dz = s["dz"].double() if case["train"] else None
    per = case["channels"] // case["groups"]
    z, dx, dres = (torch.empty_like(x) for _ in range(3))
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    for g in range(case["groups"]):
        at = slice(g * per, (g + 1) * per)
        part = x[:, at]
        centred = part - part.mean((1, 2, 3), keepdim=True)
        scale = torch.rsqrt((centred * centred).mean((1, 2, 3), keepdim=True) + EPS)
        n = centred * scale
        pre = n * gamma[at, None, None] + beta[at, None, None]
        if residual is not None:
            pre = pre + residual[:, at]
        act = {"relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "none": lambda v: v}[case["activation"]]
        z[:, at] = act(pre)
        if dz is None:
            continue
        sig = torch.sigmoid(pre)
        slope = {"relu": (pre > 0).double(), "silu": sig + pre * sig * (1 - sig), "none": torch.ones_like(pre)}[case["activation"]]
        d = dz[:, at] * slope
        dres[:, at] = d
        dgamma[at], dbeta[at] = (d * n).sum((0, 2, 3)), d.sum((0, 2, 3))
        d = d * gamma[at, None, None]
        dx[:, at] = scale * (d - d.mean((1, 2, 3), keepdim=True) - n * (d * n).mean((1, 2, 3), keepdim=True))
    if dz is None:
        return {"z": z}
    out = {"z": z, "x": dx, "gamma": dgamma, "beta": dbeta}
    if residual is not None:
        out["residual"] = dres
    return out


def _exact_conv(case, s):
    x, w, bias = _wide(s, "x", "weight", "bias")
    k = case["taps"]
    if case["step"]:
        state = s["state"].double()
        pre = bias + w[:, k - 1] * x
        for i in range(k - 1):
            pre = pre + w[:, i] * state[:, i]
        new = torch.cat([state, x[:, None]], 1)[:, 1:]
        return {"y": pre * torch.sigmoid(pre), "state": new}
    b, t, d = x.shape
    pre = bias.expand(b, t, d).clone()
    for i in range(k):                                   # tap i looks k - 1 - i steps back
        back = k - 1 - i
        if back < t:
            pre[:, back:] += w[:, i] * x[:, :t - back]
    sig = torch.sigmoid(pre)
    if not case["train"]:
        state = x.new_zeros(b, k - 1, d)
        for i in range(k - 1):
            if t - (k - 1) + i >= 0:
                state[:, i] = x[:, t - (k - 1) + i]
        return {"y": pre * sig, "state": state}
    dpre = s["dy"].double() * (sig + pre * sig * (1 - sig))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for i in range(k):
        back = k - 1 - i
        if back < t:
            dx[:, :t - back] += w[:, i] * dpre[:, back:]
            dw[:, i] = (dpre[:, back:] * x[:, :t - back]).sum((0, 1))
    return {"y": pre * sig, "x": dx, "weight": dw, "bias": dpre.sum((0, 1))}


def _exact_scan(case, s):
    u, delta, A, B, C, D, z, bias = _wide(s, "u", "delta", "A", "B", "C", "D", "z", "bias")
    raw = delta + bias
    dt = torch.nn.functional.softplus(raw, threshold=40.0)
    sig = torch.sigmoid(z)
    if case["form"] == "step":
        h = torch.exp(dt[:, :, None] * A) * s["state"].double() + dt[:, :, None] * u[:, :, None] * B[:, None, :]
        y = torch.einsum("bdn,bn->bd", h, C) + D * u
        return {"y": y * z * sig, "state": h}
    b, t, d = u.shape
    length = s["lengths"] if s["lengths"] is not None else torch.full((b,), t, device=u.device)
    h, y, kept = u.new_zeros(b, d, case["states"]), torch.zeros_like(u), []
    for i in range(t):
        live = (i < length)[:, None, None]
        new = torch.exp(dt[:, i, :, None] * A) * h + (dt[:, i] * u[:, i])[:, :, None] * B[:, i, None, :]
        h = torch.where(live, new, h)
        if case["form"] == "train":
            kept.append(h)
        y[:, i] = torch.einsum("bdn,bn->bd", h, C[:, i]) + D * u[:, i]
    inside = (torch.arange(t, device=u.device) < length[:, None])[:, :, None]
    out = torch.where(inside, y * z * sig, torch.zeros_like(y))
    if case["form"] == "prompt":
        return {"y": out, "state": h}
    dout = torch.where(inside, s["dy"].double(), torch.zeros_like(y))
    dy = dout * z * sig
    dz = dout * y * (sig + z * sig * (1 - sig))
    du, draw_, dB, dC = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(B), torch.zeros_like(C)
    dA, carry = torch.zeros_like(A), torch.zeros_like(h)
    for i in reversed(range(t)):
        a = torch.exp(dt[:, i, :, None] * A)
        dC[:, i] = torch.einsum("bd,bdn->bn", dy[:, i], kept[i])
        dh = carry + dy[:, i, :, None] * C[:, i, None, :]
        before = kept[i - 1] if i > 0 else torch.zeros_like(h)
        dB[:, i] = torch.einsum("bdn,bd->bn", dh, dt[:, i] * u[:, i])
        da = dh * before * a
        dA += (da * dt[:, i, :, None]).sum(0)
        along = torch.einsum("bdn,bn->bd", dh, B[:, i])
        du[:, i] = along * dt[:, i] + D * dy[:, i]
        draw_[:, i] = ((da * A).sum(2) + along * u[:, i]) * torch.sigmoid(raw[:, i])
        carry = torch.where((i < length)[:, None, None], a * dh, torch.zeros_like(dh))
    draw_ = torch.where(inside, draw_, torch.zeros_like(draw_))
    live = inside.double()
    return {"y": out, "u": du * live, "delta": draw_, "A": dA, "B": dB * live, "C": dC * live, "D": (dy * u).sum((0, 1)), "z": dz,
            "bias": draw_.sum((0, 1))}


def _exact_distill(case, s):
    logits, values = _wide(s, "logits", "values")
    temperature, hard = case["temperature"], case["hard_weight"]
    loss, d = logits.new_zeros(()), torch.empty_like(logits)
    for at in torch.arange(case["rows"], device=logits.device).split(512):
        x, classes = logits[at], s["classes"][at]
        p = torch.softmax(values[at] / temperature, 1)
        log_q = torch.log_softmax(x / temperature, 1)
        kl = (p * (torch.log(p) - log_q.gather(1, classes))).sum(1)
        part = torch.exp(log_q)
        part.scatter_add_(1, classes, -p)
        part *= (1 - hard) * temperature
        loss += (1 - hard) * temperature ** 2 * kl.sum()
        if hard > 0:
            label = s["labels"][at][:, None]
            log_q = torch.log_softmax(x, 1)
            loss -= hard * log_q.gather(1, label).sum()
            part += hard * torch.exp(log_q)
            part.scatter_add_(1, label, torch.full_like(label, -hard, dtype=part.dtype))
        d[at] = part / case["rows"]
    return {"loss": loss / case["rows"], "logits": d}


# ---------------------------------------------------------------------------------------------------- what a pass has to do
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "norm":
        n = case["batch"] * case["channels"] * case["height"] * case["width"]
        tensors, ops = 2 + case["residual"], 10
        if case["train"]:
            tensors, ops = tensors + 2 + case["residual"], 30
        return {"bytes": size * n * tensors + 16 * case["channels"], "flops": ops * n}
    if case["kind"] == "conv":
        n, k = case["batch"] * case["length"] * case["channels"], case["taps"]
        tensors, ops = (2 * k if case["step"] else 2), 2 * k + 5
        if case["train"]:
            tensors, ops = 4, 6 * k + 15
        return {"bytes": size * n * tensors + 4 * case["channels"] * (k + 1), "flops": ops * n}
    if case["kind"] == "scan":
        n, states = case["batch"] * case["length"] * case["channels"], case["states"]
        narrow = 2 * case["batch"] * case["length"] * states
        held = case["batch"] * case["channels"] * states
        parameters = 4 * case["channels"] * (states + 2)
        if case["form"] == "train":
            return {"bytes": size * (8 * n + 2 * narrow) + 2 * parameters, "flops": n * (24 * states + 40)}
        moved = size * (4 * n + narrow) + parameters + 4 * held * (2 if case["form"] == "step" else 1)
        return {"bytes": moved, "flops": n * (7 * states + 15)}
    n = case["rows"] * case["classes"]
    both = 2 if case["hard_weight"] > 0 else 1
    return {"bytes": 2 * size * n + case["rows"] * (case["top"] * (size + 8) + 8), "flops": n * (3 + 5 * both)}
