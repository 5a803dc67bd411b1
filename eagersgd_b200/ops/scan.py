"""Selective state-space scan with the short causal convolution ahead of it: a sequence layer without an LSTM's serial products.

A layer projects its input, runs ``causal_conv`` over the steps, makes ``delta``, ``B`` and ``C`` from the result, and scans:

    dt   = softplus(delta + delta_bias)
    h[t] = exp(dt[t] A) h[t - 1] + dt[t] u[t] B[t]
    y[t] = sum over the states of C[t] h[t], + D u[t],  times silu(z[t])

Sequences are ``[B, T, D]`` (any strides between the rows: slices of a projection and time-first tensors are read as they lie), bf16
or fp32 alike for all of a call's sequences; parameters and states are fp32 (a convolution's state has its inputs' type).  ``lengths``
(int64 [B]) ends each sequence by itself: what lies behind is not read, the outputs there are zero, and the state is that of the last
step before it.

For serving, ``return_state=True`` gives what the ``..._step`` functions go on from, one step of every sequence at a time; ``state=``
starts a sequence from one.  States carry no gradient.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F

from .. import _build
from .functional import activation_code, native_float, refuse_derivative

_TAKEN = (None, "silu")


def _wide(*tensors):
    """In fp32, or in fp64 where the first is."""
    dtype = torch.float64 if tensors[0].dtype == torch.float64 else torch.float32
    return [None if t is None else t.to(dtype) for t in tensors]


def _inside(length: int, lengths: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    t = torch.arange(length, device=like.device)
    return (t < lengths.unsqueeze(1)) if lengths is not None else torch.ones(like.shape[0], length, dtype=torch.bool, device=like.device)


def _one_step(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Sequences of no step with a step of zeros."""
    return None if x is None else F.pad(x, (0, 0, 0, 1))


def _no_step(x: torch.Tensor) -> torch.Tensor:
    return torch.zeros(x.shape[0], dtype=torch.int64, device=x.device)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y[t] = act(bias + sum over k of weight[:, k] * x[t - K + 1 + k]), every channel by itself.

    ``x`` [B, T, D], ``weight`` fp32 [D, K] with K from 2 to 4, ``bias`` fp32 [D], ``activation`` "silu" or None; ``state`` [B, K - 1, D]:
    the inputs ahead of the first (default: zeros).  With ``return_state`` also the last K - 1 inputs, for ``causal_conv_step``."""
    act = activation_code("causal_conv", activation, _TAKEN)
    if native_float(x):
        r = _build.load_torch().causal_conv(x, weight, bias, act, state, lengths, return_state)
        return tuple(r) if return_state else r[0]
    refuse_derivative("causal_conv", "a state", state)
    taps, length = weight.shape[1], x.shape[1]
    if length == 0:                 # as one step that none of the sequences has
        y, last = causal_conv(_one_step(x), weight, bias, activation, state, _no_step(x), True)
        return (y[:, :0], last) if return_state else y[:, :0]
    xw, w, b = _wide(x, weight, bias)
    inside = _inside(length, lengths, x)
    ahead = xw.new_zeros(x.shape[0], taps - 1, x.shape[2]) if state is None else state.detach().to(xw.dtype)
    padded = torch.cat([ahead, torch.where(inside.unsqueeze(2), xw, 0.0)], 1)
    y = (padded.unfold(1, taps, 1) * w).sum(3)
    y = y if b is None else y + b
    y = torch.where(inside.unsqueeze(2), F.silu(y) if activation == "silu" else y, 0.0).to(x.dtype)
    if not return_state:
        return y
    at = inside.sum(1, keepdim=True) + torch.arange(taps - 1, device=x.device)
    return y, padded.detach().gather(1, at.unsqueeze(2).expand(-1, -1, x.shape[2])).to(x.dtype)


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = "silu", out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``causal_conv`` of one more input ``x`` [B, D]: (y [B, D], the new state).  The new state is a new tensor, or ``out``, which may be
    ``state`` itself."""
    act = activation_code("causal_conv_step", activation, _TAKEN)
    if native_float(x):
        return _build.load_torch().causal_conv_step(x, state, weight, bias, act, out)
    y, new = causal_conv(x.unsqueeze(1), weight, bias, activation, state, None, True)
    return y.squeeze(1), new if out is None else out.copy_(new)


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
                   softplus: bool = True, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The scan above.  ``u``, ``delta`` and ``z`` [B, T, D], ``B`` and ``C`` [B, T, N], ``A`` fp32 [D, N] (below zero, or the states grow) with
    N up to 64, ``D`` and ``delta_bias`` fp32 [D], ``state`` fp32 [B, D, N].  ``softplus=False``: dt is delta + delta_bias.  With
    ``return_state`` also the last state, for ``selective_scan_step``."""
    if native_float(u):
        r = _build.load_torch().selective_scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, return_state)
        return tuple(r) if return_state else r[0]
    refuse_derivative("selective_scan", "a state", state)
    if u.shape[1] == 0:
        y, h = selective_scan(*map(_one_step, (u, delta)), A, *map(_one_step, (B, C)), D, _one_step(z), delta_bias, softplus, state, _no_step(u), True)
        return (y[:, :0], h) if return_state else y[:, :0]
    uw, dw, Aw, Bw, Cw, Dw, zw, bw = _wide(u, delta, A, B, C, D, z, delta_bias)
    inside = _inside(u.shape[1], lengths, u)
    if lengths is not None:         # a value behind the end meets nothing: times the zero of a gradient it could still be no number
        uw, dw, Bw, Cw, zw = (None if v is None else torch.where(inside.unsqueeze(2), v, 0.0) for v in (uw, dw, Bw, Cw, zw))
    dt = dw if bw is None else dw + bw
    dt = F.softplus(dt) if softplus else dt
    h = uw.new_zeros(u.shape[0], *A.shape) if state is None else state.detach().to(uw.dtype)
    outs = []
    for t in range(u.shape[1]):
        live = inside[:, t].view(-1, 1, 1)
        new = torch.exp(dt[:, t].unsqueeze(2) * Aw) * h + (dt[:, t] * uw[:, t]).unsqueeze(2) * Bw[:, t].unsqueeze(1)
        h = torch.where(live, new, h)
        y = (h * Cw[:, t].unsqueeze(1)).sum(2)
        y = y if Dw is None else y + Dw * uw[:, t]
        y = y if zw is None else y * F.silu(zw[:, t])
        outs.append(torch.where(live.squeeze(2), y, 0.0))
    y = torch.stack(outs, 1).to(u.dtype)
    return (y, h.detach()) if return_state else y


def selective_scan_step(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
                        softplus: bool = True, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``selective_scan`` of one more step, ``u``, ``delta`` and ``z`` [B, D], ``B`` and ``C`` [B, N]: (y [B, D], the new state).  The new state is a
    new tensor, or ``out``, which may be ``state`` itself."""
    if native_float(u):
        return _build.load_torch().selective_scan_step(u, delta, A, B, C, state, D, z, delta_bias, softplus, out)
    y, new = selective_scan(u.unsqueeze(1), delta.unsqueeze(1), A, B.unsqueeze(1), C.unsqueeze(1), D, None if z is None else z.unsqueeze(1),
                            delta_bias, softplus, state, None, True)
    return y.squeeze(1), new if out is None else out.copy_(new)
