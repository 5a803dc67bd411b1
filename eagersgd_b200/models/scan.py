"""Sequence classifier on selective scans: the LSTM classifier's interface without its serial products.

A layer normalises its input, projects it to twice its width, runs a short causal convolution over one half, makes the scan's time
steps, inputs and outputs from the result, scans, gates with the other half, and adds its projection back to the input.  All steps of
all sequences go through every product at once; only the scan itself knows an order.  A stream of steps (``step``) keeps a state of
fixed size a layer.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
import torch.nn as nn

from ..ops import functional as ops
from ..ops import scan
from .resnet import GroupNormAct

State = List[Tuple[torch.Tensor, torch.Tensor]]


def _project(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """[rows, in] -> [rows, out] in x's type."""
    if x.shape[0] == 0:                      # the kernels refuse a product of no row
        return nn.functional.linear(x, w)
    return ops.conv1x1(x.reshape(x.shape[0], x.shape[1], 1, 1), w.reshape(*w.shape, 1, 1)).reshape(x.shape[0], w.shape[0])


class ScanLayer(nn.Module):
    def __init__(self, hidden: int, width: int, states: int = 16, taps: int = 4, step_rank: Optional[int] = None):
        super().__init__()
        self.hidden, self.width, self.states = hidden, width, states
        self.rank = step_rank or max(8, (width // 16 + 7) // 8 * 8)
        uniform = lambda *s: nn.Parameter(torch.empty(*s).uniform_(-1, 1) / math.sqrt(s[-1]))  # noqa: E731
        self.norm = GroupNormAct(1, hidden)
        self.w_in = uniform(2 * width, hidden)
        self.conv_weight, self.conv_bias = uniform(width, taps), nn.Parameter(torch.zeros(width))
        self.w_bc = uniform(self.rank + 2 * states, width)
        self.w_step = uniform(width, self.rank)
        # time steps between 0.001 and 0.1 to begin with, as the inverse of softplus gives them
        dt = torch.exp(torch.rand(width) * math.log(100.0) + math.log(0.001))
        self.step_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.log_rate = nn.Parameter(torch.log(torch.arange(1, states + 1).float()).repeat(width, 1))
        self.skip = nn.Parameter(torch.ones(width))
        self.w_out = uniform(hidden, width)

    def compute_dtype_(self, dtype):
        """Low-precision weights for the products; all else stays fp32."""
        for p in (self.w_in, self.w_bc, self.w_step, self.w_out):
            p.data = p.data.to(dtype)
        return self

    def _ahead(self, h):
        x = self.norm(h.reshape(h.shape[0], self.hidden, 1, 1), relu=False)
        return _project(x.reshape(h.shape), self.w_in)

    def _operands(self, u):
        """Time steps, B and C out of the convolution's output [rows, width]."""
        p = _project(u, self.w_bc)
        r, n = self.rank, self.states
        return _project(p[:, :r].contiguous(), self.w_step), p[:, r:r + n], p[:, r + n:r + 2 * n]

    def forward(self, h, lengths=None, return_state=False):
        """h [B, T, hidden] -> the same, and the layer's state behind the last step of every sequence."""
        b, t = h.shape[:2]
        rows = lambda v: v.flatten(0, 1)  # noqa: E731
        steps = lambda v: v.unflatten(0, (b, t))  # noqa: E731
        xz = steps(self._ahead(rows(h)))
        conv = scan.causal_conv(xz[..., :self.width], self.conv_weight, self.conv_bias, lengths=lengths, return_state=return_state)
        u, conv_state = conv if return_state else (conv, None)
        delta, B, C = (steps(v) for v in self._operands(rows(u)))
        y = scan.selective_scan(u, delta, -torch.exp(self.log_rate), B, C, D=self.skip, z=xz[..., self.width:], delta_bias=self.step_bias,
                                lengths=lengths, return_state=return_state)
        y, scan_state = y if return_state else (y, None)
        h = h + steps(_project(rows(y), self.w_out))
        return (h, (conv_state, scan_state)) if return_state else h

    def step(self, h, state):
        """One step h [B, hidden]; ``state`` is moved on in place."""
        xz = self._ahead(h)
        u, _ = scan.causal_conv_step(xz[:, :self.width], state[0], self.conv_weight, self.conv_bias, out=state[0])
        delta, B, C = self._operands(u)
        y, _ = scan.selective_scan_step(u, delta, -torch.exp(self.log_rate), B, C, state[1], D=self.skip, z=xz[:, self.width:],
                                        delta_bias=self.step_bias, out=state[1])
        return h + _project(y, self.w_out)


class ScanClassifier(nn.Module):
    """Stacked scan layers over per-frame feature vectors, linear head on the last step; stands where ``LSTMClassifier`` does.
    ``dropout``: between the layers, in training, as there."""

    dropout = 0.0                            # also of networks that were saved without it

    def __init__(self, input_dim: int = 2048, hidden: int = 1024, layers: int = 2, num_classes: int = 101, width: Optional[int] = None,
                 states: int = 16, taps: int = 4, dropout: float = 0.0):
        super().__init__()
        self.hidden, self.dropout = hidden, dropout
        self.w_embed = nn.Parameter(torch.empty(hidden, input_dim).uniform_(-1, 1) / math.sqrt(input_dim))
        self.layers = nn.ModuleList(ScanLayer(hidden, width or 2 * hidden, states, taps) for _ in range(layers))
        self.fc = nn.Linear(hidden, num_classes)

    def compute_dtype_(self, dtype):
        self.w_embed.data = self.w_embed.data.to(dtype)
        for layer in self.layers:
            layer.compute_dtype_(dtype)
        self.fc.to(dtype)
        return self

    def _stack(self, x, lengths=None, return_state=False):
        b, t = x.shape[:2]
        h = _project(x.flatten(0, 1).flatten(1), self.w_embed).unflatten(0, (b, t))
        states = []
        for i, layer in enumerate(self.layers):
            h = layer(self._between(i, h), lengths, return_state)
            if return_state:
                h, s = h
                states.append(s)
        return h, states

    def _between(self, i, h):
        return nn.functional.dropout(h, self.dropout) if i > 0 and self.dropout > 0 and self.training else h

    def hidden_states(self, x, lengths=None):
        """x [B, T, input_dim] -> the top layer's outputs [T, B, hidden]."""
        return self._stack(x, lengths)[0].transpose(0, 1)

    def _last(self, h, lengths):
        if lengths is None:
            return h[:, -1]
        return h[torch.arange(h.shape[0], device=h.device), lengths.clamp(1, h.shape[1]) - 1]

    def _logits(self, h):
        if h.shape[0] == 0:
            return nn.functional.linear(h, self.fc.weight, self.fc.bias).to(torch.float32 if ops.native(h) else h.dtype)
        return ops.linear(h, self.fc.weight, self.fc.bias)

    def forward(self, x, lengths=None):
        """x [B, T, input_dim] -> logits [B, classes] of every sequence's last step."""
        return self._logits(self._last(self._stack(x, lengths)[0], lengths).contiguous())

    @torch.no_grad()
    def prompt(self, x, lengths=None) -> Tuple[torch.Tensor, State]:
        """Logits as ``forward`` gives them, and the state that ``step`` goes on from."""
        h, states = self._stack(x, lengths, True)
        return self._logits(self._last(h, lengths).contiguous()), states

    @torch.no_grad()
    def step(self, x, state: State) -> torch.Tensor:
        """Logits after one step more, x [B, input_dim]; ``state`` is moved on in place."""
        h = _project(x, self.w_embed)
        for i, (layer, s) in enumerate(zip(self.layers, state)):
            h = layer.step(self._between(i, h), s)
        return self._logits(h)
