"""Selective state space layers: the PyTorch module a model is trained with, and its
export to the engine's model files.

A layer is  xz = in_proj(x);  u = silu(causal_conv(xz[:D]));  [r, B, C] = x_proj(u);
dt = dt_proj(r);  y = selective_scan(u, dt, B, C) * silu(xz[D:]);  out_proj(y).
The reference has no such layer; the engine runs it as CausalConv and SelectiveScan
steps between Gemms (``eight_bit``: between 8-bit Gemms, rounding weights and
activations to e4m3).  A model exported with ``with_state`` takes and returns the
layers' states, so that a solver can feed it one step (or any number) at a time, as
it does an LSTM's h and c.
"""
from __future__ import annotations

import math
from typing import Sequence

import numpy as np
import torch
from torch import nn
from torch.nn import functional as F

from . import writer


class SelectiveLayer(nn.Module):
    """width -> width; `expand` * width channels, `states` states per channel."""

    def __init__(self, width: int, states: int = 16, taps: int = 4, expand: int = 2, dt_rank: int = 0):
        super().__init__()
        D = expand * width
        R = dt_rank or max(1, math.ceil(width / 16))
        self.width, self.channels, self.states, self.taps, self.dt_rank = width, D, states, taps, R
        self.in_proj = nn.Linear(width, 2 * D, bias=False)
        self.conv1d = nn.Conv1d(D, D, taps, groups=D, padding=taps - 1)
        self.x_proj = nn.Linear(D, R + 2 * states, bias=False)
        self.dt_proj = nn.Linear(R, D)
        self.A_log = nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32).repeat(D, 1)))
        self.D = nn.Parameter(torch.ones(D))
        self.out_proj = nn.Linear(D, width, bias=False)
        with torch.no_grad():  # steps between 0.001 and 0.1
            base = torch.exp(torch.rand(D) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
            self.dt_proj.bias.copy_(base + torch.log(-torch.expm1(-base)))

    def forward(self, x, conv_state=None, scan_state=None):
        """x (N, T, width); states (N, taps - 1, D) and (N, states, D), or None (zeros).
        -> y (N, T, width), the states after the last step."""
        n, T, _ = x.shape
        D, S = self.channels, self.states
        xz = self.in_proj(x)
        first = x.new_zeros(n, self.taps - 1, D) if conv_state is None else conv_state
        ext = torch.cat([first, xz[..., :D]], 1)
        u = F.silu(F.conv1d(ext.transpose(1, 2), self.conv1d.weight, self.conv1d.bias, groups=D).transpose(1, 2))
        dbc = self.x_proj(u)
        delta = F.softplus(self.dt_proj(dbc[..., :self.dt_rank]), threshold=50.0)
        B, C = dbc[..., self.dt_rank:self.dt_rank + S], dbc[..., self.dt_rank + S:]
        A = -torch.exp(self.A_log)
        h = x.new_zeros(n, D, S) if scan_state is None else scan_state.transpose(1, 2)
        ys = []
        for t in range(T):
            h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * u[:, t])[..., None] * B[:, t, None]
            ys.append((h * C[:, t, None]).sum(-1) + self.D * u[:, t])
        y = torch.stack(ys, 1) * F.silu(xz[..., D:])
        return self.out_proj(y), ext[:, T:], h.transpose(1, 2)


def export_selective(layers: Sequence[SelectiveLayer], head: Sequence, batch: int, seq_len: int, mode: str = "last",
                     with_state: bool = False, eight_bit: bool = False) -> writer.Graph:
    """Graph of stacked layers.  mode "last": the head runs on the last step's output,
    (batch, width); "y": the whole sequence (batch, seq_len, width), no head.  with_state
    adds, per layer, the inputs conv_state<i> (batch, taps - 1, channels; none with a
    single tap) and scan_state<i> (batch, states, channels), and the states after the last
    step as outputs, in front of the result (outputs come in the order of their nodes).
    The engine holds Gemms of at most 880 outputs in fp32, so 2 * expand * width is at
    most that unless `eight_bit`."""
    if mode not in ("last", "y") or (mode == "y" and len(head)):
        raise ValueError("mode is 'last', or 'y' without a head")
    if batch < 1 or seq_len < 1:
        raise ValueError(f"batch and seq_len are at least 1, got {batch} and {seq_len}")
    if not layers or any(ly.width != layers[0].width for ly in layers):
        raise ValueError("layers are one or more, of the same width")
    b = writer._Builder()
    N, T, W = batch, seq_len, layers[0].width
    inputs = [("input", [N, T, W])]
    b.vi["input"] = [N, T, W]
    x = b.add("Transpose", ["input"], [[T, N, W]], {"perm": [1, 0, 2]})[0]
    states_out = []

    def linear(v, lin, with_bias=True):
        M = lin.weight.shape[0]
        bias = np.zeros(M, np.float32) if lin.bias is None or not with_bias else writer._np32(lin.bias)
        if eight_bit:
            return b.add("Gemm8", [v, b.weight(writer._np32(lin.weight)), b.weight(bias)], [[T, N, M]], {"params": [0, 0]})[0]
        v = b.add("Alias", [v], [b.vi[v]])[0]  # a Gemm takes its operand's name over
        return b.add("Gemm", [v, b.weight(writer._np32(lin.weight)), b.weight(bias)], [[T, N, M]], {"transB": 1})[0]

    for i, ly in enumerate(layers):
        D, S, R = ly.channels, ly.states, ly.dt_rank
        conv_st, scan_st = ([f"conv_state{i}"] if with_state and ly.taps > 1 else []), ([f"scan_state{i}"] if with_state else [])
        for name, rows in [(v, ly.taps - 1) for v in conv_st] + [(v, S) for v in scan_st]:
            inputs.append((name, [N, rows, D]))
            b.vi[name] = [N, rows, D]
        xz = linear(x, ly.in_proj)
        wc = writer._np32(ly.conv1d.weight).reshape(D, ly.taps)
        bc = np.zeros(D, np.float32) if ly.conv1d.bias is None else writer._np32(ly.conv1d.bias)
        u, cs = b.add("CausalConv", [xz] + conv_st + [b.weight(wc), b.weight(bc)], [[T, N, D], [N, ly.taps - 1, D]], {"params": [0, 4]})
        dbc = linear(u, ly.x_proj)
        # the step's part of x_proj's output: its leading features
        r = b.add("Slice", [dbc], [[T, N, R]], {"axes": [2], "starts": [0], "ends": [R]})[0]
        dt = linear(r, ly.dt_proj, with_bias=False)  # its bias goes with softplus into the scan
        A = (-np.exp(ly.A_log.detach().cpu().double().numpy())).astype(np.float32)
        y, hs = b.add("SelectiveScan", [u, dt, dbc, dbc, xz, scan_st[0] if scan_st else "", b.weight(A), b.weight(writer._np32(ly.D)),
                                        b.weight(writer._np32(ly.dt_proj.bias))], [[T, N, D], [N, S, D]],
                      {"params": [0, R, R + S, D, 1, 1]})
        states_out += ([(cs, [N, ly.taps - 1, D])] if ly.taps > 1 else []) + [(hs, [N, S, D])]
        x = linear(y, ly.out_proj)
    if mode == "y":
        out = b.add("Transpose", [x], [[N, T, W]], {"perm": [1, 0, 2]})[0]
        shape = [N, T, W]
    else:
        idx = b.const(np.array(T - 1))
        out = b.add("Gather", [x, idx], [[N, W]], {"axis": 0})[0]
        shape = [N, W]
        for m in head:
            out, shape = writer._emit_module(b, m, out, shape)
    outputs = (states_out if with_state else []) + [(out, list(shape))]
    return writer.Graph(b.nodes, inputs, outputs, b.inits, b.vi, b.consts, b.true_weights)
