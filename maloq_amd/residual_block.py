"""A residual block of two linear layers between group norms, over grids or sets of positions, channels last.

    y = x + W2 act(norm2(W1 act(norm1(x)) + b1)) + b2

:class:`ResidualBlock` runs on :func:`maloq_amd.norm.group_norm`, whose activation is part of it, and
:func:`maloq_amd.dense.linear_act`, whose epilogue adds x; with ``checkpoint=torch.int8`` the layers keep their inputs for
the backward in 8 bits.  :meth:`ResidualBlock.quantized` gives the serving form, whose products take int8 or e4m3 operands.
"""
from __future__ import annotations

import math

import torch

from .dense import linear_act, linear_quantized, quantize_rows
from .norm import ACTIVATIONS, group_norm


class ResidualBlock(torch.nn.Module):
    """x [samples, ..., channels]; ``channels`` -> ``inner`` -> ``channels`` (each at most 16384 for :meth:`quantized`), both of
    ``groups`` groups; act: "none", "relu", "silu" or "gelu"; dtype float32, bfloat16 or float16; checkpoint: None or
    torch.int8.  Parameters: norm1_weight, norm1_bias [channels], w1 [inner, channels], b1 [inner], norm2_weight,
    norm2_bias [inner], w2 [channels, inner], b2 [channels]."""

    def __init__(self, channels: int, inner: int, groups: int, act: str = "silu", eps: float = 1e-5, device=None,
                 dtype: torch.dtype | None = None, checkpoint: torch.dtype | None = None):
        super().__init__()
        if act not in ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
        if groups < 1 or channels < 1 or inner < 1 or channels % groups or inner % groups:
            raise ValueError(f"{channels} and {inner} channels do not make {groups} groups")
        if checkpoint not in (None, torch.int8):
            raise ValueError(f"activations are kept as they are (None) or in 8 bits (torch.int8), not as {checkpoint}")
        kw = {"device": device, "dtype": dtype}
        self.groups, self.act, self.eps, self.checkpoint = groups, act, float(eps), checkpoint
        for i, (n, m) in enumerate(((channels, inner), (inner, channels)), 1):
            setattr(self, f"norm{i}_weight", torch.nn.Parameter(torch.ones(n, **kw)))
            setattr(self, f"norm{i}_bias", torch.nn.Parameter(torch.zeros(n, **kw)))
            setattr(self, f"w{i}", torch.nn.Parameter(torch.nn.init.normal_(torch.empty(m, n, **kw), std=1 / math.sqrt(n))))
            setattr(self, f"b{i}", torch.nn.Parameter(torch.zeros(m, **kw)))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        a = group_norm(x, self.groups, self.norm1_weight, self.norm1_bias, self.eps, act=self.act)
        h = linear_act(a, self.w1, self.b1, checkpoint=self.checkpoint)
        a = group_norm(h, self.groups, self.norm2_weight, self.norm2_bias, self.eps, act=self.act)
        return linear_act(a, self.w2, self.b2, residual=x, checkpoint=self.checkpoint)

    def quantized(self, dtype: torch.dtype = torch.int8) -> "QuantizedResidualBlock":
        """The serving form of the present weights, its products' operands int8 or float8_e4m3fn."""
        return QuantizedResidualBlock(self, dtype)


class QuantizedResidualBlock(torch.nn.Module):
    """:class:`ResidualBlock` with 8-bit operands (one fp32 scale a row of activations and of weights); norms, sums,
    activations and the residual as there.  No gradient."""

    def __init__(self, block: ResidualBlock, dtype: torch.dtype = torch.int8):
        super().__init__()
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"8-bit operands are float8_e4m3fn or int8, not {dtype}")
        if max(block.w1.shape) > 16384:
            raise ValueError(f"rows of {max(block.w1.shape)} activations are too long to quantise (16384)")
        self.groups, self.act, self.eps = block.groups, block.act, block.eps
        for name in ("norm1_weight", "norm1_bias", "norm2_weight", "norm2_bias", "b1", "b2"):
            self.register_buffer(name, getattr(block, name).detach().clone())
        for name in ("w1", "w2"):
            q, scale = quantize_rows(getattr(block, name).detach(), dtype)
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        dt = self.w1.dtype
        with torch.no_grad():
            a = group_norm(x, self.groups, self.norm1_weight, self.norm1_bias, self.eps, act=self.act)
            h = linear_quantized(*quantize_rows(a, dt), self.w1, self.w1_scale, self.b1, dtype=x.dtype)
            a = group_norm(h, self.groups, self.norm2_weight, self.norm2_bias, self.eps, act=self.act)
            return linear_quantized(*quantize_rows(a, dt), self.w2, self.w2_scale, self.b2, residual=x, dtype=x.dtype)
