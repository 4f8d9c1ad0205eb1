"""The feed-forward sublayer on a residual stream, trained and served in 8 bits.

    h = x + residual;    y = h + W2 act(W1 norm(h) + b1) + b2

:class:`FeedForward` runs on :func:`maloq_amd.norm.rms_norm` and :func:`maloq_amd.dense.linear_act`:
the additions, biases and the activation are in the kernels' epilogues, so a layer is three
forward launches for large batches.  :meth:`FeedForward.quantized` gives the serving form, whose products take e4m3
operands: the norm writes its output in 8 bits, the activation's output is quantised a row at a time.
"""
from __future__ import annotations

import math

import torch

from .dense import ACTIVATIONS, linear_act, linear_quantized, quantize_rows
from .norm import rms_norm, rms_norm_quantized


class FeedForward(torch.nn.Module):
    """``width`` -> ``inner`` -> ``width`` (each at most 16384 for :meth:`quantized`); act: "none",
    "relu", "silu" or "gelu"; dtype float32, bfloat16 or float16.  Parameters: norm_weight [width],
    w1 [inner, width], b1 [inner], w2 [width, inner], b2 [width]."""

    def __init__(self, width: int, inner: int, act: str = "silu", bias: bool = True, eps: float = 1e-6, device=None,
                 dtype: torch.dtype | None = None):
        super().__init__()
        if act not in ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
        if width < 1 or width > 16384 or inner < 1:
            raise ValueError(f"width must be 1 to 16384 and inner positive, got {width} and {inner}")
        kw = {"device": device, "dtype": dtype}
        self.act, self.eps = act, float(eps)
        self.norm_weight = torch.nn.Parameter(torch.ones(width, **kw))
        self.w1 = torch.nn.Parameter(torch.empty(inner, width, **kw))
        self.w2 = torch.nn.Parameter(torch.empty(width, inner, **kw))
        self.b1 = torch.nn.Parameter(torch.zeros(inner, **kw)) if bias else None
        self.b2 = torch.nn.Parameter(torch.zeros(width, **kw)) if bias else None
        for w in (self.w1, self.w2):
            torch.nn.init.normal_(w, std=1 / math.sqrt(w.shape[1]))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """The stream after the sublayer, of x's sizes [.., width]."""
        if residual is None:
            h, n = x, rms_norm(x, self.norm_weight, self.eps)
        else:
            n, h = rms_norm(x, self.norm_weight, self.eps, residual=residual)
        return linear_act(linear_act(n, self.w1, self.b1, act=self.act), self.w2, self.b2, residual=h)

    def quantized(self) -> "QuantizedFeedForward":
        """The serving form of the present weights."""
        return QuantizedFeedForward(self)


class QuantizedFeedForward(torch.nn.Module):
    """:class:`FeedForward` with e4m3 operands (one fp32 scale a row of activations and of weights); sums, activation
    and residual as there.  No gradient."""

    def __init__(self, layer: FeedForward):
        super().__init__()
        if layer.w1.shape[0] > 16384:
            raise ValueError(f"rows of {layer.w1.shape[0]} activations are too long to quantise (16384)")
        self.act, self.eps = layer.act, layer.eps
        for name in ("norm_weight", "b1", "b2"):
            p = getattr(layer, name)
            self.register_buffer(name, None if p is None else p.detach().clone())
        for name in ("w1", "w2"):
            q, scale = quantize_rows(getattr(layer, name).detach())
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        got = rms_norm_quantized(x, self.norm_weight, self.eps, residual=residual)
        q, scale, h = got if residual is not None else (*got, x)
        a = linear_quantized(q, scale, self.w1, self.w1_scale, self.b1, act=self.act, dtype=x.dtype)
        return linear_quantized(*quantize_rows(a), self.w2, self.w2_scale, self.b2, residual=h, dtype=x.dtype)
