"""Root-mean-square norm of a residual stream, with its gradients, and its output in 8 bits.

    h = x + residual;    y = h / sqrt(mean(h^2) + eps) * weight     (over the last dimension)

One pass over the data each way; statistics and sums are fp32, every output is rounded once.  The
backward starts from the stored ``h`` (rounded to the tensors' type) and one fp32 number a row; in
float16 with a residual, whose sums may pass 65504, from the normed row ``h / sqrt(..)`` of that
type instead, which the forward writes too where a gradient is wanted.

The 8-bit form writes ``y`` as e4m3 numbers or integers with one fp32 scale a row, ``y = q * scale``, for
:func:`maloq_amd.dense.linear_quantized`.

Beside it, group norm with an activation, channels last:

    y = act((x - mean) / sqrt(var + eps) * weight + bias)     (over a sample's positions and a group's channels)

The reference's norms are torch modules (helm/nn/layer_norm.py:18-338) over the rows of a degree;
these take the rows of any tensor's last dimension, and its groups of channels.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


class _RmsNorm(torch.autograd.Function):
    """The operators with their gradients where something traces the call; eager calls go through
    the same in C++."""

    @staticmethod
    def forward(ctx, x, w, eps, residual):
        from . import ops
        ctx.residual = residual is not None
        ctx.unit = ctx.residual and x.dtype == torch.float16
        y, h, rstd, *unit = ops.rms_norm_fwd(x, w, eps, residual, ctx.unit)
        ctx.save_for_backward(unit[0] if ctx.unit else h if ctx.residual else x, w, rstd)
        return (y, h) if ctx.residual else y

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *g_h):
        from . import ops
        h, w, rstd = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[0] or ctx.needs_input_grad[3], ctx.needs_input_grad[1]
        dx, dw = ops.rms_norm_bwd(g, g_h[0] if ctx.residual else None, h, w, rstd, need_x, need_w, ctx.unit)
        dx = dx if need_x else None
        return dx, dw if need_w else None, None, dx if ctx.residual else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """``y``, or with a residual ``(y, h)``.

    x: float32, bfloat16 or float16 on the GPU, its last dimension (at most 16384 values) normed;
    weight: that dimension, of x's type; residual: of x's sizes and type.  Differentiable once, in
    reverse mode: vmap, forward mode and the other transforms of torch.func raise.
    Where x + residual passes the type's range (65504 in float16) h is infinite; y and the gradients,
    which take the sum as it is, stay finite.
    A training step that is captured into a HIP graph needs, as any other of torch's, that no
    eager graph of the same leaves is alive.
    """
    _lib.require_cuda(x, weight, residual)
    from . import ops
    if not _lib.eager(x, weight, residual):
        return _RmsNorm.apply(x, weight, float(eps), residual)
    out = ops._ops._rms_norm(x, weight, float(eps), residual)
    return out[0] if residual is None else (out[0], out[1])


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                       dtype: torch.dtype = torch.float8_e4m3fn):
    """``(q, scale)``, or with a residual ``(q, scale, h)``: the norm's output in 8 bits.

    q: dtype (float8_e4m3fn or int8) of x's sizes; scale: float32, one a row (x's sizes without the last), such
    that the row's largest value is 448 (int8: 127), and at least 2^-100 / 448 (127).  A row that holds an infinity
    or a NaN has a NaN scale.  No gradient.
    """
    _lib.require_cuda(x, weight, residual)
    from . import ops
    with torch.no_grad():
        q, scale, h = ops.rms_norm_quantized(x, weight, float(eps), residual, dtype)
    return (q, scale) if residual is None else (q, scale, h)


class _GroupNorm(torch.autograd.Function):
    """The operators with their gradients where something traces the call; eager calls go through
    the same in C++."""

    @staticmethod
    def forward(ctx, x, groups, w, b, eps, act):
        from . import ops
        y, stats = ops.group_norm_fwd(x, groups, w, b, eps, act)
        ctx.groups, ctx.act = groups, act
        ctx.save_for_backward(x, w, b, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        from . import ops
        x, w, b, stats = ctx.saved_tensors
        nx, _, nw, nb = ctx.needs_input_grad[:4]
        dx, dwb = ops.group_norm_bwd(g, x, w, b, stats, ctx.groups, ctx.act, nx, nw or nb)
        return dx if nx else None, None, dwb[0] if nw else None, dwb[1] if nb else None, None, None


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               act: str = "none") -> torch.Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)``, channels last.

    x: [samples, ..., channels] (at least two dimensions), float32, bfloat16 or float16 on the GPU, rows of channels contiguous
    (others are copied); groups: a divisor of the channels.  Mean and variance (of the values, not an estimate from a sample)
    are those of a sample's positions and of a group's consecutive channels.  weight, bias: [channels], of x's type, or None;
    act: "none", "relu", "silu" or "gelu" (by erf).  Every sample has as many positions.  One mean and one bias for all
    components of a channel: for scalars, not for the rows of degree 1 and more of an equivariant feature.
    Statistics, sums and the activation are fp32, every output is rounded once.  The backward starts from x and the statistics and
    keeps nothing else; its sums are in a fixed order.  Differentiable once, in reverse mode: vmap, forward mode and the other
    transforms of torch.func raise.
    A training step that is captured into a HIP graph needs, as any other of torch's, that no
    eager graph of the same leaves is alive.
    """
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    if groups % 1 != 0:
        raise ValueError(f"the number of groups must be a whole one, got {groups}")
    _lib.require_cuda(x, weight, bias)
    from . import ops
    code = ACTIVATIONS[act]
    if not _lib.eager(x, weight, bias):
        return _GroupNorm.apply(x, int(groups), weight, bias, float(eps), code)
    return ops._ops._group_norm(x, int(groups), weight, bias, float(eps), code)
