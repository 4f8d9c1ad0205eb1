"""Root-mean-square norm of a residual stream, with its gradients, and its output in 8 bits.

    h = x + residual;    y = h / sqrt(mean(h^2) + eps) * weight     (over the last dimension)

One pass over the data each way; statistics and sums are fp32, every output is rounded once.  The
backward starts from the stored ``h`` (rounded to the tensors' type) and one fp32 number a row; in
float16 with a residual, whose sums may pass 65504, from the normed row ``h / sqrt(..)`` of that
type instead, which the forward writes too where a gradient is wanted.

The 8-bit form writes ``y`` as e4m3 numbers with one fp32 scale a row, ``y = q * scale``, for
:func:`maloq_amd.dense.linear_quantized`.

The reference's norms are torch modules (helm/nn/layer_norm.py:18-338) over the rows of a degree;
this one takes the rows of any tensor's last dimension.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib


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


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """``(q, scale)``, or with a residual ``(q, scale, h)``: the norm's output in 8 bits.

    q: float8_e4m3fn of x's sizes; scale: float32, one a row (x's sizes without the last), such
    that the row's largest value is 448, and at least 2^-100 / 448.  A row that holds an infinity
    or a NaN has a NaN scale.  No gradient.
    """
    _lib.require_cuda(x, weight, residual)
    from . import ops
    with torch.no_grad():
        q, scale, h = ops.rms_norm_quantized(x, weight, float(eps), residual)
    return (q, scale) if residual is None else (q, scale, h)
