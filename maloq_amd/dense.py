"""Linear layers with bias, activation and residual in the product's epilogue, and their 8-bit form.

    y = act(x W^T + b) + residual

``linear_act`` trains (float32, bfloat16, float16; float32 products on the bf16 matrix cores at
fp32 exactness); ``quantize_rows`` and ``linear_quantized`` serve: e4m3 operands with one fp32
scale a row of x (:func:`maloq_amd.norm.rms_norm_quantized`) and a row of the weight.

Products, sums and activations are fp32 and the result is rounded once, but for the sums of e4m3
products inside a matrix instruction: eight consecutive ones are added as multiples of 2^-13 of the
largest's power of two (the eights in fp32), beside the 2^-4 by which the operands are rounded.  The
backward of an activation starts from the product as it was stored, in the tensors' type, and the
products of the gradients take the activation's gradient rounded to that type (in float16 beyond
65504 that is an infinity, as of any tensor of that type).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _act(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


class _LinearAct(torch.autograd.Function):
    """The operators with their gradients where something traces the call; eager calls go through
    the same in C++."""

    @staticmethod
    def forward(ctx, x, w, b, act, residual):
        from . import ops
        y, z = ops.linear_act_fwd(x, w, b, act, residual, True)
        ctx.act, ctx.bias, ctx.residual = act, b is not None, residual is not None
        ctx.save_for_backward(x, w, z if act else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        from . import ops
        x, w, z = ctx.saved_tensors
        need = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.bias and ctx.needs_input_grad[2]]
        got = ops.linear_act_bwd(g, x, w, z, ctx.act, *need) if any(need) else [None] * 3
        dx, dw, db = (t if n else None for t, n in zip(got, need))
        return dx, dw, db, None, g if ctx.residual else None


def linear_act(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None = None, act: str = "none",
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x w^T + b) + residual``.

    x: [..., k] on the GPU, float32, bfloat16 or float16; w: [n, k], b: [n], residual: [..., n], all
    of x's type; act: "none", "relu", "silu" or "gelu" (by erf).  Differentiable once, in reverse
    mode: vmap, forward mode and the other transforms of torch.func raise.
    Rows of whole 16 bytes (k a multiple of 8, in float32 of 4) are read where they lie.  For other k
    a call without gradients copies x and w to such in each call from 17 rows on (float32: always; 64 rows
    of 4095 to 16384 bfloat16: 78 us, of 4096 27), and up to 16 rows read at odd addresses (one row 63, 22):
    pad such weights once where they serve.  A training step copies once, for its backward too.
    A training step that is captured into a HIP graph needs, as any other of torch's, that no
    eager graph of the same leaves is alive.
    """
    code = _act(act)
    _lib.require_cuda(x, w, b, residual)
    from . import ops
    if not _lib.eager(x, w, b, residual):
        return _LinearAct.apply(x, w, b, code, residual)
    return ops._ops._linear_act(x, w, b, code, residual)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``, ``x = q * scale``: float8_e4m3fn of x's sizes and one float32 scale a row of
    its last dimension (at most 16384 values), as :func:`maloq_amd.norm.rms_norm_quantized` makes
    them.  For weights [n, k] once, when they are loaded."""
    _lib.require_cuda(x)
    from . import ops
    with torch.no_grad():
        q, scale = ops.quantize_rows(x)
    return q, scale


def linear_quantized(q: torch.Tensor, scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                     b: torch.Tensor | None = None, act: str = "none", residual: torch.Tensor | None = None,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act((q scale) (wq w_scale)^T + b) + residual`` of type ``dtype`` (float32, bfloat16 or
    float16), which b and residual have too.  q: [..., k] and wq: [n, k] float8_e4m3fn, their
    scales float32, one a row.  k that is no multiple of 16 costs as in :func:`linear_act` (64 rows of 4095 to
    16384 42 us, of 4096 20).  No gradient."""
    code = _act(act)
    _lib.require_cuda(q, scale, wq, w_scale, b, residual)
    from . import ops
    with torch.no_grad():
        return ops.linear_quantized(q, scale, wq, w_scale, b, code, residual, dtype)
