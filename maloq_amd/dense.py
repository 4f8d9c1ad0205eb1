"""Linear layers with bias, activation and residual in the product's epilogue, and their 8-bit form.

    y = act(x W^T + b) + residual

``linear_act`` trains (float32, bfloat16, float16; float32 products on the bf16 matrix cores at
fp32 exactness); ``quantize_rows`` and ``linear_quantized`` serve: e4m3 or int8 operands with one fp32
scale a row of x (:func:`maloq_amd.norm.rms_norm_quantized`) and a row of the weight.  e4m3 numbers are within 2^-4 of a
value down to 2^-15 of the row's largest; integers are within 1 / 254 of the row's largest: for rows whose values are of one size.

Products, sums and activations are fp32 and the result is rounded once, but for the sums of int8 products, which are exact, and of e4m3
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
from .norm import ACTIVATIONS


def _act(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


class _LinearAct(torch.autograd.Function):
    """The operators with their gradients where something traces the call; eager calls go through
    the same in C++."""

    @staticmethod
    def forward(ctx, x, w, b, act, residual, packed):
        from . import ops
        ctx.act, ctx.bias, ctx.residual, ctx.packed = act, b is not None, residual is not None, packed
        if packed:
            y, z8, ze, x8, xe = ops.linear_packed_fwd(x, w, b, act, residual, ctx.needs_input_grad[1])
            ctx.save_for_backward(x8, xe, w, z8, ze)
        else:
            y, z = ops.linear_act_fwd(x, w, b, act, residual, True)
            ctx.save_for_backward(x, w, z if act else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        from . import ops
        need = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.bias and ctx.needs_input_grad[2]]
        got = [None] * 3
        if any(need):
            got = (ops.linear_packed_bwd if ctx.packed else ops.linear_act_bwd)(g, *ctx.saved_tensors, ctx.act, *need)
        dx, dw, db = (t if n else None for t, n in zip(got, need))
        return dx, dw, db, None, g if ctx.residual else None, None


def linear_act(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None = None, act: str = "none",
               residual: torch.Tensor | None = None, checkpoint: torch.dtype | None = None) -> torch.Tensor:
    """``act(x w^T + b) + residual``.

    x: [..., k] on the GPU, float32, bfloat16 or float16; w: [n, k], b: [n], residual: [..., n], all
    of x's type; act: "none", "relu", "silu" or "gelu" (by erf).  Differentiable once, in reverse
    mode: vmap, forward mode and the other transforms of torch.func raise.
    Rows of whole 16 bytes (k a multiple of 8, in float32 of 4) are read where they lie.  For other k
    a call without gradients copies x and w to such in each call from 17 rows on (float32: always; 64 rows
    of 4095 to 16384 bfloat16: 78 us, of 4096 27), and up to 16 rows read at odd addresses (one row 63, 22):
    pad such weights once where they serve.  A training step copies once, for its backward too.
    checkpoint: torch.int8 keeps for the backward, instead of x and of the activation's argument z, their
    :func:`pack_rows`: 33/32 of a byte a value.  y is the same (up to 16 rows the order of its sums is another), and so are
    gradients that use neither; others are those of the kept values (each within 2^-7 to 2^-6 of half the largest of
    its 32): dw takes x from them, and dx, dw and db the activation's slope, but for relu's, which stays exact.
    A training step that is captured into a HIP graph needs, as any other of torch's, that no
    eager graph of the same leaves is alive.
    """
    code = _act(act)
    if checkpoint not in (None, torch.int8):
        raise ValueError(f"activations are kept as they are (None) or in 8 bits (torch.int8), not as {checkpoint}")
    _lib.require_cuda(x, w, b, residual)
    from . import ops
    if not _lib.eager(x, w, b, residual):
        return _LinearAct.apply(x, w, b, code, residual, checkpoint is not None)
    return ops._ops._linear_act(x, w, b, code, residual, checkpoint is not None)


def pack_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, e)``: x (float32, bfloat16 or float16) in 8 bits, as :func:`linear_act` keeps activations for its backward.

    Blocks of 32 consecutive values of a row, the last one perhaps shorter: q int8 of x's sizes, e uint8 [.., ceil(n / 32)],
    ``x = q * 2^(e - 133)``.  The step is a power of two, chosen by the block's largest finite value, which becomes 63 to 126
    steps; q is the nearest integer (ties to even).  127 and -127 are infinities, -128 NaN.  No gradient.
    """
    _lib.require_cuda(x)
    from . import ops
    with torch.no_grad():
        q, e = ops.pack_rows(x)
    return q, e


def unpack_rows(q: torch.Tensor, e: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values of :func:`pack_rows`, exact in dtype (float32, bfloat16 or float16), but that those which pass the type's
    range become its largest (in float32 bfloat16's)."""
    _lib.require_cuda(q, e)
    from . import ops
    with torch.no_grad():
        return ops.unpack_rows(q, e, dtype)


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``, ``x = q * scale``: dtype (float8_e4m3fn or int8) of x's sizes and one float32 scale a row of
    its last dimension (at most 16384 values), as :func:`maloq_amd.norm.rms_norm_quantized` makes
    them.  An int8 value is the integer nearest to 127 x / (the row's largest |x|), ties to the even one.
    For weights [n, k] once, when they are loaded."""
    _lib.require_cuda(x)
    from . import ops
    with torch.no_grad():
        q, scale = ops.quantize_rows(x, dtype)
    return q, scale


def linear_quantized(q: torch.Tensor, scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                     b: torch.Tensor | None = None, act: str = "none", residual: torch.Tensor | None = None,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act((q scale) (wq w_scale)^T + b) + residual`` of type ``dtype`` (float32, bfloat16 or
    float16), which b and residual have too.  q: [..., k] and wq: [n, k] both float8_e4m3fn or both int8 (then k is
    at most 131071, and the sums are exact), their scales float32, one a row.  k that is no multiple of 16 costs as in :func:`linear_act` (64 rows of 4095 to
    16384 42 us, of 4096 20).  No gradient."""
    code = _act(act)
    _lib.require_cuda(q, scale, wq, w_scale, b, residual)
    from . import ops
    with torch.no_grad():
        return ops.linear_quantized(q, scale, wq, w_scale, b, code, residual, dtype)
