"""What a decoder layer runs between its packed projections: the residual sum with its norms, and the product of gate and up.

The reference leaves both to the model: `residual + hidden` and the RMSNorm of src/Metis/models/llama.py:23-31, and
`act_fn(gate_proj(x)) * up_proj(x)` of its MLP.  Here each is one kernel, forward and backward, in binary32 arithmetic with every
result rounded once.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, post_weight, gate, scale, eps):
        h, n = ops.residual_norm(x, y, weight, post_weight, gate, scale, eps)
        want_gate = gate is not None and ctx.needs_input_grad[4]
        ctx.save_for_backward(h, y if post_weight is not None or want_gate else None, weight, post_weight, gate)
        ctx.scale, ctx.eps, ctx.y_dtype = scale, eps, y.dtype
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_n):
        if grad_h is None and grad_n is None:
            return (None,) * 7
        h, y, weight, post_weight, gate = ctx.saved_tensors
        return (*ops.residual_norm_backward(h, y, weight, post_weight, gate, ctx.scale, ctx.eps, grad_h, grad_n, ctx.y_dtype, ctx.needs_input_grad[:5]), None, None)


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, *, post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """The residual stream behind a block and the input of the next one, from one pass:

        h = x + residual_scale * gate * z        z = y, or RMSNorm(y) * post_weight (a norm behind the block)
        n = RMSNorm(h) * weight                  (the norm in front of the next block, or of the head)

    x, y      [..., C] of one shape: the residual stream and the block's output, bf16 or float32 (the stream may be float32 beside a
              bf16 block); C a multiple of 8 up to 8192
    weight, post_weight   [C] in y's type
    gate      in y's type: [C], or x's leading sizes followed by ones ([B, 1, C]: one for each sequence of [B, S, C])

    Returns (h in x's type, n in y's type); n is the norm of h as it is stored.  Differentiable (once) in all tensors."""
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or weight.requires_grad or (post_weight is not None and post_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        return _ResidualNorm.apply(x, y, weight, post_weight, gate, float(residual_scale), float(eps))
    return ops.residual_norm(x, y, weight, post_weight, gate, float(residual_scale), float(eps))


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        return ops.swiglu(gate, up)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        gate, up = ctx.saved_tensors
        g, u = ops.swiglu_backward(gate, up, grad)
        return g if ctx.needs_input_grad[0] else None, u if ctx.needs_input_grad[1] else None


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up, the activation of a gated MLP: [..., C] bf16 or float32 of one shape and type, rows of any stride (the halves of
    one product are taken as they are).  The result is dense.  Differentiable (once) in both."""
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return _SwiGLU.apply(gate, up)
    return ops.swiglu(gate, up)
