"""What a decoder layer runs between its packed projections: the residual sum with its norms, and the product of gate and up.

The reference leaves both to the model: `residual + hidden` and the RMSNorm of src/Metis/models/llama.py:23-31, and
`act_fn(gate_proj(x)) * up_proj(x)` of its MLP.  Here each is one kernel, forward and backward, in binary32 arithmetic with every
result rounded once; their autograd nodes are compiled (csrc/host_autograd.cpp).
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, ops


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
    scale, eps = float(residual_scale), float(eps)
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or weight.requires_grad or (post_weight is not None and post_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        ops._check_residual_norm(x, y, weight, post_weight, gate, y.dtype)
        return _lib.host().recorded_residual_norm(x, y, weight, post_weight, gate, ops.residual_norm_gate_rows(x, gate), scale, eps)
    return ops.residual_norm(x, y, weight, post_weight, gate, scale, eps)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up, the activation of a gated MLP: [..., C] bf16 or float32 of one shape and type, rows of any stride (the halves of
    one product are taken as they are).  The result is dense.  Differentiable (once) in both."""
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        ops._check_swiglu(gate, up)
        return _lib.host().recorded_swiglu(gate, up)
    return ops.swiglu(gate, up)


class GatedMLP(nn.Module):
    """A gated MLP with SiLU on its own projections: down_proj(swiglu(gate_proj(x), up_proj(x))).  The projections keep their names, so the
    parameters do too."""

    def __init__(self, gate_proj: nn.Module, up_proj: nn.Module, down_proj: nn.Module):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        gate, up = self.gate_proj(x), self.up_proj(x)
        if gate.is_cuda and gate.dtype == up.dtype and gate.dtype in ops._FLOATS:
            return self.down_proj(swiglu(gate, up))
        return self.down_proj(nn.functional.silu(gate) * up)


def fuse_gated_mlps(model: nn.Module) -> int:
    """Replace every MLP that holds gate_proj, up_proj and down_proj around a SiLU (`act_fn`), and nothing else with parameters, by GatedMLP on
    the same projections.  Returns the number replaced."""
    replaced = 0
    for parent in list(model.modules()):
        for name, mlp in list(parent.named_children()):
            parts = dict(mlp.named_children())
            act = getattr(mlp, "act_fn", None)
            silu = isinstance(act, nn.SiLU) or act is nn.functional.silu or type(act).__name__ == "SiLUActivation"
            if isinstance(mlp, GatedMLP) or not silu or not {"gate_proj", "up_proj", "down_proj"} <= parts.keys() <= {"gate_proj", "up_proj", "down_proj", "act_fn"}:
                continue
            fused = GatedMLP(parts["gate_proj"], parts["up_proj"], parts["down_proj"])
            fused.train(mlp.training)
            setattr(parent, name, fused)
            replaced += 1
    return replaced
