"""What a decoder layer runs between its packed projections: the residual sum with its norms, and the product of gate and up.

The reference leaves both to the model: `residual + hidden` and the RMSNorm of src/Metis/models/llama.py:23-31, and
`act_fn(gate_proj(x)) * up_proj(x)` of its MLP.  Here each is one kernel, forward and backward, in binary32 arithmetic with every
result rounded once; their autograd nodes are compiled (csrc/host_autograd.cpp).
"""
from __future__ import annotations

import inspect

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .bitlinear import _transformed


class _ResidualNorm(torch.autograd.Function):
    """residual_norm where a tracer or a transform sees the call: the compiled node (csrc/host_autograd.cpp) would be a constant to the first and is not
    met at all by a tensor that carries a tangent and no requires_grad.  The tracer records this one, the others have its refusal."""

    @staticmethod
    def forward(ctx, x, y, weight, post_weight, gate, scale, eps):
        h, n = ops.residual_norm(x, y, weight, post_weight, gate, scale, eps)
        ctx.save_for_backward(h, y if post_weight is not None or gate is not None else None, weight, post_weight, gate)
        ctx.more = scale, eps, y.dtype
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_n):
        if grad_h is None and grad_n is None:
            return (None,) * 7
        h, y, weight, post_weight, gate = ctx.saved_tensors
        scale, eps, y_dtype = ctx.more
        return (*ops.residual_norm_backward(h, y, weight, post_weight, gate, scale, eps, grad_h, grad_n, y_dtype, ctx.needs_input_grad[:5]), None, None)


class _SwiGLU(torch.autograd.Function):
    """swiglu where a tracer or a transform sees the call, as _ResidualNorm."""

    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        return ops.swiglu(gate, up)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return ops.swiglu_backward(*ctx.saved_tensors, grad)


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, *, post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """The residual stream behind a block and the input of the next one, from one pass:

        h = x + residual_scale * gate * z        z = y, or RMSNorm(y) * post_weight (a norm behind the block)
        n = RMSNorm(h) * weight                  (the norm in front of the next block, or of the head)

    x, y      [..., C] of one shape: the residual stream and the block's output, bf16 or float32 (the stream may be float32 beside a
              bf16 block); C a multiple of 8 up to 8192
    weight, post_weight   [C] in y's type
    gate      in y's type: [C], or x's leading sizes followed by ones ([B, 1, C]: one for each sequence of [B, S, C])

    Returns (h in x's type, n in y's type); n is the norm of h as it is stored.  Differentiable (once, in reverse) in all tensors."""
    scale, eps = float(residual_scale), float(eps)
    if _transformed():
        return _ResidualNorm.apply(x, y, weight, post_weight, gate, scale, eps)
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or weight.requires_grad or (post_weight is not None and post_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        ops._check_residual_norm(x, y, weight, post_weight, gate, y.dtype)
        return _lib.host().recorded_residual_norm(x, y, weight, post_weight, gate, ops.residual_norm_gate_rows(x, gate), scale, eps)
    return ops.residual_norm(x, y, weight, post_weight, gate, scale, eps)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up, the activation of a gated MLP: [..., C] bf16 or float32 of one shape and type, rows of any stride (the halves of
    one product are taken as they are).  The result is dense.  Differentiable (once, in reverse) in both."""
    if _transformed():
        return _SwiGLU.apply(gate, up)
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


# what a module may have registered that its replacement would not run, by nn.Module's names
_REGISTERED = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks", "_state_dict_hooks", "_state_dict_pre_hooks",
               "_load_state_dict_pre_hooks", "_load_state_dict_post_hooks")


@torch.no_grad()
def _is_gated_mlp(mlp: nn.Module) -> bool:
    """Whether the module computes down_proj(silu(gate_proj(x)) * up_proj(x)) of its one argument and holds nothing else that counts.  Its class's
    forward is asked, on a twin with the module's attributes and small projections in 64 bits on the CPU, in training and in evaluation: factors, clamps and
    dropout kept in plain attributes show there, and the module's own projections are not run."""
    kind = type(mlp)
    if (any(t is not None for t in (*mlp._parameters.values(), *mlp._buffers.values())) or any(getattr(mlp, name, None) for name in _REGISTERED)
            or "forward" in vars(mlp) or kind.__call__ is not nn.Module.__call__):
        return False
    try:
        (argument,) = list(inspect.signature(kind.forward).parameters.values())[1:]
        if argument.kind not in (argument.POSITIONAL_ONLY, argument.POSITIONAL_OR_KEYWORD):
            return False
        with torch.device("cpu"):
            small = {}
            for k, (name, n, m) in enumerate((("gate_proj", 4, 6), ("up_proj", 4, 6), ("down_proj", 6, 4))):
                small[name] = nn.Linear(n, m, bias=False, dtype=torch.float64, device="meta").to_empty(device="cpu")
                small[name].weight.copy_(torch.sin(torch.arange(1.0 + 7 * k, 1 + 7 * k + n * m, dtype=torch.float64) ** 2).reshape(m, n))
            # from rows of zeros to rows far beyond any clamp
            scale = torch.tensor([0.0, 1e-2, 1.0, 3e1, 1e3, 1e6], dtype=torch.float64).reshape(1, 6, 1)
            x = torch.cos(torch.arange(48, dtype=torch.float64) ** 2).reshape(2, 6, 4) * scale
            want = small["down_proj"](nn.functional.silu(small["gate_proj"](x)) * small["up_proj"](x))
            twin = object.__new__(kind)
            twin.__dict__.update(vars(mlp), _modules={**mlp._modules, **small})
            for training in (True, False):
                twin.__dict__["training"] = training
                with torch.random.fork_rng(devices=[]):
                    got = kind.forward(twin, x.clone())
                # (a forward that goes through binary32 on its way is the formula too)
                if not isinstance(got, torch.Tensor) or got.shape != want.shape or not bool(((got - want).abs() <= 1e-5 * want.abs().amax(-1, keepdim=True)).all()):
                    return False
    except Exception:                                              # (asks its projections for more than a product, or its caller for more than x)
        return False
    return True


def fuse_gated_mlps(model: nn.Module) -> int:
    """Replace every MLP that holds gate_proj, up_proj and down_proj around a SiLU (`act_fn`) by GatedMLP on the same projections, where that is all
    it does: one with parameters, buffers, hooks or a forward of its own beside them, or whose forward computes anything else, stays as it is.  Returns the number
    replaced."""
    replaced = 0
    for parent in list(model.modules()):
        for name, mlp in list(parent.named_children()):
            parts = dict(mlp.named_children())
            act = getattr(mlp, "act_fn", None)
            silu = isinstance(act, nn.SiLU) or act is nn.functional.silu or type(act).__name__ == "SiLUActivation"
            if isinstance(mlp, GatedMLP) or not silu or not {"gate_proj", "up_proj", "down_proj"} <= parts.keys() <= {"gate_proj", "up_proj", "down_proj", "act_fn"}:
                continue
            if not _is_gated_mlp(mlp):
                continue
            fused = GatedMLP(parts["gate_proj"], parts["up_proj"], parts["down_proj"])
            fused.train(mlp.training)
            setattr(parent, name, fused)
            replaced += 1
    return replaced
