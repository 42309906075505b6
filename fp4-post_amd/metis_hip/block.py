"""What a decoder layer runs between its packed projections: the residual sum with its norms, the product of gate and up, and the turn of queries and keys.

The reference leaves both to the model: `residual + hidden` and the RMSNorm of src/Metis/models/llama.py:23-31, and
`act_fn(gate_proj(x)) * up_proj(x)` of its MLP, and the rotary embedding between its q / k projections and attention.  Here each is one kernel, forward and backward, in binary32 arithmetic with every
result rounded once; their autograd nodes are compiled (csrc/host_autograd.cpp).
"""
from __future__ import annotations

import inspect
import math

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


class _Rotary(torch.autograd.Function):
    """rotary where a tracer or a transform sees the call, as _ResidualNorm."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, factor):
        ctx.save_for_backward(positions, inv_freq)
        ctx.more = interleaved, factor
        return ops.rotary(q, k, positions, inv_freq, interleaved, factor)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        positions, inv_freq = ctx.saved_tensors
        return (*ops.rotary(grad_q, grad_k, positions, inv_freq, *ctx.more, True), None, None, None, None)


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


def rotary_frequencies(turned: int, base: float = 10000.0, scaling: dict | None = None, *, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, factor) for rotary: the frequencies base^(-2 i / turned), float64 [turned / 2], and what multiplies the turned vectors (1.0, but for
    "yarn").  `scaling` stretches them for contexts beyond the trained length, by its "type" (or "rope_type", as model settings have it):

        "linear"  every frequency divided by "factor"
        "llama3"  frequencies of wavelengths beyond original / low_freq_factor divided by "factor", those below original / high_freq_factor left, between
                  them a mixture, linear in original / wavelength; original = "original_max_position_embeddings"
        "yarn"    the pairs that turn more than "beta_fast" (32) times within the original length left, those that turn less than "beta_slow" (1) times
                  divided by "factor", between them a mixture, linear in the pair's number; the factor of the vectors is "attention_factor", or
                  0.1 log(factor) + 1"""
    if turned <= 0 or turned % 2 or not base > 0.0:
        raise ValueError(f"rotary_frequencies: a positive even number of columns and a positive base, not {turned} and {base}")
    freq = [float(base) ** (-2 * i / turned) for i in range(turned // 2)]
    factor = 1.0
    kind = None if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind not in (None, "default"):
        if kind not in ("linear", "llama3", "yarn"):
            raise ValueError(f"rotary_frequencies: scaling is 'linear', 'llama3' or 'yarn', not {kind!r}")
        need = {"linear": ("factor",), "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
                "yarn": ("factor", "original_max_position_embeddings")}[kind]
        missing = [name for name in need if scaling.get(name) is None]
        if missing:
            raise ValueError(f"rotary_frequencies: {kind!r} needs {', '.join(missing)}")
        stretch = float(scaling["factor"])
        if not stretch >= 1.0:
            raise ValueError(f"rotary_frequencies: a factor of at least 1, not {stretch}")
        if kind == "linear":
            keep = [0.0] * len(freq)
        elif kind == "llama3":
            low, high, original = (float(scaling[name]) for name in need[1:])
            if not high > low:
                raise ValueError(f"rotary_frequencies: high_freq_factor above low_freq_factor, not {high} and {low}")
            keep = [min(max((original * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in freq]
        else:
            original = float(scaling["original_max_position_embeddings"])
            fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

            def pair(turns):                                       # the pair that turns so often within the original length
                return turned * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
            first, last = pair(fast), pair(slow)
            if scaling.get("truncate", True):
                first, last = math.floor(first), math.ceil(last)
            first, last = max(first, 0), min(last, turned - 1)
            last = last + 0.001 if first == last else last
            keep = [1.0 - min(max((i - first) / (last - first), 0.0), 1.0) for i in range(len(freq))]
            given = scaling.get("attention_factor")
            if given is None and (scaling.get("mscale") or scaling.get("mscale_all_dim")):
                raise ValueError("rotary_frequencies: settings with mscale say what they mean by it: attention_factor")
            factor = float(given) if given is not None else (0.1 * math.log(stretch) + 1.0 if stretch > 1.0 else 1.0)
        freq = [f * w + f / stretch * (1.0 - w) for f, w in zip(freq, keep)]
    return torch.tensor(freq, dtype=torch.float64, device=device), factor


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False, factor: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys turned by the angles of their positions:

        (y1, y2) = factor * (x1 cos a - x2 sin a, x2 cos a + x1 sin a),     a = position * inv_freq[i]

    q, k       [..., heads, dim] of one type, bf16 or float32, alike but for their heads (parts of one product's rows are taken as they are); dim even, up to 512
    positions  int64, of the leading sizes of q ([B, S] for [B, S, heads, dim]) or of the last of them ([S], [1, S])
    inv_freq   float32 or float64 [n], n at most dim / 2: the first 2 n columns of each head are turned, the pairs (i, i + n) or, interleaved, (2 i, 2 i + 1);
               the columns behind them are copied.  rotary_frequencies gives it, with `factor`; a model's own buffer is taken too

    The angles are formed in 64 bits.  The results are dense.  Differentiable (once, in reverse) in q and k."""
    factor = float(factor)
    if _transformed():
        if inv_freq.requires_grad:
            raise ValueError("rotary: no gradient of inv_freq")
        return _Rotary.apply(q, k, positions, inv_freq, bool(interleaved), factor)
    out = _lib.host().recorded_rotary(q, k, positions, inv_freq, interleaved, factor, False)
    if out is not None:
        return out
    if inv_freq.requires_grad:                                     # (refused, or positions made dense first)
        raise ValueError("rotary: no gradient of inv_freq")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        ops._check_rotary("rotary", q, k, positions, inv_freq)
        return _lib.host().recorded_rotary(q, k, ops._flat_positions("rotary", positions, q.shape[:-2]), inv_freq, interleaved, factor, True)
    return ops.rotary(q, k, positions, inv_freq, interleaved, factor)


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
