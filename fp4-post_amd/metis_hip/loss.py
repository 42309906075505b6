"""Log-probabilities of tokens under a model's head, and losses on them, without a tensor of logits.

The reference's trainers take them from the logits that the model returns: log_softmax over [tokens, vocabulary] and a gather of the
sampled tokens (its GRPO and DPO entries, src/grpo/grpo.py and src/dpo/dpo.py, through TRL), or cross entropy.  A head of 131072 rows makes
that 2 GB in binary32 for 4096 tokens, several times over with the gradient.  Here the head's product, the softmax and the gather are one
operator on the last hidden states and the head's weight.
"""
from __future__ import annotations

import copy
import inspect
from collections.abc import Mapping

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import ops
from .bitlinear import _transformed


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, temperature, entropy):
        logp, lse, ent, index = ops.head_logprobs(hidden, weight, targets, ignore_index, temperature, entropy)
        ctx.save_for_backward(hidden, weight, targets, lse, ent, index)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return (logp, ent) if entropy else logp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logp, grad_entropy=None):
        if grad_logp is None and grad_entropy is None:
            return (None,) * 6
        hidden, weight, targets, lse, ent, index = ctx.saved_tensors
        gx, gw = ops.head_logprobs_backward(hidden, weight, targets, ctx.temperature, lse, ent, index, grad_logp, grad_entropy, *ctx.needs_input_grad[:2])
        return gx, gw, None, None, None, None


def token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                   entropy: bool = False):
    """log softmax(hidden weight^T / temperature) at each token's target, float32 of targets' shape; with entropy=True also the entropy of each
    token's distribution.

    hidden    bf16 [..., H], the last hidden states (behind the final norm); H a multiple of 16
    weight    bf16 [V, H], the head's weight; any V up to 2^22
    targets   int64 [...]; a token whose target is ignore_index has 0 and no gradient, and its hidden state is not looked at.  Any other
              target outside the vocabulary makes its results NaN.

    Differentiable (once, in reverse) in hidden and weight; the logits are formed in pieces, in both directions, and never kept."""
    if _transformed() or (torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)):
        return _TokenLogprobs.apply(hidden, weight, targets, int(ignore_index), float(temperature), bool(entropy))
    logp, _, ent, _ = ops.head_logprobs(hidden, weight, targets, ignore_index, temperature, entropy)
    return (logp, ent) if entropy else logp


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(hidden weight^T / temperature) with the targets, as torch.nn.functional.cross_entropy on the logits would
    give it ("mean": over the targets that are not ignored; NaN where all are), float32.  Operands as in token_logprobs."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_cross_entropy: reduction is 'mean', 'sum' or 'none', not {reduction!r}")
    loss = -token_logprobs(hidden, weight, targets, temperature=temperature, ignore_index=ignore_index)
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / (targets != ignore_index).sum()


class _Known(nn.Module):
    """A decoder's stand-in that returns `out`: in place of the whole of it and of any module inside; whatever else is asked of it is the decoder's own."""

    def __init__(self, out, decoder):
        super().__init__()
        self.__dict__["__known"] = out, decoder                    # (a name that no decoder's attribute has; not registered as its module)

    def __getattr__(self, name):
        value = getattr(self.__dict__["__known"][1], name)
        return self if isinstance(value, nn.Module) else value

    def forward(self, *args, **kwargs):
        return self.__dict__["__known"][0]


def _with_hidden(out, hidden: torch.Tensor):
    """A decoder's output like `out` that holds these last hidden states, and nothing else where its class can be made of them alone."""
    if isinstance(out, tuple):
        return out._replace(**{out._fields[0]: hidden}) if hasattr(out, "_fields") else (hidden, *out[1:])
    try:
        return type(out)(last_hidden_state=hidden)
    except TypeError:
        other = copy.copy(out)
        other.last_hidden_state = hidden
        return other


@torch.no_grad()
def _logits_are_the_product(model, head, weight: torch.Tensor, out, masked: bool, inputs: dict) -> bool:
    """Whether the model's logits are its last hidden states times the head's weight, with no factor, cap, shift or cut on the way.  Its class's forward is
    asked, on a twin with the model's attributes whose decoder returns known hidden states (as `out`, its output, holds them) and whose head is a small one, on the
    CPU: no setting has to be known by its name.  A model without a forward of its own has nothing to say against it."""
    model = getattr(model, "_orig_mod", model)                     # (compiled)
    kind = type(model)
    if not isinstance(model, nn.Module) or kind.forward is nn.Module.forward:
        return True
    rows, H, V = 3, 2, weight.shape[0]
    try:
        with torch.device("cpu"):
            # a row of zeros (a shift), rows of usual size and beyond any cap; as many columns as the head has
            hidden = torch.cos(torch.arange(rows * H, dtype=torch.float64) ** 2).reshape(1, rows, H) * torch.tensor([0.0, 1e1, 1e5], dtype=torch.float64)[:, None]
            small = nn.Linear(H, V, bias=False, dtype=torch.float64, device="meta")
            small.weight = nn.Parameter(torch.linspace(-1.0, 1.0, V * H, dtype=torch.float64).reshape(V, H), requires_grad=False)
            known = _Known(_with_hidden(out, hidden), model.base_model)
            modules = {name: known if m is model.base_model else small if m is head else m for name, m in model._modules.items()}
            if known not in modules.values() or small not in modules.values():
                return False
            twin = object.__new__(kind)
            twin.__dict__.update(vars(model), _modules=modules)
            given = {"input_ids": torch.zeros(1, rows, dtype=torch.int64), **({"attention_mask": torch.ones(1, rows, dtype=torch.int64)} if masked else {}), **inputs}
            takes = inspect.signature(kind.forward).parameters
            every = any(p.kind is p.VAR_KEYWORD for p in takes.values())
            got = kind.forward(twin, **{name: v for name, v in given.items() if every or name in takes})
            if isinstance(got, tuple):
                got = got[0]
            elif isinstance(got, Mapping):
                got = got.get("logits")
            got = got if isinstance(got, torch.Tensor) else getattr(got, "logits", None)
            want = small(hidden)
            # (a forward that rounds its logits to bf16 returns the product too: half a step of it is 2^-8, and binary32's is lost in that)
            return isinstance(got, torch.Tensor) and got.shape == want.shape and bool(((got - want).abs_().amax(-1) <= 2.0 ** -7 * want.abs().amax(-1)).all())
    except Exception:                                              # (takes its decoder apart, or wants more than a decoder's call)
        return False


def model_token_logprobs(model, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None, labels: torch.Tensor | None = None, *,
                         temperature: float = 1.0, ignore_index: int = -100, entropy: bool = False, **inputs):
    """token_logprobs of a causal language model's next tokens, [B, S - 1] for input_ids [B, S], without its logits: the model's decoder
    (`base_model`) gives the last hidden states, its output embedding's weight is the head.  What a DPO or GRPO step takes of the policy and of the
    reference model.

    labels defaults to input_ids; positions with ignore_index have 0 and no gradient (and are not computed), and so do those that
    attention_mask leaves out: where the token is masked, or the position before it, whose hidden state would predict it (padding on the left: a
    row's first token has nothing to be predicted from).  inputs: further arguments of the decoder.

    Only for models whose logits are that product and nothing more: their own forward is asked each time, on stand-ins of the decoder and the head
    (on the CPU, beside the decoder's work on the device), and models that scale, cap, shift or cut their logits are refused."""
    head = model.get_output_embeddings()
    if getattr(head, "bias", None) is not None:
        raise ValueError("model_token_logprobs: a head without bias")
    config = getattr(model, "config", None)
    if getattr(config, "final_logit_softcapping", None) or any(getattr(config, k, None) not in (None, 1, 1.0) for k in ("logit_scale", "logits_scaling")):
        raise ValueError("model_token_logprobs: a head whose logits are used as they are, not capped or scaled")
    weight = getattr(head, "weight", None)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"model_token_logprobs: an output embedding with one weight [V, H], not {type(head).__name__}")
    if type(head).forward is not nn.Linear.forward or "forward" in vars(head) or head._forward_hooks or head._forward_pre_hooks:
        raise ValueError(f"model_token_logprobs: a plain linear head without hooks, whose forward multiplies by its weight and does nothing else, not {type(head).__name__}")
    out = model.base_model(input_ids=input_ids, attention_mask=attention_mask, **inputs)
    hidden = out[0] if isinstance(out, tuple) else out.last_hidden_state
    if not _logits_are_the_product(model, head, weight, out, attention_mask is not None, inputs):
        raise ValueError(f"model_token_logprobs: {type(model).__name__} does not return its decoder's last hidden states times its head's weight as logits; "
                         "use token_logprobs on the hidden states that its head is given")
    targets = (input_ids if labels is None else labels)[:, 1:]
    if attention_mask is not None:
        targets = targets.masked_fill((attention_mask[:, 1:] == 0) | (attention_mask[:, :-1] == 0), ignore_index)
    return token_logprobs(hidden[:, :-1], weight, targets, temperature=temperature, ignore_index=ignore_index, entropy=entropy)
