"""Operators between and behind the packed projections of a training or serving step, as cases that can be timed.

    listed()            the cases that stand for the whole range
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the operator in elementary operations, or (own) through metis_hip
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   the outputs from the definition, in 64 bits

The kinds:
    norm    residual_norm: h = x + scale * gate * postnorm(y), n = norm(h); with "grad" also the gradients for given ones of h and n
    swiglu  swiglu: silu(gate) * up, the operands the halves of one product's rows ("split") or two tensors
    loss    token_logprobs: log-probability of each token's target under softmax(hidden weight^T / temperature), and the
            distribution's entropy; with "grad" also the gradients of hidden and weight
"""
import os
import sys

import torch

own = False

_EPS = 1e-6
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    path = os.path.join(os.getcwd(), "fp4-post_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import metis_hip
    return metis_hip


def listed():
    return [
        # behind the attention of one decoded token, 1.5B-class layer: the launch counts
        {"name": "norm_token", "kind": "norm", "seqs": 1, "tokens": 1, "cols": 1536, "residual": "bf16", "branch": "bf16", "post": False, "gate": "", "scale": 1.0, "grad": False},
        # a prompt through a layer with a norm behind its block too and a residual scale, odd length
        {"name": "norm_prompt_post", "kind": "norm", "seqs": 1, "tokens": 4099, "cols": 3584, "residual": "bf16", "branch": "bf16", "post": True, "gate": "", "scale": 0.5, "grad": False},
        # the residual sum and next norm of a 7B-class layer in a training step of 8192 tokens
        {"name": "norm_train", "kind": "norm", "seqs": 2, "tokens": 4096, "cols": 3584, "residual": "bf16", "branch": "bf16", "post": False, "gate": "", "scale": 1.0, "grad": True},
        # binary32 residual stream, a norm behind the block and a gate for each sequence, ragged rows
        {"name": "norm_train_gated", "kind": "norm", "seqs": 3, "tokens": 701, "cols": 4096, "residual": "f32", "branch": "bf16", "post": True, "gate": "seq", "scale": 1.0, "grad": True},
        # five decoded tokens between gate/up and down of a 1.5B-class layer
        {"name": "swiglu_tokens", "kind": "swiglu", "rows": 5, "cols": 8960, "dtype": "bf16", "split": False, "grad": False},
        # the same step of a 7B-class layer in training, the operands halves of one gate/up product
        {"name": "swiglu_train", "kind": "swiglu", "rows": 4096, "cols": 18944, "dtype": "bf16", "split": True, "grad": True},
        # binary32 arithmetic, ragged
        {"name": "swiglu_train_f32", "kind": "swiglu", "rows": 2103, "cols": 8960, "dtype": "f32", "split": False, "grad": True},
        # log-probabilities of the tokens that five sequences have just decoded
        {"name": "loss_tokens", "kind": "loss", "tokens": 5, "hidden": 1536, "vocab": 131072, "temperature": 1.0, "entropy": False, "grad": False},
        # a small head with an odd vocabulary, one ragged sequence in training
        {"name": "loss_train_small", "kind": "loss", "tokens": 411, "hidden": 1536, "vocab": 32003, "temperature": 1.0, "entropy": False, "grad": True},
        # the reference model's scores of a batch of completions: forward alone
        {"name": "loss_score", "kind": "loss", "tokens": 4096, "hidden": 3584, "vocab": 131072, "temperature": 1.0, "entropy": False, "grad": False},
        # a policy step with the entropy bonus at a sampling temperature, few tokens against a large head
        {"name": "loss_train_entropy", "kind": "loss", "tokens": 600, "hidden": 2048, "vocab": 128003, "temperature": 0.8, "entropy": True, "grad": True},
        # a training step of 4096 tokens against the head of a 7B-class model
        {"name": "loss_train", "kind": "loss", "tokens": 4096, "hidden": 3584, "vocab": 131072, "temperature": 1.0, "entropy": False, "grad": True},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random() / step)) * step))


def draw(rng):
    kind = rng.choice(("norm", "norm", "swiglu", "loss", "loss", "loss"))
    grad = rng.random() < 0.6
    if kind == "norm":
        residual, branch = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")))
        return {"kind": kind, "seqs": rng.randint(1, 4), "tokens": _log(rng, 1, 2048), "cols": _log(rng, 256, 8192, 16), "residual": residual, "branch": branch,
                "post": rng.random() < 0.5, "gate": rng.choice(("", "", "channel", "seq")), "scale": rng.choice((1.0, 1.0, 0.5)), "grad": grad}
    if kind == "swiglu":
        return {"kind": kind, "rows": _log(rng, 1, 4096), "cols": _log(rng, 256, 18944, 8), "dtype": rng.choice(("bf16", "bf16", "f32")), "split": rng.random() < 0.5, "grad": grad}
    return {"kind": kind, "tokens": _log(rng, 1, 4096), "hidden": _log(rng, 512, 3584, 16), "vocab": _log(rng, 1000, 131072), "temperature": rng.choice((1.0, 1.0, 0.8)),
            "entropy": rng.random() < 0.4, "grad": grad}


# ---------------------------------------------------------------------------------------------- inputs
class _Source:
    """Values from one seed, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(dtype)

    def activation(self, *shape, dtype=torch.bfloat16):
        """N(0, 1) with 0.1 % of the channels 20 times larger: outlier channels as language models have them."""
        x = torch.randn(*shape, generator=self.g, device="cuda")
        x[..., torch.randperm(shape[-1], generator=self.g, device="cuda")[: max(1, shape[-1] // 1000)]] *= 20.0
        return x.to(dtype)

    def integers(self, high, *shape):
        return torch.randint(high, shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")


def prepare(case, seed):
    src = _Source(seed)
    state = dict(case)
    if case["kind"] == "norm":
        shape, cols = (case["seqs"], case["tokens"], case["cols"]), case["cols"]
        res, br = _DTYPES[case["residual"]], _DTYPES[case["branch"]]
        state.update(x=src.activation(*shape, dtype=res), y=src.normal(*shape, scale=0.5, dtype=br), weight=1 + src.normal(cols, scale=0.1, dtype=br), post_weight=None, gate_vector=None)
        if case["post"]:
            state["post_weight"] = 1 + src.normal(cols, scale=0.1, dtype=br)
        if case["gate"]:
            state["gate_vector"] = src.normal(*((case["seqs"], 1, cols) if case["gate"] == "seq" else (cols,)), scale=0.5, dtype=br)
        if case["grad"]:
            state.update(gh=src.normal(*shape, scale=1e-2, dtype=res), gn=src.normal(*shape, scale=1e-2, dtype=br))
            state["leaves"] = [state[k].requires_grad_() for k in ("x", "y", "weight", "post_weight", "gate_vector") if state[k] is not None]
    elif case["kind"] == "swiglu":
        rows, cols, dt = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        if case["split"]:
            both = src.normal(rows, 2 * cols, scale=1.5, dtype=dt)
            gate, up = both[:, :cols], both[:, cols:]
        else:
            gate, up = src.normal(rows, cols, scale=1.5, dtype=dt), src.normal(rows, cols, scale=1.5, dtype=dt)
        state.update(gate=gate, up=up)
        if case["grad"]:
            state["ga"] = src.normal(rows, cols, scale=1e-2, dtype=dt)
            state["leaves"] = [gate.requires_grad_(), up.requires_grad_()]
    else:
        T, H, V = case["tokens"], case["hidden"], case["vocab"]
        weight = src.normal(V, H, scale=0.02)
        targets = src.integers(V, T)
        # half of the tokens are ones that the model all but expects, the others far from it
        pull = (src.uniform(T, 1) < 0.5).float() * src.uniform(T, 1) * 25.0 / (0.02 * H ** 0.5)
        hidden = (src.normal(T, H, dtype=torch.float32) + pull * weight[targets].float() / 0.02 / H ** 0.5).bfloat16()
        targets = torch.where(src.uniform(T) < 0.1, -100, targets)                       # prompt and padding positions
        state.update(hidden_states=hidden, weight=weight, targets=targets)
        if case["grad"]:
            state["g_logp"] = src.normal(T, scale=1.0 / T, dtype=torch.float32)          # advantages over the number of tokens
            state["g_entropy"] = src.normal(T, scale=0.01 / T, dtype=torch.float32) if case["entropy"] else None
            state["leaves"] = [hidden.requires_grad_(), weight.requires_grad_()]
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _calls(state)
    with torch.no_grad():
        return {"norm": _norm, "swiglu": _swiglu, "loss": _loss}[state["kind"]](state)


def _calls(s):
    m = _package()
    with torch.set_grad_enabled(s["grad"]):
        if s["kind"] == "norm":
            h, n = m.residual_norm(s["x"], s["y"], s["weight"], post_weight=s["post_weight"], gate=s["gate_vector"], residual_scale=s["scale"], eps=_EPS)
            return [h, n] + (list(torch.autograd.grad((h, n), s["leaves"], (s["gh"], s["gn"]))) if s["grad"] else [])
        if s["kind"] == "swiglu":
            a = m.swiglu(s["gate"], s["up"])
            return [a] + (list(torch.autograd.grad(a, s["leaves"], s["ga"])) if s["grad"] else [])
        out = m.token_logprobs(s["hidden_states"], s["weight"], s["targets"], temperature=s["temperature"], entropy=s["entropy"])
        out = list(out) if s["entropy"] else [out]
        if not s["grad"]:
            return out
        given = [s["g_logp"], s["g_entropy"]] if s["entropy"] else [s["g_logp"]]
        return out + list(torch.autograd.grad(out, s["leaves"], given))


def _unit(t):
    """(t / sqrt(mean(t^2) + eps), 1 / sqrt(...)) over the last dimension."""
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + _EPS)
    return t * r, r


def _unit_back(u, hat, r):
    """Gradient through _unit: u is the gradient of its result."""
    return r * (u - hat * (u * hat).mean(-1, keepdim=True))


def _norm(s):
    x, y, w = s["x"].float(), s["y"].float(), s["weight"].float()
    p = None if s["post_weight"] is None else s["post_weight"].float()
    g = None if s["gate_vector"] is None else s["gate_vector"].float()
    if p is not None:
        yh, ry = _unit(y)
        z = yh * p
    else:
        z = y
    factor = s["scale"] if g is None else s["scale"] * g
    h = (x + factor * z).to(s["x"].dtype)
    hh, rh = _unit(h.float())
    out = [h, (hh * w).to(s["y"].dtype)]
    if not s["grad"]:
        return out
    gn = s["gn"].float()
    d = s["gh"].float() + _unit_back(gn * w, hh, rh)
    dz = factor * d
    out += [d.to(s["x"].dtype), (dz if p is None else _unit_back(dz * p, yh, ry)).to(s["y"].dtype), (gn * hh).sum((0, 1)).to(s["weight"].dtype)]
    if p is not None:
        out.append((dz * yh).sum((0, 1)).to(s["post_weight"].dtype))
    if g is not None:
        dg = s["scale"] * d * z
        out.append((dg.sum(1, keepdim=True) if g.dim() == 3 else dg.sum((0, 1))).to(s["gate_vector"].dtype))
    return out


def _swiglu(s):
    g, u = s["gate"].float(), s["up"].float()
    sg = 1 / (1 + torch.exp(-g))
    out = [(g * sg * u).to(s["gate"].dtype)]
    if s["grad"]:
        da = s["ga"].float()
        out += [(da * u * sg * (1 + g * (1 - sg))).to(s["gate"].dtype), (da * g * sg).to(s["up"].dtype)]
    return out


def _loss(s):
    x, w, t = s["hidden_states"].float(), s["weight"].float(), s["targets"]
    live = t != -100
    at = torch.where(live, t, 0).unsqueeze(1)
    logits = x @ w.t()
    if s["temperature"] != 1.0:
        logits = logits / s["temperature"]
    top = logits.amax(1, keepdim=True)
    lse = (top + torch.log(torch.exp(logits - top).sum(1, keepdim=True)))
    out = [torch.where(live, (logits.gather(1, at) - lse).squeeze(1), 0.0)]
    if not (s["grad"] or s["entropy"]):
        return out
    logp = logits.sub_(lse)
    prob = torch.exp(logp)
    ent = None
    if s["entropy"]:
        ent = -(prob * logp).sum(1, keepdim=True)
        out.append(torch.where(live, ent.squeeze(1), 0.0))
    if s["grad"]:
        gl = torch.where(live, s["g_logp"], 0.0).unsqueeze(1)
        if ent is not None:
            d = prob * -(gl + torch.where(live, s["g_entropy"], 0.0).unsqueeze(1) * (logp + ent))
        else:
            d = prob.mul_(-gl)
        d.scatter_add_(1, at, gl)
        if s["temperature"] != 1.0:
            d = d / s["temperature"]
        out += [(d @ w).to(torch.bfloat16), (d.t() @ x).to(torch.bfloat16)]
    return out


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"bf16": 2, "f32": 4}
    if case["kind"] == "norm":
        n, r, b = case["seqs"] * case["tokens"] * case["cols"], size[case["residual"]], size[case["branch"]]
        moved, ops = n * (2 * r + 2 * b), 10 * n
        if case["grad"]:
            # gh, gn and what the forward read; both gradients (they are one tensor where nothing lies between the sum and y)
            same = r == b and not case["post"] and not case["gate"] and case["scale"] == 1.0
            moved, ops = moved + n * (r + b + r + (0 if same else b)), ops + 25 * n
        return {"bytes": moved, "flops": ops}
    if case["kind"] == "swiglu":
        n, b = case["rows"] * case["cols"], size[case["dtype"]]
        return {"bytes": n * b * (6 if case["grad"] else 3), "flops": n * (20 if case["grad"] else 6)}
    T, H, V = case["tokens"], case["hidden"], case["vocab"]
    times = 2 if case["grad"] else 1                                                     # both operands read, and their gradients written
    return {"bytes": times * 2 * (T + V) * H + 12 * T, "flops": (6 if case["grad"] else 2) * T * V * H}


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "norm":
            return _exact_norm(s)
        if case["kind"] == "swiglu":
            g, u = s["gate"].double(), s["up"].double()
            sig = torch.sigmoid(g)
            out = [sig * g * u]
            return out + [s["ga"].double() * u * (sig + g * sig * (1 - sig)), s["ga"].double() * (sig * g)] if case["grad"] else out
        return _exact_loss(s)


def _exact_norm(s):
    def rms(t):
        return (t.square().sum(-1, keepdim=True) / t.shape[-1] + _EPS).sqrt()

    y = s["y"].double()
    gate = torch.ones((), dtype=torch.float64, device="cuda") if s["gate_vector"] is None else s["gate_vector"].double()
    factor = gate * s["scale"]
    ny = rms(y) if s["post"] else None
    z = y / ny * s["post_weight"].double() if s["post"] else y
    total = s["x"].double() + factor * z
    h = total.to(s["x"].dtype).double()                                                  # the residual stream as it is stored
    nh, w = rms(h), s["weight"].double()
    out = [total, h / nh * w]
    if not s["grad"]:
        return out
    cols, gn = h.shape[-1], s["gn"].double()
    dx = s["gh"].double() + gn * w / nh - h * (gn * w * h).sum(-1, keepdim=True) / (cols * nh ** 3)
    dz = dx * factor
    if s["post"]:
        v = dz * s["post_weight"].double()
        out += [dx, v / ny - y * (v * y).sum(-1, keepdim=True) / (cols * ny ** 3)]
    else:
        out += [dx, dz]
    out.append((gn * h / nh).flatten(0, 1).sum(0))
    if s["post"]:
        out.append((dz * y / ny).flatten(0, 1).sum(0))
    if s["gate_vector"] is not None:
        dg = dx * z * s["scale"]
        out.append(dg.sum(1, keepdim=True) if s["gate_vector"].dim() == 3 else dg.flatten(0, 1).sum(0))
    return out


def _exact_loss(s):
    """In slices of the vocabulary, so that 64 bits of a large head fit."""
    x, t = s["hidden_states"].double() / s["temperature"], s["targets"]
    V, step = s["weight"].shape[0], 16384
    live = t >= 0
    lse, dot, hit = torch.full_like(x[:, 0], -torch.inf), torch.zeros_like(x[:, 0]), torch.zeros_like(x[:, 0])
    for v0 in range(0, V, step):
        l = x @ s["weight"][v0:v0 + step].double().t()
        inside = live & (t >= v0) & (t < v0 + l.shape[1])
        hit[inside] = l[inside, t[inside] - v0]
        new = torch.logaddexp(lse, torch.logsumexp(l, 1))
        dot = dot * torch.exp(lse - new) + (torch.exp(l - new[:, None]) * l).sum(1)
        lse = new
    ent = lse - dot
    out = [torch.where(live, hit - lse, 0.0)]
    if s["entropy"]:
        out.append(torch.where(live, ent, 0.0))
    if not s["grad"]:
        return out
    gl = torch.where(live, s["g_logp"].double(), 0.0)
    ge = torch.where(live, s["g_entropy"].double(), 0.0) if s["entropy"] else torch.zeros_like(gl)
    gx, gw = torch.zeros_like(x), torch.empty(V, x.shape[1], dtype=torch.float64, device="cuda")
    for v0 in range(0, V, step):
        w = s["weight"][v0:v0 + step].double()
        lp = x @ w.t() - lse[:, None]
        d = torch.exp(lp) * (-gl[:, None] - ge[:, None] * (lp + ent[:, None]))
        rows = torch.nonzero(live & (t >= v0) & (t < v0 + w.shape[0])).squeeze(1)
        d[rows, t[rows] - v0] += gl[rows]
        gx += d @ w / s["temperature"]
        gw[v0:v0 + step] = d.t() @ x
    return out + [gx, gw]
