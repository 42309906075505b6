"""residual_norm, swiglu and token_logprobs together, as a training step of a causal language model runs them: behind and between the layers'
projections, and as the loss on the head."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
EPS = 1e-6


class Layer(nn.Module):
    """A block that mixes (in attention's place a projection), and a gated MLP; norms in front of both and behind the MLP."""

    def __init__(self, hidden, inter, linear):
        super().__init__()
        self.mix = linear(hidden, hidden)
        self.gate_proj, self.up_proj, self.down_proj = linear(hidden, inter), linear(hidden, inter), linear(inter, hidden)
        self.norm_mlp = nn.Parameter(torch.ones(hidden))
        self.norm_behind = nn.Parameter(torch.ones(hidden))
        self.gate_vector = nn.Parameter(torch.ones(hidden))
        self.norm_next = nn.Parameter(torch.ones(hidden))

    def forward(self, h, n):
        from metis_hip import residual_norm, swiglu
        h, n = residual_norm(h, self.mix(n), self.norm_mlp, eps=EPS)
        return residual_norm(h, self.down_proj(swiglu(self.gate_proj(n), self.up_proj(n))), self.norm_next, post_weight=self.norm_behind, gate=self.gate_vector,
                             residual_scale=0.5, eps=EPS)

    def plain(self, h, n):
        def norm(t, w):
            return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        h = h + self.mix(n)
        n = norm(h, self.norm_mlp)
        z = self.down_proj(nn.functional.silu(self.gate_proj(n)) * self.up_proj(n))
        h = h + 0.5 * self.gate_vector * norm(z, self.norm_behind)
        return h, norm(h, self.norm_next)


class Decoder(nn.Module):
    def __init__(self, vocab, hidden, inter, layers, linear):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.first = nn.Parameter(torch.ones(hidden))
        self.layers = nn.ModuleList(Layer(hidden, inter, linear) for _ in range(layers))

    def forward(self, input_ids, attention_mask=None, plain=False):
        h = self.embed(input_ids)
        n = (h / (h.float() if not plain else h).square().mean(-1, keepdim=True).add(EPS).sqrt()).to(h.dtype) * self.first
        for layer in self.layers:
            h, n = layer.plain(h, n) if plain else layer(h, n)
        return (n,)


class Model(nn.Module):
    def __init__(self, vocab=515, hidden=128, inter=320, layers=2, linear=lambda k, n: nn.Linear(k, n, bias=False)):
        super().__init__()
        self.base_model = Decoder(vocab, hidden, inter, layers, linear)
        self.lm_head = nn.Linear(hidden, vocab, bias=False)

    def get_output_embeddings(self):
        return self.lm_head


def batch(seed, vocab=515, B=3, S=70):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(vocab, (B, S), generator=g)
    mask = torch.ones(B, S, dtype=torch.int64)
    mask[1, 41:] = 0
    mask[2, 3:] = 0
    return ids.cuda(), mask.cuda(), torch.randn(B, S - 1, generator=g).cuda()


def test_step_against_64_bits():
    """The same parameters in 64 bits.  Relative to the largest value a path multiplies through, each of its roundings to bf16 is at most 2^-8; the longest
    path has 2 for the first norm, 6 in each layer (mix, h and n, gate or up, their product, down, h and n of which two follow each other: 8 counted), the same number
    again backward, and the head's dl and gradient: 2 + 2 * 8 + 2 + 2 * 8 + 2 = 38.  They are independent: sqrt(38) 2^-8 in the 2-norm, and twice that is allowed,
    for the norms and gates, whose derivatives are of about one."""
    import copy
    from metis_hip import model_token_logprobs
    torch.manual_seed(3)
    model = Model()
    for p in model.parameters():
        if p.dim() == 1:
            p.data += 0.1 * torch.randn_like(p)
    model = model.to(BF)
    exact = copy.deepcopy(model).double().cuda()
    model = model.cuda()
    ids, mask, g = batch(4)
    logp = model_token_logprobs(model, ids, mask)
    (logp * g).sum().backward()
    hidden, = exact.base_model(ids, plain=True)
    want = torch.log_softmax(exact.lm_head(hidden[:, :-1]), -1).gather(2, ids[:, 1:, None]).squeeze(2) * mask[:, 1:]
    (want * g.double()).sum().backward()
    most = 2 * 38 ** 0.5 * 2.0 ** -8
    assert float((logp.double() - want).norm() / want.norm()) <= most
    assert not bool(logp[mask[:, 1:] == 0].any())
    for (name, p), (_, q) in zip(model.named_parameters(), exact.named_parameters()):
        assert p.grad is not None and p.grad.dtype == BF
        assert float((p.grad.double() - q.grad).norm() / q.grad.norm()) <= most, name


def test_step_with_packed_projections():
    """The same step on BitLinear projections that share a packed activation: the MLP and the norm module of the package give the bits of the calls that
    they are made of, and every parameter has a finite gradient."""
    from metis_hip import BitLinear, FusedRMSNormQuant, GatedMLP, LinearLowbit, MetisArgs, residual_norm, swiglu
    args = MetisArgs.direct_fp4(forward_svd_rank=32)
    torch.manual_seed(5)

    def layer(k, n):
        made = BitLinear(k, n, args=args, bias=False, dtype=BF, compute_dtype=BF)
        make = dict(args=args, device="cuda", storage_dtype=BF, compute_dtype=BF)
        made.warmup_linear, made.vlinear = LinearLowbit(k, n, bias=False, **make), LinearLowbit(k, 32, bias=False, **make)
        made.ulinear = nn.Linear(32, n, bias=False, device="cuda", dtype=BF)
        made.s = nn.Parameter((5.0 * 0.9 ** torch.arange(32, device="cuda", dtype=torch.float32)).to(BF))
        with torch.no_grad():
            made.warmup_linear.weight.copy_(torch.randn(n, k) * 0.02)
            made.vlinear.weight.copy_(torch.randn(32, k) * k ** -0.5)
            made.ulinear.weight.copy_(torch.randn(n, 32) * n ** -0.5)
        made.is_svd_quant = True
        return made

    mlp = GatedMLP(layer(256, 512), layer(256, 512), layer(512, 256))
    group = {"name": "mlp.gate_up", "mean_cache": {}, "input_ref": None, "quantized_input": None, "members": [mlp.gate_proj, mlp.up_proj]}
    for m in group["members"]:
        m.activation_group = group
    norm = FusedRMSNormQuant(nn.Parameter((1 + 0.1 * torch.randn(256, device="cuda")).to(BF)), EPS, group)
    x, y = torch.randn(2, 160, 256, device="cuda").to(BF), torch.randn(2, 160, 256, device="cuda").to(BF)
    with torch.no_grad():
        h, n = norm(y, x)
        want = residual_norm(x, y, norm.weight, eps=EPS)
        assert torch.equal(h, want[0]) and torch.equal(n, want[1])
        assert torch.equal(mlp(n), mlp.down_proj(swiglu(mlp.gate_proj(n), mlp.up_proj(n))))
    head, t = torch.randn(700, 256, device="cuda").to(BF).requires_grad_(), torch.randint(700, (2, 160), device="cuda")
    from metis_hip import linear_cross_entropy
    x.requires_grad_()
    h, n = norm(y, x)
    h, n = norm(mlp(n), h)
    loss = linear_cross_entropy(n, head, t)
    loss.backward()
    leaves = [x, head, norm.weight, *mlp.parameters()]
    assert bool(loss.isfinite()) and all(p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any()) for p in leaves if p.requires_grad)


def test_mlps_of_a_model_are_replaced():
    """fuse_gated_mlps keeps parameters and names, and the result of the MLP up to the product's roundings: silu, its product and the sums behind them in
    bf16 before, one rounding now; two half steps more on each term of down_proj's sums."""
    from metis_hip import GatedMLP, fuse_gated_mlps

    class Mlp(nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj, self.down_proj = nn.Linear(64, 160, bias=False), nn.Linear(64, 160, bias=False), nn.Linear(160, 64, bias=False)
            self.act_fn = nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))

    class Other(Mlp):
        def __init__(self):
            super().__init__()
            self.act_fn = nn.GELU()

    torch.manual_seed(6)
    model = nn.ModuleDict({"a": nn.ModuleDict({"mlp": Mlp()}), "b": nn.ModuleDict({"mlp": Other()})}).to(BF).cuda()
    names = [n for n, _ in model.named_parameters()]
    x = torch.randn(50, 64, device="cuda").to(BF)
    before = model["a"]["mlp"](x)
    assert fuse_gated_mlps(model) == 1 and fuse_gated_mlps(model) == 0
    assert isinstance(model["a"]["mlp"], GatedMLP) and isinstance(model["b"]["mlp"], Other) and [n for n, _ in model.named_parameters()] == names
    mlp = model["a"]["mlp"]
    after = mlp(x)
    with torch.no_grad():
        terms = (nn.functional.silu(mlp.gate_proj(x).float()) * mlp.up_proj(x).float()).abs() @ mlp.down_proj.weight.float().abs().t()
        assert bool(((after.float() - before.float()).abs() <= 2.0 ** -8 * (4 * terms + 2 * before.float().abs())).all())


def test_padding_on_the_left_reaches_nothing():
    """Hidden states of padding that are NaN, on the left and on the right: the log-probabilities are those of the rows without padding (the same
    products of the same rows, in tiles of other neighbours: a logit is a binary32 sum of 64 products whose magnitudes make less than 8 together, off by at
    most 64 2^-24 8 = 2^-15, and so is the lse; both on two sides: 2^-13), and no gradient is touched."""
    from metis_hip import model_token_logprobs, token_logprobs
    torch.manual_seed(9)
    vocab, H, B, S = 515, 64, 3, 40
    hidden = torch.randn(B, S, H).to(BF).cuda()
    mask = torch.ones(B, S, dtype=torch.int64)
    mask[0, :13] = 0
    mask[1, :39] = 0
    mask[2, 30:] = 0
    mask = mask.cuda()
    ids = torch.randint(vocab, (B, S)).cuda()
    padded = hidden.masked_fill(mask[:, :, None] == 0, float("nan")).requires_grad_()

    class Known(nn.Module):
        def forward(self, input_ids, attention_mask=None):
            return (padded,)

    model = Model(vocab=vocab, hidden=H, inter=64, layers=1).to(BF).cuda()
    model.base_model = Known()
    logp = model_token_logprobs(model, ids, mask)
    logp.sum().backward()
    live = (mask[:, 1:] != 0) & (mask[:, :-1] != 0)
    assert not bool(logp[~live].any()) and bool(logp.isfinite().all())
    for b, (first, end) in enumerate(((13, S), (39, S), (0, 30))):
        assert int(live[b].sum()) == end - first - 1
        with torch.no_grad():
            alone = token_logprobs(hidden[b, first:end - 1], model.lm_head.weight, ids[b, first + 1:end])
        assert bool(((logp[b, first:end - 1] - alone).abs() <= 2.0 ** -13).all())
    assert bool(padded.grad.isfinite().all()) and not bool(padded.grad[:, :-1][~live].any())
    assert bool(model.lm_head.weight.grad.isfinite().all()) and bool(model.lm_head.weight.grad.any())


def test_refusals_of_heads():
    from metis_hip import model_token_logprobs
    model = Model(hidden=64, inter=64, layers=1).to(BF).cuda()
    ids, mask, _ = batch(7, B=3, S=50)
    model.lm_head = nn.Linear(64, 515, bias=True, device="cuda", dtype=BF)
    with pytest.raises(ValueError, match="bias"):
        model_token_logprobs(model, ids, mask)


def test_forward_and_backward_in_a_graph():
    """The three operators with their recorded backward, captured on leaves of their own and replayed on changed values, eager steps on copies between the
    replays; every replay has the eager step's bits."""
    from metis_hip import residual_norm, swiglu, token_logprobs
    gen = torch.Generator().manual_seed(31)

    def values():
        def normal(*shape, scale=1.0):
            return (torch.randn(*shape, generator=gen) * scale).to(BF).cuda()
        x, y, weight, up, head = normal(2, 65, 256), normal(2, 65, 256), 1 + normal(256, scale=0.1), normal(2, 65, 256), normal(1003, 256, scale=0.1)
        targets = torch.randint(1003, (2, 65), generator=gen)
        targets[0, :9] = -100
        return [x, y, weight, up, head], targets.cuda(), torch.randn(2, 65, generator=gen).cuda()

    def step(leaves, targets, g):
        x, y, weight, up, head = leaves
        h, n = residual_norm(x, y, weight)
        logp, ent = token_logprobs(swiglu(n, up) + h, head, targets, entropy=True)
        return [logp.detach(), *torch.autograd.grad((logp, ent), leaves, (g, 0.1 * g))]

    def eager(tensors, targets, g):
        return step([t.detach().clone().requires_grad_() for t in tensors], targets, g)

    tensors, targets, g = values()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager(tensors, targets, g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    leaves = [t.requires_grad_() for t in tensors]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(leaves, targets, g)
    for _ in range(3):
        more, new_targets, new_g = values()
        with torch.no_grad():
            for a, b in zip((*leaves, targets, g), (*more, new_targets, new_g)):
                a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager(leaves, targets, g)))


def test_traced_calls_run_again():
    """What torch.jit.trace records of the three operators runs them on the inputs that it is given: the bits of the calls themselves, values and gradients."""
    from metis_hip import residual_norm, swiglu, token_logprobs
    torch.manual_seed(41)
    weight, post, head = ((1 + 0.1 * torch.randn(256)).to(BF).cuda(), (1 + 0.1 * torch.randn(256)).to(BF).cuda(), torch.randn(515, 256).to(BF).cuda())

    def step(x, y, gate, targets):
        h, n = residual_norm(x, y, weight, post_weight=post, gate=gate, residual_scale=0.5)
        h, n = residual_norm(h, swiglu(n, h), weight)
        logp, ent = token_logprobs(n, head, targets, entropy=True)
        return logp + 0.1 * ent, h

    def values():
        return *(torch.randn(2, n, 256).to(BF).cuda().requires_grad_() for n in (35, 35, 1)), torch.randint(515, (2, 35)).cuda()

    traced = torch.jit.trace(step, values(), check_trace=False)
    for _ in range(2):
        x, y, gate, targets = values()
        results = []
        for run in (traced, step):
            loss, h = run(x, y, gate, targets)
            results.append([loss.detach(), h.detach(), *torch.autograd.grad((loss.sum(), h), (x, y, gate), (torch.ones((), device="cuda"), torch.ones_like(h)))])
        assert all(torch.equal(a, b) for a, b in zip(*results))
    with torch.no_grad():
        traced = torch.jit.trace(step, values(), check_trace=False)
        new = values()
        assert all(torch.equal(a, b) for a, b in zip(traced(*new), step(*new)))


def test_tangents_are_refused_on_the_device():
    """Forward mode meets a refusal, with and without reverse mode beside it, and a level that none of the tensors is part of changes nothing."""
    import torch.autograd.forward_ad as fwd
    from metis_hip import residual_norm, swiglu, token_logprobs
    x, y, head = torch.randn(5, 64).to(BF).cuda(), torch.randn(5, 64).to(BF).cuda(), torch.randn(70, 64).to(BF).cuda()
    w, targets = torch.ones(64, dtype=BF, device="cuda"), torch.randint(70, (5,)).cuda()
    calls = {"norm": lambda x: residual_norm(x, y, w)[1], "gate": lambda x: swiglu(x, y), "loss": lambda x: token_logprobs(x, head, targets)}
    for call in calls.values():
        for leaf in (x, x.clone().requires_grad_()):
            want = call(leaf)
            with fwd.dual_level():
                assert torch.equal(call(leaf), want)
                with pytest.raises(NotImplementedError, match="jvp"):
                    call(fwd.make_dual(leaf, torch.ones_like(leaf)))
