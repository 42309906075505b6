"""The rollout's operators together: a group of completions of one prompt, from a cache whose pages they share, with packed and with dense projections."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
EPS = 1e-6


class Layer(nn.Module):
    """A decoder layer: attention of new tokens over a cache, a gated MLP, norms in front of both."""

    def __init__(self, hidden, heads, kv, dim, inter, inv_freq, linear):
        super().__init__()
        from metis_hip import CachedAttention, GatedMLP
        self.attention = CachedAttention(linear(hidden, heads * dim), linear(hidden, kv * dim), linear(hidden, kv * dim), linear(heads * dim, hidden), dim, inv_freq)
        self.mlp = GatedMLP(linear(hidden, inter), linear(hidden, inter), linear(inter, hidden))
        self.norm_mlp, self.norm_next = nn.Parameter(torch.ones(hidden)), nn.Parameter(torch.ones(hidden))

    def forward(self, h, n, attend):
        from metis_hip import residual_norm
        h, n = residual_norm(h, attend(self.attention, n), self.norm_mlp, eps=EPS)
        return residual_norm(h, self.mlp(n), self.norm_next, eps=EPS)


class Model(nn.Module):
    def __init__(self, vocab=515, hidden=256, heads=6, kv=2, dim=64, inter=512, layers=2, linear=lambda k, n: nn.Linear(k, n, bias=False)):
        super().__init__()
        from metis_hip import rotary_frequencies
        inv, _ = rotary_frequencies(dim, 1e4)
        self.embed, self.lm_head = nn.Embedding(vocab, hidden), nn.Linear(hidden, vocab, bias=False)
        self.layers = nn.ModuleList(Layer(hidden, heads, kv, dim, inter, inv, linear) for _ in range(layers))
        self.sizes = heads, kv, dim

    def start(self, tokens):
        h = self.embed(tokens)
        return h, (h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + EPS)).to(h.dtype)

    def prompt(self, tokens, cache, step):
        """The prompt's tokens of one sequence through the layers, their keys and values into the cache."""
        from metis_hip import rotary_append
        heads, kv, dim = self.sizes
        h, n = self.start(tokens)
        for number, layer in enumerate(self.layers):
            def attend(a, n):
                q, k, v = (proj(n).unflatten(-1, (-1, dim)) for proj in (a.q_proj, a.k_proj, a.v_proj))
                q = rotary_append(q, k, v, step.positions, a.inv_freq, step.slots, cache.keys[number], cache.values[number])
                return a.o_proj(plain_attention(q, *read(cache, number, step.tables[0], len(tokens)), causal=True))
            h, n = layer(h, n, attend)
        return self.lm_head(n)

    def decode(self, tokens, cache, step):
        h, n = self.start(tokens)
        for number, layer in enumerate(self.layers):
            h, n = layer(h, n, lambda a, n: a(n, cache, number, step))
        return self.lm_head(n)


def read(cache, number, table, length):
    used = table[:-(-length // cache.page)].long()
    return cache.keys[number, used].transpose(1, 2).flatten(0, 1)[:length], cache.values[number, used].permute(0, 3, 1, 2).flatten(0, 1)[:length]


def plain_attention(q, k, v, causal=False):
    """[tokens, heads, dim] over [length, kv, dim], in binary32."""
    group = q.shape[1] // k.shape[1]
    k, v = (t.float().repeat_interleave(group, 1).transpose(0, 1).contiguous() for t in (k, v))
    s = q.float().transpose(0, 1).contiguous() @ k.transpose(1, 2).contiguous() * q.shape[2] ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool, device=q.device).triu(1), -torch.inf)
    return (torch.softmax(s, -1) @ v).transpose(0, 1).flatten(1).to(BF)


@torch.no_grad()
def rollout(model, cache, prompt, group, steps, uniforms, **settings):
    """(tokens [group, steps], their log-probabilities, the logits that they were drawn from)."""
    from metis_hip import sample_tokens
    (first,) = cache.new()
    logits = model.prompt(prompt, cache, cache.extend([first], [len(prompt)]))[-1:].expand(group, -1)
    seqs = [first, *cache.fork(first, group - 1)]
    out = []
    for k in range(steps):
        tokens, logp = sample_tokens(logits, uniforms[k], **settings)
        out.append((tokens, logp, logits))
        if k + 1 < steps:
            logits = model.decode(tokens, cache, cache.extend(seqs))
    return seqs, [torch.stack(t, 1) for t in zip(*out)]


def test_a_group_of_completions():
    """Tokens of five completions of a prompt that ends inside a page; each completion again from its beginning, as a prompt of its own, has the same logits: two ways
    of some forty bf16 roundings each through two layers, 2^-9 relative to a row's largest logit apiece, in random directions: under 2^-5; and the log-probabilities
    are those of the head's operator on the logits' softmax."""
    from metis_hip import PagedCache
    torch.manual_seed(1)
    model = Model().to(BF).cuda()
    with torch.no_grad():
        model.lm_head.weight.mul_(12)
    prompt = torch.randint(515, (37,)).cuda()
    cache = PagedCache(2, 64, 2, 64)
    uniforms = torch.rand(30, 5).cuda()
    seqs, (tokens, logp, logits) = rollout(model, cache, prompt, 5, 30, uniforms, temperature=0.9, top_p=0.95)
    assert tokens.shape == (5, 30) and len({tuple(t) for t in tokens.tolist()}) == 5
    with torch.no_grad():
        for i in range(5):
            (again,) = cache.new()
            whole = torch.cat((prompt, tokens[i, :-1]))
            want = model.prompt(whole, cache, cache.extend([again], [len(whole)]))[len(prompt) - 1:]
            off = (logits[i].float() - want.float()).abs().amax(1) / want.float().abs().amax(1)
            assert float(off.max()) < 2.0 ** -5, float(off.max())
            for number in range(2):
                # the same tokens' keys and values, from shared pages and from pages of its own
                a, b = ([t.float() for t in read(cache, number, torch.tensor(cache.pages(s)).cuda(), len(whole))] for s in (seqs[i], again))
                for x, y in zip(a, b):
                    assert torch.equal(x[:37], y[:37]) or float((x[:37] - y[:37]).norm() / y[:37].norm()) < 2.0 ** -6
                    assert float((x - y).norm() / y.norm()) < 2.0 ** -6
            cache.free([again])
    exact = torch.log_softmax(logits.double() / 0.9, -1).gather(-1, tokens[..., None])[..., 0]
    assert bool(((logp.double() - exact).abs() <= 2.0 ** -23 * (1 + exact.abs())).all())
    again = rollout(model, cache, prompt, 5, 30, uniforms, temperature=0.9, top_p=0.95)
    assert torch.equal(again[1][0], tokens) and torch.equal(again[1][1], logp)
    cache.free(seqs + again[0])
    assert cache.free_pages == 64


def test_a_cache_made_dense_goes_on():
    """Sequences freed in the middle of a rollout and the pages moved together: the next step's bits are those of a cache that was left as it was."""
    from metis_hip import PagedCache
    torch.manual_seed(2)
    model = Model().to(BF).cuda()
    prompt, new = torch.randint(515, (53,)).cuda(), torch.randint(515, (3,)).cuda()
    got = []
    for dense in (False, True):
        cache = PagedCache(2, 40, 2, 64)
        with torch.no_grad():
            other, first = cache.new(2)
            cache.extend([other], [100])
            model.prompt(prompt, cache, cache.extend([first], [53]))
            seqs = [first, *cache.fork(first, 2)]
            model.decode(new, cache, cache.extend(seqs))
            cache.free([other])
            if dense:
                assert cache.compact() > 0
            got.append(model.decode(new.flip(0), cache, cache.extend(seqs)))
    assert torch.equal(*got)


@pytest.mark.parametrize("dtype", [BF, torch.float8_e4m3fn])
def test_packed_projections(dtype):
    """BitLinear's projections around the cache's attention: the module's result is o_proj of plain attention over what the cache holds, within a bf16 rounding (2^-8)
    of the attention's magnitudes carried through o_proj's quantizer: the same packed operand but where a code tips over, under 2^-4 of the norm."""
    from metis_hip import BitLinear, CachedAttention, MetisArgs, PagedCache, replace_model_with_metis, rotary, rotary_frequencies
    torch.manual_seed(3)
    inv, _ = rotary_frequencies(64, 1e4)
    module = CachedAttention(*(nn.Linear(256, n, bias=False) for n in (384, 128, 128)), nn.Linear(384, 256, bias=False), 64, inv)
    module = replace_model_with_metis(nn.Sequential(module).to(BF).cuda(), MetisArgs.direct_fp4(forward_svd_rank=16))[0]
    assert all(isinstance(p, BitLinear) for p in (module.q_proj, module.k_proj, module.v_proj, module.o_proj))
    cache = PagedCache(1, 64, 2, 64, dtype=dtype, key_scale=0.5 if dtype != BF else 1.0, value_scale=0.25 if dtype != BF else 1.0)
    seqs = cache.new(7)
    with torch.no_grad():
        for k in range(20):
            x = torch.randn(7, 256).to(BF).cuda()
            step = cache.extend(seqs)
            got = module(x, cache, 0, step)
        q, k = (p(x).to(BF).unflatten(-1, (-1, 64)) for p in (module.q_proj, module.k_proj))
        q, _ = rotary(q, k, step.positions, inv.cuda())
        o = []
        for i in range(7):
            keys, values = read(cache, 0, step.tables[i], 20)
            o.append(plain_attention(q[i:i + 1], keys.float() * cache.key_scale, values.float() * cache.value_scale))
        want = module.o_proj(torch.cat(o))
        assert got.shape == (7, 256) and got.dtype == want.dtype
        assert float((got.float() - want.float()).norm() / want.float().norm()) < 2.0 ** -4


def test_a_captured_step():
    """One decode step with its draw, captured once and replayed as a sequence grows: the eager steps' bits."""
    from metis_hip import CacheStep, PagedCache, sample_tokens
    torch.manual_seed(4)
    model = Model().to(BF).cuda()
    prompt = torch.randint(515, (21,)).cuda()
    uniforms = torch.rand(12, 3).cuda()
    wide = 16

    def begin():
        cache = PagedCache(2, 64, 2, 64)
        with torch.no_grad():
            (first,) = cache.new()
            model.prompt(prompt, cache, cache.extend([first], [21]))
        return cache, [first, *cache.fork(first, 2)]

    def padded(step):
        return CacheStep(step.positions, step.slots, torch.nn.functional.pad(step.tables, (0, wide - step.tables.shape[1])).contiguous(), step.lengths)

    def run(tokens, cache, step, u):
        return sample_tokens(model.decode(tokens, cache, step), u, temperature=0.8, top_k=40)

    cache, seqs = begin()
    tokens, want = torch.tensor([1, 2, 3]).cuda(), []
    with torch.no_grad():
        for k in range(12):
            tokens, logp = run(tokens, cache, padded(cache.extend(seqs)), uniforms[k])
            want.append((tokens, logp))
    cache, seqs = begin()
    step, held = padded(cache.extend(seqs)), torch.tensor([1, 2, 3]).cuda()
    u = uniforms[0].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), torch.no_grad():
        run(held, cache, step, u)                                        # (what the libraries set up on first use)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = run(held, cache, step, u)
    for k in range(12):
        if k:
            new = padded(cache.extend(seqs))
            for a, b in zip((step.positions, step.slots, step.tables, step.lengths, held, u), (new.positions, new.slots, new.tables, new.lengths, out[0].clone(), uniforms[k])):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])


def test_traced_calls_and_tangents():
    """What a tracer records runs again on new inputs; forward-mode differentiation is refused."""
    import torch.autograd.forward_ad as fwd
    from metis_hip import paged_attention, rotary_append, rotary_frequencies, sample_tokens
    torch.manual_seed(5)
    inv = rotary_frequencies(64)[0].cuda()
    keys, values = torch.randn(9, 2, 16, 64).to(BF).cuda(), torch.randn(9, 2, 64, 16).to(BF).cuda()
    tables, lengths, slots = torch.arange(8).view(2, 4).int().cuda(), torch.tensor([50, 3]).int().cuda(), torch.tensor([49, 66]).cuda()
    head = torch.randn(101, 256).to(BF).cuda()

    def step(q, k, v, at, u):
        q = rotary_append(q, k, v, at, inv, slots, keys, values)
        o = paged_attention(q, keys, values, tables, lengths)
        return (o, *sample_tokens(o.flatten(1) @ head.t(), u))

    def given():
        return *(torch.randn(2, h, 64).to(BF).cuda() for h in (4, 2, 2)), torch.randint(100, (2,)).cuda(), torch.rand(2).cuda()

    traced = torch.jit.trace(step, given(), check_trace=False)
    for _ in range(2):
        new = given()
        assert all(torch.equal(a, b) for a, b in zip(traced(*new), step(*new)))
    q, k, v, at, u = given()
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: rotary_append(dual, k, v, at, inv, slots, keys, values), lambda: paged_attention(dual, keys, values, tables, lengths),
                     lambda: sample_tokens(fwd.make_dual(torch.zeros(2, 5).cuda(), torch.ones(2, 5).cuda()), u)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()


def test_calls_of_several_threads():
    """Four threads, each on a stream of its own, make the calls of a step at once (the interpreter is given up inside them): the results of one after the other."""
    import threading
    from metis_hip import paged_attention, rotary, rotary_append, rotary_frequencies, sample_tokens
    inv = rotary_frequencies(64)[0].cuda()

    def step(seed, rounds):
        g = torch.Generator().manual_seed(seed)
        q, k, v = (torch.randn(9, h, 64, generator=g).to(BF).cuda() for h in (6, 2, 2))
        keys, values = torch.zeros(20, 2, 16, 64, dtype=BF, device="cuda"), torch.zeros(20, 2, 64, 16, dtype=BF, device="cuda")
        positions, slots = torch.arange(9).cuda(), torch.randperm(160, generator=g)[:9].cuda()
        tables, lengths = torch.arange(20, dtype=torch.int32).reshape(2, 10).cuda(), torch.tensor([160, 33], dtype=torch.int32).cuda()
        logits, u = 3 * torch.randn(70, 5003, generator=g).to(BF).cuda(), torch.rand(70, generator=g).cuda()
        for _ in range(rounds):
            leaf = q.clone().requires_grad_()
            turned, _ = rotary(leaf, k, positions, inv)
            (grad,) = torch.autograd.grad(turned, leaf, q)
            new = rotary_append(q, k, v, positions, inv, slots, keys, values)
            o = paged_attention(new[:2], keys, values, tables, lengths)
            out = [turned.detach(), grad, new, o, *sample_tokens(logits, u, top_p=0.9), *sample_tokens(logits[:2], u[:2], top_k=30)]
        return out

    want = [step(seed, 1) for seed in range(4)]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = step(i, 20)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                         # (shown by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for mine, exact in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(mine, exact))


def test_arguments_of_other_kinds():
    """What the compiled calls leave to Python gives the same: parameters, numbers of other types, tuples of pages, strided and misaligned tensors, positions of a batch."""
    from metis_hip import copy_pages, paged_attention, rotary, rotary_append, rotary_frequencies, sample_tokens
    g = torch.Generator().manual_seed(3)
    inv = rotary_frequencies(64)[0].cuda()
    q, k, v = (torch.randn(4, 5, h, 64, generator=g).to(BF).cuda() for h in (6, 2, 2))
    positions = torch.randint(900, (4, 5), generator=g).cuda()
    want = rotary(q, k, positions, inv)
    with torch.no_grad():
        for args in ((nn.Parameter(q), k, positions, inv), (q, k, positions.t().contiguous().t(), inv), (q.transpose(0, 1).contiguous().transpose(0, 1), k, positions, inv),
                     (torch.cat((q, k), 2)[:, :, :6], torch.cat((q, k), 2)[:, :, 6:], positions, inv), (torch.stack((q, q), -1)[..., 0], k, positions, inv)):
            assert all(torch.equal(a, b) for a, b in zip(rotary(*args), want))
    flat, slots = [t.flatten(0, 1) for t in (q, k, v)], torch.randperm(48, generator=g)[:20].cuda()
    def fresh():
        return torch.zeros(3, 2, 16, 64, dtype=BF, device="cuda"), torch.zeros(3, 2, 64, 16, dtype=BF, device="cuda")
    keys, values = fresh()
    new = rotary_append(*flat, positions.flatten(), inv, slots, keys, values)
    wide = torch.zeros(20, 10, 65, dtype=BF, device="cuda")
    wide[:, :6, 1:], wide[:, 6:8, 1:], wide[:, 8:, 1:] = flat
    for args in ((wide[:, :6, 1:], wide[:, 6:8, 1:], wide[:, 8:, 1:], positions.flatten(), inv, slots), (*flat, positions.flatten(), inv, torch.stack((slots, slots), 1)[:, 0])):
        other = fresh()
        assert torch.equal(rotary_append(*args, *other), new) and torch.equal(other[0], keys) and torch.equal(other[1], values)
    tables, lengths = torch.tensor([[0, 1, 2], [2, 0, 0]], dtype=torch.int32).cuda(), torch.tensor([48, 9], dtype=torch.int32).cuda()
    o = paged_attention(new[:2], keys, values, tables, lengths)
    for args in ((wide[:2, :6, 1:].copy_(new[:2]), keys, values, tables, lengths), (new[:2], keys, values, torch.stack((tables, tables), -1)[..., 0], torch.stack((lengths, lengths), 1)[:, 0])):
        assert torch.equal(paged_attention(*args), o)
    assert torch.equal(paged_attention(new[:2], keys, values, tables, lengths, scale=torch.tensor(0.125)), o)
    pool = [torch.stack((t, t + 1)) for t in (keys, values)]
    moved = [t.clone() for t in pool]
    copy_pages(*moved, [0], [2])
    for sources, destinations in (((0,), (2,)), (torch.tensor([0]), torch.tensor([2]))):
        other = [t.clone() for t in pool]
        copy_pages(*other, sources, destinations)
        assert all(torch.equal(a, b) for a, b in zip(other, moved))
    logits, u = torch.randn(6, 700, generator=g).cuda(), torch.rand(6, generator=g).cuda()
    want = sample_tokens(logits, u, temperature=0.5, top_k=20)
    for settings in (dict(temperature=torch.full((6,), 0.5, device="cuda"), top_k=20), dict(temperature=0.5, top_k=torch.full((6,), 20, device="cuda"))):
        assert all(torch.equal(a, b) for a, b in zip(sample_tokens(logits, u, **settings), want))
    for other in (logits.t().contiguous().t(), torch.cat((logits, logits), 1)[:, :700], torch.cat((logits[:, :1], logits), 1)[:, 1:]):
        assert all(torch.equal(a, b) for a, b in zip(sample_tokens(other, torch.stack((u, u), 1)[:, 0], temperature=0.5, top_k=20), want))


def test_a_captured_draw_from_a_nucleus():
    """Rows in parts and rows alone, captured and replayed on other logits, with eager calls of the same sizes between the replays."""
    from metis_hip import sample_tokens
    g = torch.Generator().manual_seed(4)
    logits = [3 * torch.randn(r, v, generator=g).cuda() for r, v in ((2, 70001), (80, 20011))]
    u = [torch.rand(r, generator=g).cuda() for r in (2, 80)]
    held = [t.clone() for t in logits]
    draws = [sample_tokens(x, n, top_p=0.9) for x, n in zip(held, u)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        draws = [sample_tokens(x, n, top_p=0.9) for x, n in zip(held, u)]
    for turn in range(4):
        for h, x in zip(held, logits):
            h.copy_(x.roll(turn * 7, 1) * (1 + turn / 2))
        graph.replay()
        eager = [sample_tokens(h, n, top_p=0.9) for h, n in zip(held, u)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got, want in zip(draws, eager) for a, b in zip(got, want))
