"""token_logprobs on the device against its definition in 64 bits.

Tolerances.  A logit is a binary32 sum of H exact products of bf16 values: off by at most H 2^-24 sum |x w| (times 1 / temperature).  With E the largest
such error of a token's logits, log-sum-exp is off by no more than E and what the exponentials, their sums (chains of under 2^9 additions, 2^-15 of a
positive sum) and the logarithm lose: 2^-14 in all, and 2^-21 of the magnitudes that are subtracted.  The entropy moves by at most E sum p |log p + H|.
dl: p is off by a factor of exp of those errors (r below); then one rounding to bf16, half a step (2^-8 of dl), but at the target, whose rounding is made
good to 2^-16 of it (half a step of half a step, bf16 again).  The products' own sums lose at most (number of terms) 2^-24 of the sum of magnitudes, and the
result is rounded to bf16 once.  The same bounds in the 2-norm, where the roundings' part is 2^-8 |dl| |w| with the spectral norm of w: much nearer, and what a
missing or doubled piece cannot meet."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF = 2.0 ** -8


def make(seed, T, H, V, scale=0.0, ignored=0.2, sharp=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=g) * (scale or 0.3 / H ** 0.5 * 4)
    t = torch.randint(V, (T,), generator=g)
    x = torch.randn(T, H, generator=g)
    if sharp:
        x += (torch.rand(T, 1, generator=g) < 0.5).float() * w[t] / w.norm(dim=1).mean() ** 2 * 6
    if T > 2:
        t[0], t[1] = 0, V - 1
    if ignored:
        t = torch.where(torch.rand(T, generator=g) < ignored, -100, t)
    return x.to(BF).cuda(), w.to(BF).cuda(), t.cuda(), torch.randn(T, generator=g).cuda(), (torch.randn(T, generator=g) * 0.3).cuda()


class Exact:
    def __init__(self, x, w, t, temperature, ignore=-100):
        self.x, self.w, self.temp = x.double(), w.double(), temperature
        self.live = t != ignore
        at = torch.where(self.live, t, 0)
        l = self.x @ self.w.t() / temperature
        mag = self.x.abs() @ self.w.abs().t() / temperature
        self.E = (mag.amax(1) * x.shape[-1] * 2.0 ** -24)
        self.lse = torch.logsumexp(l, 1)
        self.lp = l - self.lse[:, None]
        self.p = self.lp.exp()
        self.hit = self.lp.gather(1, at[:, None]).squeeze(1)
        self.ent = -(self.p * self.lp).sum(1)
        self.onehot = torch.zeros_like(l).scatter_(1, at[:, None], 1.0)
        self.tol = 2 * self.E + 2.0 ** -14 + 2.0 ** -21 * (self.lse.abs() + l.abs().amax(1))

    def outputs(self):
        zero = torch.zeros_like(self.lse)
        return torch.where(self.live, self.hit, zero), torch.where(self.live, self.ent, zero)

    def check(self, logp, ent=None):
        hit, H = self.outputs()
        assert bool(((logp.double() - hit).abs() <= self.tol).all()), float(((logp.double() - hit).abs() / self.tol).max())
        assert not bool(logp[~self.live].any())
        if ent is not None:
            tol = self.tol * (1 + (self.p * (self.lp + self.ent[:, None]).abs()).sum(1)) + 2.0 ** -14 * (1 + self.ent)
            assert bool(((ent.double() - H).abs() <= tol).all()), float(((ent.double() - H).abs() / tol).max())

    def check_gradients(self, g, e, gx, gw):
        g = torch.where(self.live, g.double(), 0.0)[:, None]
        e = torch.zeros_like(g) if e is None else torch.where(self.live, e.double(), 0.0)[:, None]
        inside = self.lp + self.ent[:, None]
        d = (g * (self.onehot - self.p) - e * self.p * inside) / self.temp
        r = (torch.expm1(2 * self.tol))[:, None]
        loss = r * self.p * (g.abs() + e.abs() * (inside.abs() + 1)) / self.temp         # before the rounding
        rounded = (HALF * (1 - self.onehot) + HALF ** 2 * self.onehot) * d.abs()
        off = rounded + (1 + HALF) * loss
        for got, left, a, rnd, b, terms in ((gx, d, off, rounded, self.w, self.w.shape[0]), (gw, d.t(), off.t(), rounded.t(), self.x, self.x.shape[0])):
            if got is None:
                continue
            live = b if b is self.w else torch.where(self.live[:, None], b, 0.0)
            want = left @ live
            bound = (a + terms * 2.0 ** -24 * left.abs()) @ live.abs()
            bound = bound + HALF * (want.abs() + bound) + 1e-30
            err = (got.double() - want).abs()
            assert bool((err <= bound).all()), float((err / bound).max())
            norm = torch.linalg.matrix_norm(live, 2)
            most = HALF * want.norm() + rnd.norm() * norm + ((a - rnd).clamp_min(0).norm() + terms * 2.0 ** -24 * left.norm()) * norm * 1.01
            assert float(err.norm()) <= float(most) + 1e-30, float(err.norm() / most)


CASES = [  # tokens, H, V, temperature, entropy
    (1, 16, 1, 1.0, True),
    (1, 16, 2, 1.0, False),
    (2, 32, 255, 1.0, True),
    (5, 64, 257, 0.7, True),
    (64, 48, 300, 1.0, False),
    (65, 80, 1000, 2.0, True),
    (128, 128, 513, 1.0, False),
    (129, 112, 777, 1.0, True),
    (257, 272, 1025, 0.8, True),
    (33, 1536, 5003, 1.0, False),
    (700, 512, 3001, 1.0, True),
    (1030, 784, 2048, 1.0, False),
    (200, 16, 600001, 1.0, False),          # pieces of the vocabulary: 300 032 columns
    (2100, 64, 70001, 1.0, True),           # and of fewer columns, several splits
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_token_logprobs(case):
    from metis_hip import token_logprobs
    T, H, V, temp, entropy = CASES[case]
    x, w, t, g, e = make(200 + case, T, H, V)
    with torch.no_grad():
        plain = token_logprobs(x, w, t, temperature=temp, entropy=entropy)
    x.requires_grad_()
    w.requires_grad_()
    out = token_logprobs(x, w, t, temperature=temp, entropy=entropy)
    out, plain = (out, plain) if entropy else ((out,), (plain,))
    assert all(torch.equal(a, b) and a.dtype == torch.float32 and a.shape == t.shape for a, b in zip(out, plain))
    gx, gw = torch.autograd.grad(out, (x, w), (g, e) if entropy else (g,))
    assert gx.dtype == gw.dtype == BF and gx.shape == x.shape and gw.shape == w.shape
    with torch.no_grad():
        ex = Exact(x, w, t, temp)
        ex.check(*out)
        ex.check_gradients(g, e if entropy else None, gx, gw)
        assert not bool(gx[t == -100].any())


@pytest.mark.parametrize("T", [1, 40, 300, 2500])
def test_the_targets_rounding(T):
    """Nearly all of these gradients comes from dl at the targets, which all but a few tokens share: their roundings would go one way in a row of either.
    In the 2-norm what remains is the results' own rounding, and a bf16 step of the others and of the shared target's remainder."""
    from metis_hip import token_logprobs
    H, V = 528, 20011
    x, w, t, _, _ = make(9, T, H, V, scale=0.05, ignored=0.1 if T > 1 else 0.0, sharp=False)
    t = torch.where((t != -100) & (torch.arange(T, device=t.device) % 7 < 5), 12345, t)
    g = torch.full((T,), 1.003, device="cuda")                 # of bf16's 1 and 1.0078: 0.003 off
    gx, gw = torch.autograd.grad(token_logprobs(x.requires_grad_(), w.requires_grad_(), t), (x, w), g)
    with torch.no_grad():
        ex = Exact(x, w, t, 1.0)
        ex.check_gradients(g, None, gx, gw)
        d = torch.where(ex.live, g.double(), 0.0)[:, None] * (ex.onehot - ex.p)
        # of the rows alone: the share of a gradient along itself, to which independent roundings of its elements (half a step at most, of either sign) add nothing
        # but by chance: six times their root mean square, 2^-8 / 3^0.5 sum(v^4)^0.5 / sum(v^2)
        for got, want in ((gx[ex.live][-1], (d @ ex.w)[ex.live][-1]), (gw[12345], d[:, 12345] @ ex.x)):
            share = float(got.double() @ want / (want @ want)) - 1
            assert abs(share) <= 6 * HALF / 3 ** 0.5 * float((want ** 4).sum().sqrt() / (want @ want)) + 2.0 ** -14, share


@pytest.mark.parametrize("want", ["hidden", "weight"])
@pytest.mark.parametrize("which", ["logp", "entropy"])
def test_one_gradient(want, which):
    from metis_hip import token_logprobs
    x, w, t, g, e = make(1, 300, 96, 1500)
    leaf = (x if want == "hidden" else w).requires_grad_()
    logp, ent = token_logprobs(x, w, t, entropy=True)
    got, = torch.autograd.grad(logp if which == "logp" else ent, leaf, g if which == "logp" else e)
    with torch.no_grad():
        zero = torch.zeros_like(g)
        Exact(x, w, t, 1.0).check_gradients(g if which == "logp" else zero, None if which == "logp" else e, got if want == "hidden" else None, got if want == "weight" else None)


def test_equal_calls_equal_bits():
    from metis_hip import ops
    x, w, t, g, e = make(2, 500, 400, 9001)
    runs = []
    for _ in range(3):
        logp, lse, ent, index = ops.head_logprobs(x, w, t, entropy=True)
        runs.append([logp, lse, ent, *ops.head_logprobs_backward(x, w, t, 1.0, lse, ent, index, g, e)])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
    only = ops.head_logprobs_backward(x, w, t, 1.0, lse, ent, index, g, e, want_hidden=False)
    assert only[0] is None and torch.equal(only[1], runs[0][4])


@pytest.mark.parametrize("T", [7, 90, 400])
def test_ignored_tokens(T):
    """What an ignored token's hidden state holds is not looked at; all ignored, none ignored, another value of the index."""
    from metis_hip import linear_cross_entropy, token_logprobs
    x, w, t, g, _ = make(3, T, 64, 700, ignored=0.5)
    t[0], t[-1] = -100, -100
    clean = x.clone().requires_grad_()
    w.requires_grad_()
    a = token_logprobs(clean, w, t)
    ga = torch.autograd.grad(a, (clean, w), g)
    dirty = x.clone()
    dirty[t == -100] = float("nan")
    dirty[0] = float("inf")
    dirty.requires_grad_()
    b = token_logprobs(dirty, w, t)
    gb = torch.autograd.grad(b, (dirty, w), g)
    assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))
    none = torch.full_like(t, 5)
    c, ent = token_logprobs(dirty, w, none, ignore_index=5, entropy=True)
    gc = torch.autograd.grad((c, ent), (dirty, w), (g, g))
    assert not any(bool(v.any()) for v in (c, ent, *gc))
    assert bool(linear_cross_entropy(dirty, w, none, ignore_index=5).isnan())
    shifted = torch.where(t == -100, 699, torch.where(t == 699, 0, t))
    d = token_logprobs(dirty, w, shifted, ignore_index=699)
    with torch.no_grad():
        Exact(torch.where((shifted == 699)[:, None], 0, x), w, shifted, 1.0, ignore=699).check(d)


def test_targets_outside_of_the_vocabulary_show():
    from metis_hip import token_logprobs
    x, w, t, g, _ = make(4, 70, 32, 300, ignored=0.0)
    good = token_logprobs(x, w, t)
    t[3], t[40], t[69] = 300, -1, 1 << 40
    x.requires_grad_()
    logp, ent = token_logprobs(x, w, t, entropy=True)
    bad = torch.zeros_like(t, dtype=torch.bool)
    bad[[3, 40, 69]] = True
    assert bool(logp[bad].isnan().all()) and bool(ent[bad].isnan().all()) and torch.equal(logp[~bad], good[~bad])
    gx, = torch.autograd.grad(logp, x, g)
    assert bool(gx[bad].isnan().all()) and bool(gx[~bad].isfinite().all())


def test_far_logits():
    """Logits of several thousand: maxima are taken out before the exponential."""
    from metis_hip import token_logprobs
    x, w, t, g, e = make(5, 130, 64, 900, scale=20.0, sharp=False)
    x.requires_grad_()
    w.requires_grad_()
    logp, ent = token_logprobs(x, w, t, entropy=True)
    gx, gw = torch.autograd.grad((logp, ent), (x, w), (g, e))
    with torch.no_grad():
        assert float(logp.min()) < -500 and bool(logp.isfinite().all()) and bool(ent.isfinite().all())
        ex = Exact(x, w, t, 1.0)
        ex.check(logp, ent)
        assert bool(gx.isfinite().all()) and bool(gw.isfinite().all())
    # one infinite and one NaN hidden state: their rows alone
    y = x.detach().clone()
    rows = (t != -100).nonzero().flatten()[:2]
    y[rows[0], 3], y[rows[1], 5] = float("inf"), float("nan")
    z = token_logprobs(y, w, t)
    keep = torch.ones_like(t, dtype=torch.bool)
    keep[rows] = False
    assert bool(z[rows].isnan().all()) and torch.equal(z[keep], logp[keep])


def test_shapes_and_strides():
    from metis_hip import linear_cross_entropy, token_logprobs
    x, w, t, g, _ = make(6, 60, 48, 333)
    want = token_logprobs(x, w, t)
    assert torch.equal(token_logprobs(x.view(3, 20, 48), w, t.view(3, 20)), want.view(3, 20))
    # next-token targets: hidden states but for the last of each sequence, a view
    three = x.view(3, 20, 48)
    assert torch.equal(token_logprobs(three[:, :-1], w, t.view(3, 20)[:, :-1]), want.view(3, 20)[:, :-1])
    wide = torch.randn(60, 72, device="cuda").to(BF)
    wide[:, 8:56] = x
    assert torch.equal(token_logprobs(wide[:, 8:56], w, t), want)
    wide[:, 3:51] = x
    assert torch.equal(token_logprobs(wide[:, 3:51], w, t), want)
    tall = torch.randn(333, 64, device="cuda").to(BF)
    tall[:, :48] = w
    assert torch.equal(token_logprobs(x, tall[:, :48], t), want)
    assert torch.equal(token_logprobs(x.t().contiguous().t(), w.t().contiguous().t(), t), want)
    assert torch.equal(token_logprobs(x[0], w, t[0]), want[0])
    assert token_logprobs(x[:0], w, t[:0]).shape == (0,)
    e = x[:0].clone().requires_grad_()
    w2 = w.clone().requires_grad_()
    ge, gw = torch.autograd.grad(token_logprobs(e, w2, t[:0]).sum(), (e, w2))
    assert ge.shape == (0, 48) and not bool(gw.any())
    # one hidden state for all tokens: the gradient of the expanded input is the sum
    one = x[:1].clone().requires_grad_()
    ga, = torch.autograd.grad(token_logprobs(one.expand(60, 48), w, t), one, g)
    many = x[:1].expand(60, 48).clone().requires_grad_()
    gb, = torch.autograd.grad(token_logprobs(many, w, t), many, g)
    assert torch.equal(ga, gb.sum(0, keepdim=True))
    live = t != -100
    for reduction in ("none", "sum", "mean"):
        loss = linear_cross_entropy(x, w, t, reduction=reduction)
        want_loss = torch.nn.functional.cross_entropy(x.double() @ w.double().t(), t, reduction=reduction)
        assert torch.allclose(loss.double(), want_loss, rtol=0, atol=float(Exact(x, w, t, 1.0).tol.max()) * (float(live.sum()) if reduction == "sum" else 1.0))


def test_refusals():
    from metis_hip import token_logprobs
    x, w, t, _, _ = make(7, 8, 32, 50)
    for bad in (lambda: token_logprobs(x.float(), w, t), lambda: token_logprobs(x, w.float(), t), lambda: token_logprobs(x[:, :16], w, t), lambda: token_logprobs(x, w, t[:4]),
                lambda: token_logprobs(x, w, t.int()), lambda: token_logprobs(x, w, t.cpu()), lambda: token_logprobs(x, w, t, temperature=0.0),
                lambda: token_logprobs(x, w, t, temperature=float("nan")), lambda: token_logprobs(x[:, :24], w[:, :24], t), lambda: token_logprobs(x, w[:0], t),
                lambda: token_logprobs(x, w[0], t)):
        with pytest.raises(ValueError):
            bad()


def test_gradients_against_differences():
    """Along the sign of the gradient, by steps that bf16 holds: the difference of the loss is the sum of |gradient| times the steps, but for half a step of the
    gradient's two roundings (2^-8 of |dl| |w| and of the result: 2^-6 of the sum is allowed, which is several times both at these sizes), a third derivative of
    a logit's move of under 0.05, and binary32's 2^-20 of the terms."""
    from metis_hip import token_logprobs
    x, w, t, g, e = make(8, 40, 32, 50, sharp=False)
    x.requires_grad_()
    w.requires_grad_()

    def loss(x, w):
        logp, ent = token_logprobs(x, w, t, temperature=0.9, entropy=True)
        return float((logp.double() * g.double() + ent.double() * e.double()).sum())

    out = token_logprobs(x, w, t, temperature=0.9, entropy=True)
    grads = torch.autograd.grad(out, (x, w), (g, e))
    with torch.no_grad():
        for k, size in ((0, 2.0 ** -6), (1, 2.0 ** -10)):
            leaf = (x, w)[k]
            step = (grads[k].sign().float() * size)
            up, down = (leaf.float() + step).to(BF), (leaf.float() - step).to(BF)
            diff = loss(*((up, w) if k == 0 else (x, up))) - loss(*((down, w) if k == 0 else (x, down)))
            want = float(((up.double() - down.double()) * grads[k].double()).sum())
            assert want > 0 and abs(diff - want) <= 2.0 ** -6 * want, (k, diff, want)


def test_captured():
    """Forward and backward in a graph, replayed on changed inputs (other tokens ignored too), eager calls between the replays."""
    from metis_hip import ops
    x, w, t, g, e = make(9, 300, 128, 2000)

    def run():
        logp, lse, ent, index = ops.head_logprobs(x, w, t, entropy=True)
        return [logp, lse, ent, *ops.head_logprobs_backward(x, w, t, 1.0, lse, ent, index, g, e)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for k in range(3):
        nx, nw, nt, ng, ne = make(20 + k, 300, 128, 2000, ignored=0.3 * k)
        for a, b in zip((x, w, t, g, e), (nx, nw, nt, ng, ne)):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run())), k
    Exact(x, w, t, 1.0).check(held[0], held[2])


def test_other_streams():
    from metis_hip import ops
    x, w, t, g, e = make(10, 260, 256, 3000)

    def run():
        logp, lse, ent, index = ops.head_logprobs(x, w, t, entropy=True)
        return [logp, ent, *ops.head_logprobs_backward(x, w, t, 1.0, lse, ent, index, g, e)]

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


def test_a_single_row_of_any_stride():
    """One token cut out of a wider row (stride 68, no multiple of eight), and a head of one such row: the bits of dense copies."""
    from metis_hip import token_logprobs
    g = torch.Generator().manual_seed(77)
    wide = torch.randn(4, 68, generator=g).to(BF).cuda()
    heads = torch.randn(300, 64, generator=g).to(BF).cuda(), wide[2:3, :64]
    for x in (wide[:1, :64], wide[:1].view(1, 1, 68)[..., :64]):
        for w in heads:
            t = torch.zeros(x.shape[:-1], dtype=torch.int64, device="cuda")
            results = []
            for change in (lambda v: v, lambda v: v.reshape(-1).clone().view(v.shape)):
                leaves = [change(v.detach()).requires_grad_() for v in (x, w)]
                logp = token_logprobs(*leaves, t)
                results.append([logp.detach(), *torch.autograd.grad(logp.sum(), leaves)])
            assert all(torch.equal(a, b) for a, b in zip(*results))
            # (E = 64 2^-24 sum |x w| < 2^-18 100, two of it and 2^-14: under 1e-3)
            assert abs(float(results[0][0].sum()) - float(torch.log_softmax(x.reshape(-1, 64).double() @ w.double().t(), 1)[0, 0])) < 1e-3


@pytest.mark.parametrize("T,H,V,temp", [(5, 528, 131075, 1.0), (61, 208, 70001, 0.7), (700, 208, 65537, 1.0), (2500, 208, 20003, 0.8)])
def test_several_tiles_to_a_workgroup(T, H, V, temp):
    """More tiles of the logits than workgroups, each of seven stages or more with half a one at the end: the next tile's first stages are under way while the
    statistics of one leave."""
    from metis_hip import token_logprobs
    x, w, t, _, _ = make(T + V, T, H, V)
    with torch.no_grad():
        Exact(x, w, t, temp).check(*token_logprobs(x, w, t, temperature=temp, entropy=True))


def test_recomputed_and_packed_away():
    """Gradients under checkpointing of both kinds, and with the saved tensors kept on the host in between: the bits of those without."""
    from torch.utils.checkpoint import checkpoint
    from metis_hip import token_logprobs
    x, w, t, g, e = make(91, 150, 80, 1001)
    leaves = [x.requires_grad_(), w.requires_grad_()]

    def step(x, w):
        return token_logprobs(x, w, t, temperature=0.8, entropy=True)

    def kept_on_the_host(x, w):
        with torch.autograd.graph.save_on_cpu():
            return step(x, w)

    want = torch.autograd.grad(step(x, w), leaves, (g, e))
    for run in (lambda *a: checkpoint(step, *a, use_reentrant=False), kept_on_the_host):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(run(x, w), leaves, (g, e)), want))
    torch.autograd.backward(checkpoint(step, x, w, use_reentrant=True), (g, e))
    assert all(torch.equal(t.grad, b) for t, b in zip(leaves, want))


@pytest.mark.parametrize("temp", [1.0, 0.5, 2.0])
@pytest.mark.parametrize("T", [7, 90, 2100])
def test_tokens_that_the_model_is_all_but_sure_of(T, temp):
    """Logits far from zero that lie close together, of whole numbers, so that every sum of products is exact: 6144 from what all rows of the head share, and
    twelve signs of each row's own, of which every one that differs from the target's takes 2 s off, s = 3 .. 10.  What is left of 1 - p is 0.03 to 1e-8.

    logp: the target's term and the maximum are the same number, so what is lost is lost in a sum that is a little over one, of at most 64 additions on any
    way (2^-24 each), and its logarithm: 2^-17 in all.  (As the difference of a logit and a log-sum-exp in binary32 it would be off by 2^-24 6144 / temperature, up to 1e-3.)
    dl at the target, g (1 - p): the same 2^-17 of g, and the remainder's rounding; elsewhere a rounding to bf16 and what the log-sum-exp's roundings make of p, three
    of 2^-24 and two constants' of 2^-25 of 6144 / temperature: under 2^-8 of it.  And the products' binary32 sums."""
    from metis_hip import token_logprobs
    g = torch.Generator().manual_seed(T)
    V, H = 1500, 64
    codes = torch.randperm(4096, generator=g)[:V]
    signs = ((codes[:, None] >> torch.arange(12)) & 1) * 2 - 1
    w = torch.cat([torch.full((V, 48), 8.0), signs.float(), torch.zeros(V, 4)], 1).to(BF).cuda()
    t = torch.randint(V, (T,), generator=g)
    s = torch.randint(3, 11, (T, 1), generator=g).float()
    x = torch.cat([torch.full((T, 48), 16.0), s * signs[t], torch.randn(T, 4, generator=g).to(BF).float()], 1).to(BF).cuda()
    t, grad = t.cuda(), torch.randn(T, generator=g).cuda()
    t[::5] = -100
    x.requires_grad_()
    w.requires_grad_()
    logp = token_logprobs(x, w, t, temperature=temp)
    gx, gw = torch.autograd.grad(logp, (x, w), grad)
    with torch.no_grad():
        live, at = t != -100, torch.where(t == -100, 0, t)[:, None]
        l = x.double() @ w.double().t() / temp
        others = torch.exp(l - l.gather(1, at)).scatter_(1, at, 0.0)                      # relative to the target's
        rest = others.sum(1, keepdim=True)
        want = torch.where(live, -torch.log1p(rest).squeeze(1), 0.0)
        assert bool(((logp.double() - want).abs() <= 2.0 ** -17 + 2.0 ** -23 * want.abs()).all()), float((logp.double() - want).abs().max())
        gd = torch.where(live, grad.double(), 0.0)[:, None] / temp
        d = (-gd * others / (1 + rest)).scatter_(1, at, gd * rest / (1 + rest))
        off = ((HALF + 2.0 ** -8) * d.abs()).scatter_(1, at, HALF ** 2 * d.abs().gather(1, at) + 2.0 ** -17 * gd.abs()) + max(T, V) * 2.0 ** -24 * d.abs()
        for got, exact, bound in ((gx, d @ w.double(), off @ w.double().abs()), (gw, d.t() @ x.double(), off.t() @ x.double().abs())):
            bound = bound + HALF * (exact.abs() + bound) + 1e-30
            assert bool(((got.double() - exact).abs() <= bound).all()), float(((got.double() - exact).abs() / bound).max())


def test_hidden_beyond_32_bits_of_elements():
    """2^32 elements of hidden and more, the same 3000 tokens again and again: every repetition has the first one's bits where the sums are the same ones, the
    log-probabilities, and but for the order of binary32 sums those of a call on 3000, hidden's gradient."""
    from metis_hip import ops
    T, H, V, times = 3000, 4096, 300, 350
    assert T * H * times > 1 << 32
    x, w, t, g, _ = make(5, T, H, V)
    many, ts, gs = x.repeat(times, 1), t.repeat(times), g.repeat(times)
    logp, lse, _, index = ops.head_logprobs(many, w, ts)
    gx, gw = ops.head_logprobs_backward(many, w, ts, 1.0, lse, None, index, gs, None)
    first = ops.head_logprobs(x, w, t)
    gx1, gw1 = ops.head_logprobs_backward(x, w, t, 1.0, first[1], None, first[3], g, None)
    assert all(torch.equal(logp[k * T:(k + 1) * T], first[0]) for k in range(times))
    # (dl is the same, its products with the head are sums of 300 terms in one order or another: a step of bf16 where they round apart)
    for k in range(times):
        assert bool(((gx[k * T:(k + 1) * T].float() - gx1.float()).abs() <= 2 * HALF * gx1.float().abs() + 300 * 2.0 ** -24 * (w.float().norm(dim=1).max() * g.abs().max())).all())
    # each element of the weight's gradient is `times` times the small call's, both rounded once and their binary32 sums in between: of a million terms in chains
    # of the tokens' order, sqrt(2^20) 2^-24 of their magnitudes
    scale = float(gw1.double().norm())
    assert float((gw.double() / times - gw1.double()).norm()) <= (2 * HALF + 2.0 ** -14 * 8) * scale
    del many, gx
    torch.cuda.empty_cache()
