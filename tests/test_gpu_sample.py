"""sample_tokens on the device against its definition in 64 bits: equal tokens.

A token may differ from the definition's only where the random number's goal, or a threshold, lies within the weights' error of a border: weights and sums are accurate to
2^-40 or better, so over the thousands of rows here with some 10^5 borders each that is not to be expected.  Log-probabilities are rounded to binary32 once: half a
step, and 2^-38 of the magnitudes.  With top_k the sum of all weights is formed in binary32: a weight t octaves deep is off by 3 roundings of its argument, 3 t log 2 2^-24,
and by 2^-22 for the exponential, the sums of eight by 2^-21; weighted by the weights themselves t is at most 22 octaves (log2 of 2^22 tokens): 2^-18.3 in all, under 2^-18."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def definition(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens, log-probabilities) in 64 bits; the settings numbers or vectors."""
    rows, V = logits.shape
    def column(s):
        return torch.as_tensor(s, dtype=torch.float64, device=logits.device).expand(rows)[:, None]
    temperature, top_k, top_p, min_p = map(column, (temperature, top_k, top_p, min_p))
    x = logits.double()
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.where(ranked == ranked[:, :1], 1.0, torch.exp((ranked - ranked[:, :1]) / temperature))
    rank = torch.arange(V, device=logits.device)
    keep = (rank < top_k) | (top_k == 0)
    upto = torch.cumsum(torch.where(keep, w, 0.0), 1)
    before = torch.nn.functional.pad(upto[:, :-1], (1, 0))
    keep &= (before < top_p * upto[:, -1:]) | (top_p >= 1.0)
    keep &= w >= min_p
    upto = torch.cumsum(torch.zeros_like(x).scatter_(1, order, torch.where(keep, w, 0.0)), 1)
    tokens = torch.searchsorted(upto, uniforms.double()[:, None] * upto[:, -1:], right=True)
    place = (order == tokens).double().argmax(1, keepdim=True)
    logp = torch.log(w.gather(1, place)) - torch.log(w.sum(1, keepdim=True))
    empty = ranked[:, 0] == -torch.inf                                 # (binary32's lowest number is -inf in bf16)
    return torch.where(empty, -1, tokens[:, 0]), torch.where(empty, torch.nan, logp[:, 0])


def check(logits, uniforms, **settings):
    from metis_hip import sample_tokens
    tokens, logp = sample_tokens(logits, uniforms, **settings)
    rows, V = uniforms.numel(), logits.shape[-1]
    assert tokens.shape == logp.shape == uniforms.shape and tokens.dtype == torch.int64 and logp.dtype == F32
    want, want_logp = definition(logits.reshape(rows, V), uniforms.reshape(rows), **{k: s.reshape(rows) if isinstance(s, torch.Tensor) else s for k, s in settings.items()})
    off = tokens.reshape(rows) != want
    assert not bool(off.any()), (settings, tokens.reshape(rows)[off][:5], want[off][:5], uniforms.reshape(rows)[off][:5])
    k = torch.as_tensor(settings.get("top_k", 0), device=logits.device).double().expand(rows if not isinstance(settings.get("top_k"), torch.Tensor) else uniforms.shape).reshape(rows)
    bound = 2.0 ** -24 * want_logp.abs() + 2.0 ** -38 * (want_logp.abs() + 1 + math.log(V)) + torch.where((k > 0) & (k < V), 2.0 ** -18, 0.0)
    assert bool((((logp.reshape(rows).double() - want_logp).abs() <= bound) | (want_logp.isnan() & logp.reshape(rows).isnan())).all())
    return tokens, logp


def rows_of(seed, rows, V, dtype, spread=2.0, peaks=6):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, V, generator=g)
    if peaks:
        x.scatter_add_(1, torch.randint(V, (rows, peaks), generator=g), 8 * torch.rand(rows, peaks, generator=g))
    return x.to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.7, top_k=300, top_p=0.8, min_p=0.001), dict(top_p=1e-9),
            dict(top_p=0.999999), dict(top_k=7, top_p=0.5), dict(min_p=1.0), dict(temperature=1e-3), dict(temperature=50.0, top_p=0.7), dict(top_k=10 ** 9, top_p=2.0)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V", [(40, 1), (40, 2), (40, 7), (200, 64), (60, 1000), (33, 4096), (20, 32003), (9, 131072)])
def test_against_the_definition(rows, V, dtype):
    logits, u = rows_of(rows + V, rows, V, dtype)
    for settings in SETTINGS:
        check(logits, u, **settings)


def test_the_whole_range_of_the_random_number():
    """One row's distribution under 4097 numbers from 0 to the largest below 1."""
    u = torch.arange(4097, dtype=torch.float32) / 4097
    u[-1] = 1 - 2.0 ** -24
    for dtype, V in ((BF, 501), (F32, 501), (F32, 20001)):
        logits, _ = rows_of(V, 1, V, dtype)
        for settings in (dict(), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.1)):
            tokens, _ = check(logits.expand(4097, V), u.cuda(), **settings)
            assert bool((tokens[1:] >= tokens[:-1]).all())


def test_equal_logits():
    """Ties go to the lower index, however many there are: rows of one value, of two, of a few, with more of them than are sorted at once."""
    for V in (3, 100, 2048, 2049, 5000, 70001):
        g = torch.Generator().manual_seed(V)
        u = torch.rand(16, generator=g).cuda()
        for values in ((0.0,), (1.5, -0.25), (0.0, -0.0), (3.0, 2.9, 2.8, -1.0)):
            logits = torch.tensor(values)[torch.randint(len(values), (16, V), generator=g)].cuda()
            for settings in (dict(), dict(top_k=max(1, V // 3)), dict(top_p=0.37), dict(top_k=max(1, V // 2), top_p=0.61), dict(top_k=2), dict(min_p=0.9)):
                check(logits, u, **settings)
                check(logits.to(BF), u, **settings)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 0.02, 1e4, 1e30])
def test_flat_and_steep_rows(scale):
    """Logits that all lie in one bin (an untrained head's), and such that all but one have no weight left."""
    for V in (300, 40000):
        g = torch.Generator().manual_seed(V)
        logits, u = (scale * torch.randn(8, V, generator=g)).cuda(), torch.rand(8, generator=g).cuda()
        for settings in (dict(), dict(top_k=V // 5), dict(top_p=0.83), dict(top_k=V // 2, top_p=0.5), dict(top_k=2500, top_p=0.9), dict(min_p=0.3)):
            check(logits, u, **settings)
            check(logits.to(BF), u, **settings)


def test_masked_and_infinite_logits():
    from metis_hip import sample_tokens
    inf = float("inf")
    logits, u = rows_of(5, 12, 3001, F32)
    masked = logits.clone()
    masked[:, 100:] = -inf
    masked[1], masked[1, 2999] = -inf, -5.0
    masked[2, :99] = torch.finfo(F32).min
    masked[3] = torch.finfo(F32).min
    for settings in (dict(), dict(top_k=50), dict(top_k=2000), dict(top_p=0.9), dict(min_p=0.01), dict(top_k=500, top_p=0.99)):
        tokens, _ = check(masked, u, **settings)
        assert int(tokens[1]) == 2999 and bool((tokens[[0, *range(4, 12)]] < 100).all())
        check(masked.to(BF), u, **settings)
    some = logits.clone()
    some[:, ::1000] = inf                                              # all the weight, evenly
    tokens, logp = sample_tokens(some, u)
    assert torch.equal(tokens, 1000 * (u * 4).long()) and bool((logp + math.log(4)).abs().max() < 2.0 ** -20)
    tokens, _ = sample_tokens(some, u, top_k=2, top_p=0.9)
    assert torch.equal(tokens, 1000 * (u * 2).long())
    none = logits.clone()
    none[0], none[3, 7], none[5] = -inf, float("nan"), float("nan")
    want = sample_tokens(logits, u, top_p=0.9)
    got = sample_tokens(none, u, top_p=0.9)
    bad = torch.zeros(12, dtype=torch.bool, device="cuda")
    bad[[0, 3, 5]] = True
    assert bool((got[0][bad] == -1).all()) and bool(got[1][bad].isnan().all())
    assert torch.equal(got[0][~bad], want[0][~bad]) and torch.equal(got[1][~bad], want[1][~bad])


def test_settings_for_each_row():
    """Tensors of any number type in any of the settings, numbers beside them; rows with settings or numbers out of range say so and leave the others alone."""
    from metis_hip import sample_tokens
    g = torch.Generator().manual_seed(6)
    logits, u = rows_of(6, 32, 5003, BF)
    t, k, p, m = (0.5 + torch.rand(32, generator=g)).cuda(), torch.randint(0, 60, (32,), generator=g).cuda(), (0.3 + 0.7 * torch.rand(32, generator=g).double()).cuda(), (0.1 * torch.rand(32, generator=g)).cuda()
    check(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check(logits, u, temperature=t)
    check(logits, u, top_k=k.int(), top_p=0.9)
    check(logits, u, top_p=p, min_p=0.01, temperature=0.8)
    whole = sample_tokens(logits, u, temperature=0.5, top_k=40, top_p=0.9, min_p=0.01)
    full = torch.full((32,), 0.5, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(whole, sample_tokens(logits, u, temperature=full, top_k=40, top_p=0.9, min_p=0.01)))
    nan, inf = float("nan"), float("inf")
    for name, bads in (("temperature", (0.0, -1.0, nan, inf)), ("top_k", (-1.0, nan)), ("top_p", (0.0, -0.5, nan)), ("min_p", (-0.1, 1.5, nan))):
        good = {"temperature": 0.5, "top_k": 40.0, "top_p": 0.9, "min_p": 0.01}
        column = torch.full((32,), good[name], dtype=torch.float64, device="cuda")
        column[:len(bads)] = torch.tensor(bads, dtype=torch.float64)
        tokens, logp = sample_tokens(logits, u, **{**good, name: column, "top_k": column if name == "top_k" else 40})
        assert bool((tokens[:len(bads)] == -1).all()) and bool(logp[:len(bads)].isnan().all())
        assert torch.equal(tokens[len(bads):], whole[0][len(bads):]) and torch.equal(logp[len(bads):], whole[1][len(bads):])
    odd = u.clone()
    odd[:4] = torch.tensor([1.0, -1e-9, nan, inf])
    tokens, logp = sample_tokens(logits, odd)
    assert bool((tokens[:4] == -1).all()) and bool(logp[:4].isnan().all()) and torch.equal(tokens[4:], sample_tokens(logits, u)[0][4:])


def test_shapes_strides_and_alignment():
    from metis_hip import sample_tokens
    g = torch.Generator().manual_seed(7)
    for dtype in (BF, F32):
        wide = (3 * torch.randn(6, 1511, generator=g)).to(dtype).cuda()
        u = torch.rand(6, generator=g).cuda()
        for first in (0, 1, 3, 4, 8):
            part = wide[:, first:first + 1499]
            tokens, logp = check(part, u, top_p=0.95)
            dense = sample_tokens(part.contiguous(), u, top_p=0.95)
            assert torch.equal(tokens, dense[0]) and torch.equal(logp, dense[1])
        check(wide[::2], u[::2].contiguous(), top_k=30)
        check(wide.t().contiguous().t(), u, top_k=30)
        check(wide.view(2, 3, 1511), u.view(2, 3), top_p=0.9)
        check(wide.view(2, 3, 1511), u.view(2, 3), top_p=0.9, temperature=(0.5 + u).view(2, 3))
        check(wide[:1].expand(6, 1511), u)
        one = sample_tokens(wide[0], u[0])
        assert one[0].shape == () and int(one[0]) == int(sample_tokens(wide[:1], u[:1])[0])
    empty = sample_tokens(torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda"))
    assert empty[0].shape == (0,) and empty[0].dtype == torch.int64 and empty[1].shape == (0,)


def test_equal_calls_streams_and_graphs():
    """The same inputs give the same bits, on any stream and in replays on changed logits, numbers and settings."""
    from metis_hip import sample_tokens
    logits, u = rows_of(8, 50, 30011, BF)
    t = (0.5 + torch.rand(50, generator=torch.Generator().manual_seed(8))).cuda()
    want = sample_tokens(logits, u, temperature=t, top_k=900, top_p=0.97)
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(sample_tokens(logits, u, temperature=t, top_k=900, top_p=0.97))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for run in got for a, b in zip(run, want))
    held = logits.clone(), u.clone(), t.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(held[0], held[1], temperature=held[2], top_k=900, top_p=0.97)
    for k in range(3):
        new = rows_of(20 + k, 50, 30011, BF)
        held[0].copy_(new[0]), held[1].copy_(new[1]), held[2].add_(0.1)
        graph.replay()
        eager = sample_tokens(held[0], held[1], temperature=held[2], top_k=900, top_p=0.97)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_the_largest_vocabulary():
    logits, u = rows_of(9, 3, 1 << 22, F32)
    for settings in (dict(), dict(top_k=100000, top_p=0.9), dict(top_p=0.5), dict(min_p=0.01)):
        check(logits, u, **settings)
    flat = torch.zeros(2, 1 << 22, device="cuda")
    check(flat, u[:2], top_p=0.6)


def test_beyond_32_bits_of_elements():
    from metis_hip import sample_tokens
    rows = 33000
    logits, _ = rows_of(10, 64, 131072, BF)
    many = logits.repeat(rows // 64 + 1, 1)
    u = torch.rand(many.shape[0], generator=torch.Generator().manual_seed(10)).cuda()
    assert many.numel() > 1 << 32
    u[-64:] = u[:64]
    tokens, logp = sample_tokens(many, u, top_p=0.9)
    assert torch.equal(tokens[-64:], tokens[:64]) and torch.equal(logp[-64:], logp[:64])
    check(logits, u[:64].contiguous(), top_p=0.9)
    del many
    torch.cuda.empty_cache()


def test_refusals():
    from metis_hip import MetisHipError, sample_tokens
    logits, u = rows_of(11, 4, 100, F32)
    for args, more in (((logits.half(), u), {}), ((logits, u.double()), {}), ((logits, u[:3]), {}), ((logits[:, :0], u), {}), ((logits, u), dict(temperature=0.0)), ((logits, u), dict(temperature=-1.0)),
                       ((logits, u), dict(temperature=float("nan"))), ((logits, u), dict(top_k=-1)), ((logits, u), dict(top_p=0.0)), ((logits, u), dict(top_p=float("nan"))),
                       ((logits, u), dict(min_p=1.1)), ((logits, u), dict(min_p=-0.1)), ((logits, u), dict(temperature=u[:3])), ((logits, u), dict(top_p=u.cpu())), ((logits, u.cpu()), {}),
                       ((logits.requires_grad_(), u), {})):
        with pytest.raises(ValueError):
            sample_tokens(*args, **more)
        logits = logits.detach()
    with pytest.raises(MetisHipError, match="no CPU path"):
        sample_tokens(logits.cpu(), u.cpu())
    with torch.no_grad():
        sample_tokens(logits.requires_grad_(), u)


@pytest.mark.parametrize("rows", [5, 70])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_thresholds_at_any_depth(rows, dtype):
    """From a token to most of the vocabulary kept, rows in parts and rows alone: thresholds among a few tokens, some thousands, and where nothing was taken out for them."""
    for spread, peaks in ((0.5, 0), (2.2, 40), (2.2, 3), (4.0, 0)):
        logits, u = rows_of(rows + peaks, rows, 131072, dtype, spread, peaks)
        for settings in [dict(top_p=p) for p in (0.3, 0.9, 0.95, 0.99, 0.9999)] + [dict(top_k=k) for k in (1024, 1025, 2900, 3900, 3901, 50000)] + \
                        [dict(top_k=3000, top_p=0.97), dict(top_k=20000, top_p=0.6), dict(top_p=0.95, min_p=0.01), dict(top_p=0.97, min_p=1e-5), dict(min_p=1e-6), dict(top_p=0.95, temperature=2.0)]:
            check(logits, u, **settings)


@pytest.mark.parametrize("rows", [3, 70])
def test_rows_with_an_order(rows):
    """Vocabularies in order: rising, falling, in steps, the largest logits side by side or at even distances, all of them at one end."""
    g = torch.Generator().manual_seed(rows)
    u = torch.rand(rows, generator=g).cuda()
    for V in (2000, 50021):
        base = torch.sort(2.0 * torch.randn(rows, V, generator=g), 1)[0]
        beside, apart, end = (2.0 * torch.randn(rows, V, generator=g) for _ in range(3))
        for at in (0, 1, V // 2, V // 2 + 1, V // 2 + 2, V - 2, V - 1):
            beside[:, at] += 12
        apart[:, ::V // 30] += 9
        end[:, -300:] += 7
        for x in (base, base.flip(1), (4 * base).round() / 4, beside, apart, end):
            for settings in (dict(), dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.999), dict(top_k=40), dict(top_k=1500), dict(top_k=600, top_p=0.9), dict(top_p=0.9, min_p=0.02)):
                check(x.cuda(), u, **settings)
                check(x.to(BF).cuda(), u, **settings)


def test_a_row_alone_and_among_others():
    """Rows that several workgroups share draw what the same rows draw that have one each."""
    from metis_hip import sample_tokens
    logits, u = rows_of(9, 80, 40009, BF, 2.2, 30)
    for settings in (dict(), dict(top_k=50), dict(top_p=0.95), dict(top_k=4000, top_p=0.9), dict(temperature=0.7, min_p=0.01)):
        tokens, logp = sample_tokens(logits, u, **settings)
        for r in range(0, 80, 9):
            token, lp = sample_tokens(logits[r:r + 1], u[r:r + 1], **settings)
            assert int(token) == int(tokens[r]) and abs(float(lp) - float(logp[r])) <= 2.0 ** -22 * (1 + abs(float(lp))) + (2.0 ** -17 if settings.get("top_k") else 0)


def test_smallest_and_largest_temperatures():
    g = torch.Generator().manual_seed(11)
    u = torch.rand(20, generator=g).cuda()
    for V in (50, 20000):
        x = torch.randn(20, V, generator=g)
        for scale, t in ((1e-35, 1e-35), (1e-30, 3e-31), (1e15, 1e15), (1.0, 2.0 ** 64), (1.0, 1e-300), (3e38, 1e-3)):
            for settings in (dict(), dict(top_k=10), dict(top_k=3000), dict(top_p=0.9), dict(top_k=30, top_p=0.8, min_p=0.05)):
                check((scale * x.clamp(-1, 1)).cuda(), u, temperature=t, **settings)


@pytest.mark.parametrize("rows,V", [(1, 65535), (1, 65536), (31, 70003), (64, 140001), (65, 140001), (2, 1 << 20)])
def test_rows_in_parts(rows, V):
    """Sizes on both sides of those from which several workgroups share a row."""
    for dtype in (BF, F32):
        logits, u = rows_of(V + rows, rows, V, dtype, 2.2, 20)
        for settings in (dict(), dict(top_k=50), dict(top_k=2000, top_p=0.9), dict(top_p=0.95), dict(top_p=0.5, min_p=0.001), dict(top_k=V // 2), dict(temperature=3.0, top_p=0.8)):
            check(logits, u, **settings)


@pytest.mark.parametrize("V", [1023, 1025, 4001, 8177, 8184, 8185, 8192, 8193, 8200])
def test_sizes_around_the_lists(V):
    """Vocabularies on both sides of what is sorted at once and of where every token is a share, at every alignment; thresholds far down, and beyond 64 octaves."""
    for dtype in (BF, F32):
        wide, u = rows_of(V, 20, V + 8, dtype, 2.2, 20)
        for first in (0, 1, 5, 8):
            logits = wide[:, first:first + V]
            for settings in (dict(top_k=20), dict(top_k=V - 1), dict(top_k=V // 2, top_p=0.9), dict(top_p=0.95), dict(top_p=0.9999), dict(temperature=0.05, top_k=V // 2), dict(temperature=0.03, top_p=0.999)):
                check(logits, u, **settings)


def test_more_rows_than_a_launch_takes():
    """A row is a workgroup, and a launch has fewer than 2^32 work-items: 2^22 + 5 rows, with numbers of their own and settings of their own."""
    rows = (1 << 22) + 5
    g = torch.Generator(device="cuda").manual_seed(12)
    logits, u = (2 * torch.randn(rows, 8, generator=g, device="cuda")).to(BF), torch.rand(rows, generator=g, device="cuda")
    check(logits, u, top_p=0.8)
    check(logits, u, temperature=0.5 + torch.rand(rows, generator=g, device="cuda"), top_k=5)


def test_a_token_next_to_min_p():
    """One other token beside a row's largest, 4096 settings of min_p within 2^-41 of its weight and 511 tokens just below them around it: it is kept, or it is not, in
    the sums and in the draw alike, so every row has one of the two.  Depths within 1/64 of half an octave, where an octave is rounded one way or the other."""
    from metis_hip import sample_tokens
    rows = 4096
    for depth in (0.4925, 0.495, 0.4975, 0.4999, 0.5001, 1.496, 3.4993):
        x = torch.tensor(-depth * math.log(2)).item()
        logits = torch.full((rows, 1024), -50.0)
        logits[:, 0], logits[:, 512:], logits[:, 600] = 0.0, x - math.log(2) / 128, x
        weight = math.exp(float(logits[0, 600]))
        min_p = (weight * (1 + torch.arange(-rows // 2, rows // 2, dtype=torch.float64) * 2.0 ** -52)).cuda()
        u = torch.full((rows,), 0.999, device="cuda")
        del_me = [torch.full((rows,), -7, dtype=d, device="cuda") for d in (torch.int64, F32, torch.int64, F32)]
        del del_me                                                      # (what is not written shows)
        tokens, logp = sample_tokens(logits.cuda(), u, min_p=min_p)
        assert bool(((tokens == 0) | (tokens == 600)).all()), tokens[(tokens != 0) & (tokens != 600)][:5]
        assert int(tokens[0]) == 600 and int(tokens[-1]) == 0 and bool((tokens[1:] <= tokens[:-1]).all())
        total = torch.logsumexp(logits[0].double(), 0)
        want = torch.where(tokens == 600, logits[0, 600].double().cuda(), 0.0) - total.cuda()
        assert bool(((logp.double() - want).abs() <= 2.0 ** -22).all())


def test_numbers_next_to_the_borders_of_many_tokens():
    """12000 kept tokens behind a heavy one, together as heavy as it, numbers whose goal lies 2^-42 to 2^-39.5 beside a border: the definition's token.  The weights are good to
    2^-44 and the whole numbers of the sums to 2^-54 apiece, in either direction; 12000 of them cut off would move the borders by 2^-38."""
    rows, V, k = 300, 14000, 12000
    g = torch.Generator().manual_seed(13)
    logits = torch.sort(-8.9 - 0.7 * torch.rand(rows, V, generator=g), 1, descending=True)[0]
    logits[:, 0] = 0.0
    upto = torch.cumsum(torch.exp(logits[:, :k].double()), 1)
    borders, whole = upto[:, 1:3000], upto[:, -1:]
    u = (borders / whole).float()
    off = (u.double() * whole - borders).abs()
    row, at = torch.nonzero((off > 2.0 ** -42) & (off < 2.0 ** -39.5), as_tuple=True)
    assert row.numel() >= 10
    check(logits[row].cuda(), u[row, at].cuda(), top_k=k)
    check(logits[row].cuda(), u[row, at].cuda(), top_k=k, top_p=1 - 1e-12)


def test_nuclei_that_end_between_two_threads_bins():
    """A row of 2^19 tokens in order, whose nucleus is set to every number within 64 steps of the weight down to a border of bins that neighbouring threads add up: two
    roundings of one sum, 2^-45 apart.  The largest number draws the nucleus's last token or the one before it; without a threshold it would draw one of the row's last.
    (The weights in the bins are good to 2^-41.5 each, so the border lies within 64 steps of where it is in 64 bits.)"""
    from metis_hip import sample_tokens
    V, rows = 1 << 19, 128
    x = torch.sort(torch.randn(V, generator=torch.Generator().manual_seed(1)), descending=True)[0].cuda()
    upto = torch.cumsum(torch.exp(x.double() - x[0].double()), 0)
    bins = torch.round((x[0].double() - x.double()) / math.log(2) * 64)
    logits, u = x.expand(rows, V).contiguous(), torch.full((rows,), 1 - 2.0 ** -24, device="cuda")
    for last in (235, 271, 275, 283, 295, 299, 363, 399, 427, 439):
        n = int((bins <= last).sum())
        p = float(upto[n - 1] / upto[-1])
        top_p = (p + torch.arange(-rows // 2, rows // 2, dtype=torch.float64) * math.ulp(p)).cuda()
        tokens, _ = sample_tokens(logits, u, top_p=top_p)
        assert bool(((tokens - n).abs() <= 2).all()), (last, n, tokens[(tokens - n).abs() > 2])


def test_the_same_rows_in_parts_and_alone():
    """80 rows of 131072 tokens have a workgroup each, one of them alone is shared by several: equal tokens, and log-probabilities within the orders of their sums."""
    from metis_hip import _lib, sample_tokens
    V = 131072
    assert _lib.load().metis_sample_tokens_workspace_bytes(80, V) == 0 and _lib.load().metis_sample_tokens_workspace_bytes(1, V) > 0
    for dtype in (BF, F32):
        logits, u = rows_of(21, 80, V, dtype, 2.2, 30)
        for settings in (dict(), dict(top_k=50), dict(top_p=0.95), dict(top_k=4000, top_p=0.9), dict(top_k=60000), dict(top_p=0.999), dict(temperature=0.7, min_p=0.01)):
            tokens, logp = sample_tokens(logits, u, **settings)
            for r in range(0, 80, 9):
                token, lp = sample_tokens(logits[r:r + 1], u[r:r + 1], **settings)
                off = 2.0 ** -23 * (1 + abs(float(lp))) + (2.0 ** -17 if settings.get("top_k") else 0)        # (a rounding each, and with top_k two binary32 sums within 2^-18)
                assert int(token) == int(tokens[r]) and abs(float(lp) - float(logp[r])) <= off


def test_rows_in_parts_side_by_side():
    """Rows that several workgroups share, called again and again on streams and from threads at once, each with a workspace of its own: the same bits, whatever the order in
    which the workgroups take tokens out."""
    import threading
    from metis_hip import _lib, sample_tokens
    calls = []
    for rows, V, settings in ((2, 70001, dict(top_p=0.95)), (2, 70001, dict(top_k=3000, top_p=0.9)), (5, 131072, dict(top_p=0.99)), (1, 262144, dict(top_k=50)), (3, 131072, dict())):
        assert _lib.load().metis_sample_tokens_workspace_bytes(rows, V) > 0
        for dtype in (BF, F32):
            calls.append((*rows_of(V + rows, rows, V, dtype, 2.2, 20), settings))
    want = [sample_tokens(x, u, **settings) for x, u, settings in calls]
    for x, u, settings in calls:
        check(x, u, **settings)
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for x, u, settings in calls:
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(sample_tokens(x, u, **settings))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, run in enumerate(got) for a, b in zip(run, want[i % len(calls)]))
    told, failed = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                told[i] = [[sample_tokens(x, u, **settings) for x, u, settings in calls] for _ in range(5)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                         # (shown by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for mine in told:
        for round_ in mine:
            assert all(torch.equal(a, b) for one, exact in zip(round_, want) for a, b in zip(one, exact))
