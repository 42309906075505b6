"""The rollout's operators without a device: what is refused, the frequencies, and the cache's books."""
import ctypes
import math
import random

import pytest
import torch

from metis_hip import (CachedAttention, MetisHipError, PagedCache, _lib, copy_pages, paged_attention, rollout, rotary, rotary_append, rotary_frequencies,
                       sample_tokens)

BF = torch.bfloat16


def test_host_tensors_are_refused():
    q, at, inv = torch.zeros(2, 4, 64, dtype=BF), torch.arange(2), torch.ones(32)
    keys, values = torch.zeros(3, 4, 16, 64, dtype=BF), torch.zeros(3, 4, 64, 16, dtype=BF)
    for call in (lambda: rotary(q, q, at, inv), lambda: rotary_append(q, q, q, at, inv, at, keys, values), lambda: paged_attention(q, keys, values, at.int()[:, None], at.int()),
                 lambda: copy_pages(keys[None], values[None], [0], [1]), lambda: sample_tokens(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(MetisHipError, match="no CPU path"):
            call()


# addresses that are never read
ROTARY = dict(q=4096, q_token=256, q_head=64, q_heads=4, k=4096, k_token=128, k_head=64, k_heads=2, positions=4096, npos=8, inv=4096, freq=1, tokens=8, dim=64, turned=64, inter=0,
              back=0, factor=1.0, dtype=0, q_out=4096, k_out=4096, stream=None)


@pytest.mark.parametrize("changes", [dict(tokens=-1), dict(q_heads=-1), dict(k_heads=65537), dict(dim=0), dict(dim=63), dict(dim=514), dict(turned=66), dict(turned=63), dict(turned=-2), dict(dtype=2),
                                     dict(dtype=3), dict(freq=0), dict(freq=3), dict(npos=0), dict(npos=3), dict(positions=None), dict(inv=None), dict(q=None), dict(k_out=None), dict(q=4097),
                                     dict(positions=4100), dict(inv=4098), dict(q_token=-1), dict(k_head=1 << 50), dict(q_token=1 << 44), dict(tokens=1 << 40, npos=1)])
def test_rotary_refuses_before_a_launch(changes):
    assert _lib.load().metis_rotary(*{**ROTARY, **changes}.values()) == _lib.E_ARG


def test_rotary_without_tokens_or_heads():
    L = _lib.load()
    assert L.metis_rotary(*{**ROTARY, "tokens": 0, "q": None}.values()) == _lib.OK
    assert L.metis_rotary(*{**ROTARY, "q_heads": 0, "k_heads": 0, "q": None, "k": None}.values()) == _lib.OK


APPEND = dict(q=4096, q_token=256, q_head=64, q_heads=4, k=4096, k_token=128, k_head=64, kv_heads=2, v=4096, v_token=128, v_head=64, positions=4096, inv=4096, freq=1, slots=4096, tokens=8,
              dim=64, turned=64, inter=0, factor=1.0, pages=4, page=16, cache=0, key_scale=1.0, value_scale=1.0, keys=4096, values=4096, q_out=4096, stream=None)


@pytest.mark.parametrize("changes", [dict(pages=0), dict(page=0), dict(page=4097), dict(cache=1), dict(cache=4), dict(key_scale=0.0), dict(value_scale=-1.0), dict(key_scale=float("nan")),
                                     dict(keys=None), dict(values=None), dict(v=None), dict(slots=None), dict(slots=4100), dict(kv_heads=0), dict(v=4097), dict(pages=1 << 44),
                                     dict(v_token=1 << 45)])
def test_append_refuses_before_a_launch(changes):
    assert _lib.load().metis_rotary_append(*{**APPEND, **changes}.values()) == _lib.E_ARG


ATTEND = dict(q=4096, q_seq=256, q_head=64, seqs=3, heads=4, kv=2, dim=64, keys=4096, values=4096, pages=9, page=16, cache=0, tables=4096, stride=4, width=4, lengths=4096, scale=0.1,
              key_scale=1.0, value_scale=1.0, out=4096, workspace=4096, bytes=1 << 20, stream=None)


@pytest.mark.parametrize("changes", [dict(seqs=-1), dict(heads=0), dict(kv=0), dict(kv=3), dict(dim=48), dict(dim=288), dict(dim=32, cache=3), dict(page=8), dict(page=24), dict(page=8192),
                                     dict(cache=1), dict(pages=-1), dict(pages=0), dict(width=-1), dict(q=None), dict(q=4104), dict(q_seq=257), dict(q_head=63), dict(keys=None), dict(values=4104),
                                     dict(tables=None), dict(tables=4098), dict(lengths=None), dict(lengths=4097), dict(out=None), dict(width=1 << 28), dict(stride=-1)])
def test_attention_refuses_before_a_launch(changes):
    assert _lib.load().metis_paged_attention(*{**ATTEND, **changes}.values()) == _lib.E_ARG


def test_attention_wants_its_workspace():
    L = _lib.load()
    long = {**ATTEND, "width": 4096}
    need = L.metis_paged_attention_workspace_bytes(3, 4, 2, 64, 4096 * 16)
    assert need >= 3 * 4 * 2 * (64 + 2) * 4 and L.metis_paged_attention_workspace_bytes(3, 4, 2, 64, 256) == 16
    for changes in (dict(workspace=None), dict(workspace=4100), dict(bytes=need - 1)):
        assert L.metis_paged_attention(*{**long, "bytes": need, **changes}.values()) == _lib.E_WORKSPACE
    for odd in ((0, 4, 2, 64, 4096), (3, 5, 2, 64, 4096), (3, 4, 0, 64, 4096), (3, 4, 2, 64, 0), (3, 4, 2, 64, 1 << 40), (-1, -4, -2, -64, -1)):
        assert L.metis_paged_attention_workspace_bytes(*odd) == 16


def test_copies_refuse_before_a_launch():
    L = _lib.load()

    def call(sources, destinations, keys=4096, values=4096, layers=2, pages=8, size=4096):
        a, b = ((ctypes.c_int64 * len(s))(*s) for s in (sources, destinations))
        return L.metis_cache_copy_pages(keys, values, layers, pages, size, ctypes.cast(a, ctypes.c_void_p), ctypes.cast(b, ctypes.c_void_p), len(sources), None)

    for args in (([0], [8]), ([-1], [1]), ([8], [1]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([4], [4]), ([0] * 9, list(range(9)))):
        assert call(*args) == _lib.E_ARG
    for more in (dict(keys=None), dict(values=4100), dict(layers=-1), dict(pages=-1), dict(size=0), dict(size=24), dict(size=1 << 32)):
        assert call([0], [1], **more) == _lib.E_ARG
    assert call([], []) == _lib.OK and call([0], [1], layers=0) == _lib.OK
    assert L.metis_cache_copy_pages(4096, 4096, 2, 8, 4096, None, None, 1, None) == _lib.E_ARG


def test_sampling_refuses_before_a_launch():
    L = _lib.load()

    def call(parameters=(1.0, 0.0, 1.0, 0.0), logits=4096, ld=100, dtype=1, rows=4, vocab=100, uniforms=4096, each=None, tokens=4096, logprobs=4096, workspace=4096, size=1 << 24):
        p = None if parameters is None else ctypes.cast((ctypes.c_double * 4)(*parameters), ctypes.c_void_p)
        return L.metis_sample_tokens(logits, ld, dtype, rows, vocab, uniforms, p, each, tokens, logprobs, workspace, size, None)

    nan = float("nan")
    for more in (dict(logits=None), dict(logits=4098), dict(ld=99), dict(ld=-1), dict(dtype=2), dict(rows=-1), dict(rows=1 << 32), dict(vocab=0), dict(vocab=(1 << 22) + 1, ld=1 << 23), dict(uniforms=None),
                 dict(uniforms=4098), dict(tokens=None), dict(tokens=4100), dict(logprobs=None), dict(parameters=None), dict(each=4100), dict(parameters=(0.0, 0, 1, 0)),
                 dict(parameters=(nan, 0, 1, 0)), dict(parameters=(float("inf"), 0, 1, 0)), dict(parameters=(1, -1, 1, 0)), dict(parameters=(1, nan, 1, 0)), dict(parameters=(1, 0, 0, 0)),
                 dict(parameters=(1, 0, nan, 0)), dict(parameters=(1, 0, 1, 1.5)), dict(parameters=(1, 0, 1, nan))):
        assert call(**more) == _lib.E_ARG
    assert call(rows=0, logits=None) == _lib.OK


def test_frequencies():
    inv, factor = rotary_frequencies(128, 1e6)
    assert factor == 1.0 and inv.dtype == torch.float64 and torch.equal(rotary_frequencies(128, 1e6, {"rope_type": "default"})[0], inv)
    assert torch.allclose(inv, 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64), rtol=1e-14, atol=0)
    assert torch.allclose(rotary_frequencies(128, 1e6, {"type": "linear", "factor": 4.0})[0], inv / 4, rtol=1e-14, atol=0)


def test_frequencies_by_wavelength():
    """Each of the three ranges, from the definition by wavelengths."""
    scaling = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    inv, _ = rotary_frequencies(128, 500000.0)
    got, factor = rotary_frequencies(128, 500000.0, scaling)
    seen = set()
    for f, g in zip(inv.tolist(), got.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4:
            want, kind = f, "kept"
        elif wave > 8192 / 1:
            want, kind = f / 8, "stretched"
        else:
            smooth = (8192 / wave - 1) / (4 - 1)
            want, kind = (1 - smooth) * f / 8 + smooth * f, "between"
        seen.add(kind)
        assert abs(g - want) <= 1e-14 * f
    assert len(seen) == 3 and factor == 1.0


def test_frequencies_by_turns():
    """Pairs that turn often in the original length stay, those that turn less than once are stretched, a line between them; the vectors' factor."""
    scaling = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    inv, _ = rotary_frequencies(128, 1e6)
    got, factor = rotary_frequencies(128, 1e6, scaling)
    assert abs(factor - (0.1 * math.log(4.0) + 1)) < 1e-15
    turns = 32768 * inv / (2 * math.pi)
    kept = ((got / inv) - 0.25) / 0.75
    assert bool((kept[turns > 40] > 1 - 1e-12).all()) and bool((kept[turns < 0.8] < 1e-12).all()) and bool((kept[1:] <= kept[:-1] + 1e-12).all())
    low = math.floor(128 * math.log(32768 / (32 * 2 * math.pi)) / (2 * math.log(1e6)))
    high = math.ceil(128 * math.log(32768 / (2 * math.pi)) / (2 * math.log(1e6)))
    for i in range(64):
        assert abs(float(kept[i]) - min(max((high - i) / (high - low), 0.0), 1.0)) < 1e-12
    assert rotary_frequencies(128, 1e6, {**scaling, "attention_factor": 1.5})[1] == 1.5
    assert rotary_frequencies(128, 1e6, {**scaling, "factor": 1.0})[1] == 1.0


@pytest.mark.parametrize("args", [(0,), (7,), (64, -1.0), (64, 1e4, {"type": "dynamic", "factor": 2.0}), (64, 1e4, {"type": "linear"}), (64, 1e4, {"type": "linear", "factor": 0.5}),
                                  (64, 1e4, {"type": "yarn", "factor": 2.0}), (64, 1e4, {"type": "llama3", "factor": 2.0, "low_freq_factor": 1.0, "original_max_position_embeddings": 4096}),
                                  (64, 1e4, {"type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 4096}),
                                  (64, 1e4, {"type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "mscale": 0.7})])
def test_frequencies_that_are_refused(args):
    with pytest.raises(ValueError):
        rotary_frequencies(*args)


# ---------------------------------------------------------------------------------------------- the cache's books
class _Books:
    """A PagedCache on the host whose copies of pages are made by hand: each place holds the number of the token that was written there."""

    def __init__(self, monkeypatch, pages=40, page=16):
        def copies(keys, values, sources, destinations):
            assert len(set(destinations)) == len(destinations) and not set(sources) & set(destinations)
            keys[:, destinations] = keys[:, sources].clone()
            values[:, destinations] = values[:, sources].clone()
            self.copied += len(sources)
        monkeypatch.setattr(rollout, "copy_pages", copies)
        self.copied = 0
        self.cache = PagedCache(1, pages, 1, 32, page=page, device="cpu")
        self.cache.keys = torch.zeros(1, pages, 1, page, 32)             # (numbers of tokens want more than 8 bits)
        self.cache.values = torch.zeros(1, pages, 1, 32, page)
        self.told = {}
        self.count = 0

    def extend(self, seqs, counts):
        step = self.cache.extend(seqs, counts)
        at = 0
        for row, (s, n) in enumerate(zip(seqs, counts)):
            for j in range(n):
                self.count += 1
                slot, position = int(step.slots[at]), int(step.positions[at])
                assert position == len(self.told[s])
                self.cache.keys[0, slot // self.cache.page, 0, slot % self.cache.page] = self.count
                self.cache.values[0, slot // self.cache.page, 0, :, slot % self.cache.page] = self.count
                self.told[s].append(self.count)
                at += 1
            assert int(step.lengths[row]) == len(self.told[s]) == self.cache.length(s)
            used = -(-len(self.told[s]) // self.cache.page)
            assert step.tables[row, :used].tolist() == list(self.cache.pages(s))
        assert at == step.slots.numel() and step.tables.dtype == step.lengths.dtype == torch.int32

    def check(self):
        c = self.cache
        users = [0] * len(c._users)
        for s, told in self.told.items():
            pages = c.pages(s)
            assert len(pages) == -(-len(told) // c.page) and len(set(pages)) == len(pages)
            keys = c.keys[0, list(pages), 0, :, 0].flatten()[:len(told)].tolist() if pages else []
            values = c.values[0, list(pages), 0, 7].flatten()[:len(told)].tolist() if pages else []
            assert keys == values == [float(t) for t in told]
            for p in pages:
                users[p] += 1
        assert users == c._users and sorted(c._free) == [p for p, n in enumerate(users) if n == 0] and c.free_pages == len(c._free)


@pytest.mark.parametrize("seed", range(6))
def test_books_under_any_order_of_calls(monkeypatch, seed):
    rng = random.Random(seed)
    books = _Books(monkeypatch, pages=rng.choice((12, 40)))
    refused = 0
    for _ in range(300):
        alive = list(books.told)
        what = rng.random()
        if what < 0.15 or not alive:
            for s in books.cache.new(rng.randint(1, 3)):
                books.told[s] = []
        elif what < 0.3:
            s = rng.choice(alive)
            for f in books.cache.fork(s, rng.randint(1, 4)):
                books.told[f] = list(books.told[s])
        elif what < 0.45:
            gone = rng.sample(alive, rng.randint(1, max(1, len(alive) // 2)))
            books.cache.free(gone)
            for s in gone:
                del books.told[s]
        elif what < 0.55:
            books.cache.compact()
            used = len(books.cache._users) - books.cache.free_pages
            assert all(p < used for s in books.told for p in books.cache.pages(s))
        else:
            some = rng.sample(alive, rng.randint(1, len(alive)))
            counts = [rng.choice((0, 1, 1, 1, 5, 17, 40)) for _ in some]
            before = books.cache.free_pages, {s: (books.cache.pages(s), books.cache.length(s)) for s in alive}
            try:
                books.extend(some, counts)
            except MemoryError:
                refused += 1
                assert before == (books.cache.free_pages, {s: (books.cache.pages(s), books.cache.length(s)) for s in alive})
        books.check()
    assert books.copied > 0 and refused > 0


def test_a_group_of_completions_shares_its_prompt(monkeypatch):
    """Fifteen forks of a prompt that ends inside a page: nothing is copied until they go on, then fifteen last pages, and the sixteenth sequence keeps the first one."""
    books = _Books(monkeypatch, pages=64)
    (s,) = books.cache.new()
    books.told[s] = []
    books.extend([s], [100])
    free = books.cache.free_pages
    group = [s, *books.cache.fork(s, 15)]
    for f in group[1:]:
        books.told[f] = list(books.told[s])
    assert books.copied == 0 and books.cache.free_pages == free
    books.extend(group, [1] * 16)
    assert books.copied == 15 and books.cache.free_pages == free - 15
    books.check()
    books.cache.free(group)
    assert books.cache.free_pages == 64


def test_books_that_are_refused(monkeypatch):
    books = _Books(monkeypatch)
    a, b = books.cache.new(2)
    for call in (lambda: books.cache.extend([a, a], 1), lambda: books.cache.extend([a, 99], 1), lambda: books.cache.extend([a], [-1]), lambda: books.cache.extend([a], [1, 2]),
                 lambda: books.cache.free([a, a]), lambda: books.cache.free([99])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        books.cache.fork(99)
    with pytest.raises(MemoryError, match="41 pages are needed and 40 free"):
        books.cache.extend([a], [40 * 16 + 1])
    empty = books.cache.extend([], [])
    assert empty.tables.shape == (0, 0) and empty.slots.numel() == 0
    assert books.cache.extend([a, b], 0).tables.shape == (2, 0)
    for args, more in (((0, 4, 1, 64), {}), ((1, 0, 1, 64), {}), ((1, 4, 0, 64), {}), ((1, 4, 1, 48), {}), ((1, 4, 1, 288), {}), ((1, 4, 1, 64), dict(page=8)), ((1, 4, 1, 64), dict(page=48)),
                       ((1, 4, 1, 96), dict(dtype=torch.float8_e4m3fn)), ((1, 4, 1, 64), dict(dtype=torch.float16)), ((1, 4, 1, 64), dict(key_scale=0.0))):
        with pytest.raises(ValueError):
            PagedCache(*args, device="cpu", **more)


def test_the_attention_modules_parameters_and_frequencies():
    linear = lambda n, m: torch.nn.Linear(n, m, bias=False)
    inv, _ = rotary_frequencies(32, 1e6)
    module = CachedAttention(linear(64, 128), linear(64, 64), linear(64, 64), linear(128, 64), 32, inv).to(BF)
    assert sorted(module.state_dict()) == ["k_proj.weight", "o_proj.weight", "q_proj.weight", "v_proj.weight"]
    assert module.q_proj.weight.dtype == BF and torch.equal(module.inv_freq, inv) and module.inv_freq.dtype == torch.float64
    cache = PagedCache(1, 4, 2, 32, device="cpu")
    step = cache.extend(cache.new(2), [1, 2])
    with pytest.raises(ValueError, match="one new token"):
        module(torch.zeros(2, 64, dtype=BF), cache, 0, step)


def test_numbers_of_sequences():
    """Fewer than none are refused, and the books are as they were; none are none."""
    cache = PagedCache(1, 4, 1, 64, device="cpu")
    (s,) = cache.new()
    cache.extend([s], [20])
    for call in (lambda: cache.new(-1), lambda: cache.fork(s, -1), lambda: cache.fork(s, -2)):
        with pytest.raises(ValueError, match="number of sequences"):
            call()
    assert cache.new(0) == cache.fork(s, 0) == []
    (t,) = cache.fork(s)
    cache.free([s])
    assert cache.free_pages == 2 and cache.pages(t) == (0, 1)
    cache.free([t])
    assert cache.free_pages == 4 and cache.new() == [2]


def test_the_attention_module_wants_one_token_of_each_sequence():
    """As many new tokens as sequences are not enough: two of one and none of the other would attend over the other's tokens.  A step made by hand need not say its counts."""
    from dataclasses import replace
    linear = lambda n, m: torch.nn.Linear(n, m, bias=False, dtype=BF)
    module = CachedAttention(linear(64, 128), linear(64, 64), linear(64, 64), linear(128, 64), 32, rotary_frequencies(32, 1e6)[0])
    cache = PagedCache(1, 8, 2, 32, device="cpu")
    a, b, c = cache.new(3)
    x = torch.zeros(2, 64, dtype=BF)
    step = cache.extend([a, b], [2, 0])
    assert step.counts == (2, 0) and step.slots.shape == step.lengths.shape
    with pytest.raises(ValueError, match="one new token"):
        module(x, cache, 0, step)
    with pytest.raises(ValueError, match="one new token"):
        module(torch.zeros(3, 64, dtype=BF), cache, 0, cache.extend([a, b, c], [0, 3, 0]))
    step = cache.extend([a, b])
    assert step.counts == (1, 1)
    for good in (step, replace(step, counts=None), replace(step, tables=torch.nn.functional.pad(step.tables, (0, 3)))):
        with pytest.raises(MetisHipError, match="no CPU path"):      # (it gets as far as the device's calls)
            module(x, cache, 0, good)


def test_calls_of_more_than_a_launch_takes():
    """A launch has fewer than 2^32 work-items.  Rotations, appends and attention beyond it say that they are too large, and nothing is launched."""
    L = _lib.load()
    wide = dict(dim=512, turned=512, q_token=511, q_heads=1, k_heads=1, k_token=511, q_head=512, k_head=512)
    assert L.metis_rotary(*{**ROTARY, **wide, "tokens": 1 << 24, "npos": 1}.values()) == _lib.E_TOO_LARGE
    assert L.metis_rotary(*{**ROTARY, "tokens": 1 << 31, "npos": 1, "q_token": 64, "k_token": 64}.values()) == _lib.E_TOO_LARGE
    assert L.metis_rotary_append(*{**APPEND, "v_token": 127, "tokens": 1 << 25}.values()) == _lib.E_TOO_LARGE
    big = 1 << 60
    assert L.metis_paged_attention(*{**ATTEND, "seqs": 1 << 23}.values()) == _lib.E_TOO_LARGE
    assert L.metis_paged_attention(*{**ATTEND, "seqs": 1 << 18, "heads": 32, "kv": 1, "width": 1024, "bytes": big}.values()) == _lib.E_TOO_LARGE
    a = (ctypes.c_int64 * 1)(0)
    assert L.metis_cache_copy_pages(4096, 4096, 1 << 20, 8, 1 << 20, ctypes.cast(a, ctypes.c_void_p), ctypes.cast((ctypes.c_int64 * 1)(1), ctypes.c_void_p), 1, None) == _lib.E_TOO_LARGE


def test_scales_that_binary32_does_not_have():
    """Scales of the cache are positive and finite, and so held in binary32: one that is nothing there would make all scores alike."""
    L = _lib.load()
    inf, nan = float("inf"), float("nan")
    for bad in (inf, 0.0, -1.0, nan, 1e-50):
        assert L.metis_rotary_append(*{**APPEND, "key_scale": bad}.values()) == L.metis_rotary_append(*{**APPEND, "value_scale": bad}.values()) == _lib.E_ARG
        assert L.metis_paged_attention(*{**ATTEND, "key_scale": bad}.values()) == L.metis_paged_attention(*{**ATTEND, "value_scale": bad}.values()) == _lib.E_ARG
    for bad in (inf, -inf, nan):
        assert L.metis_paged_attention(*{**ATTEND, "scale": bad}.values()) == _lib.E_ARG
    for bad in (1e-50, 1e300, nan):
        for more in (dict(key_scale=bad), dict(value_scale=bad)):
            with pytest.raises(ValueError, match="scales"):
                PagedCache(1, 4, 1, 64, device="cpu", **more)


def test_gradients_of_any_argument_are_refused():
    """Frequencies, settings and caches too: whoever asks for their gradients would get none."""
    q, at, inv, u = torch.zeros(2, 4, 64, dtype=BF), torch.arange(2), torch.ones(32), torch.zeros(2)
    keys, values, logits = torch.zeros(3, 4, 16, 64, dtype=BF), torch.zeros(3, 4, 64, 16, dtype=BF), torch.zeros(2, 5)
    ask = lambda t: t.clone().requires_grad_()
    for call in (lambda: rotary_append(q, q, q, at, ask(inv), at, keys, values), lambda: rotary_append(q, q, q, at, inv, at, ask(keys), values),
                 lambda: rotary_append(q, q, q, at, inv, at, keys, ask(values)), lambda: copy_pages(ask(keys[None]), values[None], [0], [1]),
                 lambda: paged_attention(q, keys, ask(values), at.int()[:, None], at.int()), lambda: sample_tokens(logits, ask(u)), lambda: sample_tokens(logits, u, temperature=ask(u)),
                 lambda: sample_tokens(logits, u, top_p=ask(u)), lambda: sample_tokens(ask(logits), u)):
        with pytest.raises(ValueError, match="no gradients"):
            call()
        with torch.no_grad(), pytest.raises(MetisHipError, match="no CPU path"):
            call()


def test_counts_that_are_no_whole_numbers():
    """Refused before a page is taken; whole numbers of other types are taken as such."""
    import numpy as np
    cache = PagedCache(1, 8, 1, 64, device="cpu")
    a, b = cache.new(2)
    cache.extend([a], [20])
    for counts in ([1.5, 1], [1, 40.5], [1, None], ["1", 1]):
        before = cache.free_pages, [(cache.pages(s), cache.length(s)) for s in (a, b)], list(cache._users)
        with pytest.raises(TypeError):
            cache.extend([a, b], counts)
        assert before == (cache.free_pages, [(cache.pages(s), cache.length(s)) for s in (a, b)], list(cache._users))
    step = cache.extend([a, b], np.array([1, 17]))
    assert step.counts == (1, 17) and step.lengths.tolist() == [21, 17] and all(type(n) is int for n in step.counts) and type(cache.length(a)) is int
