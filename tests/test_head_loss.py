"""token_logprobs: what is refused, and the sizes a caller asks for, without a device."""
import pytest
import torch

from metis_hip import MetisHipError, _lib, linear_cross_entropy, model_token_logprobs, token_logprobs


def test_host_tensors_are_refused():
    x, w, t = torch.zeros(3, 32, dtype=torch.bfloat16), torch.zeros(7, 32, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(MetisHipError, match="no CPU path"):
        token_logprobs(x, w, t)
    with pytest.raises(MetisHipError, match="no CPU path"):
        linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")


@pytest.mark.parametrize("setting", [dict(final_logit_softcapping=30.0), dict(logit_scale=0.0625), dict(logits_scaling=8.0)])
def test_heads_that_do_more_than_a_product_are_refused(setting):
    from types import SimpleNamespace
    model = SimpleNamespace(config=SimpleNamespace(**setting), get_output_embeddings=lambda: SimpleNamespace(weight=None, bias=None))
    with pytest.raises(ValueError, match="not capped or scaled"):
        model_token_logprobs(model, torch.zeros(1, 4, dtype=torch.int64))


@pytest.mark.parametrize("head", [None, torch.nn.Identity(), torch.nn.LayerNorm(8, bias=False)])
def test_heads_without_one_matrix_are_refused(head):
    from types import SimpleNamespace
    with pytest.raises(ValueError, match="one weight"):
        model_token_logprobs(SimpleNamespace(get_output_embeddings=lambda: head), torch.zeros(1, 4, dtype=torch.int64))


def _forward(**changes):
    a = dict(hidden=4096, ldh=64, weight=4096, ldw=64, targets=4096, ignore=-100, tokens=4, H=64, V=100, temperature=1.0, logp=4096, lse=4096, entropy=None, index=4096,
             workspace=4096, bytes=1 << 30, stream=None)
    a.update(changes)
    return _lib.load().metis_head_logprobs(*a.values())


BAD = [dict(H=60), dict(H=0), dict(H=65552, ldh=65552, ldw=65552), dict(V=0), dict(V=(1 << 22) + 1), dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(hidden=None), dict(weight=None),
       dict(targets=None), dict(index=None), dict(ldh=56), dict(ldw=56), dict(ldh=68), dict(ldw=68), dict(hidden=4104), dict(weight=4104), dict(targets=4100), dict(index=4112),
       dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(temperature=4e-39)]


@pytest.mark.parametrize("changes", BAD + [dict(logp=None), dict(lse=None), dict(lse=4098), dict(entropy=4098)])
def test_the_forward_refuses_before_a_launch(changes):
    assert _forward(**changes) == _lib.E_ARG


def test_workspaces():
    L = _lib.load()
    need = L.metis_head_logprobs_workspace_bytes(4, 64, 100, 0)
    assert 0 < need < L.metis_head_logprobs_workspace_bytes(4, 64, 100, 1)
    assert L.metis_head_logprobs_workspace_bytes(0, 64, 100, 0) == 0 and L.metis_head_logprobs_workspace_bytes(4, 60, 100, 0) == 0
    assert L.metis_head_index_bytes(10) >= (64 + 20) * 4 and L.metis_head_index_bytes(-1) == 0
    for changes in (dict(workspace=None), dict(bytes=need - 1), dict(workspace=4096 + 16)):
        assert _forward(**changes) == _lib.E_WORKSPACE
    assert _forward(tokens=0, hidden=None, workspace=None) == _lib.OK
    back = L.metis_head_logprobs_backward_workspace_bytes
    assert back(4, 64, 100, 1, 1) >= back(4, 64, 100, 0, 1) > 0 and back(4, 64, 100, 1, 0) > 0 and back(0, 64, 100, 1, 1) == 0
    # a piece of the gradient of the logits, not the whole: 4096 x 131072 of it would be 1 GiB (and three numbers a token)
    assert back(4096, 3584, 131072, 0, 0) <= (256 << 20) + 12 * 4096
    # and with many tokens at most twice the binary32 gradient of hidden
    assert back(1 << 20, 4096, 131072, 0, 0) <= 8 * (1 << 20) * 4096 + 12 * (1 << 20)


def _backward(**changes):
    a = dict(hidden=4096, ldh=64, weight=4096, ldw=64, targets=4096, tokens=4, H=64, V=100, temperature=1.0, lse=4096, entropy=None, g_logp=4096, g_entropy=None, index=4096,
             gh=4096, gw=4096, workspace=4096, bytes=1 << 40, stream=None)
    a.update(changes)
    return _lib.load().metis_head_logprobs_backward(*a.values())


@pytest.mark.parametrize("changes", BAD + [dict(tokens=0), dict(lse=None), dict(g_entropy=4096), dict(gh=4104), dict(gw=4104), dict(g_logp=4098)])
def test_the_backward_refuses_before_a_launch(changes):
    assert _backward(**changes) == _lib.E_ARG


def test_the_backward_wants_its_workspace():
    need = _lib.load().metis_head_logprobs_backward_workspace_bytes(4, 64, 100, 1, 1)
    for changes in (dict(workspace=None), dict(bytes=need - 1), dict(workspace=4096 + 16)):
        assert _backward(**changes) == _lib.E_WORKSPACE
    assert _backward(gh=None, gw=None, workspace=None) == _lib.OK


def _seen_targets(monkeypatch, ids, mask, **more):
    """The targets and hidden states that model_token_logprobs hands on, without a device."""
    from types import SimpleNamespace
    from metis_hip import loss
    got = {}

    def take(hidden, weight, targets, **_):
        got.update(hidden=hidden, targets=targets)
        return targets
    monkeypatch.setattr(loss, "token_logprobs", take)
    hidden = torch.zeros(*ids.shape, 8)
    model = SimpleNamespace(get_output_embeddings=lambda: torch.nn.Linear(8, 32, bias=False), base_model=lambda **_: (hidden,))
    model_token_logprobs(model, ids, mask, **more)
    return got["targets"].tolist()


@pytest.mark.parametrize("mask,want", [([0, 0, 1, 1, 1], [-100, -100, 6, 7]),        # padded on the left: the first real token has no context
                                       ([1, 1, 1, 0, 0], [4, 5, -100, -100]),        # on the right
                                       ([1, 0, 1, 1, 0], [-100, -100, 6, -100]),     # a hole: neither into it nor out of it
                                       ([0, 0, 0, 0, 0], [-100] * 4), ([0, 0, 0, 0, 1], [-100] * 4), ([1] * 5, [4, 5, 6, 7]), (None, [4, 5, 6, 7])])
def test_tokens_count_where_they_and_the_position_before_them_are_there(monkeypatch, mask, want):
    ids = torch.tensor([[3, 4, 5, 6, 7]])
    for dtype in (torch.int64, torch.bool):
        assert _seen_targets(monkeypatch, ids, None if mask is None else torch.tensor([mask], dtype=dtype)) == [want]


def test_labels_and_the_mask_both_leave_tokens_out(monkeypatch):
    ids, labels = torch.tensor([[3, 4, 5, 6, 7]]), torch.tensor([[-100, -100, -100, 9, 10]])
    assert _seen_targets(monkeypatch, ids, torch.tensor([[0, 1, 1, 1, 1]]), labels=labels) == [[-100, -100, 9, 10]]
    assert _seen_targets(monkeypatch, ids, torch.tensor([[0, 0, 0, 1, 1]]), labels=labels) == [[-100, -100, -100, 10]]
    assert _seen_targets(monkeypatch, ids, torch.tensor([[1, 1, 1, 1, 0]]), labels=labels, ignore_index=10) == [[-100, -100, 9, 10]]


class _Decoder(torch.nn.Module):
    def __init__(self, output):
        super().__init__()
        self.embed, self.output, self.lm_head_multiplier = torch.nn.Embedding(20, 8), output, 0.25
        if output == "inside":                                           # as models whose decoder lies one level further down
            self.decoder = _Decoder("object")

    def forward(self, input_ids, attention_mask=None):
        from types import SimpleNamespace
        hidden = self.embed(input_ids)
        return (hidden, None) if self.output == "tuple" else SimpleNamespace(last_hidden_state=hidden)


class _Causal(torch.nn.Module):
    """A causal language model whose logits are its head's product, returned in one of the usual ways."""

    def __init__(self, output="object", returned="object"):
        super().__init__()
        self.base_model, self.lm_head, self.returned, self.calls = _Decoder(output), torch.nn.Linear(8, 20, bias=False), returned, []
        self.factor = 2.0

    def get_output_embeddings(self):
        return self.lm_head

    def hidden(self, input_ids, attention_mask):
        out = (self.base_model.decoder if self.base_model.output == "inside" else self.base_model)(input_ids, attention_mask=attention_mask)
        return out[0] if isinstance(out, tuple) else out.last_hidden_state

    def logits(self, hidden):
        return self.lm_head(hidden)

    def forward(self, input_ids, attention_mask=None, labels=None):
        from types import SimpleNamespace
        logits = self.logits(self.hidden(input_ids, attention_mask)).float()
        return {"object": SimpleNamespace(logits=logits), "tuple": (logits, None), "tensor": logits, "dict": {"logits": logits}, "nothing": None}[self.returned]


class _TimesHead(_Causal):
    def logits(self, hidden):
        return self.lm_head(hidden) * self.factor


class _TimesDecoders(_Causal):
    def logits(self, hidden):
        return self.lm_head(hidden) * self.base_model.lm_head_multiplier


class _TimesHidden(_Causal):
    def logits(self, hidden):
        return self.lm_head(hidden / 3.0)


class _Capped(_Causal):
    def logits(self, hidden):
        return 50.0 * torch.tanh(self.lm_head(hidden) / 50.0)


class _Shifted(_Causal):
    def __init__(self):
        super().__init__()
        self.shift = torch.full((20,), 1e-3)

    def logits(self, hidden):
        return self.lm_head(hidden) + self.shift


class _Cut(_Causal):
    def logits(self, hidden):
        return self.lm_head(hidden)[..., :17]


class _Normed(_Causal):
    def logits(self, hidden):
        return self.lm_head(torch.nn.functional.layer_norm(hidden, hidden.shape[-1:]))


class _ByHand(_Causal):                                                  # asks its decoder for its parts
    def hidden(self, input_ids, attention_mask):
        return self.base_model.embed.weight[input_ids]


def _asked(model, mask=True):
    """model_token_logprobs without a device: it ends in token_logprobs' refusal of host tensors."""
    ids = torch.tensor([[3, 4, 5, 6, 7, 8], [1, 2, 3, 4, 5, 6]])
    with pytest.raises(MetisHipError, match="no CPU path"):
        model_token_logprobs(model, ids, torch.ones_like(ids) if mask else None)


@pytest.mark.parametrize("mask", [True, False])
@pytest.mark.parametrize("output", ["object", "tuple", "inside"])
@pytest.mark.parametrize("returned", ["object", "tuple", "tensor", "dict"])
def test_models_whose_logits_are_the_product_are_taken(output, returned, mask):
    model = _Causal(output, returned)
    attributes = dict(vars(model))
    _asked(model, mask)
    assert dict(vars(model)) == attributes and set(model._modules) == {"base_model", "lm_head"}


@pytest.mark.parametrize("kind", [_TimesHead, _TimesDecoders, _TimesHidden, _Capped, _Shifted, _Cut, _Normed, _ByHand])
def test_models_whose_logits_are_something_else_are_refused(kind):
    with pytest.raises(ValueError, match="logits"):
        model_token_logprobs(kind(), torch.tensor([[3, 4, 5, 6]]))


def test_models_that_return_no_logits_are_refused():
    with pytest.raises(ValueError, match="logits"):
        model_token_logprobs(_Causal(returned="nothing"), torch.tensor([[3, 4, 5, 6]]))


def test_a_factor_of_one_is_no_factor():
    model = _TimesHead()
    model.factor = 1.0
    _asked(model)


@pytest.mark.parametrize("name,setting,taken", [("Llama", {}, True), ("Qwen2", {}, True), ("OPT", {"word_embed_proj_dim": 32, "ffn_dim": 48}, True),
                                                ("Mixtral", {"num_local_experts": 2}, True), ("Gemma2", {"head_dim": 8, "final_logit_softcapping": None}, True),
                                                ("Gemma2", {"head_dim": 8}, False), ("Granite", {"logits_scaling": 8.0}, False), ("Cohere", {}, False)])
def test_models_of_a_library(name, setting, taken):
    transformers = pytest.importorskip("transformers")
    config = getattr(transformers, f"{name}Config")(vocab_size=20, hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                                                    pad_token_id=0, bos_token_id=0, eos_token_id=0, tie_word_embeddings=False, **setting)
    model = getattr(transformers, f"{name}ForCausalLM")(config)
    if taken:
        _asked(model)
    else:
        with pytest.raises(ValueError, match="logits"):
            model_token_logprobs(model, torch.tensor([[3, 4, 5, 6]]))


class _Adapted(torch.nn.Module):
    """A head in an adapter's wrapper that hands out the weight of what it wraps."""

    def __init__(self, head):
        super().__init__()
        self.head, self.a, self.b = head, torch.nn.Linear(8, 2, bias=False), torch.nn.Linear(2, 20, bias=False)

    weight = property(lambda self: self.head.weight)
    bias = property(lambda self: self.head.bias)

    def forward(self, x):
        return self.head(x) + self.b(self.a(x))


class _Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2.0 * super().forward(x)


def _lowbit_head():
    from metis_hip import LinearLowbit, MetisArgs
    return LinearLowbit(8, 20, bias=False, args=MetisArgs(), device="cpu")


def _changed(change):
    head = torch.nn.Linear(8, 20, bias=False)
    change(head)
    return head


@pytest.mark.parametrize("make", [lambda: _Adapted(torch.nn.Linear(8, 20, bias=False)), lambda: _Doubled(8, 20, bias=False), _lowbit_head,
                                  lambda: _changed(lambda h: h.register_forward_hook(lambda m, a, y: 2 * y)),
                                  lambda: _changed(lambda h: h.register_forward_pre_hook(lambda m, a: (2 * a[0],))),
                                  lambda: _changed(lambda h: setattr(h, "forward", lambda x: torch.nn.functional.linear(x, 2 * h.weight)))],
                         ids=["adapter", "subclass", "quantized", "hook", "pre_hook", "forward"])
def test_heads_that_compute_something_else_with_their_weight_are_refused(make):
    model = _Causal()
    model.lm_head = make()
    with pytest.raises(ValueError, match="plain linear"):
        model_token_logprobs(model, torch.tensor([[3, 4, 5, 6]]))


def test_parametrized_heads_are_taken():
    """The weight of a parametrization is what its forward multiplies by."""
    class Scaled(torch.nn.Module):
        def forward(self, w):
            return 2 * w
    model = _Causal()
    torch.nn.utils.parametrize.register_parametrization(model.lm_head, "weight", Scaled())
    _asked(model)


def test_a_single_row_has_no_stride_that_counts():
    """A row cut out of a wider one, or the last position of one sequence: the entry point wants strides in eights, and of one row there is none."""
    from metis_hip import ops
    wide = torch.zeros(3, 68, dtype=torch.bfloat16)
    for t in (wide[:1, :64], wide.flatten()[:68].view(1, 1, 68)[..., :64], torch.zeros(1, 7, 61, 64, dtype=torch.bfloat16)[:, 2:3, 5:6]):
        taken, ld = ops._head_operand(t)
        assert ld == 64 and taken.shape == (1, 64) and taken.data_ptr() % 16 == 0
    taken, ld = ops._head_operand(wide[:, :64])                          # (more rows are copied for it)
    assert ld == 64 and taken.is_contiguous()
    taken, ld = ops._head_operand(torch.zeros(3, 72, dtype=torch.bfloat16)[:, :64])
    assert ld == 72 and taken.stride() == (72, 1)


@pytest.mark.parametrize("T,H,V", [(1, 16, 1), (5, 1536, 131072), (64, 3584, 131072), (65, 2048, 131072), (540, 2048, 65536), (600, 2048, 128003), (2048, 4096, 131072), (2049, 512, 4000),
                                   (4096, 3584, 131072), (1 << 17, 4096, 152064)])
def test_the_backwards_workspace_is_what_the_header_says(T, H, V):
    """With the partial sums of grad_hidden, which want_hidden adds: at most 64 copies, and at most one for each 512 columns of a piece."""
    ask = _lib.load().metis_head_logprobs_backward_workspace_bytes
    rows = -(-T // 64) * 64 + (192 if T > 64 else 0) if T <= 2048 else -(-T // 256) * 256
    piece = max(256 << 20, 8 * rows * H) // (2 * rows) // 256 * 256 or 256
    width = min(piece, -(-V // 256) * 256)
    copies = max(1, min(64, width // 512))
    for weight in (0, 1):
        without = 2 * rows * width + 12 * rows + weight * (4 * rows * H + 4 * (-(-V // 256) * 256)) + 6 * 256
        assert 0 < ask(T, H, V, 0, weight) <= without
        assert 4 * rows * H <= ask(T, H, V, 1, weight) - ask(T, H, V, 0, weight) <= 4 * rows * H * copies


def test_decoder_outputs_of_a_class_of_their_own_are_taken():
    """One that cannot be made of the hidden states alone, and a tuple with names."""
    from collections import namedtuple

    class Output:
        def __init__(self, last_hidden_state, aux):
            self.last_hidden_state, self.aux = last_hidden_state, aux

    for output in (Output, namedtuple("Named", ["last_hidden_state", "aux"])):
        class Decoder(_Decoder):
            def forward(self, input_ids, attention_mask=None, output=output):
                return output(self.embed(input_ids), 3)

        for kind, taken in ((_Causal, True), (_TimesHead, False)):
            class Model(kind):
                def hidden(self, input_ids, attention_mask):
                    return self.base_model(input_ids, attention_mask=attention_mask).last_hidden_state

            model = Model()
            model.base_model = Decoder("object")
            if taken:
                _asked(model)
            else:
                with pytest.raises(ValueError, match="logits"):
                    model_token_logprobs(model, torch.tensor([[3, 4, 5, 6]]))
