"""residual_norm, swiglu and the modules that call them: what is refused or left as it is, without a device."""
import ctypes

import pytest
import torch

from metis_hip import GatedMLP, MetisHipError, _lib, fuse_gated_mlps, ops, residual_norm, swiglu


def test_host_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(MetisHipError, match="no CPU path"):
        residual_norm(x, x, w)
    with pytest.raises(MetisHipError, match="no CPU path"):
        swiglu(x, x)


@pytest.mark.parametrize("shape,gate,rows", [((2, 3, 8), (8,), 1), ((2, 3, 8), (2, 1, 8), 2), ((2, 3, 8), (1, 1, 8), 1), ((2, 3, 8), (2, 3, 8), 6),
                                             ((5, 8), (5, 8), 5), ((5, 8), (1, 8), 1), ((8,), (8,), 1), ((1, 3, 8), (1, 3, 8), 3)])
def test_gate_rows(shape, gate, rows):
    assert ops.residual_norm_gate_rows(torch.empty(shape), torch.empty(gate)) == rows


@pytest.mark.parametrize("shape,gate", [((2, 3, 8), (2, 8)), ((2, 3, 8), (3, 1, 8)), ((2, 3, 8), (1, 3, 8)), ((5, 8), (1, 5, 8)), ((5, 8), (4, 8))])
def test_gates_of_other_shapes_are_refused(shape, gate):
    with pytest.raises(ValueError, match="leading sizes"):
        ops.residual_norm_gate_rows(torch.empty(shape), torch.empty(gate))


def _norm_args(**changes):
    """metis_residual_norm's arguments for 4 x 64 in bf16 with addresses that are never read."""
    args = dict(x=4096, x_dtype=0, y=4096, y_dtype=0, weight=4096, post=None, gate=None, gate_rows=0, scale=1.0, eps=1e-6, rows=4, cols=64, h=4096, n=4096, stream=None)
    args.update(changes)
    return tuple(args.values())


@pytest.mark.parametrize("changes", [dict(cols=60), dict(cols=0), dict(cols=8200), dict(rows=-1), dict(rows=1 << 31), dict(x_dtype=2), dict(y_dtype=1), dict(x=None), dict(y=None),
                                     dict(weight=None), dict(h=None), dict(n=None), dict(x=4098), dict(weight=4104), dict(gate=4096), dict(gate_rows=2),
                                     dict(gate=4096, gate_rows=3), dict(gate=4096, gate_rows=-1), dict(post=4100)])
def test_the_abi_refuses_before_a_launch(changes):
    assert _lib.load().metis_residual_norm(*_norm_args(**changes)) == _lib.E_ARG


def test_no_rows_are_no_work():
    assert _lib.load().metis_residual_norm(*_norm_args(rows=0, x=None, y=None)) == _lib.OK


def _backward_args(**changes):
    args = dict(h=4096, x_dtype=0, y=None, y_dtype=0, weight=4096, post=None, gate=None, gate_rows=0, scale=1.0, eps=1e-6, rows=4, cols=64, gh=4096, gn=4096, gx=4096, gy=4096,
                gw=4096, gp=None, gg=None, workspace=4096, bytes=1 << 30, stream=None)
    args.update(changes)
    return tuple(args.values())


@pytest.mark.parametrize("changes", [dict(rows=0), dict(cols=12), dict(h=None), dict(post=4096), dict(gp=4096), dict(gg=4096), dict(gate=4096, gate_rows=2, gg=4096),
                                     dict(gh=4097), dict(gx=4100), dict(gw=4104)])
def test_the_backward_refuses_before_a_launch(changes):
    assert _lib.load().metis_residual_norm_backward(*_backward_args(**changes)) == _lib.E_ARG


def test_the_backward_wants_its_workspace():
    L = _lib.load()
    need = L.metis_residual_norm_backward_workspace_bytes(4, 64, 0)
    assert need > 0 and L.metis_residual_norm_backward_workspace_bytes(0, 64, 0) == 0 and L.metis_residual_norm_backward_workspace_bytes(4, 60, 0) == 0
    assert L.metis_residual_norm_backward_workspace_bytes(4, 64, 3) == 0                        # 3 does not divide 4
    for changes in (dict(workspace=None), dict(bytes=need - 1), dict(workspace=4100)):
        assert L.metis_residual_norm_backward(*_backward_args(**changes)) == _lib.E_WORKSPACE


@pytest.mark.parametrize("changes", [dict(rows=-1), dict(cols=-1), dict(dtype=2), dict(gate=None), dict(up=None), dict(out=None), dict(gate=4097), dict(ldg=63), dict(ldu=63),
                                     dict(cols=1 << 31), dict(rows=1 << 40, cols=1 << 20, ldg=1 << 20, ldu=1 << 20)])
def test_swiglu_refuses_before_a_launch(changes):
    args = dict(gate=4096, ldg=64, up=4096, ldu=64, rows=4, cols=64, dtype=0, out=4096, stream=None)
    args.update(changes)
    L = _lib.load()
    assert L.metis_swiglu(*args.values()) == _lib.E_ARG
    back = (args["gate"], args["ldg"], args["up"], args["ldu"], ctypes.c_void_p(4096), args["rows"], args["cols"], args["dtype"], args["out"], 4096, None)
    assert L.metis_swiglu_backward(*back) == _lib.E_ARG


def test_swiglu_refuses_more_pieces_than_it_counts():
    rows = (1 << 31) // 8
    assert _lib.load().metis_swiglu(4096, 64, 4096, 64, rows, 64, 0, 4096, None) == _lib.E_TOO_LARGE


class _Mlp(torch.nn.Module):
    def __init__(self):
        super().__init__()
        Linear = torch.nn.Linear
        self.gate_proj, self.up_proj, self.down_proj, self.act_fn = Linear(16, 24, bias=False), Linear(16, 24), Linear(24, 16, bias=False), torch.nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class _Cast(_Mlp):                                                       # the same formula, written in another way
    def forward(self, hidden_states):
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1])
        gate = torch.nn.functional.silu(self.gate_proj(x).float()).to(x.dtype)
        return self.down_proj(self.up_proj(x) * gate).view(shape)


class _GateMultiplier(_Mlp):
    multiplier = 1.5

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x) * self.multiplier) * self.up_proj(x))


class _DownMultiplier(_Mlp):
    def __init__(self):
        super().__init__()
        self.multipliers = [1.0, 0.5]

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x) * self.multipliers[0]) * self.up_proj(x)) * self.multipliers[1]


class _Clamped(_Mlp):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x).clamp(max=200.0)) * self.up_proj(x))


class _Dropout(_Mlp):
    def forward(self, x):
        return self.down_proj(torch.nn.functional.dropout(self.act_fn(self.gate_proj(x)) * self.up_proj(x), 0.1, self.training))


class _Swapped(_Mlp):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class _Residual(_Mlp):
    def forward(self, x):
        return x + super().forward(x)


class _Optional(_Mlp):
    def forward(self, x, scale=None):
        x = super().forward(x)
        return x if scale is None else x * scale


class _Pair(_Mlp):
    def forward(self, x):
        return super().forward(x), None


class _OwnParameter(_Mlp):                                               # (not used: it would vanish from the model all the same)
    def __init__(self):
        super().__init__()
        self.scale = torch.nn.Parameter(torch.ones(()))


class _OwnBuffer(_Mlp):
    def __init__(self):
        super().__init__()
        self.register_buffer("scale", torch.ones(()))


def _hooked(register):
    def make():
        mlp = _Mlp()
        getattr(mlp, register)(lambda *_: None)
        return mlp
    return make


def _with_its_own_forward():
    mlp = _Mlp()
    mlp.forward = lambda x: x
    return mlp


def _in_a_model(mlp, train):
    model = torch.nn.Module()
    model.layer = torch.nn.Module()
    model.layer.mlp = mlp
    return model.train(train)


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("make", [_Mlp, _Cast])
def test_mlps_that_are_the_formula_are_replaced(make, train):
    mlp = make()
    model = _in_a_model(mlp, train)
    names, calls = [n for n, _ in model.named_parameters()], []
    for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj):
        p.register_forward_hook(lambda *_: calls.append(1))
    before = torch.get_rng_state()
    assert fuse_gated_mlps(model) == 1 and isinstance(model.layer.mlp, GatedMLP) and model.layer.mlp.training == train
    assert not calls and torch.equal(torch.get_rng_state(), before)      # (the projections themselves were not asked)
    assert [n for n, _ in model.named_parameters()] == names and model.layer.mlp.gate_proj is mlp.gate_proj


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("make", [_GateMultiplier, _DownMultiplier, _Clamped, _Dropout, _Swapped, _Residual, _Optional, _Pair, _OwnParameter, _OwnBuffer, _with_its_own_forward,
                                  *(_hooked(r) for r in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook",
                                                         "register_state_dict_pre_hook"))])
def test_mlps_that_do_more_stay_as_they_are(make, train):
    torch.manual_seed(1)
    mlp = make()
    model = _in_a_model(mlp, train)
    names, x = sorted(model.state_dict()), torch.randn(3, 5, 16)
    attributes = dict(vars(mlp))
    assert fuse_gated_mlps(model) == 0 and model.layer.mlp is mlp
    assert sorted(model.state_dict()) == names and dict(vars(mlp)) == attributes
    if make not in (_Dropout, _Pair):
        with torch.no_grad():
            assert torch.equal(model.layer.mlp(x), mlp(x))


def test_mlps_of_a_library_are_told_apart():
    """The same children and activation in both: one multiplies in its forward."""
    transformers = pytest.importorskip("transformers")
    from transformers.models.falcon_h1.modeling_falcon_h1 import FalconH1MLP
    from transformers.models.llama.modeling_llama import LlamaMLP
    small = dict(hidden_size=16, intermediate_size=24, num_attention_heads=2, num_key_value_heads=2)
    assert fuse_gated_mlps(_in_a_model(LlamaMLP(transformers.LlamaConfig(**small)), True)) == 1
    assert fuse_gated_mlps(_in_a_model(FalconH1MLP(transformers.FalconH1Config(**small, mlp_multipliers=[2.0, 0.5])), True)) == 0


@pytest.mark.parametrize("cols", [64, 60])
@pytest.mark.parametrize("stream,branch,weight", [(torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16, torch.bfloat16),
                                                  (torch.float32, torch.float32, torch.float32), (torch.float32, torch.bfloat16, torch.float32)])
def test_the_norm_modules_pair_has_its_types_without_the_kernel_too(stream, branch, weight, cols):
    """FusedRMSNormQuant(y, residual) where the kernel does not take the tensors: the stream in its own type and the norm in the branch's, as the kernel
    gives them; each value that of binary64 but for its roundings: the sum's, x * rstd's where the module rounds it, and the result's, and binary32's own."""
    from metis_hip import FusedRMSNormQuant
    g = torch.Generator().manual_seed(7)
    x, y = torch.randn(3, 5, cols, generator=g).to(stream), torch.randn(3, 5, cols, generator=g).to(branch)
    w = torch.nn.Parameter((1 + 0.1 * torch.randn(cols, generator=g)).to(weight))
    with torch.no_grad():
        h, n = FusedRMSNormQuant(w, 1e-6, {"name": "mlp.gate_up"})(y, x)
    assert h.dtype == stream and n.dtype == branch and h.shape == n.shape == x.shape
    total = x.double() + y.double()
    assert bool(((h.double() - total).abs() <= torch.finfo(stream).eps / 2 * total.abs()).all())
    want = h.double() / (h.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    assert bool(((n.double() - want).abs() <= (1.01 * torch.finfo(branch).eps + 2.0 ** -20) * want.abs()).all())


@pytest.mark.parametrize("name", ["residual_norm", "residual_norm_backward", "swiglu", "swiglu_backward", "head_logprobs", "head_logprobs_backward"])
def test_operators_take_all_their_arguments_by_name(name):
    """Their first one too, which says on which device the call runs."""
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    t, f = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    given = {"residual_norm": dict(y=x, weight=w, x=x), "swiglu": dict(up=x, gate=x), "swiglu_backward": dict(grad=x, up=x, gate=x),
             "residual_norm_backward": dict(y=None, weight=w, post_weight=None, gate=None, scale=1.0, eps=1e-6, grad_h=x, grad_n=x, y_dtype=x.dtype, h=x),
             "head_logprobs": dict(weight=x, targets=t, hidden=x),
             "head_logprobs_backward": dict(weight=x, targets=t, temperature=1.0, lse=f, entropy=None, index=t, grad_logp=f, grad_entropy=None, hidden=x)}[name]
    with pytest.raises(MetisHipError, match="no CPU path"):
        getattr(ops, name)(**given)
    with pytest.raises(TypeError):
        getattr(ops, name)()
