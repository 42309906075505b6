// residual_norm, swiglu and rotary as nodes of torch's autograd, in compiled code.  Host code only: the arithmetic is libmetis_hip.so's, the checks of arguments are
// made by the Python functions that call these (metis_hip/block.py, metis_hip/ops.py); rotary's are made here first, and what does not pass them is Python's (host time of a rotation and
// its gradient 44 to 75 us on different hosts before, 39 to 62 now, of which the engine's way to its thread and back is 28).
//
// All are kernels of some tens of microseconds in a training step, and a node written in Python costs more than that: recorded, run backward in the
// engine's own thread (which has to get the interpreter first) and allocated for.  One token x 1536, forward and all gradients: 101 us through
// torch.autograd.Function in Python, 49 of them an empty one's, and 123 with a norm behind the block and a gate; here 73 and 93.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <optional>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/metis_hip.h"
#include "host_autograd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_of(at::ScalarType t) { return t == at::kBFloat16 ? METIS_DTYPE_BF16 : METIS_DTYPE_F32; }

// the current stream of the tensor's device
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
// contiguous and 16-byte aligned; a copy only where it has to be one
Tensor flat(const Tensor& t)
{
    if (!t.defined() || (t.is_contiguous() && aligned(t))) return t;
    Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}
const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A return code as the package's own exception, in the forward and through the engine in the backward (the type is asked for with the interpreter held).
struct EntryError : torch::PyTorchError {
    using PyTorchError::PyTorchError;
    PyObject* python_type() override
    {
        static PyObject* const type = [] {
            PyObject* lib = PyImport_ImportModule("metis_hip._lib");
            PyObject* found = lib ? PyObject_GetAttrString(lib, "MetisHipError") : nullptr;
            Py_XDECREF(lib);
            if (!found) PyErr_Clear();
            return found ? found : PyExc_RuntimeError;
        }();
        return type;
    }
};
void checked(int rc, const char* what)
{
    if (rc != METIS_OK) throw EntryError(std::string(what) + ": " + metis_error_string(rc) + " (code " + std::to_string(rc) + ")");
}

// Gradients that may be differentiated no further: where a second time is prepared, using them says so.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto refuse = std::make_shared<torch::autograd::DelayedError>("metis_hip: trying to differentiate twice what is differentiable once", static_cast<int64_t>(grads.size()));
    return (*refuse)(std::move(grads));
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& weight, const std::optional<Tensor>& post_weight,
                                 const std::optional<Tensor>& gate_vector, int64_t gate_rows, double scale, double eps)
    {
        const Tensor post = post_weight.value_or(Tensor()), gate = gate_vector.value_or(Tensor());
        const c10::DeviceGuard on(x.device());
        const int64_t cols = x.size(-1), rows = x.numel() / cols;
        const Tensor h = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), n = at::empty(x.sizes(), y.options().memory_format(at::MemoryFormat::Contiguous));
        ctx->set_materialize_grads(false);
        const Tensor a = flat(x), b = flat(y), w = flat(weight), p = flat(post), g = flat(gate);
        checked(metis_residual_norm(in(a), dtype_of(x.scalar_type()), in(b), dtype_of(y.scalar_type()), in(w), in(p), in(g), gate_rows, static_cast<float>(scale),
                                    static_cast<float>(eps), rows, cols, out(h), out(n), stream_of(x)), "metis_residual_norm");
        const bool keep = post.defined() || (gate.defined() && gate.requires_grad());
        ctx->save_for_backward({h, keep ? y : Tensor(), weight, post, gate});
        ctx->saved_data["more"] = std::vector<double>{scale, eps, static_cast<double>(gate_rows), y.scalar_type() == at::kBFloat16 ? 1.0 : 0.0};
        return {h, n};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list given(8);
        if (!grads[0].defined() && !grads[1].defined()) return given;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor h = flat(saved[0]), weight = flat(saved[2]), post = flat(saved[3]), gate = flat(saved[4]), gh = flat(grads[0]), gn = flat(grads[1]);
        const c10::DeviceGuard on(h.device());
        const std::vector<double> more = ctx->saved_data["more"].toDoubleVector();
        const double scale = more[0], eps = more[1];
        const int64_t gate_rows = static_cast<int64_t>(more[2]), cols = h.size(-1), rows = h.numel() / cols;
        const at::ScalarType branch = more[3] != 0.0 ? at::kBFloat16 : at::kFloat;
        const at::TensorOptions stream_type = h.options().memory_format(at::MemoryFormat::Contiguous), branch_type = stream_type.dtype(branch);
        const bool same = !post.defined() && !gate.defined() && scale == 1.0 && h.scalar_type() == branch;      // the gradient of y is that of x
        // (inputs are counted without those that are not there)
        const bool want_x = ctx->needs_input_grad(0), want_y = ctx->needs_input_grad(1), want_g = gate.defined() && ctx->needs_input_grad(post.defined() ? 4 : 3);
        const Tensor y = post.defined() || want_g ? flat(saved[1]) : Tensor();
        Tensor gx, gy, gw, gp, gg;
        if (want_x || (same && want_y)) gx = at::empty(h.sizes(), stream_type);
        if (want_y && !same) gy = at::empty(h.sizes(), branch_type);
        if (ctx->needs_input_grad(2)) gw = at::empty({cols}, branch_type);
        if (post.defined() && ctx->needs_input_grad(3)) gp = at::empty({cols}, branch_type);
        if (want_g) gg = at::empty(gate.sizes(), branch_type);
        if (rows == 0) {
            for (Tensor* t : {&gx, &gy, &gw, &gp, &gg})
                if (t->defined()) t->zero_();
        }
        const size_t need = metis_residual_norm_backward_workspace_bytes(rows, cols, gate_rows);
        const Tensor workspace = at::empty({static_cast<int64_t>(need)}, stream_type.dtype(at::kByte));
        if (rows > 0)
            checked(metis_residual_norm_backward(in(h), dtype_of(h.scalar_type()), in(y), dtype_of(branch), in(weight), in(post), in(gate), gate_rows, static_cast<float>(scale),
                                                 static_cast<float>(eps), rows, cols, in(gh), in(gn), out(gx), out(gy), out(gw), out(gp), out(gg), out(workspace), need, stream_of(h)),
                    "metis_residual_norm_backward");
        if (want_x) given[0] = gx;
        if (want_y) given[1] = same ? gx : gy;
        given[2] = gw;
        given[3] = gp;
        given[4] = gg;
        return once(std::move(given));
    }
};

// the tensor with dense rows of any stride (halves of one product's rows are taken as they are), and that stride
std::pair<Tensor, int64_t> strided(const Tensor& t, int64_t rows, int64_t cols)
{
    if (t.is_contiguous()) return {t, cols};
    Tensor r = t.reshape({rows, cols});
    if (r.stride(1) != 1 || (rows > 1 && r.stride(0) < cols)) r = r.contiguous();
    return {r, std::max(r.stride(0), cols)};
}

struct SwiGLU : torch::autograd::Function<SwiGLU> {
    static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up)
    {
        const c10::DeviceGuard on(gate.device());
        const Tensor a = at::empty(gate.sizes(), gate.options().memory_format(at::MemoryFormat::Contiguous));
        ctx->save_for_backward({gate, up});
        if (gate.numel() == 0) return a;
        const int64_t cols = gate.size(-1), rows = gate.numel() / cols;
        const auto g = strided(gate, rows, cols), u = strided(up, rows, cols);
        checked(metis_swiglu(in(g.first), g.second, in(u.first), u.second, rows, cols, dtype_of(gate.scalar_type()), out(a), stream_of(gate)), "metis_swiglu");
        return a;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &gate = saved[0], &up = saved[1], da = grads[0].contiguous();
        const c10::DeviceGuard on(gate.device());
        const at::TensorOptions type = gate.options().memory_format(at::MemoryFormat::Contiguous);
        const Tensor dg = at::empty(gate.sizes(), type), du = at::empty(gate.sizes(), type);
        if (gate.numel() == 0) return once({ctx->needs_input_grad(0) ? dg : Tensor(), ctx->needs_input_grad(1) ? du : Tensor()});
        const int64_t cols = gate.size(-1), rows = gate.numel() / cols;
        const auto g = strided(gate, rows, cols), u = strided(up, rows, cols);
        checked(metis_swiglu_backward(in(g.first), g.second, in(u.first), u.second, in(da), rows, cols, dtype_of(gate.scalar_type()), out(dg), out(du), stream_of(gate)),
                "metis_swiglu_backward");
        return once({ctx->needs_input_grad(0) ? dg : Tensor(), ctx->needs_input_grad(1) ? du : Tensor()});
    }
};

// [..., heads, dim] as [tokens, heads, dim] with dense dimensions, and the strides of its tokens and heads (of a single one: none that counts)
struct HeadRows {
    Tensor t;
    int64_t token = 0, head = 0, heads = 0;
    HeadRows(const Tensor& given, int64_t tokens)
    {
        if (!given.defined()) return;
        heads = given.size(-2);
        const int64_t dim = given.size(-1);
        token = heads * dim;
        head = dim;
        t = given;
        if (t.is_contiguous()) return;
        t = given.reshape({tokens, heads, dim});
        if (t.stride(2) != 1) t = t.contiguous();
        if (tokens > 1) token = t.stride(0);
        if (heads > 1) head = t.stride(1);
    }
};

struct Rotary : torch::autograd::Function<Rotary> {
    // both results, undefined where there is nothing to turn
    static variable_list turn(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double factor, bool back)
    {
        const Tensor& any = q.defined() ? q : k;
        const c10::DeviceGuard on(any.device());
        const int64_t dim = any.size(-1), heads = any.size(-2), tokens = any.numel() > 0 ? any.numel() / (heads * dim) : 0;
        const at::TensorOptions type = any.options().memory_format(at::MemoryFormat::Contiguous);
        const Tensor to_q = q.defined() ? at::empty(q.sizes(), type) : Tensor(), to_k = k.defined() ? at::empty(k.sizes(), type) : Tensor();
        if (tokens > 0) {
            const HeadRows a(q, tokens), b(k, tokens);
            checked(metis_rotary(in(a.t), a.token, a.head, a.heads, in(b.t), b.token, b.head, b.heads, positions.const_data_ptr<int64_t>(), positions.numel(), in(inv_freq),
                                 inv_freq.scalar_type() == at::kDouble ? METIS_DTYPE_F64 : METIS_DTYPE_F32, tokens, dim, 2 * inv_freq.numel(), interleaved, back,
                                 static_cast<float>(factor), dtype_of(any.scalar_type()), out(to_q), out(to_k), stream_of(any)), "metis_rotary");
        }
        return {to_q, to_k};
    }

    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double factor)
    {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, inv_freq});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["factor"] = factor;
        return turn(q, k, positions, inv_freq, interleaved, factor, false);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list given(6);
        const Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), gk = ctx->needs_input_grad(1) ? grads[1] : Tensor();
        if (!gq.defined() && !gk.defined()) return given;
        const variable_list saved = ctx->get_saved_variables();
        const variable_list turned = turn(gq, gk, saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["factor"].toDouble(), true);
        given[0] = turned[0];
        given[1] = turned[1];
        return once(std::move(given));
    }
};

// Whether rotary takes the arguments as they are, positions dense (what is wrong with others the Python functions say).
bool plain_rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq)
{
    const int64_t lead = q.dim() - 2;
    const auto type = q.scalar_type(), freq = inv_freq.scalar_type();
    if (!q.is_cuda() || !k.is_cuda() || !positions.is_cuda() || !inv_freq.is_cuda() || lead < 1 || k.dim() != lead + 2 || k.scalar_type() != type ||
        (type != at::kBFloat16 && type != at::kFloat) || (freq != at::kDouble && freq != at::kFloat) || positions.scalar_type() != at::kLong || inv_freq.requires_grad())
        return false;
    const auto device = q.get_device();
    const int64_t dim = q.size(lead + 1), n = inv_freq.numel();
    if (k.get_device() != device || positions.get_device() != device || inv_freq.get_device() != device || k.size(lead + 1) != dim || dim % 2 || dim <= 0 || dim > 512 || q.size(lead) <= 0 ||
        q.size(lead) > 65536 || k.size(lead) <= 0 || k.size(lead) > 65536 || inv_freq.dim() != 1 || n <= 0 || 2 * n > dim || !inv_freq.is_contiguous() || !positions.is_contiguous())
        return false;
    int64_t ones = 0;
    while (ones < positions.dim() && positions.size(ones) == 1) ++ones;
    const int64_t own = positions.dim() - ones;
    if (own > lead) return false;
    for (int64_t i = 0; i < lead; ++i)
        if (k.size(i) != q.size(i) || (i >= lead - own && positions.size(i - (lead - own) + ones) != q.size(i))) return false;
    return true;
}

// The interpreter's lock given up: an allocation may wait for the device.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// a tensor or None; false with a Python error set
bool tensor_of(PyObject* o, Tensor* t)
{
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "a tensor or None, not %s", Py_TYPE(o)->tp_name);
        return false;
    }
    *t = THPVariable_Unpack(o);
    return true;
}

}  // namespace

PyObject* metis_recorded_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Tensor t[5];
    if (n != 8) {
        PyErr_SetString(PyExc_TypeError, "recorded_residual_norm(x, y, weight, post_weight, gate, gate_rows, scale, eps)");
        return nullptr;
    }
    for (int i = 0; i < 5; ++i)
        if (!tensor_of(a[i], &t[i])) return nullptr;
    const long long gate_rows = PyLong_AsLongLong(a[5]);
    const double scale = PyFloat_AsDouble(a[6]), eps = PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) return nullptr;
    if (!t[0].defined() || !t[1].defined() || !t[2].defined()) {
        PyErr_SetString(PyExc_TypeError, "recorded_residual_norm: x, y and weight are tensors");
        return nullptr;
    }
    variable_list r;
    {
        Unlocked unlocked;
        r = ResidualNorm::apply(t[0], t[1], t[2], t[3].defined() ? std::optional<Tensor>(t[3]) : std::nullopt, t[4].defined() ? std::optional<Tensor>(t[4]) : std::nullopt,
                                static_cast<int64_t>(gate_rows), scale, eps);
    }
    PyObject* h = THPVariable_Wrap(std::move(r[0]));
    PyObject* normed = h ? THPVariable_Wrap(std::move(r[1])) : nullptr;
    PyObject* both = normed ? PyTuple_Pack(2, h, normed) : nullptr;
    Py_XDECREF(h);
    Py_XDECREF(normed);
    return both;
    END_HANDLE_TH_ERRORS
}

PyObject* metis_recorded_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Tensor gate, up;
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "recorded_swiglu(gate, up)");
        return nullptr;
    }
    if (!tensor_of(a[0], &gate) || !tensor_of(a[1], &up)) return nullptr;
    if (!gate.defined() || !up.defined()) {
        PyErr_SetString(PyExc_TypeError, "recorded_swiglu: gate and up are tensors");
        return nullptr;
    }
    Tensor r;
    {
        Unlocked unlocked;
        r = SwiGLU::apply(gate, up);
    }
    return THPVariable_Wrap(std::move(r));
    END_HANDLE_TH_ERRORS
}

PyObject* metis_recorded_rotary(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Tensor t[4];
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "recorded_rotary(q, k, positions, inv_freq, interleaved, factor, checked)");
        return nullptr;
    }
    for (int i = 0; i < 4; ++i) {
        if (!tensor_of(a[i], &t[i])) return nullptr;
        if (!t[i].defined()) {
            PyErr_SetString(PyExc_TypeError, "recorded_rotary: q, k, positions and inv_freq are tensors");
            return nullptr;
        }
    }
    const int interleaved = PyObject_IsTrue(a[4]);
    const double factor = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) return nullptr;
    if (a[6] != Py_True) {
        for (int i = 0; i < 4; ++i)
            if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
        if (!plain_rotary(t[0], t[1], t[2], t[3])) Py_RETURN_NONE;
    }
    variable_list r;
    {
        Unlocked unlocked;
        if (at::GradMode::is_enabled() && (t[0].requires_grad() || t[1].requires_grad())) r = Rotary::apply(t[0], t[1], t[2], t[3], interleaved != 0, factor);
        else r = Rotary::turn(t[0], t[1], t[2], t[3], interleaved != 0, factor, false);
    }
    PyObject* q = THPVariable_Wrap(std::move(r[0]));
    PyObject* k = q ? THPVariable_Wrap(std::move(r[1])) : nullptr;
    PyObject* both = k ? PyTuple_Pack(2, q, k) : nullptr;
    Py_XDECREF(q);
    Py_XDECREF(k);
    return both;
    END_HANDLE_TH_ERRORS
}
