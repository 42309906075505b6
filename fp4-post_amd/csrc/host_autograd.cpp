// residual_norm and swiglu as nodes of torch's autograd, in compiled code.  Host code only: the arithmetic is libmetis_hip.so's, the checks of arguments are
// made by the Python functions that call these (metis_hip/block.py, metis_hip/ops.py).
//
// Both are kernels of some tens of microseconds in a training step, and a node written in Python costs more than that: recorded, run backward in the
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
