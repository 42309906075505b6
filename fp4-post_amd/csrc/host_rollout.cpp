// The rollout's operators from Python in one step, for calls that need nothing but the entry point: operands on the current device, of the types and layouts that it takes as
// they are, with no gradients to refuse.  Anything else is answered by None, and the Python functions (metis_hip/rollout.py, metis_hip/ops.py) say what is wrong with it, or copy what has
// to be copied.  Host code only; a decode step makes these calls for every layer, and the checks written in Python cost more than the launches.  Host time of a call, through the Python
// functions before and after: rotary_append of a token 15.5 -> 7.7 us, paged_attention of one sequence 12.5 -> 7.5, sample_tokens of a row 18 -> 14 (three launches), copy_pages of 15 pages
// 16 -> 7.1.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cmath>
#include <vector>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/metis_hip.h"
#include "host_autograd.h"

namespace {

using at::Tensor;

// The interpreter's lock given up: an allocation may wait for the device.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* not_here() { Py_RETURN_NONE; }

// tensors on one device, the current one, none of which asks for gradients
bool take(PyObject* const* a, Py_ssize_t n, const Tensor** t)
{
    const bool grad = at::GradMode::is_enabled();
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_CheckExact(a[i])) return false;
        t[i] = &THPVariable_Unpack(a[i]);
        if (!t[i]->is_cuda() || t[i]->get_device() != t[0]->get_device() || (grad && t[i]->requires_grad())) return false;
    }
    return t[0]->get_device() == c10::hip::current_device();
}
bool number(PyObject* o, double* v)
{
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
    *v = PyFloat_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}
// (in binary32, as the entry points take them)
bool finite32(double v) { return std::isfinite(static_cast<float>(v)); }
bool positive(double v) { return static_cast<float>(v) > 0.0f && finite32(v); }
uintptr_t address(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// [.., heads, dim] with dense dimensions; the strides of its rows and heads (of a single one: none that counts)
bool rows(const Tensor& t, int64_t* row, int64_t* head)
{
    if (t.stride(2) != 1) return false;
    *row = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
    *head = t.size(1) > 1 ? t.stride(1) : t.size(2);
    return true;
}
int cache_type(const Tensor& keys, const Tensor& values)
{
    if (keys.scalar_type() != values.scalar_type() || keys.dim() != 4 || values.dim() != 4 || !keys.is_contiguous() || !values.is_contiguous() || keys.size(0) != values.size(0) ||
        keys.size(1) != values.size(1) || keys.size(2) != values.size(3) || keys.size(3) != values.size(2))
        return -1;
    return keys.scalar_type() == at::kBFloat16 ? METIS_DTYPE_BF16 : keys.scalar_type() == at::kFloat8_e4m3fn ? METIS_DTYPE_E4M3 : -1;
}
template <class T> const T* data(const Tensor& t) { return static_cast<const T*>(t.const_data_ptr()); }
// of a tensor that the call writes: one that shares its numbers until it is written (a lazy clone) gets its own
template <class T> T* written(const Tensor& t) { return static_cast<T*>(t.mutable_data_ptr()); }

}  // namespace

// rotary_append(q, k, v, positions, inv_freq, slots, keys, values, interleaved, factor, key_scale, value_scale)
PyObject* metis_host_rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    const Tensor* t[8];
    double factor, key_scale, value_scale;
    if (n != 12 || !take(a, 8, t) || !PyBool_Check(a[8]) || !number(a[9], &factor) || !number(a[10], &key_scale) || !number(a[11], &value_scale)) return not_here();
    const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &positions = *t[3], &inv_freq = *t[4], &slots = *t[5], &keys = *t[6], &values = *t[7];
    const int type = cache_type(keys, values);
    if (type < 0 || q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || q.scalar_type() != at::kBFloat16 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16)
        return not_here();
    const int64_t tokens = q.size(0), dim = q.size(2), half = inv_freq.numel();
    const bool wide = inv_freq.scalar_type() == at::kDouble;
    if (tokens == 0 || k.size(0) != tokens || k.size(2) != dim || keys.size(1) != k.size(1) || keys.size(3) != dim || positions.scalar_type() != at::kLong || slots.scalar_type() != at::kLong ||
        positions.dim() != 1 || slots.dim() != 1 || positions.size(0) != tokens || slots.size(0) != tokens || !positions.is_contiguous() || !slots.is_contiguous() || inv_freq.dim() != 1 ||
        (!wide && inv_freq.scalar_type() != at::kFloat) || !inv_freq.is_contiguous() || half == 0 || 2 * half > dim || !positive(key_scale) || !positive(value_scale))
        return not_here();
    int64_t qt, qh, kt, kh, vt, vh;
    if (!rows(q, &qt, &qh) || !rows(k, &kt, &kh) || !rows(v, &vt, &vh)) return not_here();
    const bool interleaved = a[8] == Py_True;
    int rc;
    Tensor out;
    {
        Unlocked unlocked;
        out = at::empty({tokens, q.size(1), dim}, q.options().memory_format(at::MemoryFormat::Contiguous));
        rc = metis_rotary_append(data<void>(q), qt, qh, q.size(1), data<void>(k), kt, kh, k.size(1), data<void>(v), vt, vh, data<int64_t>(positions), data<void>(inv_freq),
                                 wide ? METIS_DTYPE_F64 : METIS_DTYPE_F32, data<int64_t>(slots), tokens, dim, 2 * half, interleaved, static_cast<float>(factor), keys.size(0), keys.size(2), type,
                                 static_cast<float>(key_scale), static_cast<float>(value_scale), written<void>(keys), written<void>(values), written<void>(out), stream_of(q));
    }
    return rc == METIS_OK ? THPVariable_Wrap(std::move(out)) : not_here();
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, keys, values, tables, lengths, scale or None, key_scale, value_scale)
PyObject* metis_host_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    const Tensor* t[5];
    double scale = 0.0, key_scale, value_scale;
    if (n != 8 || !take(a, 5, t) || (a[5] != Py_None && !number(a[5], &scale)) || !number(a[6], &key_scale) || !number(a[7], &value_scale)) return not_here();
    const Tensor &q = *t[0], &keys = *t[1], &values = *t[2], &tables = *t[3], &lengths = *t[4];
    const int type = cache_type(keys, values);
    if (type < 0 || q.dim() != 3 || q.scalar_type() != at::kBFloat16 || q.size(0) == 0 || q.size(2) != keys.size(3) || tables.dim() != 2 || tables.size(0) != q.size(0) ||
        tables.scalar_type() != at::kInt || (tables.size(1) > 1 && tables.stride(1) != 1) || lengths.dim() != 1 || lengths.size(0) != q.size(0) || lengths.scalar_type() != at::kInt ||
        !lengths.is_contiguous() || !positive(key_scale) || !positive(value_scale) || !finite32(scale))
        return not_here();
    const int64_t seqs = q.size(0), heads = q.size(1), dim = q.size(2), width = tables.size(1), page = keys.size(2);
    int64_t qs, qh;
    if (!rows(q, &qs, &qh) || qs % 8 || qh % 8 || address(q) % 16 || dim == 0) return not_here();
    if (a[5] == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(dim));
    int rc;
    Tensor out;
    {
        Unlocked unlocked;
        const at::TensorOptions options = q.options().memory_format(at::MemoryFormat::Contiguous);
        const size_t need = metis_paged_attention_workspace_bytes(seqs, heads, keys.size(1), dim, width * page);
        out = at::empty({seqs, heads, dim}, options);
        Tensor workspace;
        if (need > 16) workspace = at::empty({static_cast<int64_t>(need)}, options.dtype(at::kByte));
        rc = metis_paged_attention(data<void>(q), qs, qh, seqs, heads, keys.size(1), dim, data<void>(keys), data<void>(values), keys.size(0), page, type, data<int32_t>(tables), tables.stride(0),
                                   width, data<int32_t>(lengths), static_cast<float>(scale), static_cast<float>(key_scale), static_cast<float>(value_scale), written<void>(out),
                                   need > 16 ? written<void>(workspace) : nullptr, need, stream_of(q));
    }
    return rc == METIS_OK ? THPVariable_Wrap(std::move(out)) : not_here();
    END_HANDLE_TH_ERRORS
}

// copy_pages(keys, values, sources, destinations): True where it is done
PyObject* metis_host_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    const Tensor* t[2];
    if (n != 4 || !take(a, 2, t) || !PyList_Check(a[2]) || !PyList_Check(a[3]) || PyList_GET_SIZE(a[2]) != PyList_GET_SIZE(a[3])) return not_here();
    const Tensor &keys = *t[0], &values = *t[1];
    if (keys.dim() != 5 || values.dim() != 5 || cache_type(keys.size(0) ? keys[0] : keys, values.size(0) ? values[0] : values) < 0 || keys.size(0) != values.size(0) || !keys.is_contiguous() ||
        !values.is_contiguous())
        return not_here();
    const Py_ssize_t count = PyList_GET_SIZE(a[2]);
    std::vector<int64_t> pages(2 * static_cast<size_t>(count));
    for (int which = 0; which < 2; ++which)
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject* o = PyList_GET_ITEM(a[2 + which], i);
            if (!PyLong_CheckExact(o)) return not_here();
            const long long p = PyLong_AsLongLong(o);
            if (p == -1 && PyErr_Occurred()) { PyErr_Clear(); return not_here(); }
            pages[static_cast<size_t>(which * count + i)] = p;
        }
    const int64_t size = keys.size(2) * keys.size(3) * keys.size(4) * static_cast<int64_t>(keys.element_size());
    const int rc = metis_cache_copy_pages(written<void>(keys), written<void>(values), keys.size(0), keys.size(1), size, pages.data(), pages.data() + count, count, stream_of(keys));
    if (rc != METIS_OK) return not_here();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p)
PyObject* metis_host_sample_tokens(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    const Tensor* t[2];
    double settings[4];
    if (n != 6 || !take(a, 2, t)) return not_here();
    for (int i = 0; i < 4; ++i)
        if (!number(a[2 + i], &settings[i])) return not_here();
    const Tensor &logits = *t[0], &uniforms = *t[1];
    const bool f32 = logits.scalar_type() == at::kFloat;
    if (logits.dim() != 2 || uniforms.dim() != 1 || uniforms.size(0) != logits.size(0) || logits.size(0) == 0 || logits.size(1) == 0 || (!f32 && logits.scalar_type() != at::kBFloat16) ||
        uniforms.scalar_type() != at::kFloat || !uniforms.is_contiguous() || (logits.size(1) > 1 && logits.stride(1) != 1) || (logits.size(0) > 1 && logits.stride(0) < logits.size(1)))
        return not_here();
    const int64_t count = logits.size(0), vocab = logits.size(1);
    int rc;
    Tensor tokens, logprobs;
    {
        Unlocked unlocked;
        const at::TensorOptions options = uniforms.options().memory_format(at::MemoryFormat::Contiguous);
        const size_t need = metis_sample_tokens_workspace_bytes(count, vocab);
        tokens = at::empty({count}, options.dtype(at::kLong));
        logprobs = at::empty({count}, options);
        Tensor workspace;
        if (need) workspace = at::empty({static_cast<int64_t>(need)}, options.dtype(at::kByte));
        rc = metis_sample_tokens(data<void>(logits), count > 1 ? logits.stride(0) : vocab, f32 ? METIS_DTYPE_F32 : METIS_DTYPE_BF16, count, vocab, data<float>(uniforms), settings, nullptr,
                                 written<int64_t>(tokens), written<float>(logprobs), need ? written<void>(workspace) : nullptr, need, stream_of(logits));
    }
    if (rc != METIS_OK) return not_here();
    PyObject* first = THPVariable_Wrap(std::move(tokens));
    PyObject* second = first ? THPVariable_Wrap(std::move(logprobs)) : nullptr;
    PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}
