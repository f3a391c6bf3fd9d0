/*
 * Python module lfm_attn_py: the calls of include/lfm_gpu_attn.h on torch
 * tensors, for laii_b200/attn.py (reads the arguments that it passes, in order).
 *
 * Checks of tensors, allocation of outputs and the call on torch's current
 * stream in one step.  A small call is as long as its way to the launch: through
 * ctypes, with the checks and allocations in Python, a row norm of 64 rows with
 * its read-back took 17.3 us for 3.3 us on the device; two launches alone take
 * 5.  So: 8 to 9 us.
 * Functions return their outputs, or the status as an int where it is not 0.
 */
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

#include "lfm_gpu_attn.h"

namespace {

using at::Tensor;

uint32_t type_of(at::ScalarType t, const char *what) {
    TORCH_CHECK_VALUE(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, what, ": ", t, " (float32, float16 or bfloat16)");
    return t == at::kFloat ? LFM_GPU_TYPE_F32 : t == at::kHalf ? LFM_GPU_TYPE_F16 : LFM_GPU_TYPE_BF16;
}
at::ScalarType scalar_of(uint32_t type) {
    return type == LFM_GPU_TYPE_F32 ? at::kFloat : type == LFM_GPU_TYPE_F16 ? at::kHalf : at::kBFloat16;
}

/* The call's arguments in order; one that is not what it should be raises. */
struct Args {
    PyObject *const *at;
    Py_ssize_t n, i = 0;
    PyObject *next() {
        TORCH_CHECK_TYPE(i < n, "too few arguments");
        return at[i++];
    }
    int64_t integer() {
        const long long v = PyLong_AsLongLong(next());
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
    float real() {
        const double v = PyFloat_AsDouble(next());
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return (float)v;
    }
    bool flag() {
        const int v = PyObject_IsTrue(next());
        if (v < 0) throw python_error();
        return v != 0;
    }
    template <class T>
    T *address() {
        PyObject *o = next();
        if (o == Py_None) return nullptr;
        void *p = PyLong_AsVoidPtr(o);
        if (!p && PyErr_Occurred()) throw python_error();
        return static_cast<T *>(p);
    }
    /* None: an undefined tensor */
    Tensor tensor(const char *what) {
        PyObject *o = next();
        if (o == Py_None) return Tensor();
        TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
        return THPVariable_Unpack(o);
    }
};

/* The address of a contiguous tensor of `dims` dimensions on the device. */
void *dense(const Tensor &t, const char *what, at::ScalarType type, int64_t index, int64_t dims) {
    if (!t.defined()) return nullptr;
    TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == type && t.get_device() == index && t.dim() == dims && t.is_contiguous(), what,
                      " must be a contiguous ", dims, "-d ", type, " tensor on CUDA device ", index);
    return t.data_ptr();
}

/* Rows [tokens][heads][dim] with the heads of a token one behind the other; heads < 0: any number. */
struct Rows {
    void *p = nullptr;
    int64_t tokens = 0, heads = 0, stride = 0;
};
Rows rows(const Tensor &t, const char *what, int64_t heads, int64_t dim, at::ScalarType type, int64_t index) {
    TORCH_CHECK_VALUE(t.defined() && t.is_cuda() && t.dim() == 3 && t.size(2) == dim && (heads < 0 || t.size(1) == heads) &&
                          t.scalar_type() == type && t.get_device() == index,
                      what, " must be ", type, " [tokens, ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", dim,
                      "] on CUDA device ", index);
    TORCH_CHECK_VALUE(t.is_contiguous() || (t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == dim)), what, ": [tokens, heads, ", dim,
                      "] with the heads of a token one behind the other");
    /* the stride of one row says nothing */
    return {t.data_ptr(), t.size(0), t.size(1), t.size(0) != 1 ? t.stride(0) : t.size(1) * dim};
}

Tensor fresh(at::IntArrayRef size, at::ScalarType type, int64_t index) {
    return at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (c10::DeviceIndex)index), std::nullopt);
}
void *stream_of(int64_t index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
PyObject *wrap(const Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

/* (handle, device, x, delta, weight, eps, x_out, type of the rows or -1, q8) -> (x_out, rows, q8) */
PyObject *add_rmsnorm(PyObject *, PyObject *const *argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{argv, n};
    auto *h = a.address<lfm_gpu_moe_t>();
    const int64_t index = a.integer();
    const Tensor x = a.tensor("x"), delta = a.tensor("delta"), weight = a.tensor("weight");
    const float eps = a.real();
    Tensor x_out = a.tensor("x_out"), xb, q8;
    const int64_t xb_type = a.integer();
    const bool want_q8 = a.flag();
    TORCH_CHECK_VALUE(x.defined(), "x must be given");
    const void *xp = dense(x, "x", at::kFloat, index, 2);
    const int64_t T = x.size(0), D = x.size(1);
    const void *dp = nullptr;
    uint32_t dt = 0;
    if (delta.defined()) {
        dt = type_of(delta.scalar_type(), "delta");
        dp = dense(delta, "delta", delta.scalar_type(), index, 2);
        TORCH_CHECK_VALUE(delta.sizes() == x.sizes(), "delta must have the shape of x");
    }
    const void *wp = dense(weight, "weight", at::kFloat, index, 1);
    TORCH_CHECK_VALUE(!wp || weight.size(0) == D, "weight must have ", D, " values");
    TORCH_CHECK_VALUE(T <= UINT32_MAX && D <= UINT32_MAX, "x: ", T, " rows of ", D);
    if (x_out.defined()) {
        dense(x_out, "x_out", at::kFloat, index, 2);
        TORCH_CHECK_VALUE(x_out.sizes() == x.sizes(), "x_out must have the shape of x");
    } else {
        x_out = fresh({T, D}, at::kFloat, index);
    }
    if (xb_type >= 0) xb = fresh({T, D}, scalar_of((uint32_t)xb_type), index);
    if (want_q8) q8 = fresh({T, D / 256, 292}, at::kByte, index);
    const lfm_gpu_status_t st = lfm_gpu_add_rmsnorm(
        h, static_cast<const float *>(xp), dp, dt, (uint32_t)T, (uint32_t)D, static_cast<const float *>(wp), eps,
        static_cast<float *>(x_out.data_ptr()), xb.defined() ? xb.data_ptr() : nullptr, xb_type >= 0 ? (uint32_t)xb_type : 0,
        want_q8 ? q8.data_ptr() : nullptr, stream_of(index));
    if (st != LFM_GPU_OK) return PyLong_FromLong(st);
    THPObjectPtr o0(wrap(x_out)), o1(wrap(xb)), o2(wrap(q8));
    if (!o0 || !o1 || !o2) return nullptr;
    return PyTuple_Pack(3, o0.get(), o1.get(), o2.get());
    END_HANDLE_TH_ERRORS
}

/* (handle, device, q8, type) -> values */
PyObject *read_q8(PyObject *, PyObject *const *argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{argv, n};
    auto *h = a.address<lfm_gpu_moe_t>();
    const int64_t index = a.integer();
    const Tensor q8 = a.tensor("q8");
    const uint32_t type = (uint32_t)a.integer();
    TORCH_CHECK_VALUE(q8.defined(), "q8 must be given");
    const void *p = dense(q8, "q8", at::kByte, index, 3);
    const int64_t T = q8.size(0), D = q8.size(1) * 256;
    TORCH_CHECK_VALUE(q8.size(2) == 292 && T <= UINT32_MAX && D <= UINT32_MAX, "q8 must be [T, D / 256, 292]");
    const Tensor out = fresh({T, D}, scalar_of(type), index);
    const lfm_gpu_status_t st = lfm_gpu_q8k_read(h, p, (uint32_t)T, (uint32_t)D, type, out.data_ptr(), stream_of(index));
    return st != LFM_GPU_OK ? PyLong_FromLong(st) : wrap(out);
    END_HANDLE_TH_ERRORS
}

/* (handle, device, cache, batch, rope, q, k, v, q_out) -> q_out; the third to fifth are addresses of descriptors */
PyObject *append(PyObject *, PyObject *const *argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{argv, n};
    auto *h = a.address<lfm_gpu_moe_t>();
    const int64_t index = a.integer();
    const auto *kv = a.address<lfm_gpu_kv_t>();
    auto *batch = a.address<lfm_gpu_kv_batch_t>();
    const auto *rope = a.address<lfm_gpu_rope_t>();
    const Tensor q = a.tensor("q"), k = a.tensor("k"), v = a.tensor("v");
    Tensor q_out = a.tensor("q_out");
    TORCH_CHECK_VALUE((q.defined() || k.defined()) && k.defined() == v.defined(), "q, or k and v, or all three");
    const Tensor &first = q.defined() ? q : k;
    const at::ScalarType dt = first.scalar_type();
    const uint32_t type = type_of(dt, "q");
    const int64_t d = kv->head_dim;
    Rows qr, outr, kr, vr;
    int64_t T = 0;
    if (k.defined()) {
        kr = rows(k, "k", kv->n_kv_heads, d, dt, index);
        vr = rows(v, "v", kv->n_kv_heads, d, dt, index);
        T = kr.tokens;
    }
    if (q.defined()) {
        qr = rows(q, "q", -1, d, dt, index);
        T = qr.tokens;
        if (!q_out.defined()) q_out = fresh(q.sizes(), dt, index);
        outr = rows(q_out, "q_out", qr.heads, d, dt, index);
        TORCH_CHECK_VALUE(outr.tokens >= T, "q_out must have the rows of q");
    }
    TORCH_CHECK_VALUE(!k.defined() || (kr.tokens == T && vr.tokens == T), "q, k and v must have the same number of tokens");
    TORCH_CHECK_VALUE(T <= UINT32_MAX && qr.heads <= UINT32_MAX, "q: ", T, " tokens of ", qr.heads, " heads");
    batch->n_tokens = (uint32_t)T;
    const lfm_gpu_status_t st =
        lfm_gpu_kv_append(h, kv, batch, rope, type, (uint32_t)qr.heads, qr.p, (size_t)qr.stride, outr.p, (size_t)outr.stride, kr.p,
                          (size_t)kr.stride, vr.p, (size_t)vr.stride, stream_of(index));
    return st != LFM_GPU_OK ? PyLong_FromLong(st) : wrap(q_out);
    END_HANDLE_TH_ERRORS
}

/* (handle, device, cache, batch, tokens, type) -> (keys, values) */
PyObject *read(PyObject *, PyObject *const *argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{argv, n};
    auto *h = a.address<lfm_gpu_moe_t>();
    const int64_t index = a.integer();
    const auto *kv = a.address<lfm_gpu_kv_t>();
    auto *batch = a.address<lfm_gpu_kv_batch_t>();
    const int64_t T = a.integer();
    const uint32_t type = (uint32_t)a.integer();
    TORCH_CHECK_VALUE(T >= 0 && T <= UINT32_MAX, T, " tokens");
    const Tensor k = fresh({T, kv->n_kv_heads, kv->head_dim}, scalar_of(type), index);
    const Tensor v = fresh({T, kv->n_kv_heads, kv->head_dim}, scalar_of(type), index);
    batch->n_tokens = (uint32_t)T;
    const lfm_gpu_status_t st = lfm_gpu_kv_read(h, kv, batch, type, k.data_ptr(), v.data_ptr(), stream_of(index));
    if (st != LFM_GPU_OK) return PyLong_FromLong(st);
    THPObjectPtr o0(wrap(k)), o1(wrap(v));
    if (!o0 || !o1) return nullptr;
    return PyTuple_Pack(2, o0.get(), o1.get());
    END_HANDLE_TH_ERRORS
}

/* (handle, device, cache, batch, q, scale, causal, window, softcap, out) -> out */
PyObject *attend(PyObject *, PyObject *const *argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{argv, n};
    auto *h = a.address<lfm_gpu_moe_t>();
    const int64_t index = a.integer();
    const auto *kv = a.address<lfm_gpu_kv_t>();
    auto *batch = a.address<lfm_gpu_kv_batch_t>();
    const Tensor q = a.tensor("q");
    const float scale = a.real();
    const bool causal = a.flag();
    const int64_t window = a.integer();
    const float softcap = a.real();
    Tensor out = a.tensor("out");
    TORCH_CHECK_VALUE(q.defined(), "q must be given");
    TORCH_CHECK_VALUE(window >= 0 && window <= UINT32_MAX, "window=", window);
    const at::ScalarType dt = q.scalar_type();
    const uint32_t type = type_of(dt, "q");
    const Rows r = rows(q, "q", -1, kv->head_dim, dt, index);
    if (!out.defined()) out = fresh(q.sizes(), dt, index);
    const Rows o = rows(out, "out", r.heads, kv->head_dim, dt, index);
    TORCH_CHECK_VALUE(o.tokens >= r.tokens, "out must have the rows of q");
    TORCH_CHECK_VALUE(r.tokens <= UINT32_MAX && r.heads <= UINT32_MAX, "q: ", r.tokens, " tokens of ", r.heads, " heads");
    batch->n_tokens = (uint32_t)r.tokens;
    const lfm_gpu_status_t st =
        lfm_gpu_attn_forward(h, kv, batch, (uint32_t)r.heads, scale, causal, (uint32_t)window, softcap, type, r.p, (size_t)r.stride, o.p,
                             (size_t)o.stride, stream_of(index));
    return st != LFM_GPU_OK ? PyLong_FromLong(st) : wrap(out);
    END_HANDLE_TH_ERRORS
}

#define FN(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FN(add_rmsnorm), FN(read_q8), FN(append), FN(read), FN(attend), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "lfm_attn_py", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_lfm_attn_py() { return PyModule_Create(&kModule); }
