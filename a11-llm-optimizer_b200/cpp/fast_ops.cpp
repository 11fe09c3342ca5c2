// fast_ops.cpp - a11spec._fast: the argument checks and calls of the layer
// operators (a11spec.ops.add_rms_norm, linear, chunk_attention) in C++.
//
// One decoded token calls each of them several times per layer, and the kernels
// take 2 to 8 us: checked in Python and called through ctypes a call takes 8 to
// 13 us on the host, from here 3 to 5 with the outputs given and 4 to 8 where it
// makes them. Semantics, arguments and errors are
// documented in a11spec/ops.py; the kernels are those of the C ABI
// (include/a11spec.h).
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <exception>
#include <sstream>
#include <string>

#include "a11spec.h"

namespace {

PyObject *error_class = nullptr;  // a11spec.A11Error

struct Refused {  // becomes an A11Error
    int code;
    std::string message;
};

template <typename... T>
[[noreturn]] void refuse(int code, const T &...parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw Refused{code, s.str()};
}

void check(int rc) {
    if (rc != A11S_OK) throw Refused{rc, a11s_last_error()};
}

// A tensor argument; null for None.
const at::Tensor *tensor(PyObject *o, const char *name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) refuse(A11S_EINVAL, name, " must be a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor &cuda_tensor(PyObject *o, const char *op, const char *name) {
    const at::Tensor *t = tensor(o, name);
    if (!t) refuse(A11S_EINVAL, op, ": ", name, " must be a tensor");
    if (!t->is_cuda()) refuse(A11S_EINVAL, op, ": CUDA tensors expected (", name, ")");
    return *t;
}

// Element stride between the rows of t [..., dim]: unit column stride, rows evenly spaced.
int64_t row_stride(const at::Tensor &t, const char *name, int64_t dim) {
    const auto sizes = t.sizes();
    if (sizes.empty() || sizes.back() != dim) refuse(A11S_EINVAL, name, " must be [..., ", dim, "], got ", sizes);
    if (t.is_contiguous() || t.numel() == 0) return dim;
    const auto strides = t.strides();
    if (strides.back() != 1 && dim > 1) refuse(A11S_EINVAL, name, " must have unit column stride");
    int64_t inner = -1, rows = 0;  // the innermost axis of more than one row; an axis of one row has no stride
    int64_t next = 0;
    for (int64_t i = (int64_t)sizes.size() - 2; i >= 0; --i) {
        if (sizes[i] == 1) continue;
        if (inner < 0) inner = strides[i];
        else if (strides[i] != next) refuse(A11S_EINVAL, name, " rows must be evenly spaced");
        next = strides[i] * sizes[i];
        rows = 1;
    }
    return rows ? inner : dim;
}
int64_t rows_of(const at::Tensor &t, const char *name, int64_t dim, at::ScalarType type, at::DeviceIndex dev) {
    if (!t.is_cuda() || t.get_device() != dev) refuse(A11S_EINVAL, name, " must be on cuda:", (int)dev);
    if (t.scalar_type() != type) refuse(A11S_EINVAL, name, " must be ", type, ", got ", t.scalar_type());
    return row_stride(t, name, dim);
}
// Pointer of a dense vector of n elements; null for null.
void *vector_of(const at::Tensor *t, const char *name, int64_t n, at::ScalarType type, at::DeviceIndex dev) {
    if (!t) return nullptr;
    if (!t->is_cuda() || t->get_device() != dev || t->scalar_type() != type || t->numel() != n || !t->is_contiguous())
        refuse(A11S_EINVAL, name, " must be ", n, " contiguous ", type, " elements on cuda:", (int)dev);
    return t->data_ptr();
}
int32_t fit(int64_t v, const char *what) {
    if (v < 0 || v > INT32_MAX) refuse(A11S_EUNSUPPORTED, what, " ", v, " does not fit 32 bits");
    return (int32_t)v;
}
PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }
PyObject *wrap_or_none(PyObject *given, const at::Tensor &made) {
    if (given != Py_None) {
        Py_INCREF(given);
        return given;
    }
    if (made.defined()) return wrap(made);
    Py_RETURN_NONE;
}
double number(PyObject *o, const char *name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(A11S_EINVAL, name, " must be a number");
    }
    return v;
}
int64_t integer(PyObject *o, const char *name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(A11S_EINVAL, name, " must be an integer");
    }
    return v;
}

template <typename F>
PyObject *guarded(F f) {
    try {
        return f();
    } catch (const Refused &r) {
        PyObject *e = error_class ? PyObject_CallFunction(error_class, "is", r.code, r.message.c_str()) : nullptr;
        if (e) {
            PyErr_SetObject(error_class, e);
            Py_DECREF(e);
        } else if (!PyErr_Occurred()) {
            PyErr_SetString(PyExc_RuntimeError, r.message.c_str());
        }
    } catch (...) {  // torch's own keep their types: an allocation that fails is torch.OutOfMemoryError
        if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}
bool arity(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
    return false;
}

// (x, weight, residual, eps, out_dtype, out, scales, sum_out) -> (out, scales, sum)
PyObject *add_rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (!arity(n_args, 8)) return nullptr;
    return guarded([&]() -> PyObject * {
        const at::Tensor &x = cuda_tensor(a[0], "add_rms_norm", "x");
        const at::Tensor *weight = tensor(a[1], "weight"), *residual = tensor(a[2], "residual"), *out = tensor(a[5], "out"),
                         *scales = tensor(a[6], "scales"), *sum = tensor(a[7], "sum_out");
        const at::ScalarType type = x.scalar_type();
        if ((type != at::kFloat && type != at::kBFloat16) || x.dim() == 0 || x.sizes().back() == 0)
            refuse(A11S_EINVAL, "add_rms_norm: x must be float32 or bfloat16 [..., dim], got ", type, " ", x.sizes());
        const auto dev = x.get_device();
        const int64_t dim = x.sizes().back(), n = x.numel(), rows = n / dim;
        const int code = type == at::kFloat ? A11S_F32 : A11S_BF16;
        c10::cuda::OptionalCUDAGuard guard(x.device());
        const int64_t xs = rows_of(x, "x", dim, type, dev);
        if (!weight) refuse(A11S_EINVAL, "weight must be a tensor");
        const void *wp = vector_of(weight, "weight", dim, type, dev);
        at::ScalarType out_type = type;
        if (a[4] != Py_None) {
            if (!THPDtype_Check(a[4])) refuse(A11S_EINVAL, "add_rms_norm: out_dtype must be a torch.dtype");
            out_type = reinterpret_cast<THPDtype *>(a[4])->scalar_type;
        } else if (out) {
            out_type = out->scalar_type();
        }
        at::Tensor new_out, new_scales, new_sum;
        if (!out) {
            new_out = at::empty(x.sizes(), x.options().dtype(out_type));
            out = &new_out;
        } else if (out->scalar_type() != out_type) {
            refuse(A11S_EINVAL, "add_rms_norm: out is ", out->scalar_type(), ", out_dtype ", out_type);
        }
        const bool e4m3 = out_type == at::kFloat8_e4m3fn;
        const int64_t os = rows_of(*out, "out", dim, e4m3 ? at::kFloat8_e4m3fn : type, dev);
        if (e4m3 && !scales) {
            new_scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
            scales = &new_scales;
        } else if (scales && !e4m3) {
            refuse(A11S_EINVAL, "add_rms_norm: scales go with e4m3 output");
        }
        float *sp = static_cast<float *>(vector_of(scales, "scales", rows, at::kFloat, dev));
        int64_t rs = 0, hs = 0;
        bool same = out->numel() == n;
        if (residual) {
            rs = rows_of(*residual, "residual", dim, type, dev);
            if (!sum) {
                new_sum = at::empty(x.sizes(), x.options());
                sum = &new_sum;
            }
            hs = rows_of(*sum, "sum_out", dim, type, dev);
            same = same && residual->numel() == n && sum->numel() == n;
        } else if (sum) {
            refuse(A11S_EINVAL, "add_rms_norm: sum_out without a residual");
        }
        if (!same) refuse(A11S_EINVAL, "add_rms_norm: x, residual, sum_out and out must have the same rows");
        check(a11s_add_rms_norm(code, x.data_ptr(), xs, residual ? residual->data_ptr() : nullptr, rs, wp, fit(rows, "rows"),
                                fit(dim, "dim"), (float)number(a[3], "eps"), sum ? sum->data_ptr() : nullptr, hs,
                                e4m3 ? A11S_E4M3 : code, out->data_ptr(), os, sp, c10::cuda::getCurrentCUDAStream(dev).stream()));
        PyObject *r = PyTuple_New(3);
        PyTuple_SET_ITEM(r, 0, wrap_or_none(a[5], new_out));
        PyTuple_SET_ITEM(r, 1, wrap_or_none(a[6], new_scales));
        PyTuple_SET_ITEM(r, 2, wrap_or_none(a[7], new_sum));
        return r;
    });
}

// (x, weight, bias, activation code, gate, gate_bias, residual, x_scale, weight_scale, gate_scale, out, ws) -> out
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (!arity(n_args, 12)) return nullptr;
    return guarded([&]() -> PyObject * {
        const at::Tensor &x = cuda_tensor(a[0], "linear", "x");
        const at::Tensor *weight = tensor(a[1], "weight"), *bias = tensor(a[2], "bias"), *gate = tensor(a[4], "gate"),
                         *gate_bias = tensor(a[5], "gate_bias"), *residual = tensor(a[6], "residual"),
                         *x_scale = tensor(a[7], "x_scale"), *w_scale = tensor(a[8], "weight_scale"),
                         *g_scale = tensor(a[9], "gate_scale"), *out = tensor(a[10], "out"), *ws = tensor(a[11], "ws");
        if (!weight || weight->dim() != 2 || x.dim() == 0) refuse(A11S_EINVAL, "linear: x [..., K] and weight [N, K] expected");
        const int64_t N = weight->size(0), K = weight->size(1);
        const at::ScalarType type = x.scalar_type();
        if (type != at::kBFloat16 && type != at::kFloat8_e4m3fn)
            refuse(A11S_EINVAL, "linear: x must be bfloat16 or float8_e4m3fn, got ", type);
        const auto dev = x.get_device();
        const int64_t rows = K ? x.numel() / K : 0;
        c10::cuda::OptionalCUDAGuard guard(x.device());
        const int64_t xs = rows_of(x, "x", K, type, dev);
        const void *wp = vector_of(weight, "weight", N * K, type, dev);
        if (gate && gate->sizes() != weight->sizes())
            refuse(A11S_EINVAL, "linear: gate ", gate->sizes(), " differs from weight ", weight->sizes());
        const void *gp = vector_of(gate, "gate", N * K, type, dev);
        at::Tensor new_out;
        if (!out) {
            auto shape = x.sizes().vec();
            shape.back() = N;
            new_out = at::empty(shape, x.options().dtype(at::kBFloat16));
            out = &new_out;
        }
        const int64_t os = rows_of(*out, "out", N, at::kBFloat16, dev);
        int64_t rs = 0;
        bool same = out->numel() == rows * N;
        if (residual) {
            rs = rows_of(*residual, "residual", N, at::kBFloat16, dev);
            same = same && residual->numel() == rows * N;
        }
        if (!same) refuse(A11S_EINVAL, "linear: out and residual must have x's ", rows, " rows");
        void *wsp = nullptr;
        size_t wsb = 0;
        if (ws) {
            wsp = vector_of(ws, "ws", ws->numel(), at::kByte, dev);
            wsb = (size_t)ws->numel();
        }
        check(a11s_linear(type == at::kBFloat16 ? A11S_BF16 : A11S_E4M3, x.data_ptr(), xs,
                          static_cast<float *>(vector_of(x_scale, "x_scale", rows, at::kFloat, dev)), wp,
                          static_cast<float *>(vector_of(w_scale, "weight_scale", N, at::kFloat, dev)), gp,
                          static_cast<float *>(vector_of(g_scale, "gate_scale", N, at::kFloat, dev)),
                          vector_of(bias, "bias", N, at::kBFloat16, dev), vector_of(gate_bias, "gate_bias", N, at::kBFloat16, dev),
                          fit(rows, "rows"), fit(K, "K"), fit(N, "N"), (int32_t)integer(a[3], "activation"),
                          residual ? residual->data_ptr() : nullptr, rs, out->data_ptr(), os, wsp, wsb,
                          c10::cuda::getCurrentCUDAStream(dev).stream()));
        return wrap_or_none(a[10], new_out);
    });
}

// (q, k_pool, v_pool, page_table, ctx_lens, n_new, scale, max_kv_len, want_lse, out, lse, ws) -> (out, lse, ws)
PyObject *chunk_attention(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (!arity(n_args, 12)) return nullptr;
    return guarded([&]() -> PyObject * {
        const at::Tensor &q = cuda_tensor(a[0], "chunk_attention", "q");
        const at::Tensor *k = tensor(a[1], "k_pool"), *v = tensor(a[2], "v_pool"), *table = tensor(a[3], "page_table"),
                         *ctx = tensor(a[4], "ctx_lens"), *n_new = tensor(a[5], "n_new"), *out = tensor(a[9], "out"),
                         *lse = tensor(a[10], "lse"), *ws = tensor(a[11], "ws");
        if (!k || !v || !table || !ctx || q.dim() != 4 || k->dim() != 4)
            refuse(A11S_EINVAL, "chunk_attention: q [B, n, Hq, D], pools [P, 16, Hkv, D], page_table and ctx_lens expected");
        const int64_t B = q.size(0), N = q.size(1), Hq = q.size(2), D = q.size(3), P = k->size(0), Hkv = k->size(2);
        if (k->size(1) != A11S_PAGE_TOKENS || k->size(3) != D || v->sizes() != k->sizes())
            refuse(A11S_EINVAL, "pool shape must be [P, 16, Hkv, D] for K and V");
        const auto dev = q.get_device();
        c10::cuda::OptionalCUDAGuard guard(q.device());
        if (q.scalar_type() != at::kBFloat16 || (D > 1 && q.stride(3) != 1) || (Hq > 1 && q.stride(2) != D))
            refuse(A11S_EINVAL, "q must be bfloat16 with a token's heads dense");
        const int64_t qs = N > 1 ? q.stride(1) : B > 1 ? q.stride(0) : Hq * D;
        if (B > 1 && q.stride(0) != N * qs) refuse(A11S_EINVAL, "q tokens must be evenly spaced");
        const void *kp = vector_of(k, "k_pool", k->numel(), at::kBFloat16, dev);
        const void *vp = vector_of(v, "v_pool", k->numel(), at::kBFloat16, dev);
        if (table->dim() != 2 || table->size(0) != B)
            refuse(A11S_EINVAL, "page_table must be [", B, ", maxpages], got ", table->sizes());
        const int64_t pages = table->size(1);
        const int32_t *tp = static_cast<int32_t *>(vector_of(table, "page_table", B * pages, at::kInt, dev));
        const int32_t *cp = static_cast<int32_t *>(vector_of(ctx, "ctx_lens", B, at::kInt, dev));
        const int32_t *np = static_cast<int32_t *>(vector_of(n_new, "n_new", B, at::kInt, dev));
        const float scale = a[6] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)number(a[6], "scale");
        const int32_t kv = fit(a[7] == Py_None ? pages * A11S_PAGE_TOKENS : integer(a[7], "max_kv_len"), "max_kv_len");
        at::Tensor new_out, new_lse, new_ws;
        if (!out) {
            new_out = at::empty(q.sizes(), q.options());
            out = &new_out;
        }
        void *op = vector_of(out, "out", q.numel(), at::kBFloat16, dev);
        if (!lse && a[8] == Py_True) {
            new_lse = at::empty({B, N, Hq}, q.options().dtype(at::kFloat));
            lse = &new_lse;
        }
        float *lp = static_cast<float *>(vector_of(lse, "lse", B * N * Hq, at::kFloat, dev));
        const int32_t b = fit(B, "batch"), n = fit(N, "n"), hq = fit(Hq, "Hq"), hkv = fit(Hkv, "Hkv"), d = fit(D, "D");
        if (!ws) {
            const int64_t need = (int64_t)a11s_chunk_attention_workspace_bytes(b, n, hq, hkv, d, kv);
            new_ws = at::empty({std::max<int64_t>(need, 256)}, q.options().dtype(at::kByte));
            ws = &new_ws;
        }
        void *wsp = vector_of(ws, "ws", ws->numel(), at::kByte, dev);
        check(a11s_chunk_attention(q.data_ptr(), qs, kp, vp, fit(P, "pages"), tp, fit(pages, "maxpages"), cp, np, b, n, hq, hkv, d, kv,
                                   scale, op, lp, wsp, (size_t)ws->numel(), c10::cuda::getCurrentCUDAStream(dev).stream()));
        PyObject *r = PyTuple_New(3);
        PyTuple_SET_ITEM(r, 0, wrap_or_none(a[9], new_out));
        PyTuple_SET_ITEM(r, 1, wrap_or_none(a[10], new_lse));
        PyTuple_SET_ITEM(r, 2, wrap_or_none(a[11], new_ws));
        return r;
    });
}

// (tensor, dim) -> the row stride the operators would use (any device).
PyObject *row_stride_py(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (!arity(n_args, 2)) return nullptr;
    return guarded([&]() -> PyObject * {
        const at::Tensor *t = tensor(a[0], "tensor");
        if (!t) refuse(A11S_EINVAL, "tensor must be a tensor");
        return PyLong_FromLongLong(row_stride(*t, "tensor", integer(a[1], "dim")));
    });
}
PyObject *set_error_class(PyObject *, PyObject *cls) {
    Py_XDECREF(error_class);
    Py_INCREF(cls);
    error_class = cls;
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"add_rms_norm", FAST(add_rms_norm)},
                         {"linear", FAST(linear)},
                         {"chunk_attention", FAST(chunk_attention)},
                         {"row_stride", FAST(row_stride_py)},
                         {"set_error_class", set_error_class, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
