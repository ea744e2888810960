// wf_torch.cpp - the Python entry of the operators around a layer of routed FP8 experts.
//
// One call checks its tensors, allocates its outputs on their device and hands raw
// pointers to the C ABI (include/wfb200.h).  It is compiled because at one token the
// kernels take a few microseconds and a call made through ctypes took 13 to 22 of them
// (argument conversion, stream look-up, an allocation per output through the
// interpreter); wanferenz_b200/ops.py documents each function.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/wfb200.h"

namespace {

using at::ScalarType;

PyObject *g_check = nullptr;  // _lib.check: raises WfError for a status

// Thrown with the Python error set.
struct Raised {};

[[noreturn]] void raise(PyObject *type, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Raised();
}

std::string shape_text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

// A CUDA tensor of one of the types (on `dev` when given), contiguous and 16-byte aligned: another
// layout, or a view that starts off a 16-byte boundary, is copied first.
at::Tensor tensor(PyObject *o, const char *name, std::initializer_list<ScalarType> types, const char *types_text,
                  const at::Device *dev = nullptr) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a tensor, not %.80s", name, Py_TYPE(o)->tp_name);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda()) raise(PyExc_ValueError, "wanferenz_b200 operators run on CUDA tensors only (%s is not)", name);
    bool ok = false;
    for (ScalarType s : types) ok |= t.scalar_type() == s;
    if (!ok) raise(PyExc_TypeError, "%s has dtype %s, expected %s", name, c10::toString(t.scalar_type()), types_text);
    if (dev && t.device() != *dev)
        raise(PyExc_ValueError, "%s is on %s, expected %s", name, t.device().str().c_str(), dev->str().c_str());
    if (t.is_neg()) return t.resolve_neg().contiguous();  // its memory holds the values' negatives
    if (!t.is_contiguous()) return t.contiguous();
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t;
}

void want_shape(const at::Tensor &t, const char *name, at::IntArrayRef s) {
    if (t.sizes() != s)
        raise(PyExc_ValueError, "%s has shape %s, expected %s", name, shape_text(t.sizes()).c_str(), shape_text(s).c_str());
}

long long integer(PyObject *o, const char *name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (PyErr_ExceptionMatches(PyExc_OverflowError)) {
            PyErr_Clear();
            raise(PyExc_ValueError, "%s out of range", name);
        }
        throw Raised();
    }
    return v;
}
double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v != 0;
}

// An output: each has an allocation of its own, so that a caller may resize, free or save one and leave
// the others alone.  (One allocation for all of a call's took 0.4 to 0.9 us less at a few tokens, and
// growing an output in place then ran into its neighbour.)
at::Tensor empty(at::IntArrayRef s, ScalarType type, const at::Device &dev) {
    return at::detail::empty_cuda(s, type, dev, std::nullopt);
}

void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int kind(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? WF_SCALE_F32 : WF_SCALE_E8M0; }

// Calls f(stream) with `dev` current and raises for a status other than WF_OK.
template <class F>
void run(const at::Device &dev, const char *name, F f) {
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
    const int rc = f((void *)c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (rc) {
        PyObject *r = PyObject_CallFunction(g_check, "is", rc, name);
        Py_XDECREF(r);
        if (!r) throw Raised();
    }
}

PyObject *pack(std::initializer_list<at::Tensor> ts) {
    PyObject *r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) throw Raised();
    Py_ssize_t i = 0;
    for (const at::Tensor &t : ts) {
        PyObject *o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
        if (!o) {
            Py_DECREF(r);
            throw Raised();
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

#define WF_ENTRY(name, count)                                                              \
    PyObject *name##_impl(PyObject *const *a);                                             \
    PyObject *name(PyObject *, PyObject *const *a, Py_ssize_t n) {                         \
        HANDLE_TH_ERRORS                                                                   \
        if (n != count) return PyErr_Format(PyExc_TypeError, #name " takes " #count " arguments"); \
        try {                                                                              \
            return name##_impl(a);                                                         \
        } catch (const Raised &) {                                                         \
            return nullptr;                                                                \
        }                                                                                  \
        END_HANDLE_TH_ERRORS                                                               \
    }                                                                                      \
    PyObject *name##_impl(PyObject *const *a)

const char *const F32_BF16 = "torch.float32 or torch.bfloat16", *const BF16 = "torch.bfloat16", *const F32 = "torch.float32";
const char *const E4M3 = "torch.float8_e4m3fn", *const SCALES = "torch.float32 or torch.float8_e8m0fnu";
const char *const I32 = "torch.int32";

// x, weight, eps, residual, norm_out, ue8m0, scale dtype -> q, s, y, h
WF_ENTRY(rms_norm_quant, 7) {
    const at::Tensor x = tensor(a[0], "x", {at::kBFloat16}, BF16);
    const at::Device dev = x.device();
    if (x.dim() < 1) raise(PyExc_ValueError, "x must have at least one dimension");
    const int64_t d = x.size(-1);
    if (d == 0 || d % 128 || d > 16384) raise(PyExc_ValueError, "last dim %lld must be a multiple of 128, at most 16384", (long long)d);
    const at::Tensor w = tensor(a[1], "weight", {at::kFloat, at::kBFloat16}, F32_BF16, &dev);
    want_shape(w, "weight", {d});
    const double eps = number(a[2]);
    at::Tensor res, h, y;
    if (a[3] != Py_None) {
        res = tensor(a[3], "residual", {at::kBFloat16}, BF16, &dev);
        want_shape(res, "residual", x.sizes());
        h = empty(x.sizes(), at::kBFloat16, dev);
    }
    const bool ue8m0 = truth(a[5]);
    if (!THPDtype_Check(a[6])) raise(PyExc_TypeError, "scale_dtype must be a torch.dtype");
    const ScalarType st = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
    if (st != at::kFloat && st != at::kFloat8_e8m0fnu) raise(PyExc_TypeError, "unsupported scale dtype %s", c10::toString(st));
    if (st != at::kFloat && !ue8m0) raise(PyExc_ValueError, "e8m0 scales need scale_fmt (power-of-two rounding)");
    c10::DimVector ss(x.sizes());
    ss.back() = d / 128;
    const at::Tensor q = empty(x.sizes(), at::kFloat8_e4m3fn, dev), s = empty(ss, st, dev);
    if (truth(a[4])) y = empty(x.sizes(), at::kBFloat16, dev);
    if (x.numel())
        run(dev, "wf_rms_norm_quant", [&](void *stream) {
            return wf_rms_norm_quant(ptr(x), ptr(res), ptr(w), w.scalar_type() == at::kBFloat16, x.numel() / d, d, (float)eps,
                                     ue8m0, ptr(q), ptr(s), kind(s), ptr(y), ptr(h), stream);
        });
    return pack({q, s, y, h});
}

// logits, topk, bias, score, n_groups, topk_groups, top2, renorm, scale -> weights, indices
WF_ENTRY(route_topk, 9) {
    const at::Tensor l = tensor(a[0], "logits", {at::kFloat, at::kBFloat16}, F32_BF16);
    const at::Device dev = l.device();
    if (l.dim() != 2) raise(PyExc_ValueError, "logits must be [T, E]");
    const int64_t t = l.size(0), e = l.size(1);
    const long long k = integer(a[1], "topk"), score = integer(a[3], "score_func"), g = integer(a[4], "n_groups");
    const long long keep = integer(a[5], "topk_groups");
    at::Tensor bias;
    if (a[2] != Py_None) {
        bias = tensor(a[2], "bias", {at::kFloat}, F32, &dev);
        want_shape(bias, "bias", {e});
    }
    if (e < 1 || e > 512) raise(PyExc_ValueError, "%lld experts: 1 to 512 are supported", (long long)e);
    if (g < 1 || g > 32 || e % g || keep < 1 || keep > g)
        raise(PyExc_ValueError, "n_groups %lld (1 to 32) must divide the %lld experts, topk_groups %lld lie in 1..n_groups", g,
              (long long)e, keep);
    if (k < 1 || k > 16 || k > keep * (e / g))
        raise(PyExc_ValueError, "topk %lld must be in 1..min(16, experts of topk_groups groups)", k);
    const bool top2 = truth(a[6]), renorm = truth(a[7]);
    const double scale = number(a[8]);
    const at::Tensor w = empty({t, k}, at::kFloat, dev), i = empty({t, k}, at::kLong, dev);
    if (t)
        run(dev, "wf_route_topk", [&](void *stream) {
            return wf_route_topk(ptr(l), l.scalar_type() == at::kBFloat16, (const float *)ptr(bias), t, (int32_t)e, (int32_t)k,
                                 (int32_t)score, (int32_t)g, (int32_t)keep, top2, renorm, (float)scale, (float *)ptr(w),
                                 (int64_t *)ptr(i), stream);
        });
    return pack({w, i});
}

// indices, n_experts, expert_offset -> offsets, tokens, slots
WF_ENTRY(expert_dispatch, 3) {
    const at::Tensor x = tensor(a[0], "indices", {at::kLong, at::kInt}, "torch.int64 or torch.int32");
    const at::Device dev = x.device();
    if (x.dim() != 2) raise(PyExc_ValueError, "indices must be [T, k]");
    const int64_t t = x.size(0), k = x.size(1);
    const long long n = integer(a[1], "n_experts"), base = integer(a[2], "expert_offset");
    if (k < 1 || k > 16 || n < 1 || n > 512 || t * k > 1 << 30)
        raise(PyExc_ValueError, "indices [%lld, %lld] over %lld experts: k in 1..16, 1 to 512 experts, at most 2^30 pairs",
              (long long)t, (long long)k, n);
    if (base < 0 || base > 0x7fffffff - 512) raise(PyExc_ValueError, "expert_offset %lld out of range", base);
    const at::Tensor offsets = empty({n + 1}, at::kInt, dev), tokens = empty({t * k}, at::kInt, dev);
    const at::Tensor slots = empty({t, k}, at::kInt, dev);
    if (!t) return pack({offsets.zero_(), tokens, slots});
    const size_t need = wf_expert_dispatch_workspace_bytes(t, (int32_t)k, (int32_t)n);
    at::Tensor ws;
    if (need) ws = empty({(int64_t)need}, at::kByte, dev);
    run(dev, "wf_expert_dispatch", [&](void *stream) {
        return wf_expert_dispatch(ptr(x), x.scalar_type() == at::kLong, t, (int32_t)k, (int32_t)n, base, (int32_t *)ptr(offsets),
                                  (int32_t *)ptr(tokens), (int32_t *)ptr(slots), ptr(ws), need, stream);
    });
    return pack({offsets, tokens, slots});
}

// a, a_s, w, w_s, offsets, rows, out -> out
WF_ENTRY(grouped_fp8_gemm, 7) {
    const at::Tensor x = tensor(a[0], "a", {at::kFloat8_e4m3fn}, E4M3);
    const at::Device dev = x.device();
    const at::Tensor w = tensor(a[2], "w", {at::kFloat8_e4m3fn}, E4M3, &dev);
    const at::Tensor offsets = tensor(a[4], "offsets", {at::kInt}, I32, &dev);
    if (x.dim() != 2 || w.dim() != 3 || offsets.dim() != 1)
        raise(PyExc_ValueError, "a must be [M, K], w [E, N, K] and offsets [E + 1]");
    const int64_t m = x.size(0), k = x.size(1), e = w.size(0), n = w.size(1);
    if (k == 0 || k % 128 || k > 1 << 20 || n == 0 || n % 8 || n > 1 << 20 || e < 1 || e > 512 || e * n > 1 << 30)
        raise(PyExc_ValueError, "E %lld, N %lld, K %lld: E in 1..512, N a multiple of 8, K a multiple of 128 (at most 2^20 each)",
              (long long)e, (long long)n, (long long)k);
    want_shape(w, "w", {e, n, k});
    want_shape(offsets, "offsets", {e + 1});
    const at::Tensor x_s = tensor(a[1], "a_s", {at::kFloat, at::kFloat8_e8m0fnu}, SCALES, &dev);
    want_shape(x_s, "a_s", {m, k / 128});
    const at::Tensor w_s = tensor(a[3], "w_s", {at::kFloat, at::kFloat8_e8m0fnu}, SCALES, &dev);
    want_shape(w_s, "w_s", {e, (n + 127) / 128, k / 128});
    at::Tensor rows;
    int64_t r = m;
    if (a[5] != Py_None) {
        rows = tensor(a[5], "rows", {at::kInt}, I32, &dev);
        if (rows.dim() != 1) raise(PyExc_ValueError, "rows must be [R]");
        r = rows.size(0);
    }
    if (m > 1 << 30 || r > 1 << 30) raise(PyExc_ValueError, "%lld rows of a, %lld rows: at most 2^30 are supported", (long long)m, (long long)r);
    at::Tensor out;
    if (a[6] == Py_None) {
        out = empty({r, n}, at::kBFloat16, dev);
    } else {
        out = tensor(a[6], "out", {at::kBFloat16}, BF16, &dev);
        want_shape(out, "out", {r, n});
        if (!out.is_same(THPVariable_Unpack(a[6]))) raise(PyExc_ValueError, "out must be contiguous and 16-byte aligned");
    }
    if (r) {
        if (!m) raise(PyExc_ValueError, "a has no rows to take");
        // a graph that saved the caller's out must see that its values change
        if (a[6] != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
        at::Tensor ws;
        const size_t need = wf_grouped_fp8_workspace_bytes(rows.defined(), r, (int32_t)e, k);
        if (need) ws = empty({(int64_t)need}, at::kByte, dev);
        run(dev, "wf_grouped_fp8_gemm", [&](void *stream) {
            return wf_grouped_fp8_gemm(ptr(x), ptr(x_s), kind(x_s), ptr(w), ptr(w_s), kind(w_s), (const int32_t *)ptr(offsets),
                                       (const int32_t *)ptr(rows), m, r, (int32_t)e, n, k, ptr(out), ptr(ws), need, stream);
        });
    }
    return THPVariable_Wrap(out);
}

// rows, slots, weights, shared, out dtype -> y
WF_ENTRY(expert_combine, 5) {
    const at::Tensor rows = tensor(a[0], "rows", {at::kBFloat16}, BF16);
    const at::Device dev = rows.device();
    const at::Tensor slots = tensor(a[1], "slots", {at::kInt}, I32, &dev);
    if (rows.dim() != 2 || slots.dim() != 2) raise(PyExc_ValueError, "rows must be [R, D] and slots [T, k]");
    const int64_t r = rows.size(0), d = rows.size(1), t = slots.size(0), k = slots.size(1);
    if (d == 0 || d % 8 || d > 1 << 20 || k < 1 || k > 16 || r > 0x7fffffff)
        raise(PyExc_ValueError, "rows [%lld, %lld], slots [%lld, %lld]: D must be a multiple of 8 up to 2^20, k in 1..16",
              (long long)r, (long long)d, (long long)t, (long long)k);
    at::Tensor w, shared;
    if (a[2] != Py_None) {
        w = tensor(a[2], "weights", {at::kFloat}, F32, &dev);
        want_shape(w, "weights", {t, k});
    }
    if (a[3] != Py_None) {
        shared = tensor(a[3], "shared", {at::kBFloat16}, BF16, &dev);
        want_shape(shared, "shared", {t, d});
    }
    if (!THPDtype_Check(a[4])) raise(PyExc_TypeError, "out_dtype must be a torch.dtype");
    const ScalarType ot = reinterpret_cast<THPDtype *>(a[4])->scalar_type;
    if (ot != at::kBFloat16 && ot != at::kFloat) raise(PyExc_TypeError, "out_dtype %s is not bfloat16 or float32", c10::toString(ot));
    const at::Tensor y = empty({t, d}, ot, dev);
    if (t)
        run(dev, "wf_expert_combine", [&](void *stream) {
            return wf_expert_combine(ptr(rows), r, (const int32_t *)ptr(slots), (const float *)ptr(w), ptr(shared), t, (int32_t)k, d,
                                     ptr(y), ot == at::kFloat, stream);
        });
    return THPVariable_Wrap(y);
}

PyObject *set_check(PyObject *, PyObject *f) {
    Py_XSETREF(g_check, Py_NewRef(f));
    Py_RETURN_NONE;
}

#define WF_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {WF_METHOD(rms_norm_quant), WF_METHOD(route_topk),     WF_METHOD(expert_dispatch),
                           WF_METHOD(grouped_fp8_gemm), WF_METHOD(expert_combine), {"set_check", set_check, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_wfb200_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__wfb200_torch() { return PyModule_Create(&g_module); }
