// Native call path of the small operators.  A decode step launches kernels of a few microseconds, and checking five tensors and
// passing a dozen arguments from Python took longer than the launch (6.3 us a call, of which the launch 2.3; this way 2.9).  Each function
// here makes the checks of its namesake in ops.py (moe.py) on the tensors themselves, takes the current stream and calls the C ABI.  It
// returns True when the kernels are enqueued and False for anything it does not accept, a failed call included: its namesake
// then runs its own checks and calls, and raises the error with its reason.  So there is one set of errors, and this file only has to
// be right about what it accepts.
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "kbn_fp8.h"

namespace {

using at::ScalarType;
using at::Tensor;

// A plain CUDA tensor argument (exactly torch.Tensor or torch.nn.Parameter), or null.
const Tensor* tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}
bool is_code(const Tensor& t) { return t.scalar_type() == ScalarType::Byte || t.scalar_type() == ScalarType::Float4_e2m1fn_x2; }
bool is_byte_scale(const Tensor& t) { return t.scalar_type() == ScalarType::Byte || t.scalar_type() == ScalarType::Float8_e8m0fnu; }

// Rows with contiguous values: [m, n], row stride ld (that of a single row is free and taken as its length).
struct Rows {
    const Tensor* t = nullptr;
    int64_t m = 0, n = 0, ld = 0;
    bool get(PyObject* o) {
        t = tensor(o);
        if (t == nullptr || t->dim() != 2) return false;
        m = t->size(0);
        n = t->size(1);
        ld = m > 1 ? t->stride(0) : n;
        return t->stride(1) == 1 || n <= 1;
    }
    bool is(int64_t rows, int64_t cols) const { return m == rows && n == cols; }
    bool dense() const { return ld == n; }
    void* ptr() const { return t->data_ptr(); }
};
struct Bf16Rows : Rows {
    bool get(PyObject* o) { return Rows::get(o) && t->scalar_type() == ScalarType::BFloat16; }
};
struct Codes : Rows {
    bool get(PyObject* o) { return Rows::get(o) && is_code(*t); }
};
// Packed scales of [rows, k] values.
struct Packed {
    const Tensor* t = nullptr;
    bool get(PyObject* o, int64_t rows, int64_t k) {
        t = tensor(o);
        return t != nullptr && t->scalar_type() == ScalarType::Byte && t->numel() >= kbn_packed_mxfp4_bytes(rows, k) && t->is_contiguous() &&
               (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) == 0;
    }
};

// The tensors' one device, made current for the call; its current stream.
class Launch {
public:
    template <typename... T>
    explicit Launch(const Tensor* first, const T*... rest) : index_(first->device().index()) {
        ok_ = index_ >= 0 && ((rest == nullptr || rest->device().index() == index_) && ...);
        if (!ok_) return;
        before_ = c10::cuda::current_device();
        if (before_ != index_) c10::cuda::set_device(index_);
        stream_ = c10::cuda::getCurrentCUDAStream(index_).stream();
    }
    ~Launch() {
        try {
            if (ok_ && before_ != index_) c10::cuda::set_device(before_);
        } catch (...) {      // the call's own result stands
        }
    }
    Launch(const Launch&) = delete;
    Launch& operator=(const Launch&) = delete;
    bool ok() const { return ok_; }
    kbn_stream_t stream() const { return stream_; }

private:
    c10::DeviceIndex index_, before_ = 0;
    bool ok_ = false;
    kbn_stream_t stream_ = nullptr;
};

// bf16 [n], contiguous, or None.
bool get_bias(PyObject* o, int64_t n, const Tensor*& t) {
    t = nullptr;
    if (o == Py_None) return true;
    t = tensor(o);
    return t != nullptr && t->scalar_type() == ScalarType::BFloat16 && t->numel() == n && t->is_contiguous();
}

// The C call itself, without the interpreter lock: a launch may have to wait for room in the stream's queue.
template <typename F>
bool enqueued(F&& f) {
    PyThreadState* const state = PyEval_SaveThread();
    const int rc = f();
    PyEval_RestoreThread(state);
    return rc == KBN_OK;
}

template <typename F>
PyObject* guarded(F&& f) {      // no C++ exception leaves the module
    try {
        if (f()) Py_RETURN_TRUE;
    } catch (...) {
    }
    Py_RETURN_FALSE;
}

typedef int (*QuantFn)(const void*, int64_t, int64_t, int64_t, void*, int64_t, void*, int64_t, void*, kbn_stream_t);

// (x, out_fp4, out_scale | None, packed_sf | None); halves: 2 for gate | up.
bool quant(QuantFn fn, int halves, PyObject* const* a, Py_ssize_t n_args) {
    Bf16Rows x;
    Codes q;
    Rows s;
    Packed p;
    if (n_args != 4 || !x.get(a[0]) || !q.get(a[1]) || x.n % (32 * halves) != 0 || x.n == 0 || x.m == 0) return false;
    const int64_t k = x.n / halves;
    if (!q.is(x.m, k / 2)) return false;
    if (a[2] != Py_None && !(s.get(a[2]) && is_byte_scale(*s.t) && s.is(x.m, k / 32))) return false;
    if (a[3] != Py_None && !p.get(a[3], x.m, k)) return false;
    if (s.t == nullptr && p.t == nullptr) return false;
    const Launch at(x.t, q.t, s.t, p.t);
    void *const xp = x.ptr(), *const qp = q.ptr(), *const sp = s.t ? s.ptr() : nullptr, *const pp = p.t ? p.t->data_ptr() : nullptr;
    return at.ok() && enqueued([&] { return fn(xp, x.m, k, x.ld, qp, q.ld, sp, s.ld, pp, at.stream()); });
}

PyObject* quant_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] { return quant(kbn_quant_mxfp4, 1, a, n); });
}
PyObject* silu_mul_quant_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] { return quant(kbn_silu_mul_quant_mxfp4, 2, a, n); });
}

// (q, scale, out)
PyObject* dequant_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Codes q;
        Rows s;
        Bf16Rows o;
        if (n != 3 || !q.get(a[0]) || !s.get(a[1]) || !is_byte_scale(*s.t) || !o.get(a[2]) || o.n % 32 != 0 || o.n == 0 || o.m == 0) return false;
        if (!q.is(o.m, o.n / 2) || !s.is(o.m, o.n / 32)) return false;
        const Launch at(o.t, q.t, s.t);
        void *const qp = q.ptr(), *const sp = s.ptr(), *const op = o.ptr();
        return at.ok() && enqueued([&] { return kbn_dequant_mxfp4(qp, q.ld, sp, s.ld, o.m, o.n, op, o.ld, at.stream()); });
    });
}

// (a_q, a_sf, b_q, b_sf, out, bias | None)
PyObject* mxfp4_gemm_nt(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Codes q, w;
        Packed qs, ws;
        Bf16Rows o;
        const Tensor* bias;
        if (n != 6 || !q.get(a[0]) || !w.get(a[2]) || q.n != w.n || q.n % 16 != 0 || q.n == 0 || !q.dense() || !w.dense() || q.m == 0 || w.m == 0) return false;
        const int64_t k = 2 * q.n;
        if (!qs.get(a[1], q.m, k) || !ws.get(a[3], w.m, k) || !o.get(a[4]) || !o.is(q.m, w.m) || !get_bias(a[5], w.m, bias)) return false;
        const Launch at(q.t, qs.t, w.t, ws.t, o.t, bias);
        void *const qp = q.ptr(), *const sp = qs.t->data_ptr(), *const wp = w.ptr(), *const wsp = ws.t->data_ptr(), *const bp = bias ? bias->data_ptr() : nullptr,
             *const op = o.ptr();
        return at.ok() && enqueued([&] { return kbn_mxfp4_gemm_nt(qp, sp, wp, wsp, bp, op, o.ld, q.m, w.m, k, at.stream()); });
    });
}

// (x, a_q, a_sf, b_q, b_sf, out, bias | None)
PyObject* mxfp4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Bf16Rows x, o;
        Codes q, w;
        Packed qs, ws;
        const Tensor* bias;
        if (n != 7 || !x.get(a[0]) || !q.get(a[1]) || !w.get(a[3]) || x.n % 32 != 0 || x.n == 0 || x.m == 0 || w.m == 0) return false;
        if (!q.is(x.m, x.n / 2) || w.n != x.n / 2 || !q.dense() || !w.dense()) return false;
        if (!qs.get(a[2], x.m, x.n) || !ws.get(a[4], w.m, x.n) || !o.get(a[5]) || !o.is(x.m, w.m) || !get_bias(a[6], w.m, bias)) return false;
        const Launch at(x.t, q.t, qs.t, w.t, ws.t, o.t, bias);
        void *const xp = x.ptr(), *const qp = q.ptr(), *const sp = qs.t->data_ptr(), *const wp = w.ptr(), *const wsp = ws.t->data_ptr(),
             *const bp = bias ? bias->data_ptr() : nullptr, *const op = o.ptr();
        return at.ok() && enqueued([&] { return kbn_mxfp4_linear(xp, x.ld, x.m, x.n, qp, sp, wp, wsp, bp, op, o.ld, w.m, at.stream()); });
    });
}

bool is_shape(const Tensor& t, int64_t a, int64_t b, int64_t c) {
    return t.dim() == 3 && t.size(0) == a && t.size(1) == b && t.size(2) == c && t.is_contiguous();
}
bool get_int(PyObject* o, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}
bool get_float(PyObject* o, float& v) {
    if (!PyFloat_CheckExact(o)) return false;
    v = static_cast<float>(PyFloat_AS_DOUBLE(o));
    return true;
}

// moe.few_tokens_moe's arguments in its order, all of them; returns the output, or False.
PyObject* few_tokens_moe(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    try {
        Bf16Rows x, out;
        Rows logits;
        int64_t top_k, n_group, topk_group;
        float renorm_floor, scale;
        if (n_args != 18 || !x.get(a[0]) || !logits.get(a[1]) || x.m == 0 || logits.m != x.m || x.m > 16 || x.n % 128 != 0) Py_RETURN_FALSE;
        const bool logits_bf16 = logits.t->scalar_type() == ScalarType::BFloat16;
        if (!logits_bf16 && logits.t->scalar_type() != ScalarType::Float) Py_RETURN_FALSE;
        const Tensor *w13 = tensor(a[2]), *s13 = tensor(a[3]), *w2 = tensor(a[4]), *s2 = tensor(a[5]);
        if (w13 == nullptr || s13 == nullptr || w2 == nullptr || s2 == nullptr || w2->dim() != 3) Py_RETURN_FALSE;
        if (!get_int(a[6], top_k) || !PyUnicode_CheckExact(a[7]) || !get_int(a[9], n_group) || !get_int(a[10], topk_group) || !PyBool_Check(a[11]) ||
            !get_float(a[12], renorm_floor) || !get_float(a[13], scale) || !PyBool_Check(a[14]))
            Py_RETURN_FALSE;
        const bool softmax = PyUnicode_CompareWithASCIIString(a[7], "softmax") == 0;
        if (!softmax && PyUnicode_CompareWithASCIIString(a[7], "sigmoid") != 0) Py_RETURN_FALSE;
        const int64_t t = x.m, h = x.n, e = logits.n;
        const bool fp8 = w13->scalar_type() == ScalarType::Float8_e4m3fn && w2->scalar_type() == ScalarType::Float8_e4m3fn;
        if (!fp8 && !(is_code(*w13) && is_code(*w2))) Py_RETURN_FALSE;
        const int64_t i = fp8 ? w2->size(2) : 2 * w2->size(2);
        if (i % 128 != 0 || i == 0 || top_k <= 0) Py_RETURN_FALSE;
        if (fp8) {
            if (!is_shape(*w13, e, 2 * i, h) || !is_shape(*w2, e, h, i) || s13->scalar_type() != ScalarType::Float || s2->scalar_type() != ScalarType::Float ||
                !is_shape(*s13, e, 2 * i / 128, h / 128) || !is_shape(*s2, e, h / 128, i / 128))
                Py_RETURN_FALSE;
        } else if (!is_shape(*w13, e, 2 * i, h / 2) || !is_shape(*w2, e, h, i / 2) || !is_byte_scale(*s13) || !is_byte_scale(*s2) ||
                   !is_shape(*s13, e, 2 * i, h / 32) || !is_shape(*s2, e, h, i / 32)) {
            Py_RETURN_FALSE;
        }
        const Tensor *bias = nullptr, *out_w = nullptr, *out_ids = nullptr;
        if (a[8] != Py_None) {
            bias = tensor(a[8]);
            if (bias == nullptr || bias->scalar_type() != ScalarType::Float || bias->numel() != e || !bias->is_contiguous()) Py_RETURN_FALSE;
        }
        if (a[15] != Py_None && !(out.get(a[15]) && out.is(t, h))) Py_RETURN_FALSE;
        if ((a[16] == Py_None) != (a[17] == Py_None)) Py_RETURN_FALSE;
        if (a[16] != Py_None) {
            out_w = tensor(a[16]);
            out_ids = tensor(a[17]);
            if (out_w == nullptr || out_ids == nullptr || out_w->scalar_type() != ScalarType::Float || out_ids->scalar_type() != ScalarType::Int ||
                out_w->dim() != 2 || out_ids->dim() != 2 || out_w->size(0) != t || out_w->size(1) != top_k || out_ids->size(0) != t || out_ids->size(1) != top_k ||
                !out_w->is_contiguous() || !out_ids->is_contiguous())
                Py_RETURN_FALSE;
        }
        const Launch at(x.t, logits.t, w13, s13, w2, s2, bias, out.t, out_w, out_ids);
        const int64_t bytes = kbn_moe_few_tokens_workspace_bytes(t, top_k, h, i);
        if (!at.ok() || bytes == 0) Py_RETURN_FALSE;
        // on the calling stream's account: the allocator hands it to nobody else before this call's kernels have run
        const Tensor workspace = at::empty({bytes}, x.t->options().dtype(ScalarType::Byte));
        const Tensor result = out.t != nullptr ? *out.t : at::empty({t, h}, x.t->options());
        void *const xp = x.ptr(), *const lp = logits.ptr(), *const w13p = w13->data_ptr(), *const s13p = s13->data_ptr(), *const w2p = w2->data_ptr(),
             *const s2p = s2->data_ptr(), *const rp = result.data_ptr(), *const wp = workspace.data_ptr();
        const float* const bp = bias != nullptr ? static_cast<const float*>(bias->data_ptr()) : nullptr;
        float* const owp = out_w != nullptr ? static_cast<float*>(out_w->data_ptr()) : nullptr;
        int32_t* const oip = out_ids != nullptr ? static_cast<int32_t*>(out_ids->data_ptr()) : nullptr;
        const int64_t ld_out = out.t != nullptr ? out.ld : h;
        const bool done = enqueued([&] {
            return kbn_moe_few_tokens(xp, x.ld, t, lp, logits_bf16, logits.ld, e, softmax, bp, n_group, topk_group, top_k, a[11] == Py_True, renorm_floor, scale,
                                      a[14] == Py_True, fp8 ? 0 : 1, w13p, s13p, w2p, s2p, h, i, rp, ld_out, owp, oip, wp, bytes, at.stream());
        });
        if (!done) Py_RETURN_FALSE;
        if (out.t != nullptr) {
            Py_INCREF(a[15]);
            return a[15];
        }
        return THPVariable_Wrap(result);
    } catch (...) {
    }
    Py_RETURN_FALSE;
}

#define KBN_CALL(name) \
    { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {KBN_CALL(quant_mxfp4), KBN_CALL(silu_mul_quant_mxfp4), KBN_CALL(dequant_mxfp4), KBN_CALL(mxfp4_gemm_nt), KBN_CALL(mxfp4_linear),
                         KBN_CALL(few_tokens_moe),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Native call path of the small operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
