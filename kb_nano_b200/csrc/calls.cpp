// Native call path of the small operators.  A decode step launches kernels of a few microseconds, and checking five tensors and
// passing a dozen arguments from Python took longer than the launch (6.3 us a call, of which the launch 2.3; this way 2.9).  Each function
// here makes the checks of its namesake in ops.py on the tensors themselves, takes the current stream and calls the C ABI.  It
// returns True when the kernels are enqueued and False for anything it does not accept, a failed call included: ops.py
// then runs its own checks and calls, and raises the error with its reason.  So there is one set of errors, and this file only has to
// be right about what it accepts.
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
        if (ok_ && before_ != index_) c10::cuda::set_device(before_);
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

#define KBN_CALL(name) \
    { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {KBN_CALL(quant_mxfp4), KBN_CALL(silu_mul_quant_mxfp4), KBN_CALL(dequant_mxfp4), KBN_CALL(mxfp4_gemm_nt), KBN_CALL(mxfp4_linear),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Native call path of the small operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
