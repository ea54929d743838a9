// enc_bind.cpp -- the host side of the encoder's layer operators where nothing has to be copied: one
// call from Python checks the tensors, makes the outputs and enqueues the kernel on torch's current
// stream.  A call of a few microseconds on the GPU is otherwise spent mostly in Python and ctypes (one
// query's norm and rotation: 3.9 us of kernel, 16 us of host).
//
// Each function returns its outputs, or None where an operand cannot be used as it lies or is not as the
// operator wants it: ragrt_b200/encoder.py then copies or says what is wrong.  An int is the library's
// status.  The library's entry points come by address (bind), from the one ctypes has loaded.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ragrt_b200.h"

namespace {

decltype(&ragrt_enc_packed_attention) f_attention = nullptr;
decltype(&ragrt_enc_qk_norm_rope) f_rope = nullptr;
decltype(&ragrt_enc_gated_ffn) f_ffn = nullptr;
decltype(&ragrt_enc_gated_ffn_backward) f_ffn_backward = nullptr;
decltype(&ragrt_enc_gated_ffn_workspace) f_ffn_workspace = nullptr;

// The current device, where the first tensor of a call lies on it; -1 otherwise.
int device_of(PyObject* o) {
    if (!THPVariable_Check(o)) return -1;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == c10::cuda::current_device() ? (int)t.get_device() : -1;
}
// A strided tensor on that device; false for anything else.
bool take(PyObject* o, int device, const at::Tensor** t) {
    if (!THPVariable_Check(o)) return false;
    *t = &THPVariable_Unpack(o);
    return device >= 0 && (*t)->is_cuda() && (*t)->get_device() == device && (*t)->layout() == at::kStrided;
}
bool aligned(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
bool solid(const at::Tensor& t) { return t.is_contiguous() && aligned(t); }
// dtype code of a 16-bit type, or -1
int code(const at::Tensor& t) {
    return t.scalar_type() == at::kHalf ? RAGRT_F16 : t.scalar_type() == at::kBFloat16 ? RAGRT_BF16 : -1;
}
// Row stride of [T, H, D] rows that can be used in place, or 0 (as _row_stride in encoder.py).
int64_t row_stride(const at::Tensor& t) {
    const int64_t T = t.size(0), H = t.size(1), D = t.size(2);
    if ((t.stride(2) != 1 && D > 1) || (t.stride(1) != D && H > 1) || !aligned(t)) return 0;
    if (T <= 1) return H * D;
    return t.stride(0) >= H * D && t.stride(0) % 8 == 0 ? t.stride(0) : 0;
}
bool fits(int64_t n) { return n >= 0 && n <= 0x7FFFFFFF; }
// A new tensor on t's device, straight from the allocator of torch's CUDA tensors.
at::Tensor fresh(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
    return at::Tensor(at::detail::empty_cuda(shape, type, t.device(), std::nullopt));
}
at::Tensor like(const at::Tensor& t, at::IntArrayRef shape) { return fresh(t, shape, t.scalar_type()); }
void* stream(int device) { return (void*)at::cuda::getCurrentCUDAStream(device).stream(); }

// A C++ exception becomes Python's error, as torch itself translates it (out of memory above all).
template <typename F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    return f();
    END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a, r, f, b, w;
    if (!PyArg_ParseTuple(args, "KKKKK", &a, &r, &f, &b, &w)) return nullptr;
    f_attention = (decltype(f_attention))a;
    f_rope = (decltype(f_rope))r;
    f_ffn = (decltype(f_ffn))f;
    f_ffn_backward = (decltype(f_ffn_backward))b;
    f_ffn_workspace = (decltype(f_ffn_workspace))w;
    Py_RETURN_NONE;
}

// packed_attention(q, k, v, cu_seqlens, causal, scale)
PyObject* packed_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 6 || !f_attention) Py_RETURN_NONE;
        const int dev = device_of(a[0]);
        const at::Tensor *q, *k, *v, *cu;
        if (!take(a[0], dev, &q) || !take(a[1], dev, &k) || !take(a[2], dev, &v) || !take(a[3], dev, &cu)) Py_RETURN_NONE;
        const int dt = code(*q);
        if (dt < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || q->dim() != 3 ||
            k->dim() != 3 || !k->sizes().equals(v->sizes()) || q->size(0) != k->size(0) || q->size(2) != k->size(2) ||
            cu->dim() != 1 || cu->size(0) < 1 || cu->scalar_type() != at::kInt || !cu->is_contiguous() ||
            !fits(q->size(0)) || !fits(q->size(1)) || !fits(q->size(2)) || !fits(k->size(1)) || !fits(cu->size(0)))
            Py_RETURN_NONE;
        const int64_t qs = row_stride(*q), ks = row_stride(*k), vs = row_stride(*v);
        if (!qs || !ks || !vs) Py_RETURN_NONE;
        const int causal = PyObject_IsTrue(a[4]);
        const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)q->size(2)) : PyFloat_AsDouble(a[5]);
        if (causal < 0 || PyErr_Occurred()) return nullptr;
        at::Tensor out = like(*q, q->sizes());
        const int rc = f_attention(q->data_ptr(), k->data_ptr(), v->data_ptr(), (const int32_t*)cu->data_ptr(), out.data_ptr(),
                                   (int32_t)q->size(0), (int32_t)cu->size(0) - 1, (int32_t)q->size(1),
                                   (int32_t)k->size(1), (int32_t)q->size(2), qs, ks, vs, q->size(1) * q->size(2),
                                   (float)scale, causal, dt, stream(dev));
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out));
    });
}

// qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9 || !f_rope) Py_RETURN_NONE;
        const int dev = device_of(a[0]);
        const at::Tensor *q, *k, *c, *s, *pos, *w[2] = {nullptr, nullptr};
        if (!take(a[0], dev, &q) || !take(a[1], dev, &k) || !take(a[2], dev, &c) || !take(a[3], dev, &s) ||
            !take(a[4], dev, &pos))
            Py_RETURN_NONE;
        const int dt = code(*q);
        if (dt < 0 || k->scalar_type() != q->scalar_type() || q->dim() != 3 || k->dim() != 3 || q->size(0) != k->size(0) ||
            q->size(2) != k->size(2) || !fits(q->size(0)) || !fits(q->size(1)) || !fits(q->size(2)) || !fits(k->size(1)))
            Py_RETURN_NONE;
        for (int i = 0; i < 2; ++i) {
            if (a[5 + i] == Py_None) continue;
            if (!take(a[5 + i], dev, &w[i]) || w[i]->scalar_type() != q->scalar_type() || w[i]->dim() != 1 ||
                w[i]->size(0) != q->size(2) || !solid(*w[i]))
                Py_RETURN_NONE;
        }
        if (c->dim() != 2 || !c->sizes().equals(s->sizes()) || c->scalar_type() != at::kFloat ||
            s->scalar_type() != at::kFloat || !solid(*c) || !solid(*s) || !fits(c->size(0)) || !fits(2 * c->size(1)) ||
            pos->dim() != 1 || pos->size(0) != q->size(0) || !pos->is_contiguous() ||
            (pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong))
            Py_RETURN_NONE;
        const int64_t qs = row_stride(*q), ks = row_stride(*k);
        if (!qs || !ks) Py_RETURN_NONE;
        const double eps = PyFloat_AsDouble(a[7]);
        const int inter = PyObject_IsTrue(a[8]);
        if (inter < 0 || PyErr_Occurred()) return nullptr;
        at::Tensor qo = like(*q, q->sizes()), ko = like(*k, k->sizes());
        const int rc = f_rope(q->data_ptr(), k->data_ptr(), w[0] ? w[0]->data_ptr() : nullptr, w[1] ? w[1]->data_ptr() : nullptr,
                              (const float*)c->data_ptr(), (const float*)s->data_ptr(), pos->data_ptr(),
                              (int32_t)pos->element_size(), qo.data_ptr(), ko.data_ptr(), (int32_t)q->size(0),
                              (int32_t)q->size(1), (int32_t)k->size(1), (int32_t)q->size(2), (int32_t)(2 * c->size(1)),
                              (int32_t)c->size(0), qs, ks, q->size(1) * q->size(2), k->size(1) * k->size(2), (float)eps,
                              inter, dt, stream(dev));
        if (rc) return PyLong_FromLong(rc);
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(qo)), THPVariable_Wrap(std::move(ko)));
    });
}

// x [M, K], w_gate and w_up [F, K] in place, one type; its code or -1
int ffn_operands(const at::Tensor& x, const at::Tensor& g, const at::Tensor& u) {
    if (x.dim() != 2 || g.dim() != 2 || !g.sizes().equals(u.sizes()) || g.size(1) != x.size(1) ||
        g.scalar_type() != x.scalar_type() || u.scalar_type() != x.scalar_type() || !solid(x) || !solid(g) || !solid(u) ||
        !fits(x.size(0)) || !fits(g.size(0)) || !fits(x.size(1)))
        return -1;
    return code(x);
}

// gated_ffn(x, w_gate, w_up, act, keep)
PyObject* gated_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 5 || !f_ffn) Py_RETURN_NONE;
        const int dev = device_of(a[0]);
        const at::Tensor *x, *g, *u;
        if (!take(a[0], dev, &x) || !take(a[1], dev, &g) || !take(a[2], dev, &u)) Py_RETURN_NONE;
        const int dt = ffn_operands(*x, *g, *u), keep = PyObject_IsTrue(a[4]);
        const long act = PyLong_AsLong(a[3]);
        if (keep < 0 || PyErr_Occurred()) return nullptr;
        if (dt < 0) Py_RETURN_NONE;
        const int64_t M = x->size(0), F = g->size(0), K = x->size(1);
        at::Tensor h = like(*x, {M, F}), gate, up;
        if (keep) {
            gate = fresh(*x, {M, F}, at::kFloat);
            up = fresh(*x, {M, F}, at::kFloat);
        }
        const int rc = f_ffn(x->data_ptr(), g->data_ptr(), u->data_ptr(), h.data_ptr(), keep ? (float*)gate.data_ptr() : nullptr,
                             keep ? (float*)up.data_ptr() : nullptr, (int32_t)M, (int32_t)F, (int32_t)K, (int32_t)act, dt,
                             stream(dev));
        if (rc) return PyLong_FromLong(rc);
        if (!keep) return THPVariable_Wrap(std::move(h));
        return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(h)), THPVariable_Wrap(std::move(gate)),
                             THPVariable_Wrap(std::move(up)));
    });
}

// gated_ffn_backward(dh, x, w_gate, w_up, gate, up, act, need_dx, need_dw)
PyObject* gated_ffn_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9 || !f_ffn_backward) Py_RETURN_NONE;
        const int dev = device_of(a[0]);
        const at::Tensor *dh, *x, *g, *u, *gate, *up;
        if (!take(a[0], dev, &dh) || !take(a[1], dev, &x) || !take(a[2], dev, &g) || !take(a[3], dev, &u) ||
            !take(a[4], dev, &gate) || !take(a[5], dev, &up))
            Py_RETURN_NONE;
        const int dt = ffn_operands(*x, *g, *u), dx = PyObject_IsTrue(a[7]), dw = PyObject_IsTrue(a[8]);
        const long act = PyLong_AsLong(a[6]);
        if (dx < 0 || dw < 0 || PyErr_Occurred()) return nullptr;
        if (dt < 0) Py_RETURN_NONE;
        const int64_t M = x->size(0), F = g->size(0), K = x->size(1);
        for (const at::Tensor* t : {dh, gate, up})
            if (t->scalar_type() != (t == dh ? x->scalar_type() : at::kFloat) || t->dim() != 2 || t->size(0) != M || t->size(1) != F || !solid(*t))
                Py_RETURN_NONE;
        // dg, du and the parts' sums, in one piece
        const int64_t bytes = f_ffn_workspace((int32_t)M, (int32_t)F, (int32_t)K, dx, dw), n = (M * F * 2 + 15) / 16 * 16;
        const at::Tensor scratch = fresh(*x, {2 * n + bytes}, at::kByte);
        char* own = (char*)scratch.data_ptr();
        at::Tensor rx, rg, ru;
        if (dx) rx = like(*x, {M, K});
        if (dw) {
            rg = like(*x, {F, K});
            ru = like(*x, {F, K});
        }
        const int rc = f_ffn_backward(dh->data_ptr(), x->data_ptr(), g->data_ptr(), u->data_ptr(),
                                      (const float*)gate->data_ptr(), (const float*)up->data_ptr(), own, own + n,
                                      dx ? rx.data_ptr() : nullptr, dw ? rg.data_ptr() : nullptr,
                                      dw ? ru.data_ptr() : nullptr, (int32_t)M, (int32_t)F, (int32_t)K, (int32_t)act,
                                      dt, bytes ? own + 2 * n : nullptr, bytes, stream(dev));
        if (rc) return PyLong_FromLong(rc);
        auto wrap = [](bool has, at::Tensor& t) {
            if (has) return THPVariable_Wrap(std::move(t));
            Py_INCREF(Py_None);
            return Py_None;
        };
        return Py_BuildValue("(NNN)", wrap(dx, rx), wrap(dw, rg), wrap(dw, ru));
    });
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "addresses of the library's entry points"},
    {"packed_attention", (PyCFunction)(void*)packed_attention, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void*)qk_norm_rope, METH_FASTCALL, nullptr},
    {"gated_ffn", (PyCFunction)(void*)gated_ffn, METH_FASTCALL, nullptr},
    {"gated_ffn_backward", (PyCFunction)(void*)gated_ffn_backward, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_enc_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__enc_bind() { return PyModule_Create(&module); }
