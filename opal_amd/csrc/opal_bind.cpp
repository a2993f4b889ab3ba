// The Python side of the score head's calls: checks of tensor arguments, results, workspaces, one C entry (include/opal_hip.h).  A call for
// one read is as long as its host side, so this is C++ rather than ctypes: a product of one row 7.8 -> 4.8 us, a layer norm 7.3 -> 4.6, of which the launch is 3.
// Engine (opal_amd/engine.py) documents the calls; the order with other streams is its business too.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>

#include "opal_hip.h"

namespace {

PyObject *check = nullptr;                     // opal_amd._lib.check: raises OpalError for a status

struct Failed {};                              // a Python error is set

[[noreturn]] void refuse(const char *format, ...)
{
    va_list args;
    va_start(args, format);
    PyErr_FormatV(PyExc_ValueError, format, args);
    va_end(args);
    throw Failed();
}

int type_of(at::ScalarType s) { return s == at::kFloat ? OPAL_F32 : s == at::kHalf ? OPAL_F16 : s == at::kBFloat16 ? OPAL_BF16 : -1; }
at::ScalarType scalar(int type) { return type == OPAL_F32 ? at::kFloat : type == OPAL_F16 ? at::kHalf : at::kBFloat16; }
const char *name_of(int type) { return type == OPAL_F32 ? "torch.float32" : type == OPAL_F16 ? "torch.float16" : "torch.bfloat16"; }

struct Env {
    opal_ctx *ctx;
    int index;                                 // of the GPU
    at::TensorOptions on(at::ScalarType s) const { return at::TensorOptions().dtype(s).device(at::Device(at::kCUDA, (c10::DeviceIndex)index)); }
    // A C entry, without the interpreter's lock (a launch waits when the queue is full); its status raises.
    template <class F> void run(F &&entry) const
    {
        PyThreadState *state = PyEval_SaveThread();
        const int rc = entry();
        PyEval_RestoreThread(state);
        if (rc == OPAL_OK) return;
        PyObject *r = PyObject_CallFunction(check, "iK", rc, (unsigned long long)(uintptr_t)ctx);
        Py_XDECREF(r);
        if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "status %d", rc);
        throw Failed();
    }
};

// sizes as the C entries take them: what does not fit is larger than they allow, and stays so
uint32_t u32(int64_t v) { return v > 0xffffffffll ? 0xffffffffu : (uint32_t)v; }

struct Matrix {
    void *p = nullptr;
    int type = 0;
    uint64_t ld = 0;
    int64_t rows = 0, cols = 0;
};

// A matrix argument, checked; -1: any number of rows or columns, any type.
Matrix matrix(const Env &e, PyObject *o, const char *name, int64_t rows = -1, int64_t cols = -1, int type = -1)
{
    const at::Tensor *t = THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
    const int kind = t ? type_of(t->scalar_type()) : -1;
    if (kind < 0 || t->layout() != at::kStrided || t->dim() != 2)
        refuse("%s must be a matrix (2-d tensor) of float32, float16 or bfloat16 on cuda:%d", name, e.index);
    if (t->is_neg()) refuse("%s is a view with the negation still to be made: call its resolve_neg()", name);       // (the imaginary part of a conjugate)
    if (!t->is_cuda() || t->get_device() != e.index) refuse("%s must be on cuda:%d", name, e.index);
    if (type >= 0 && kind != type) refuse("%s is %s: must be %s", name, name_of(kind), name_of(type));
    const int64_t n = t->size(0), c = t->size(1), ld = n <= 1 ? c : t->stride(0);
    if ((rows >= 0 && n != rows) || (cols >= 0 && c != cols))
        refuse("%s is (%lld, %lld): must have %lld rows and %lld columns (-1: any)", name, (long long)n, (long long)c, (long long)rows, (long long)cols);
    if (c < 1 || (c > 1 && t->stride(1) != 1) || ld < c) refuse("%s needs at least one column, columns of stride 1 and rows that do not overlap", name);
    return {t->data_ptr(), kind, (uint64_t)ld, n, c};
}

Matrix optional_matrix(const Env &e, PyObject *o, const char *name, int64_t rows, int64_t cols, int type = -1)
{
    return o == Py_None ? Matrix() : matrix(e, o, name, rows, cols, type);
}

// A vector argument, checked; null for None.
void *vector(const Env &e, PyObject *o, const char *name, int64_t n, at::ScalarType s = at::kFloat)
{
    if (o == Py_None) return nullptr;
    const at::Tensor *t = THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
    if (t && t->is_neg()) refuse("%s is a view with the negation still to be made: call its resolve_neg()", name);
    if (!t || t->layout() != at::kStrided || t->dim() != 1 || t->size(0) != n || t->scalar_type() != s || !t->is_contiguous() || !t->is_cuda() || t->get_device() != e.index)
        refuse("%s must be a contiguous %s vector of %lld on cuda:%d", name, s == at::kFloat ? "torch.float32" : "torch.int32", (long long)n, e.index);
    return t->data_ptr();
}

int out_type(PyObject *o, int none)
{
    if (o == Py_None) return none;
    const int type = THPDtype_Check(o) ? type_of(reinterpret_cast<THPDtype *>(o)->scalar_type) : -1;
    if (type < 0) refuse("%R: must be float32, float16 or bfloat16", o);
    return type;
}

// A new matrix.  Rows begin on 16 bytes, which the kernels' wide reads need; rows of 1 KB or more on 128, so that a tile's part of a
// row is whole cache lines (60 001 x 1563 float32 logits: 273 -> 252 us).
at::Tensor new_matrix(const Env &e, int64_t n, int64_t cols, int type)
{
    const int64_t each = type == OPAL_F32 ? 4 : 2, step = (cols * each >= 1024 ? 128 : 16) / each, ld = (cols + step - 1) / step * step;
    return at::empty_strided({n, cols}, {ld, 1}, e.on(scalar(type)));
}
at::Tensor new_vector(const Env &e, int64_t n, at::ScalarType s = at::kFloat) { return at::empty({n}, e.on(s)); }

void *at_of(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
uint64_t ld_of(const at::Tensor &t) { return t.defined() ? (uint64_t)t.stride(0) : 0; }

// Results: an undefined tensor is None.
template <class... T> PyObject *results(const T &...t)
{
    PyObject *r = PyTuple_New(sizeof...(T));
    if (!r) throw Failed();
    Py_ssize_t i = 0;
    for (const at::Tensor *x : {&t...}) {
        PyObject *o = x->defined() ? THPVariable_Wrap(*x) : (Py_INCREF(Py_None), Py_None);
        if (!o) {
            Py_DECREF(r);
            throw Failed();
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

bool is_true(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Failed();
    return v == 1;
}
double number(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Failed();
    return v;
}
int integer(PyObject *o)
{
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Failed();
    return (int)v;
}

// Every call: (ctx, index of the GPU, arguments ...), by position.
typedef PyObject *Body(const Env &, PyObject *const *);
template <Body *body, Py_ssize_t COUNT> PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    try {
        if (n != COUNT + 2) {
            PyErr_Format(PyExc_TypeError, "%zd arguments instead of %zd", n, COUNT + 2);
            return nullptr;
        }
        const Env e{(opal_ctx *)PyLong_AsVoidPtr(args[0]), integer(args[1])};
        if (PyErr_Occurred()) return nullptr;
        at::AutoDispatchBelowADInplaceOrView plain;      // results that autograd does not know of
        return body(e, args + 2);
    } catch (const Failed &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// x, gamma, beta, eps, out_dtype, want_stats -> y, mean, rstd
PyObject *layer_norm(const Env &e, PyObject *const *a)
{
    const Matrix x = matrix(e, a[0], "x");
    void *gamma = vector(e, a[1], "gamma", x.cols), *beta = vector(e, a[2], "beta", x.cols);
    const float eps = (float)number(a[3]);
    const int type = out_type(a[4], x.type);
    const at::Tensor y = new_matrix(e, x.rows, x.cols, type);
    at::Tensor mean, rstd;
    if (is_true(a[5])) {
        mean = new_vector(e, x.rows);
        rstd = new_vector(e, x.rows);
    }
    e.run([&] { return opal_layer_norm(e.ctx, x.p, x.type, x.ld, (const float *)gamma, (const float *)beta, x.rows, u32(x.cols), eps, at_of(y), type, ld_of(y),
                           (float *)at_of(mean), (float *)at_of(rstd)); });
    return results(y, mean, rstd);
}

// dy, x, gamma, mean, rstd, out_dtype, want_dx, want_params -> dx, dgamma, dbeta
PyObject *layer_norm_backward(const Env &e, PyObject *const *a)
{
    const Matrix x = matrix(e, a[1], "x"), dy = matrix(e, a[0], "dy", x.rows, x.cols);
    if (a[3] == Py_None || a[4] == Py_None) refuse("mean and rstd of the forward pass are needed (layer_norm(..., want_stats=True))");
    void *gamma = vector(e, a[2], "gamma", x.cols), *mean = vector(e, a[3], "mean", x.rows), *rstd = vector(e, a[4], "rstd", x.rows);
    const int type = out_type(a[5], x.type);
    at::Tensor dx, dgamma, dbeta, work;
    if (is_true(a[6])) dx = new_matrix(e, x.rows, x.cols, type);
    uint64_t bytes = 0;
    if (is_true(a[7])) {
        dgamma = new_vector(e, x.cols);
        dbeta = new_vector(e, x.cols);
        bytes = opal_layer_norm_backward_workspace(x.rows, u32(x.cols));
        if (bytes) work = new_vector(e, (int64_t)bytes, at::kByte);
    }
    e.run([&] { return opal_layer_norm_backward(e.ctx, dy.p, dy.type, dy.ld, x.p, x.type, x.ld, (const float *)gamma, (const float *)mean, (const float *)rstd, x.rows,
                                    u32(x.cols), at_of(dx), type, ld_of(dx), (float *)at_of(dgamma), (float *)at_of(dbeta), at_of(work), bytes); });
    return results(dx, dgamma, dbeta);
}

// x, w, bias, residual, activation, out_dtype, want_pre -> y, pre
PyObject *linear(const Env &e, PyObject *const *a)
{
    const Matrix x = matrix(e, a[0], "x"), w = matrix(e, a[1], "w", -1, x.cols, x.type);
    void *bias = vector(e, a[2], "bias", w.rows);
    const Matrix res = optional_matrix(e, a[3], "residual", x.rows, w.rows);
    const int act = integer(a[4]), type = out_type(a[5], x.type);
    const at::Tensor y = new_matrix(e, x.rows, w.rows, type);
    at::Tensor pre;
    if (is_true(a[6])) pre = new_matrix(e, x.rows, w.rows, x.type);
    e.run([&] { return opal_linear(e.ctx, x.p, x.ld, w.p, w.ld, x.type, (const float *)bias, act, res.p, res.type, res.ld, x.rows, u32(x.cols), u32(w.rows),
                       at_of(y), type, ld_of(y), at_of(pre), ld_of(pre)); });
    return results(y, pre);
}

// dy, w, pre, residual, activation, out_dtype -> dx
PyObject *linear_grad_input(const Env &e, PyObject *const *a)
{
    const Matrix dy = matrix(e, a[0], "dy"), w = matrix(e, a[1], "w", dy.cols, -1, dy.type);
    const int act = integer(a[4]), type = out_type(a[5], dy.type);
    if (act && a[2] == Py_None) refuse("an activation's gradient needs pre (linear(..., want_pre=True))");
    const Matrix pre = act ? matrix(e, a[2], "pre", dy.rows, w.cols, dy.type) : Matrix();
    const Matrix res = optional_matrix(e, a[3], "residual", dy.rows, w.cols);
    const at::Tensor dx = new_matrix(e, dy.rows, w.cols, type);
    e.run([&] { return opal_linear_grad_input(e.ctx, dy.p, dy.ld, w.p, w.ld, dy.type, pre.p, pre.ld, act, res.p, res.type, res.ld, dy.rows, u32(w.cols),
                                  u32(dy.cols), at_of(dx), type, ld_of(dx)); });
    return results(dx);
}

// dy, x, want_bias -> dw, dbias
PyObject *linear_grad_weight(const Env &e, PyObject *const *a)
{
    const Matrix x = matrix(e, a[1], "x"), dy = matrix(e, a[0], "dy", x.rows, -1, x.type);
    const at::Tensor dw = at::empty({dy.cols, x.cols}, e.on(at::kFloat));
    at::Tensor db, work;
    if (is_true(a[2])) db = new_vector(e, dy.cols);
    const uint64_t bytes = opal_linear_grad_weight_workspace(x.rows, u32(x.cols), u32(dy.cols), x.type);
    if (bytes) work = new_vector(e, (int64_t)bytes, at::kByte);
    e.run([&] { return opal_linear_grad_weight(e.ctx, dy.p, dy.ld, x.p, x.ld, x.type, x.rows, u32(x.cols), u32(dy.cols), (float *)at_of(dw), (uint64_t)x.cols,
                                   (float *)at_of(db), at_of(work), bytes); });
    return results(dw, db);
}

// scores, labels, scale, out_dtype, want_grad -> loss, grad
PyObject *softmax_loss(const Env &e, PyObject *const *a)
{
    const Matrix s = matrix(e, a[0], "scores");
    if (a[1] == Py_None) refuse("labels are needed");
    void *labels = vector(e, a[1], "labels", s.rows, at::kInt);
    const float scale = (float)number(a[2]);
    const int type = out_type(a[3], s.type);
    const at::Tensor loss = new_vector(e, s.rows);
    at::Tensor grad;
    if (is_true(a[4])) grad = new_matrix(e, s.rows, s.cols, type);
    e.run([&] { return opal_softmax_loss(e.ctx, s.p, s.type, s.ld, s.rows, u32(s.cols), (const int32_t *)labels, scale, (float *)at_of(loss), at_of(grad), type, ld_of(grad)); });
    return results(loss, grad);
}

// scores -> class, probability
PyObject *softmax_class(const Env &e, PyObject *const *a)
{
    const Matrix s = matrix(e, a[0], "scores");
    const at::Tensor cls = new_vector(e, s.rows, at::kInt), prob = new_vector(e, s.rows);
    e.run([&] { return opal_softmax_class(e.ctx, s.p, s.type, s.ld, s.rows, u32(s.cols), (int32_t *)at_of(cls), (float *)at_of(prob)); });
    return results(cls, prob);
}

PyObject *on_error(PyObject *, PyObject *f)
{
    Py_INCREF(f);
    Py_XSETREF(check, f);
    Py_RETURN_NONE;
}

#define OPAL_CALL(NAME, COUNT) {#NAME, (PyCFunction)(void (*)(void)) & call<NAME, COUNT>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OPAL_CALL(layer_norm, 6),
                         OPAL_CALL(layer_norm_backward, 8),
                         OPAL_CALL(linear, 7),
                         OPAL_CALL(linear_grad_input, 6),
                         OPAL_CALL(linear_grad_weight, 3),
                         OPAL_CALL(softmax_loss, 5),
                         OPAL_CALL(softmax_class, 1),
                         {"on_error", on_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// What it was built from (a hash that the build computes) and for: opal_amd._lib.bind compares both.
PyMODINIT_FUNC PyInit__bind()
{
    PyObject *m = PyModule_Create(&module);
    if (m && (PyModule_AddStringConstant(m, "source", OPAL_BIND_SOURCE) || PyModule_AddStringConstant(m, "torch", OPAL_BIND_TORCH))) Py_CLEAR(m);
    return m;
}
