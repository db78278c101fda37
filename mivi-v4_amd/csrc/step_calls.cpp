// The Python binding of the step's calls (mivi_hip_rms_norm and the others of
// that part of include/mivi_hip.h): tensors in, checks of their types, shapes,
// strides and devices, the call. Through ctypes the same checks and 20 to 35
// converted arguments take 10 us of a call whose kernel takes 4.
//
// Every function takes the stream's handle first and returns the call's status;
// mivi_hip/step.py documents their arguments.
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "../../include/mivi_hip.h"

namespace {

// What Python raises as ValueError.
struct Refused : std::exception {
    std::string text;
    explicit Refused(std::string t) : text(std::move(t)) {}
    const char* what() const noexcept override { return text.c_str(); }
};
// A Python error is set already.
struct Raised {};

const at::Tensor* tensor(PyObject* o, const char* what) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) throw Refused(std::string(what) + " is a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& needed(PyObject* o, const char* what) {
    const at::Tensor* t = tensor(o, what);
    if (!t) throw Refused(std::string(what) + " is a tensor");
    return *t;
}

int32_t type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MIVI_GGML_F32;
        case at::kHalf: return MIVI_GGML_F16;
        case at::kBFloat16: return MIVI_GGML_BF16;
        default: throw Refused("tensors are float32, float16 or bfloat16");
    }
}

void on_device(const at::Tensor& t, const at::Tensor& like, const char* what) {
    if (t.device() != like.device()) throw Refused(std::string(what) + " is on another device");
}

// [rows, dim] or [rows, heads, dim] with a contiguous last dimension.
struct Rows {
    void* p = nullptr;
    size_t span = 0, row = 0, head = 0;
};
Rows rows(const at::Tensor& t, const char* what) {
    const int64_t d = t.dim();
    if (t.size(d - 1) > 1 && t.stride(d - 1) != 1)
        throw Refused(std::string(what) + " has a contiguous last dimension");
    Rows r;
    r.p = t.data_ptr(), r.row = (size_t)t.stride(0), r.head = d == 3 ? (size_t)t.stride(1) : 0;
    if (t.numel())
        r.span = (size_t)(t.size(0) - 1) * r.row + (d == 3 ? (size_t)(t.size(1) - 1) * r.head : 0) + (size_t)t.size(d - 1);
    return r;
}
Rows rows_like(const at::Tensor* t, const at::Tensor& like, const char* what) {
    if (!t) return {};
    if (t->sizes() != like.sizes() || t->scalar_type() != like.scalar_type())
        throw Refused(std::string(what) + " has another shape or type");
    on_device(*t, like, what);
    return rows(*t, what);
}

// A contiguous array; numel -1: any number.
void* array(const at::Tensor& t, at::ScalarType type, const at::Tensor& like, const char* what, int64_t numel = -1) {
    if (t.scalar_type() != type || !t.is_contiguous())
        throw Refused(std::string(what) + " is a contiguous tensor of " + c10::toString(type));
    on_device(t, like, what);
    if (numel >= 0 && t.numel() != numel)
        throw Refused(std::string(what) + " has " + std::to_string(t.numel()) + " values, not " + std::to_string(numel));
    return t.data_ptr();
}

// Dimensions of a scale of [rows, dim / group] (0: one a row).
size_t group_of(const at::Tensor& scales, int64_t n_rows, int64_t dim, const char* what) {
    const int64_t n = scales.dim() == 1 ? 1 : scales.dim() == 2 ? scales.size(1) : 0;
    if (n == 0 || scales.size(0) != n_rows || dim % n) throw Refused(std::string(what) + " is [rows, dim / group]");
    return n == 1 ? 0 : (size_t)(dim / n);
}

size_t size(PyObject* o) {
    const size_t v = PyLong_AsSize_t(o);
    if (v == (size_t)-1 && PyErr_Occurred()) throw Raised();
    return v;
}
void* handle(PyObject* o) {
    void* v = PyLong_AsVoidPtr(o);
    if (!v && PyErr_Occurred()) throw Raised();
    return v;
}
float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return (float)v;
}

// Other Python threads run meanwhile: a launch waits where its queue is full.
struct Unlocked {
    PyThreadState* s = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(s); }
};

// ------------------------------------------------------------------- calls
// stream, out, x, weight, eps, residual, residual_out
int32_t rms_norm(PyObject* const* a) {
    const at::Tensor& x = needed(a[2], "x");
    if (x.dim() != 2 && x.dim() != 3) throw Refused("x is [rows, dim] or [rows, heads, dim]");
    const int64_t dim = x.size(x.dim() - 1), heads = x.dim() == 3 ? x.size(1) : 1;
    const Rows in = rows(x, "x"), o = rows_like(&needed(a[1], "out"), x, "out");
    const Rows r = rows_like(tensor(a[5], "residual"), x, "residual");
    const Rows s = rows_like(tensor(a[6], "residual_out"), x, "residual_out");
    const float* w = (const float*)array(needed(a[3], "weight"), at::kFloat, x, "weight", dim);
    const float eps = number(a[4]);
    void* stream = handle(a[0]);
    const Unlocked u;
    return mivi_hip_rms_norm(type_of(x), o.p, o.span, o.row, o.head, in.p, in.span, in.row, in.head, r.p, r.span, r.row,
                             r.head, s.p, s.span, s.row, s.head, w, (size_t)dim, eps, (size_t)x.size(0), (size_t)heads,
                             (size_t)dim, stream);
}

// stream, codes, scales, x, weight, eps, residual, residual_out
int32_t rms_norm_q8(PyObject* const* a) {
    const at::Tensor &codes = needed(a[1], "codes"), &scales = needed(a[2], "scales"), &x = needed(a[3], "x");
    if (x.dim() != 2 || codes.sizes() != x.sizes()) throw Refused("x and codes are [rows, dim]");
    const int64_t n = x.size(0), dim = x.size(1);
    const Rows in = rows(x, "x"), r = rows_like(tensor(a[6], "residual"), x, "residual");
    const Rows s = rows_like(tensor(a[7], "residual_out"), x, "residual_out");
    const float* w = (const float*)array(needed(a[4], "weight"), at::kFloat, x, "weight", dim);
    uint8_t* c = (uint8_t*)array(codes, at::kChar, x, "codes");
    float* f = (float*)array(scales, at::kFloat, x, "scales");
    const float eps = number(a[5]);
    void* stream = handle(a[0]);
    const Unlocked u;
    return mivi_hip_rms_norm_q8(type_of(x), c, (size_t)codes.numel(), f, (size_t)scales.numel(),
                                group_of(scales, n, dim, "scales"), in.p, in.span, in.row, r.p, r.span, r.row, s.p,
                                s.span, s.row, w, (size_t)dim, eps, (size_t)n, (size_t)dim, stream);
}

// stream, q, k, freqs, positions, starts, lens, half, scale, q_out, k_out
int32_t rope(PyObject* const* a) {
    const at::Tensor *q = tensor(a[1], "q"), *k = tensor(a[2], "k"), *one = q ? q : k;
    if (!one) throw Refused("neither q nor k");
    if (one->dim() != 3) throw Refused("q and k are [rows, heads, head_dim], of one type and device");
    const int64_t n = one->size(0), hd = one->size(2);
    Rows in[2], out[2];
    size_t heads[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        const at::Tensor* t = i ? k : q;
        const at::Tensor* o = tensor(a[9 + i], i ? "k_out" : "q_out");
        if (!t) continue;
        if (t->dim() != 3 || t->size(0) != n || t->size(2) != hd || t->scalar_type() != one->scalar_type() ||
            t->device() != one->device())
            throw Refused("q and k are [rows, heads, head_dim], of one type and device");
        in[i] = rows(*t, i ? "k" : "q"), out[i] = o ? rows_like(o, *t, i ? "k_out" : "q_out") : in[i];
        heads[i] = (size_t)t->size(1);
    }
    const at::Tensor& f = needed(a[3], "freqs");
    const void* freqs = array(f, at::kDouble, *one, "freqs");
    const at::Tensor *pos = tensor(a[4], "positions"), *starts = tensor(a[5], "starts"), *lens = tensor(a[6], "lens");
    if (!pos == !starts || !starts != !lens) throw Refused("either positions, or starts and lens");
    const int32_t *p = nullptr, *st = nullptr, *ln = nullptr;
    size_t seqs = 0;
    if (pos) {
        p = (const int32_t*)array(*pos, at::kInt, *one, "positions", n);
    } else {
        st = (const int32_t*)array(*starts, at::kInt, *one, "starts");
        if (starts->numel() == 0) throw Refused("starts has a value more than there are sequences");
        seqs = (size_t)starts->numel() - 1;
        ln = (const int32_t*)array(*lens, at::kInt, *one, "lens", (int64_t)seqs);
    }
    const int half = PyObject_IsTrue(a[7]);
    if (half < 0) throw Raised();
    const float scale = number(a[8]);
    void* stream = handle(a[0]);
    if (n == 0) return MIVI_OK;  // no address stands for no positions
    const Unlocked u;
    return mivi_hip_rope(type_of(*one), out[0].p, out[0].span, out[0].row, out[0].head, in[0].p, in[0].span, in[0].row,
                         in[0].head, heads[0], out[1].p, out[1].span, out[1].row, out[1].head, in[1].p, in[1].span,
                         in[1].row, in[1].head, heads[1], (size_t)n, (size_t)hd, 2 * (size_t)f.numel(), half, freqs,
                         (size_t)f.numel(), scale, p, pos ? (size_t)n : 0, st, ln, seqs, stream);
}

// stream, out, packed, scale type, zeros, rows, cols, group, x, x_scales
int32_t w4_matmul_rows(PyObject* const* a) {
    const at::Tensor &out = needed(a[1], "out"), &packed = needed(a[2], "packed"), &x = needed(a[8], "x");
    const at::Tensor* xs = tensor(a[9], "x_scales");
    const size_t n = size(a[5]), cols = size(a[6]), group = size(a[7]);
    if (x.dim() != 2 || out.dim() != 2 || x.size(0) != out.size(0)) throw Refused("x is [batch, cols], out [batch, rows]");
    if ((size_t)x.size(1) != cols || (size_t)out.size(1) != n)
        throw Refused("weights are " + std::to_string(n) + " x " + std::to_string(cols));
    on_device(x, packed, "x");
    on_device(out, packed, "out");
    const size_t batch = (size_t)x.size(0);
    const Rows o = rows(out, "out");
    const uint8_t* w = (const uint8_t*)packed.data_ptr();
    const size_t bytes = (size_t)packed.numel();
    const int32_t st = (int32_t)size(a[3]), zeros = (int32_t)size(a[4]);
    void* stream = handle(a[0]);
    const Unlocked u;
    if (!xs) {
        if (x.scalar_type() != out.scalar_type()) throw Refused("x and out are of one type");
        const Rows in = rows(x, "x");
        return mivi_hip_w4_matmul_rows(type_of(out), o.p, o.span, o.row, w, bytes, st, zeros, in.p, in.span, in.row, batch,
                                       n, cols, group, stream);
    }
    const uint8_t* c = (const uint8_t*)array(x, at::kChar, packed, "x");
    const float* f = (const float*)array(*xs, at::kFloat, packed, "x_scales");
    return mivi_hip_w4_matmul_rows_q8(type_of(out), o.p, o.span, o.row, w, bytes, st, zeros, c, (size_t)x.numel(), f,
                                      (size_t)xs->numel(), group_of(*xs, (int64_t)batch, (int64_t)cols, "x_scales"), batch,
                                      n, cols, group, stream);
}

// stream, tokens, counts, target, drafted, accept, pick, starts, draft, workspace
int32_t verify_rows(PyObject* const* a) {
    const at::Tensor &tokens = needed(a[1], "tokens"), &counts = needed(a[2], "counts"), &p = needed(a[3], "target");
    const at::Tensor &drafted = needed(a[4], "drafted"), &accept = needed(a[5], "accept"), &pick = needed(a[6], "pick");
    const at::Tensor &starts = needed(a[7], "starts"), *q = tensor(a[8], "draft"), *ws = tensor(a[9], "workspace");
    if (p.dim() != 2 || p.scalar_type() != at::kFloat) throw Refused("target is [rows, vocab] of float32");
    const int64_t n = p.size(0), seqs = starts.numel() - 1;
    if (seqs < 0) throw Refused("starts has a value more than there are sequences");
    const Rows tp = rows(p, "target"), tq = rows_like(q, p, "draft");
    if (ws && (!ws->is_contiguous() || ws->device() != p.device()))
        throw Refused("workspace is a contiguous tensor on the other tensors' device");
    void* stream = handle(a[0]);
    const Unlocked u;
    return mivi_hip_verify_rows((int32_t*)array(tokens, at::kInt, p, "tokens", n), (size_t)n,
                                (int32_t*)array(counts, at::kInt, p, "counts", seqs), (size_t)seqs, (const float*)tp.p,
                                tp.span, tp.row, (const float*)tq.p, tq.span, tq.row,
                                (const int32_t*)array(drafted, at::kInt, p, "drafted", n), (size_t)n,
                                (const float*)array(accept, at::kFloat, p, "accept", n), (size_t)n,
                                (const float*)array(pick, at::kFloat, p, "pick", seqs), (size_t)seqs,
                                (const int32_t*)array(starts, at::kInt, p, "starts"), (size_t)seqs, (size_t)n,
                                (size_t)p.size(1), ws ? ws->data_ptr() : nullptr,
                                ws ? (size_t)ws->numel() * ws->element_size() : 0, stream);
}

template <int32_t (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    try {
        if (n != N) throw Refused("takes " + std::to_string(N) + " arguments");
        return PyLong_FromLong(F(a));
    } catch (const Raised&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
}

#define CALL(NAME, N) {#NAME, (PyCFunction)(void*)call<NAME, N>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(rms_norm, 7),        CALL(rms_norm_q8, 8),  CALL(rope, 11),
                         CALL(w4_matmul_rows, 10), CALL(verify_rows, 10), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_step", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step() { return PyModule_Create(&module); }
