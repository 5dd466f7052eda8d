// _tensors: the calls of pkv/__init__.py that take torch tensors, from the
// tensors to the C entry points of the library. A call of a dozen arrays costs
// more host time in Python's attribute lookups and ctypes' conversions than its
// launch takes (plan_step: 10.5 us of host time so, 4 here).
//
// Every function checks its tensors (types, sizes, gaps, one device) before it
// calls, and returns an int: 0, the entry point's status (above 0), or below 0
// what is wrong with which tensor: -(8 i + reason) for the i-th one, counted
// from 0 in the function's order of tensors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

#include "../../include/pkv.h"

namespace {

enum Reason { NO_TENSOR = 1, SHAPE = 2, DEVICE = 3, NOT_GPU = 4 };

// The library that the package has loaded (bind).
struct {
    decltype(&pkv_plan_step) plan_step;
    decltype(&pkv_plan_truncate) plan_truncate;
    decltype(&pkv_rope_spans) rope_spans;
    decltype(&pkv_rope_positions) rope_positions;
    decltype(&pkv_rope_rows) rope_rows;
    decltype(&pkv_attn_packed) attn_packed;
} lib;

// The arguments of one call, taken in order; the first thing that is wrong is
// kept, and later takes then do nothing.
class Call {
public:
    Call(PyObject* const* args, Py_ssize_t n) : args_(args), n_(n) {
        dev_ = integer();
        stream_ = reinterpret_cast<void*>(static_cast<uintptr_t>(integer()));
    }
    int64_t integer() {
        PyObject* o = next();
        if (!o || bad()) return 0;
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) error_ = true;
        return v;
    }
    // An integer that goes to an int of the entry point.
    int small() { return fit(integer()); }
    int fit(int64_t v) {
        if (v < INT_MIN || v > INT_MAX) large_ = true;
        return static_cast<int>(v);
    }
    float real() {
        PyObject* o = next();
        if (!o || bad()) return 0;
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) error_ = true;
        return static_cast<float>(v);
    }
    // The next tensor, unchecked but for being one (its sizes may be needed
    // first); null for None.
    const at::Tensor* tensor() {
        PyObject* o = next();
        if (!o || bad()) return nullptr;
        at_++;
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) {
            wrong(NO_TENSOR);
            return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided) wrong(SHAPE);
        return bad() ? nullptr : &t;
    }
    // Checks of the tensor taken last.
    bool holds(bool good) {
        if (!bad() && !good) wrong(SHAPE);
        return !bad();
    }
    template <class T>
    T* words(const at::Tensor* t, at::ScalarType type, int64_t numel) {
        if (!t || !holds(t->scalar_type() == type && t->is_contiguous() && (numel < 0 || t->numel() == numel)) || !here(*t))
            return nullptr;
        return static_cast<T*>(t->data_ptr());
    }
    // A tensor that must be there.
    int32_t* ints(int64_t numel) { return need(words<int32_t>(tensor(), at::kInt, numel), numel); }
    int32_t* ints_or_none(int64_t numel) { return words<int32_t>(tensor(), at::kInt, numel); }
    float* floats_or_none(int64_t numel) { return words<float>(tensor(), at::kFloat, numel); }
    // [T, H, D] rows whose last dim has no gaps; a stride that nobody steps by
    // is given as a dense one.
    struct Rows {
        void* at = nullptr;
        int64_t row = 0, head = 0;
    };
    Rows rows(const at::Tensor* t, at::ScalarType type, int64_t T, int64_t H, int64_t D) {
        Rows r;
        if (!t || !holds(t->scalar_type() == type && t->dim() == 3 && t->size(0) == T && t->size(1) == H && t->size(2) == D &&
                         t->stride(2) == 1) ||
            !here(*t))
            return r;
        r.at = t->data_ptr();
        r.row = T > 1 ? t->stride(0) : H * D;
        r.head = H > 1 ? t->stride(1) : D;
        return r;
    }
    bool bad() const { return error_ || fail_; }
    void* stream() const { return stream_; }
    // After the last argument: whether the entry point may be called.
    bool ready() {
        if (!bad() && used_ != n_) {
            PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
            error_ = true;
        }
        if (!bad() && dev_ < 0) {
            at_ = 1;
            wrong(NOT_GPU);
        }
        return !bad() && !large_;
    }
    PyObject* refused() const {
        if (error_) return nullptr;
        return PyLong_FromLong(fail_ ? -fail_ : PKV_ERR_UNSUPPORTED);
    }

private:
    PyObject* next() {
        if (bad()) return nullptr;
        if (used_ == n_) {
            PyErr_SetString(PyExc_TypeError, "too few arguments");
            error_ = true;
            return nullptr;
        }
        return args_[used_++];
    }
    template <class T>
    T* need(T* p, int64_t) {
        if (!p && !bad() && last_none()) wrong(NO_TENSOR);
        return p;
    }
    bool last_none() const { return used_ > 0 && args_[used_ - 1] == Py_None; }
    bool here(const at::Tensor& t) {
        if (t.get_device() != dev_) wrong(DEVICE);
        return !bad();
    }
    void wrong(Reason r) { fail_ = 8 * (at_ - 1) + r; }

    PyObject* const* args_;
    Py_ssize_t n_, used_ = 0;
    long at_ = 0, fail_ = 0;  // tensors taken; 8 i + reason of the one that will not do
    int64_t dev_ = -1;
    void* stream_ = nullptr;
    bool error_ = false, large_ = false;
};

template <class F>
PyObject* called(F&& f) {
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = f();
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(status);
}

// plan_step(dev, stream, block_table, pos, len, held, ntok, slot_map, tok_seq, cu, limits, len_out, held_out, status,
//           free_list, free_count, free_count_out, block_size, num_blocks)
PyObject* plan_step(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const at::Tensor* t = c.tensor();
    const bool two = t && t->dim() == 2;
    c.holds(two);
    const int64_t n = two ? t->size(0) : 0, width = two ? t->size(1) : 0;
    int32_t* table = c.words<int32_t>(t, at::kInt, -1);
    t = c.tensor();
    const int64_t T = t ? t->numel() : 0;
    c.holds(t != nullptr);
    int32_t* pos = c.words<int32_t>(t, at::kInt, -1);
    int32_t *len = c.ints(n), *held = c.ints(n), *ntok = c.ints(n), *slot = c.ints(T), *seq = c.ints(T), *cu = c.ints(n + 1),
            *limits = c.ints(n), *len_out = c.ints(n), *held_out = c.ints(n), *status = c.ints(n);
    const at::Tensor* list = c.tensor();
    int32_t* free_list = c.words<int32_t>(list, at::kInt, -1);
    int32_t *count = c.ints_or_none(1), *count_out = c.ints_or_none(1);
    const int block_size = c.small();
    const int64_t num_blocks = c.integer();
    const int rows = c.fit(n), wide = c.fit(width), tokens = c.fit(T);
    if (!c.ready()) return c.refused();
    if (list && list->numel() < num_blocks) return PyLong_FromLong(PKV_ERR_INVALID);
    return called([&] {
        return lib.plan_step(len, held, ntok, rows, table, wide, block_size, num_blocks, free_list, count, tokens, pos, slot,
                             seq, cu, limits, len_out, held_out, count_out, status, c.stream());
    });
}

// plan_truncate(dev, stream, block_table, new_len, len, held, free_list, free_count, block_size, num_blocks)
PyObject* plan_truncate(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const at::Tensor* t = c.tensor();
    const bool two = t && t->dim() == 2;
    c.holds(two);
    const int64_t n = two ? t->size(0) : 0, width = two ? t->size(1) : 0;
    int32_t* table = c.words<int32_t>(t, at::kInt, -1);
    int32_t *new_len = c.ints(n), *len = c.ints(n), *held = c.ints(n);
    const at::Tensor* list = c.tensor();
    c.holds(list != nullptr);
    int32_t* free_list = c.words<int32_t>(list, at::kInt, -1);
    int32_t* count = c.ints(1);
    const int block_size = c.small();
    const int64_t num_blocks = c.integer();
    const int rows = c.fit(n), wide = c.fit(width);
    if (!c.ready()) return c.refused();
    if (list->numel() < num_blocks) return PyLong_FromLong(PKV_ERR_INVALID);
    return called([&] {
        return lib.plan_truncate(new_len, len, held, rows, table, wide, block_size, num_blocks, free_list, count, c.stream());
    });
}

// The spans' tensors: [n, 5] rows and offsets [requests + 1].
struct Spans {
    int64_t n = 0, requests = 0;
    int32_t *cu = nullptr, *spans = nullptr, *base = nullptr;
    explicit Spans(Call& c) {
        const at::Tensor* t = c.tensor();
        c.holds(t && t->numel() >= 1);
        requests = t ? t->numel() - 1 : 0;
        cu = c.words<int32_t>(t, at::kInt, -1);
        t = c.tensor();
        c.holds(t && t->dim() == 2 && t->size(1) == 5);
        n = t && t->dim() == 2 ? t->size(0) : 0;
        spans = c.words<int32_t>(t, at::kInt, 5 * n);
        base = c.ints(n);
    }
};

// rope_spans(dev, stream, span_cu, spans, base)
PyObject* rope_spans(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const Spans s(c);
    const int requests = c.fit(s.requests), n = c.fit(s.n);
    if (!c.ready()) return c.refused();
    return called([&] { return lib.rope_spans(s.cu, s.spans, requests, n, s.base, c.stream()); });
}

// rope_positions(dev, stream, span_cu, spans, base, pos, tok_seq, rope)
PyObject* rope_positions(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const Spans s(c);
    const at::Tensor* t = c.tensor();
    const int64_t T = t ? t->numel() : 0;
    c.holds(t != nullptr);
    int32_t *pos = c.words<int32_t>(t, at::kInt, -1), *seq = c.ints(T);
    t = c.tensor();
    c.holds(t && t->dim() == 2 && t->size(0) == 3 && t->size(1) >= T);
    const int64_t wide = t && t->dim() == 2 ? t->size(1) : 0;
    int32_t* rope = c.words<int32_t>(t, at::kInt, -1);
    const int requests = c.fit(s.requests), n = c.fit(s.n), rows = c.fit(T), stride = c.fit(wide);
    if (!c.ready()) return c.refused();
    return called(
        [&] { return lib.rope_positions(pos, seq, rows, s.cu, s.spans, s.base, requests, n, rope, stride, c.stream()); });
}

// q [T, Hq, D] and k [T, Hkv, D] of one type of rows, which says the type, T, D
// and the heads of the tensors after them.
struct QK {
    at::ScalarType type = at::kBFloat16;
    int64_t T = 0, Hq = 0, Hkv = 0, D = 0;
    bool served = true;  // a type of rows that the entry points know
    Call::Rows q, k;
    explicit QK(Call& c) {
        const at::Tensor* t = c.tensor();
        if (!c.holds(t && t->dim() == 3)) return;
        type = t->scalar_type();
        served = type == at::kBFloat16 || type == at::kHalf;
        T = t->size(0), Hq = t->size(1), D = t->size(2);
        q = c.rows(t, type, T, Hq, D);
        t = c.tensor();
        if (!c.holds(t && t->dim() == 3)) return;
        Hkv = t->size(1);
        k = c.rows(t, type, T, Hkv, D);
    }
    int dtype() const { return type == at::kBFloat16 ? PKV_BF16 : PKV_FP16; }
};

// rope_rows(dev, stream, q, k, q_out, k_out, rope, axes, inv_freq, q_norm, k_norm, eps, adjacent)
PyObject* rope_rows(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const QK x(c);
    if (!c.bad() && !x.served) return PyLong_FromLong(PKV_ERR_UNSUPPORTED);
    const at::Tensor* t = c.tensor();
    c.holds(t != nullptr);
    const Call::Rows qo = c.rows(t, x.type, x.T, x.Hq, x.D);
    t = c.tensor();
    c.holds(t != nullptr);
    const Call::Rows ko = c.rows(t, x.type, x.T, x.Hkv, x.D);
    t = c.tensor();
    c.holds(t && t->dim() == 2 && t->size(0) == 3 && t->size(1) >= x.T);
    const int64_t wide = t && t->dim() == 2 ? t->size(1) : 0;
    int32_t* rope = c.words<int32_t>(t, at::kInt, -1);
    t = c.tensor();
    c.holds(t != nullptr);
    const int64_t half = t ? t->numel() : 0;
    int32_t* axes = c.words<int32_t>(t, at::kInt, -1);
    t = c.tensor();
    c.holds(t != nullptr);
    float* inv = c.words<float>(t, at::kFloat, half);
    float *qn = c.floats_or_none(x.D), *kn = c.floats_or_none(x.D);
    const float eps = c.real();
    const int adjacent = c.small();
    const int T = c.fit(x.T), Hq = c.fit(x.Hq), Hkv = c.fit(x.Hkv), D = c.fit(x.D), rot = c.fit(2 * half), stride = c.fit(wide);
    if (!c.ready()) return c.refused();
    return called([&] {
        return lib.rope_rows(x.q.at, x.q.row, x.q.head, x.k.at, x.k.row, x.k.head, qo.at, qo.row, qo.head, ko.at, ko.row,
                             ko.head, Hq, Hkv, D, x.dtype(), qn, kn, eps, rope, stride, axes, inv, rot, adjacent, T,
                             c.stream());
    });
}

// attn_packed(dev, stream, q, k, v, out, gate, cu, scale)
PyObject* attn_packed(PyObject* const* args, Py_ssize_t nargs) {
    Call c(args, nargs);
    const QK x(c);
    if (!c.bad() && !x.served) return PyLong_FromLong(PKV_ERR_UNSUPPORTED);
    const at::Tensor* t = c.tensor();
    c.holds(t != nullptr);
    const Call::Rows v = c.rows(t, x.type, x.T, x.Hkv, x.D);
    t = c.tensor();
    c.holds(t != nullptr);
    const Call::Rows out = c.rows(t, x.type, x.T, x.Hq, x.D);
    const Call::Rows gate = c.rows(c.tensor(), x.type, x.T, x.Hq, x.D);
    t = c.tensor();
    c.holds(t && t->numel() >= 1);
    const int64_t seqs = t ? t->numel() - 1 : 0;
    int32_t* cu = c.words<int32_t>(t, at::kInt, -1);
    const float scale = c.real();
    const int T = c.fit(x.T), Hq = c.fit(x.Hq), Hkv = c.fit(x.Hkv), D = c.fit(x.D), n = c.fit(seqs);
    if (!c.ready()) return c.refused();
    return called([&] {
        return lib.attn_packed(x.q.at, x.q.row, x.q.head, x.k.at, x.k.row, x.k.head, v.at, v.row, v.head, gate.at, gate.row,
                               gate.head, out.at, out.row, out.head, cu, n, T, Hq, Hkv, D, x.dtype(), scale, c.stream());
    });
}

// bind(path): the entry points of the library at `path`, which is loaded.
PyObject* bind(PyObject* const* args, Py_ssize_t nargs) {
    const char* path = nargs == 1 ? PyUnicode_AsUTF8(args[0]) : nullptr;
    if (!path) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "bind(path)");
        return nullptr;
    }
    void* h = dlopen(path, RTLD_NOW);
    if (!h) {
        PyErr_SetString(PyExc_ImportError, dlerror());
        return nullptr;
    }
    const char* missing = nullptr;
    auto find = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
        if (!f) missing = name;
    };
    find(lib.plan_step, "pkv_plan_step");
    find(lib.plan_truncate, "pkv_plan_truncate");
    find(lib.rope_spans, "pkv_rope_spans");
    find(lib.rope_positions, "pkv_rope_positions");
    find(lib.rope_rows, "pkv_rope_rows");
    find(lib.attn_packed, "pkv_attn_packed");
    if (missing) {
        PyErr_SetString(PyExc_ImportError, missing);
        return nullptr;
    }
    Py_RETURN_NONE;
}

// torch throws on tensors without storage or with symbolic sizes.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        return F(args, nargs);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
#define METHOD(f) {#f, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),           METHOD(plan_step), METHOD(plan_truncate), METHOD(rope_spans),
                         METHOD(rope_positions), METHOD(rope_rows), METHOD(attn_packed),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
