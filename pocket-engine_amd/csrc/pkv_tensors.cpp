// _tensors: what pkv/__init__.py asks of torch tensors, a call for all of a
// step's arguments at once. The same questions through Python's attributes cost
// 0.4 us a tensor, more than the launch for calls of a dozen arrays (plan_step:
// 7 us of host time, 1.3 here).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// Element types by the codes the Python side passes.
bool type_is(const at::Tensor& t, long code) {
    const at::ScalarType s = t.scalar_type();
    return code == 0   ? s == at::kBFloat16
           : code == 1 ? s == at::kHalf
           : code == 2 ? s == at::kInt
                       : s == at::kFloat;
}

// The failing argument (counted from 0) and what is wrong with it, as one
// number: 8 index + reason.
enum { NO_TENSOR = 1, SHAPE = 2, DEVICE = 3 };
PyObject* wrong(Py_ssize_t index, int reason) { return PyLong_FromSsize_t(8 * index + reason); }

// words(dev, type, t, n, t, n, ..): the data pointers, as a tuple, of arrays
// without gaps on device dev of n elements each (below 0: any); None stays.
PyObject* words(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs < 2 || nargs % 2) {
        PyErr_SetString(PyExc_TypeError, "words(dev, type, tensor, numel, ...)");
        return nullptr;
    }
    const long dev = PyLong_AsLong(args[0]), type = PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t count = (nargs - 2) / 2;
    PyObject* out = PyTuple_New(count);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < count; i++) {
        PyObject* item = args[2 + 2 * i];
        if (item == Py_None) {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(out, i, Py_None);
            continue;
        }
        const long long n = PyLong_AsLongLong(args[3 + 2 * i]);
        int reason = 0;
        if (PyErr_Occurred()) {
            Py_DECREF(out);
            return nullptr;
        }
        if (!THPVariable_Check(item)) {
            reason = NO_TENSOR;
        } else {
            const at::Tensor& t = THPVariable_Unpack(item);
            if (t.layout() != at::kStrided || !type_is(t, type) || !t.is_contiguous() || (n >= 0 && t.numel() != n))
                reason = SHAPE;
            else if (t.get_device() != dev)
                reason = DEVICE;
            else
                PyTuple_SET_ITEM(out, i, PyLong_FromVoidPtr(t.data_ptr()));
        }
        if (reason) {
            Py_DECREF(out);
            return wrong(i, reason);
        }
    }
    return out;
}

// rows(dev, type, T, D, t, H, t, H, ..): (pointer, row stride, head stride) of
// every [T, H, D] view whose last dim has no gaps, in one tuple (a stride that
// nobody steps by is given as a dense one); None: (None, 0, 0).
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs < 4 || nargs % 2) {
        PyErr_SetString(PyExc_TypeError, "rows(dev, type, T, D, tensor, heads, ...)");
        return nullptr;
    }
    const long dev = PyLong_AsLong(args[0]), type = PyLong_AsLong(args[1]);
    const long long T = PyLong_AsLongLong(args[2]), D = PyLong_AsLongLong(args[3]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t count = (nargs - 4) / 2;
    PyObject* out = PyTuple_New(3 * count);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < count; i++) {
        PyObject* item = args[4 + 2 * i];
        if (item == Py_None) {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(out, 3 * i, Py_None);
            PyTuple_SET_ITEM(out, 3 * i + 1, PyLong_FromLong(0));
            PyTuple_SET_ITEM(out, 3 * i + 2, PyLong_FromLong(0));
            continue;
        }
        const long long H = PyLong_AsLongLong(args[5 + 2 * i]);
        int reason = 0;
        if (PyErr_Occurred()) {
            Py_DECREF(out);
            return nullptr;
        }
        if (!THPVariable_Check(item)) {
            reason = NO_TENSOR;
        } else {
            const at::Tensor& t = THPVariable_Unpack(item);
            if (t.layout() != at::kStrided || !type_is(t, type) || t.dim() != 3 || t.size(0) != T || t.size(1) != H ||
                t.size(2) != D || t.stride(2) != 1) {
                reason = SHAPE;
            } else if (t.get_device() != dev) {
                reason = DEVICE;
            } else {
                PyTuple_SET_ITEM(out, 3 * i, PyLong_FromVoidPtr(t.data_ptr()));
                PyTuple_SET_ITEM(out, 3 * i + 1, PyLong_FromLongLong(T > 1 ? t.stride(0) : H * D));
                PyTuple_SET_ITEM(out, 3 * i + 2, PyLong_FromLongLong(H > 1 ? t.stride(1) : D));
            }
        }
        if (reason) {
            Py_DECREF(out);
            return wrong(i, reason);
        }
    }
    return out;
}

// torch throws on tensors without storage or with symbolic sizes.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    try {
        return F(self, args, nargs);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"words", (PyCFunction)(void (*)(void))guarded<words>, METH_FASTCALL, "pointers of arrays without gaps"},
    {"rows", (PyCFunction)(void (*)(void))guarded<rows>, METH_FASTCALL, "pointers and strides of [T, H, D] rows"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
