// CPython calls of the readout operators' C entry points: through ctypes the
// twenty arguments of a product take 2 to 3 us to convert, here a few tenths (one
// row's product 11.7 -> 9.2 us a call).
// The functions are handed over by address from the library that _lib.py
// loaded, so both bindings call the same copy of it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/mdsoap.h"

#include <cstdint>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

namespace {

// One argument: None is a null pointer, pointers and integers are ints; bytes are handed over by their address.
template <class T>
T value_of(PyObject* o) {
    if constexpr (std::is_pointer_v<T>) {
        if (o == Py_None) return nullptr;
        if (PyBytes_Check(o)) return reinterpret_cast<T>(PyBytes_AS_STRING(o));
        return reinterpret_cast<T>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o)));
    } else if constexpr (std::is_floating_point_v<T>) {
        return static_cast<T>(PyFloat_AsDouble(o));
    } else {
        return static_cast<T>(PyLong_AsLongLong(o));
    }
}

template <int ID, class F>
struct Entry;

template <int ID, class... Args>
struct Entry<ID, int(Args...)> {
    static inline int (*function)(Args...) = nullptr;

    template <size_t... I>
    static PyObject* run(PyObject* const* args, std::index_sequence<I...>) {
        const std::tuple<Args...> values{value_of<Args>(args[I])...};
        if (PyErr_Occurred()) return nullptr;
        return PyLong_FromLong(function(std::get<I>(values)...));
    }

    static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count) {
        if (!function) {
            PyErr_SetString(PyExc_RuntimeError, "readout calls are not bound to the library");
            return nullptr;
        }
        if (count != (Py_ssize_t)sizeof...(Args)) {
            PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", (Py_ssize_t)sizeof...(Args), count);
            return nullptr;
        }
        return run(args, std::index_sequence_for<Args...>{});
    }
};

using Norm = Entry<0, decltype(mdsoap_rms_norm)>;
using NormBackward = Entry<1, decltype(mdsoap_rms_norm_backward)>;
using Quantize = Entry<2, decltype(mdsoap_quantize)>;
using Matmul = Entry<3, decltype(mdsoap_matmul)>;
using AdamWStep = Entry<4, decltype(mdsoap_adamw_step)>;

template <class E>
void bind_one(PyObject* address) {
    using F = decltype(E::function);
    E::function = value_of<F>(address);
}

// bind(rms_norm, rms_norm_backward, quantize, matmul, adamw_step): the functions' addresses.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (count != 5) {
        PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
        return nullptr;
    }
    bind_one<Norm>(args[0]);
    bind_one<NormBackward>(args[1]);
    bind_one<Quantize>(args[2]);
    bind_one<Matmul>(args[3]);
    bind_one<AdamWStep>(args[4]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// ---- what the optimizer looks at before every step: a few methods of each of
// its tensors, called from here without lists and sets in between (twelve
// tensors, addresses of parameters and moments among it: 10.4 -> 7.9 us a step).

PyObject *g_numel, *g_is_contiguous, *g_get_device, *g_data_ptr, *g_dtype;

// use(numel, is_contiguous, get_device, data_ptr): methods of a tensor.
PyObject* use(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (count != 4) {
        PyErr_SetString(PyExc_TypeError, "use takes four methods");
        return nullptr;
    }
    PyObject** const to[4] = {&g_numel, &g_is_contiguous, &g_get_device, &g_data_ptr};
    for (int i = 0; i < 4; ++i) {
        Py_INCREF(args[i]);
        Py_XSETREF(*to[i], args[i]);
    }
    if (!g_dtype && !(g_dtype = PyUnicode_InternFromString("dtype"))) return nullptr;
    Py_RETURN_NONE;
}

// A list, and that `use` was called.
bool ready(PyObject* list) {
    if (!g_dtype) PyErr_SetString(PyExc_RuntimeError, "readout calls know no tensor methods");
    else if (!PyList_Check(list)) PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
    else return true;
    return false;
}

// method(tensor) as an integer; the Python error is set where there is none.
unsigned long long ask(PyObject* method, PyObject* tensor) {
    PyObject* const answer = PyObject_Vectorcall(method, &tensor, 1, nullptr);
    if (!answer) return 0;
    const unsigned long long value = PyLong_AsUnsignedLongLongMask(answer);
    Py_DECREF(answer);
    return value;
}

// addresses(tensors): their data pointers, in a row.
PyObject* addresses(PyObject*, PyObject* tensors) {
    if (!ready(tensors)) return nullptr;
    const Py_ssize_t count = PyList_GET_SIZE(tensors);
    PyObject* const out = PyBytes_FromStringAndSize(nullptr, count * 8);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < count && !PyErr_Occurred(); ++i) {
        const uint64_t at = ask(g_data_ptr, PyList_GET_ITEM(tensors, i));
        std::memcpy(PyBytes_AS_STRING(out) + 8 * i, &at, 8);
    }
    if (!PyErr_Occurred()) return out;
    Py_DECREF(out);
    return nullptr;
}

// gather(tensors, sizes, device): their data pointers and their type; 1 where
// there are not as many tensors of these sizes, 2 where they are not contiguous,
// of one type and on the device.
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (count != 3 || !PyList_Check(args[1])) {
        PyErr_SetString(PyExc_TypeError, "gather takes tensors, a list of sizes and a device");
        return nullptr;
    }
    PyObject *const tensors = args[0], *const sizes = args[1];
    if (!ready(tensors)) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(tensors);
    const long long device = PyLong_AsLongLong(args[2]);
    if (n != PyList_GET_SIZE(sizes)) return PyLong_FromLong(1);
    for (Py_ssize_t i = 0; i < n; ++i)
        if ((long long)ask(g_numel, PyList_GET_ITEM(tensors, i)) != PyLong_AsLongLong(PyList_GET_ITEM(sizes, i)))
            return PyErr_Occurred() ? nullptr : PyLong_FromLong(1);
    PyObject* kind = nullptr;  // borrowed: a type lives as long as torch does
    PyObject* const out = PyBytes_FromStringAndSize(nullptr, n * 8);
    if (!out) return nullptr;
    bool fit = true;
    for (Py_ssize_t i = 0; i < n && fit; ++i) {
        PyObject* const tensor = PyList_GET_ITEM(tensors, i);
        PyObject* const own = PyObject_GetAttr(tensor, g_dtype);
        if (!own) break;
        Py_DECREF(own);
        if (i == 0) kind = own;
        fit = own == kind && ask(g_is_contiguous, tensor) && (long long)ask(g_get_device, tensor) == device;
        const uint64_t at = fit ? ask(g_data_ptr, tensor) : 0;
        std::memcpy(PyBytes_AS_STRING(out) + 8 * i, &at, 8);
    }
    if (PyErr_Occurred() || !fit) {
        Py_DECREF(out);
        return PyErr_Occurred() ? nullptr : PyLong_FromLong(2);
    }
    return Py_BuildValue("(NO)", out, kind ? kind : Py_None);
}

// identical(a, b): whether two lists hold the very same objects.
PyObject* identical(PyObject*, PyObject* const* args, Py_ssize_t count) {
    if (count != 2) {
        PyErr_SetString(PyExc_TypeError, "identical takes two lists");
        return nullptr;
    }
    bool same = PyList_Check(args[0]) && PyList_Check(args[1]) && PyList_GET_SIZE(args[0]) == PyList_GET_SIZE(args[1]);
    for (Py_ssize_t i = 0; same && i < PyList_GET_SIZE(args[0]); ++i)
        same = PyList_GET_ITEM(args[0], i) == PyList_GET_ITEM(args[1], i);
    return PyBool_FromLong(same);
}

template <class E>
PyCFunction entry() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&E::call));
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    {"rms_norm", entry<Norm>(), METH_FASTCALL, nullptr},
    {"rms_norm_backward", entry<NormBackward>(), METH_FASTCALL, nullptr},
    {"quantize", entry<Quantize>(), METH_FASTCALL, nullptr},
    {"matmul", entry<Matmul>(), METH_FASTCALL, nullptr},
    {"adamw_step", entry<AdamWStep>(), METH_FASTCALL, nullptr},
    {"use", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&use)), METH_FASTCALL, nullptr},
    {"addresses", addresses, METH_O, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&gather)), METH_FASTCALL, nullptr},
    {"identical", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&identical)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_readout_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__readout_call() { return PyModule_Create(&module); }
