// CPython calls of the readout operators' C entry points: through ctypes the
// twenty arguments of a product take 2 to 3 us to convert, here a few tenths (one
// row's product 11.7 -> 9.2 us a call).
// The functions are handed over by address from the library that _lib.py
// loaded, so both bindings call the same copy of it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/mdsoap.h"

#include <cstdint>
#include <tuple>
#include <type_traits>
#include <utility>

namespace {

// One argument: None is a null pointer, pointers and integers are ints.
template <class T>
T value_of(PyObject* o) {
    if constexpr (std::is_pointer_v<T>) {
        return o == Py_None ? nullptr : reinterpret_cast<T>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o)));
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
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_readout_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__readout_call() { return PyModule_Create(&module); }
