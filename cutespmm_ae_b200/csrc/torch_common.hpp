// What the files of the torch binding share: errors of the C ABI as Python exceptions, the current stream, arguments of CPython fast
// calls, operators looked up once.
#pragma once
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/cutespmm.h"

namespace bind {

using at::Tensor;

inline PyObject *g_error_class = nullptr;  // CuteSpmmError(status, message)

// The GIL is held.
inline void set_status_error(int status)
{
    const char *msg = cutespmm_last_error();
    if (!msg || !*msg) msg = cutespmm_status_string(status);
    PyObject *e = g_error_class ? PyObject_CallFunction(g_error_class, "is", status, msg) : nullptr;
    if (e) {
        PyErr_SetObject(reinterpret_cast<PyObject *>(Py_TYPE(e)), e);
        Py_DECREF(e);
    } else if (!PyErr_Occurred()) {
        PyErr_SetString(PyExc_RuntimeError, msg);
    }
}

inline void check_status(int status)  // with or without the GIL
{
    if (status == CUTESPMM_OK) return;
    PyGILState_STATE g = PyGILState_Ensure();
    set_status_error(status);
    python_error err;
    err.persist();
    PyGILState_Release(g);
    throw err;
}

inline void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

template <class Sig> c10::TypedOperatorHandle<Sig> handle(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

inline const Tensor &tensor(PyObject *o, const char *what)
{
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a torch tensor");
    return THPVariable_Unpack(o);
}
inline Tensor tensor_or_none(PyObject *o, const char *what) { return o == Py_None ? Tensor() : tensor(o, what); }
inline int64_t integer(PyObject *o)
{
    const int64_t v = o == Py_None ? 0 : (int64_t)PyLong_AsUnsignedLongLong(o);
    if (PyErr_Occurred()) throw python_error();
    return v;
}
inline void *pointer(PyObject *o) { return reinterpret_cast<void *>(integer(o)); }
inline void want_args(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n); }
// a stream the caller named: its handle (the default stream's is 0, which the calls above read as "the current one")
inline void *named_stream(PyObject *o)
{
    if (o == Py_None) return nullptr;
    void *s = pointer(o);
    return s ? s : reinterpret_cast<void *>(0x1);  // cudaStreamLegacy
}

// fn without the interpreter lock, as ctypes makes its calls: a launch that waits for room in its stream's queue must not hold
// up other threads, and threads that drive a stream each run side by side.  The calls below take their arguments out of
// Python first and hold references of their own to the tensors.
template <class Fn> auto without_gil(Fn &&fn)
{
    struct Released {
        PyThreadState *state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
    } released;
    return fn();
}

// Adds the calls of torch_pattern.cpp to the module.
int add_pattern_calls(PyObject *module);

}  // namespace bind
