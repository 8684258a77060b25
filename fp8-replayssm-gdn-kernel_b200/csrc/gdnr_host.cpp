// Host-side call path of the prompt / mixed-batch operators: fills the gdnr_tensor
// views of a call from torch tensors and calls the C entry point on the current stream
// of their device.  In Python the views of eleven tensors take 10 us, more than the kernel of
// a call on a few tokens; here about 0.5 us.
//
//   _host.built_for   the torch and the Python it was compiled against
//   _host.call(address, tensors, tail) -> status
//     address   of an entry point int f(const void* args, void* stream)
//     tensors   tuple of CUDA tensors or None (absent), the leading gdnr_tensor fields
//     tail      bytes of the argument structure behind them
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstring>

#include "../../include/gdnr.h"

namespace {

int dtype_of(c10::ScalarType t) {
  switch (t) {
    case c10::ScalarType::Float: return GDNR_F32;
    case c10::ScalarType::Half: return GDNR_F16;
    case c10::ScalarType::BFloat16: return GDNR_BF16;
    case c10::ScalarType::Float8_e4m3fn: return GDNR_E4M3;
    case c10::ScalarType::Int: return GDNR_I32;
    case c10::ScalarType::Bool: case c10::ScalarType::Byte: return GDNR_U8;
    case c10::ScalarType::Char: return GDNR_I8;
    default: return GDNR_DT_NONE;
  }
}

constexpr Py_ssize_t MAX_TENSORS = 16, MAX_TAIL = 64;

// Sizes, strides and addresses throw for tensors that have none (transforms' wrappers, sparse ones), as the guard
// does for a missing device: all of it becomes a Python exception.
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3 || !PyTuple_Check(args[1]) || !PyBytes_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError, "call(address, tensors, tail)");
    return nullptr;
  }
  void* const address = PyLong_AsVoidPtr(args[0]);
  if (!address) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
    return nullptr;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(args[1]), tail = PyBytes_GET_SIZE(args[2]);
  if (n > MAX_TENSORS || tail > MAX_TAIL) {
    PyErr_SetString(PyExc_ValueError, "too many arguments");
    return nullptr;
  }
  alignas(16) unsigned char buf[MAX_TENSORS * sizeof(gdnr_tensor) + MAX_TAIL];
  std::memset(buf, 0, size_t(n) * sizeof(gdnr_tensor));
  int device = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* const o = PyTuple_GET_ITEM(args[1], i);
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "argument %zd is not a tensor", i);
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) {
      PyErr_Format(PyExc_ValueError, "libgdnr operates on CUDA tensors; got a tensor on %s", t.device().str().c_str());
      return nullptr;
    }
    if (device < 0) device = t.device().index();
    if (t.device().index() != device) {
      PyErr_Format(PyExc_ValueError, "tensors of one call have to be on one device; got cuda:%d and %s", device,
                   t.device().str().c_str());
      return nullptr;
    }
    gdnr_tensor d = {};
    d.dtype = dtype_of(t.scalar_type());
    if (d.dtype == GDNR_DT_NONE) {
      PyErr_Format(PyExc_ValueError, "dtype %s is not supported by libgdnr", c10::toString(t.scalar_type()));
      return nullptr;
    }
    if (t.dim() > 4) {
      PyErr_SetString(PyExc_ValueError, "libgdnr tensors have at most 4 dimensions");
      return nullptr;
    }
    d.data = t.data_ptr();
    if (!d.data) {
      if (t.numel() > 0) {  // a fake tensor, a wrapper subclass, a storage resized to nothing
        PyErr_Format(PyExc_ValueError, "argument %zd has elements but no memory", i);
        return nullptr;
      }
      d.data = reinterpret_cast<void*>(16);  // an empty tensor is present
    }
    d.ndim = int32_t(t.dim());
    for (int64_t k = 0; k < t.dim(); ++k) {
      d.shape[k] = t.size(k);
      d.stride[k] = t.stride(k);
    }
    std::memcpy(buf + size_t(i) * sizeof(gdnr_tensor), &d, sizeof(d));
  }
  if (device < 0) {
    PyErr_SetString(PyExc_ValueError, "no tensors");
    return nullptr;
  }
  std::memcpy(buf + size_t(n) * sizeof(gdnr_tensor), PyBytes_AS_STRING(args[2]), size_t(tail));
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  void* const stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  return PyLong_FromLong(reinterpret_cast<int (*)(const void*, void*)>(address)(buf, stream));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL, "call(address, tensors, tail) -> status"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Call path of libgdnr's prompt operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  PyObject* const m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", GDNR_BUILT_FOR) < 0) {  // the torch and the Python: build.py
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
