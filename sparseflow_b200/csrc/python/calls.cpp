// Python calls of the operators around the gated FFN (include/sparseflow_b200.h, group 1b) without ctypes: eager calls of kernels of a few
// microseconds are bound by the host, and ctypes converts 25 arguments in 2.7 us where this takes 0.2 us.  Same names, arguments in the same order;
// pointers are ints or None.  An int that its parameter cannot hold raises OverflowError.
//
// Only the stable interface of CPython from 3.10 on is used, so that one build serves every interpreter that finds it in the tree.
#define Py_LIMITED_API 0x030A0000
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../../include/sparseflow_b200.h"

namespace {

template <class T>
bool convert(PyObject* o, T& v) {
  if constexpr (std::is_pointer_v<T>) {
    if (o == Py_None) { v = nullptr; return true; }
    v = static_cast<T>(PyLong_AsVoidPtr(o));
  } else if constexpr (std::is_floating_point_v<T>) {
    v = static_cast<T>(PyFloat_AsDouble(o));
  } else {
    const long long n = PyLong_AsLongLong(o);
    if (n < std::numeric_limits<T>::min() || n > std::numeric_limits<T>::max()) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_OverflowError, "%lld is beyond a C int", n);
      return false;
    }
    v = static_cast<T>(n);
  }
  return !PyErr_Occurred();
}

template <class R, class... A, size_t... I>
PyObject* call(R (*f)(A...), PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
  if (n != static_cast<Py_ssize_t>(sizeof...(A))) return PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", static_cast<Py_ssize_t>(sizeof...(A)), n);
  std::tuple<A...> v;
  if (!(convert(args[I], std::get<I>(v)) && ...)) return nullptr;
  R r;
  Py_BEGIN_ALLOW_THREADS      // a launch may wait for room in the stream's queue
  r = f(std::get<I>(v)...);
  Py_END_ALLOW_THREADS
  if constexpr (std::is_same_v<R, size_t>) return PyLong_FromSize_t(r);
  else return PyLong_FromLong(r);
}
template <class R, class... A>
PyObject* call(R (*f)(A...), PyObject* const* args, Py_ssize_t n) {
  return call(f, args, n, std::index_sequence_for<A...>());
}
template <auto F>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) { return call(F, args, n); }

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<&name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    ENTRY(sfb200_group_workspace_bytes), ENTRY(sfb200_group_rows), ENTRY(sfb200_moe_route), ENTRY(sfb200_grouped_scratch_bytes),
    ENTRY(sfb200_grouped_sparse_gemm), ENTRY(sfb200_grouped_sparse_gemm_swiglu), ENTRY(sfb200_moe_combine), ENTRY(sfb200_block_norm),
    ENTRY(sfb200_lora_workspace_bytes), ENTRY(sfb200_lora_add), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
