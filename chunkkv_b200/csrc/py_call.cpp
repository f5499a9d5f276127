// CPython calls of the entry points that a decode step makes by the dozen.
//
// Converting some twenty arguments through ctypes takes 1.3 to 2.6 us a call, as long as the
// smaller kernels run.  Here each entry point gets a wrapper made from its declared
// parameter types: pointers from ints or None, integers with a range check, floats.  The
// addresses come from the loaded library (bind), so this module links against nothing.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <iterator>
#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "chunkkv_b200.h"

namespace {

template <typename T>
bool convert(PyObject* o, T& out) {
  if constexpr (std::is_pointer_v<T>) {
    if (o == Py_None) {
      out = nullptr;
      return true;
    }
    out = reinterpret_cast<T>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o)));
  } else if constexpr (std::is_floating_point_v<T>) {
    out = static_cast<T>(PyFloat_AsDouble(o));
  } else {
    static_assert(std::is_integral_v<T> && std::is_signed_v<T>);
    const long long x = PyLong_AsLongLong(o);
    if (x < std::numeric_limits<T>::min() || x > std::numeric_limits<T>::max()) {
      PyErr_Format(PyExc_OverflowError, "%lld does not fit %d bits", x, static_cast<int>(8 * sizeof(T)));
      return false;
    }
    out = static_cast<T>(x);
  }
  return PyErr_Occurred() == nullptr;
}

// One wrapper per entry point; Tag keeps those of equal types apart.
template <auto Tag, typename F>
struct Call;
template <auto Tag, typename... A>
struct Call<Tag, int (*)(A...)> {
  static inline int (*fn)(A...) = nullptr;
  static PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != Py_ssize_t(sizeof...(A))) {
      PyErr_Format(PyExc_TypeError, "%zd arguments, %zu expected", n, sizeof...(A));
      return nullptr;
    }
    return go(args, std::index_sequence_for<A...>{});
  }
  template <size_t... I>
  static PyObject* go(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<A...> v{};
    if (!(convert(args[I], std::get<I>(v)) && ...)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  }
};

struct Entry {
  const char* name;
  PyMethodDef def;
  void (*set)(uintptr_t);
};
#define CKV_ENTRY(name)                                                                                  \
  []() -> Entry {                                                                                        \
    using W = Call<__LINE__, decltype(&name)>;                                                           \
    return {#name,                                                                                       \
            {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&W::run)), METH_FASTCALL, nullptr}, \
            [](uintptr_t p) { W::fn = reinterpret_cast<decltype(&name)>(p); }};                          \
  }()
Entry entries[] = {
    CKV_ENTRY(ckv_kv8_write),
    CKV_ENTRY(ckv_kv8_read),
    CKV_ENTRY(ckv_block_digest),
    CKV_ENTRY(ckv_attention_kv8),
    CKV_ENTRY(ckv_block_select),
    CKV_ENTRY(ckv_attention_blocks),
    CKV_ENTRY(ckv_attention_blocks_kv8),
    CKV_ENTRY(ckv_attention_sparse),
    CKV_ENTRY(ckv_attention_sparse_kv8),
};

// bind(name, address) -> the entry point as a builtin function
PyObject* bind(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "sK", &name, &address)) return nullptr;
  for (Entry& e : entries)
    if (std::strcmp(e.name, name) == 0) {
      e.set(static_cast<uintptr_t>(address));
      return PyCFunction_New(&e.def, nullptr);
    }
  PyErr_Format(PyExc_KeyError, "%s", name);
  return nullptr;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind(name, address) -> callable"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_call", "Direct calls of libchunkkv_b200.so", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call() {
  PyObject* m = PyModule_Create(&module_def);
  if (m == nullptr) return nullptr;
  PyObject* names = PyTuple_New(Py_ssize_t(std::size(entries)));
  for (size_t i = 0; names != nullptr && i < std::size(entries); ++i)
    PyTuple_SET_ITEM(names, Py_ssize_t(i), PyUnicode_FromString(entries[i].name));
  if (names == nullptr || PyModule_AddObject(m, "names", names) < 0) {
    Py_XDECREF(names);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
