// The Python host's short way to mtl_launch: a launch whose buffers are torch tensors,
// checked and packed in one call.
//
// launch(plan, args, ndrange, stream, workspace) returns mtl_launch's status, or None where
// anything is not as plain as this: every buffer argument a contiguous CUDA tensor on the
// current device of the element type the kernel wants (or None, where the kernel allows it),
// every scalar an int or a float, ndrange an int. The caller then takes its long way, which
// knows the other kinds of buffers and says what is wrong. So this file refuses nothing and
// allows nothing that the long way would not.

#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdint>
#include <cstring>
#include <vector>

#include "../../../include/mantle_cuda.h"

namespace {

using Launch = mtl_status (*)(int32_t, const mtl_arg*, int32_t, const int64_t*, int32_t, void*, uint64_t, void*);
constexpr int kMost = 32;

struct Plan {
  Launch entry;
  int32_t kernel;
  int buffers, args;
  char letter[kMost];   // what each buffer holds: f, h, i, or o, t, p, q by the argument below
  int by[kMost];
  char kind[kMost];     // the signature: B, b, i, f
};

// Whether an element type can stand for the letter: f Float32, h bfloat16 (or its bits), i
// Int32, 4 and 5 codes in e4m3 and e5m2 (or bytes).
bool stands_for(c10::ScalarType t, char letter) {
  using S = c10::ScalarType;
  switch (letter) {
    case 'f': return t == S::Float;
    case 'h': return t == S::BFloat16 || t == S::UInt16 || t == S::Short;
    case 'i': return t == S::Int;
    case '4': return t == S::Byte || t == S::Char || t == S::Float8_e4m3fn;
    case '5': return t == S::Byte || t == S::Char || t == S::Float8_e5m2;
  }
  return false;
}

// plan(entry address, kernel, signature, letters, by): what launch() is to check.
PyObject* plan(PyObject*, PyObject* args) {
  unsigned long long entry;
  int kernel;
  const char *signature, *letters;
  PyObject* by;
  if (!PyArg_ParseTuple(args, "KissO!", &entry, &kernel, &signature, &letters, &PyTuple_Type, &by)) return nullptr;
  auto* p = new Plan();
  p->entry = reinterpret_cast<Launch>(entry);
  p->kernel = kernel;
  p->buffers = (int)std::strlen(letters);
  p->args = (int)std::strlen(signature);
  if (p->args > kMost || p->buffers > p->args || PyTuple_GET_SIZE(by) != p->buffers) {
    delete p;
    PyErr_SetString(PyExc_ValueError, "plan: signature, letters and by do not fit together");
    return nullptr;
  }
  std::memcpy(p->kind, signature, p->args);
  std::memcpy(p->letter, letters, p->buffers);
  for (int i = 0; i < p->buffers; ++i) {
    p->by[i] = (int)PyLong_AsLong(PyTuple_GET_ITEM(by, i));
    if (PyErr_Occurred() || p->by[i] >= p->args) {
      delete p;
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "plan: no such argument");
      return nullptr;
    }
  }
  return PyCapsule_New(p, "plan", [](PyObject* c) { delete static_cast<Plan*>(PyCapsule_GetPointer(c, "plan")); });
}

// An int that fits 32 bits. (A bool is one, as it is for struct.)
bool int32_of(PyObject* o, int32_t* v) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || x < INT32_MIN || x > INT32_MAX) return false;
  *v = (int32_t)x;
  return true;
}

// The tensor's address and bytes where it is a contiguous one on `device` (which is asked
// for with the first).
// A tensor that has no such thing (a sparse one, one without storage) throws: it is not plain.
bool tensor_of(PyObject* o, int* device, char letter, uint64_t* ptr, uint64_t* bytes) try {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || !t.is_contiguous() || t.layout() != c10::kStrided) return false;
  if (*device < 0) *device = c10::cuda::current_device();
  if (t.get_device() != *device) return false;
  if (letter && !stands_for(t.scalar_type(), letter)) return false;
  *ptr = reinterpret_cast<uint64_t>(t.data_ptr());
  *bytes = (uint64_t)t.nbytes();
  return *ptr || !*bytes;  // values without an address: a tensor without storage
} catch (...) {
  return false;
}

PyObject* launch(PyObject*, PyObject* const* in, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  const auto* p = static_cast<const Plan*>(PyCapsule_GetPointer(in[0], "plan"));
  if (!p) return nullptr;
  PyObject* args = in[1];
  if (!PyTuple_Check(args) || PyTuple_GET_SIZE(args) != p->args || !PyLong_Check(in[2])) Py_RETURN_NONE;
  int over = 0;
  const long long range = PyLong_AsLongLongAndOverflow(in[2], &over);
  const unsigned long long stream = PyLong_Check(in[3]) ? PyLong_AsUnsignedLongLong(in[3]) : ~0ull;
  if (over || PyErr_Occurred() || stream == ~0ull) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  mtl_arg a[kMost];
  std::memset(a, 0, sizeof(mtl_arg) * p->args);
  for (int i = p->buffers; i < p->args; ++i) {
    PyObject* o = PyTuple_GET_ITEM(args, i);
    if (p->kind[i] == 'f') {
      a[i].kind = MTL_ARG_F32;
      if (!PyFloat_Check(o)) Py_RETURN_NONE;
      const double v = PyFloat_AS_DOUBLE(o);
      if (v > 3.4e38 || v < -3.4e38) Py_RETURN_NONE;
      a[i].v.f32 = (float)v;
    } else {
      a[i].kind = MTL_ARG_I32;
      if (p->kind[i] != 'i' || !int32_of(o, &a[i].v.i32)) Py_RETURN_NONE;
    }
  }
  int device = -1;
  for (int i = 0; i < p->buffers; ++i) {
    PyObject* o = PyTuple_GET_ITEM(args, i);
    if (o == Py_None) {
      if (p->kind[i] != 'b') Py_RETURN_NONE;
      a[i].kind = MTL_ARG_NULL;
      continue;
    }
    char letter = p->letter[i];
    if (p->by[i] >= 0) {
      const int32_t which = a[p->by[i]].v.i32;
      if (which != 0 && which != 1) Py_RETURN_NONE;
      letter = letter == 'o' || letter == 't' ? "fh"[which] : "45"[which];
    }
    a[i].kind = MTL_ARG_PTR;
    if (!tensor_of(o, &device, letter, &a[i].v.ptr, &a[i].bytes)) Py_RETURN_NONE;
  }
  uint64_t scratch = 0, size = 0;
  if (in[4] != Py_None && !tensor_of(in[4], &device, 0, &scratch, &size)) Py_RETURN_NONE;
  const int64_t nd[3] = {range, 1, 1};
  mtl_status st;
  Py_BEGIN_ALLOW_THREADS;
  st = p->entry(p->kernel, a, p->args, nd, 1, reinterpret_cast<void*>(scratch), size, reinterpret_cast<void*>(stream));
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong((long)st);
}

PyMethodDef methods[] = {{"plan", plan, METH_VARARGS, nullptr},
                         {"launch", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(launch)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Tensors are read by the layout of the torch that this was compiled against, so no other will do.
PyMODINIT_FUNC PyInit__launch(void) {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  Py_XDECREF(torch);
  if (!version) return nullptr;
  const bool same = PyUnicode_Check(version) && PyUnicode_CompareWithASCIIString(version, BUILT_FOR_TORCH) == 0;
  if (!same) PyErr_Format(PyExc_ImportError, "_launch was built for torch " BUILT_FOR_TORCH ", not %S", version);
  Py_DECREF(version);
  return same ? PyModule_Create(&module) : nullptr;
}
