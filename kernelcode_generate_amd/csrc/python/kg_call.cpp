// kernelcode_generate_amd._kg_call: an entry of libkg_gfx950.so called with torch tensors, numbers and None, their slots packed here
// from the tensors' own sizes and strides. native.call_entry packs the same slots in Python, 0.4 us a tensor (a call of 11 operands
// 9.2 us, 4 of them the library's), and does so wherever this module says that it does not know an argument.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "kg_gfx950.h"

namespace {

constexpr Py_ssize_t kMostArgs = 32;
constexpr int64_t kMostAxes = 8;  // of a tensor; no entry takes as many
using Entry = int (*)(const KgArgSlot*, unsigned long long);

int dtype_code(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return KG_DTYPE_F32;
    case at::kDouble: return KG_DTYPE_F64;
    case at::kInt: return KG_DTYPE_I32;
    case at::kLong: return KG_DTYPE_I64;
    case at::kHalf: return KG_DTYPE_F16;
    case at::kBFloat16: return KG_DTYPE_BF16;
    case at::kChar: return KG_DTYPE_I8;
    case at::kFloat8_e4m3fn: return KG_DTYPE_E4M3;
    default: return 0;
  }
}

const long long kAbsent[2] = {0, 1};  // extent and stride of an absent memory slot
const long long kScalar[1] = {0};     // of a tensor of rank 0

// A tensor's extents and strides, copied: the entry runs without the interpreter's lock, and another thread may change the tensor's view.
struct Axes {
  long long shape[kMostAxes], stride[kMostAxes];
};

// False: an argument that native.py takes its own way (a subclass, another number type, an integer past 64 bits).
bool fill(KgArgSlot* slot, Axes* axes, PyObject* arg) {
  *slot = KgArgSlot{};
  if (arg == Py_None) {
    slot->kind = KG_ARG_MEMORY;
    slot->shape = &kAbsent[0];
    slot->stride = &kAbsent[1];
    slot->rank = 1;
  } else if (PyLong_CheckExact(arg)) {
    int past = 0;
    slot->kind = KG_ARG_INT;
    slot->int_value = PyLong_AsLongLongAndOverflow(arg, &past);
    return past == 0;
  } else if (PyFloat_CheckExact(arg)) {
    slot->kind = KG_ARG_FLOAT;
    slot->float_value = PyFloat_AS_DOUBLE(arg);
  } else if (THPVariable_CheckExact(arg)) {
    const at::Tensor& t = THPVariable_Unpack(arg);
    const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
    if (t.dim() > kMostAxes) return false;
    for (int64_t i = 0; i < t.dim(); ++i) {
      axes->shape[i] = sizes[i];
      axes->stride[i] = strides[i];
    }
    slot->kind = KG_ARG_MEMORY;
    slot->dtype_code = dtype_code(t.scalar_type());
    slot->rank = (unsigned long long)t.dim();
    slot->shape = t.dim() == 0 ? kScalar : axes->shape;
    slot->stride = t.dim() == 0 ? kScalar : axes->stride;
    slot->data = t.mutable_data_ptr();  // (an entry may write it: a lazy copy is made here, as by data_ptr())
    return slot->dtype_code != 0;
  } else {
    return false;
  }
  return true;
}

// call(address of the entry, arguments as a tuple) -> its status, or None: an argument that is not known here
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 2 || !PyLong_Check(args[0]) || !PyTuple_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "call(address, arguments)");
    return nullptr;
  }
  const Entry entry = reinterpret_cast<Entry>(PyLong_AsVoidPtr(args[0]));
  const Py_ssize_t slots = PyTuple_GET_SIZE(args[1]);
  if (entry == nullptr || slots > kMostArgs) Py_RETURN_NONE;
  KgArgSlot slot[kMostArgs];
  Axes axes[kMostArgs];
  try {
    for (Py_ssize_t i = 0; i < slots; ++i)
      if (!fill(&slot[i], &axes[i], PyTuple_GET_ITEM(args[1], i))) Py_RETURN_NONE;
  } catch (...) {  // (a tensor without extents or memory of its own)
    Py_RETURN_NONE;
  }
  int status;
  Py_BEGIN_ALLOW_THREADS  // (the tuple keeps the tensors)
  status = entry(slot, (unsigned long long)slots);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

PyMethodDef kMethods[] = {{"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call)), METH_FASTCALL,
                           "call(address, arguments) -> status, or None where an argument is not known"},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kg_call", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

// "version commit" of the torch that runs, as build.py writes KG_TORCH from the one that it compiles against.
PyObject* running_torch() {
  PyObject *torch = PyImport_ImportModule("torch"), *text = nullptr;
  PyObject* version = torch != nullptr ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  PyObject* versions = version != nullptr ? PyObject_GetAttrString(torch, "version") : nullptr;
  PyObject* commit = versions != nullptr ? PyObject_GetAttrString(versions, "git_version") : nullptr;
  if (versions != nullptr) {
    PyErr_Clear();  // (a torch may name no commit)
    text = commit == nullptr || commit == Py_None ? PyUnicode_FromFormat("%S", version) : PyUnicode_FromFormat("%S %S", version, commit);
  }
  Py_XDECREF(commit);
  Py_XDECREF(versions);
  Py_XDECREF(version);
  Py_XDECREF(torch);
  return text;
}

}  // namespace

// Tensors are read by torch's inlined layouts and Python's objects by its macros, which no missing symbol tells apart: another version
// of either is refused.
PyMODINIT_FUNC PyInit__kg_call() {
  const char* const python = Py_GetVersion();
  const size_t own = sizeof(KG_PYTHON) - 1;  // "3.10."
  if (strncmp(python, KG_PYTHON, own) != 0) {
    PyErr_Format(PyExc_ImportError, "built against Python %sx, this is %s", KG_PYTHON, python);
    return nullptr;
  }
  PyObject* const torch = running_torch();
  if (torch == nullptr) return nullptr;
  const bool same = PyUnicode_CompareWithASCIIString(torch, KG_TORCH) == 0;
  if (!same) PyErr_Format(PyExc_ImportError, "built against torch %s, this is %S", KG_TORCH, torch);
  Py_DECREF(torch);
  return same ? PyModule_Create(&kModule) : nullptr;
}
