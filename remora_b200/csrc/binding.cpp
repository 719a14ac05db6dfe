// binding.cpp — the host side of a call from Python: lays out the descriptors
// of a call's tensors in one buffer.  In Python this costs a microsecond per
// tensor, more than the rest of a single-token call.
//
//   describe(device, operands, table) -> (buffer, address, ...) or None
//
// operands: a tuple of (name, tensor or None, rank) or, for other types than
// f32, (name, tensor or None, rank, dtype).  The buffer (bytes, to be kept until
// the call returns) holds a RemoraMemRefN for each tensor; its address follows
// in the tuple, None for None.  With table = k > 0 the first k addresses form an
// argument struct at the buffer's start, whose address stands for them.  None is
// returned when an operand is not a tensor of its type, rank and device: the
// caller says which.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

namespace {

constexpr Py_ssize_t kMaxOperands = 32;
constexpr int64_t kMaxRank = 10;

PyObject *layout(PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 3 || !PyTuple_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "describe(device, operands, table)");
    return nullptr;
  }
  const long device = PyLong_AsLong(args[0]);
  PyObject *operands = args[1];
  const long table = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const Py_ssize_t n = PyTuple_GET_SIZE(operands);
  if (n > kMaxOperands || table < 0 || table > n) {
    PyErr_SetString(PyExc_ValueError, "describe: too many operands, or a table longer than they are");
    return nullptr;
  }
  const at::Tensor *tensors[kMaxOperands];
  int64_t starts[kMaxOperands];  // all that may throw is done before memory is taken
  int64_t words = table;
  for (Py_ssize_t k = 0; k < n; ++k) {
    PyObject *item = PyTuple_GET_ITEM(operands, k);
    const Py_ssize_t fields = PyTuple_Check(item) ? PyTuple_GET_SIZE(item) : 0;
    if (fields != 3 && fields != 4) {
      PyErr_SetString(PyExc_TypeError, "describe: an operand is (name, tensor, rank) or (name, tensor, rank, dtype)");
      return nullptr;
    }
    PyObject *value = PyTuple_GET_ITEM(item, 1);
    tensors[k] = nullptr;
    if (value == Py_None) continue;
    if (!THPVariable_Check(value)) Py_RETURN_NONE;
    const at::Tensor &t = THPVariable_Unpack(value);
    const long rank = PyLong_AsLong(PyTuple_GET_ITEM(item, 2));
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type = at::kFloat;
    if (fields == 4) {
      PyObject *d = PyTuple_GET_ITEM(item, 3);
      if (!THPDtype_Check(d)) {
        PyErr_SetString(PyExc_TypeError, "describe: the fourth field is a torch dtype");
        return nullptr;
      }
      type = reinterpret_cast<THPDtype *>(d)->scalar_type;
    }
    if (t.scalar_type() != type || t.dim() != rank || rank > kMaxRank || t.get_device() != device ||
        !t.has_storage())
      Py_RETURN_NONE;
    tensors[k] = &t;
    starts[k] = t.numel() ? (int64_t)reinterpret_cast<uintptr_t>(t.storage().data()) : 0;
    t.strides();
    words += 3 + 2 * rank;
  }
  PyObject *buffer = PyBytes_FromStringAndSize(nullptr, words * 8);
  if (buffer == nullptr) return nullptr;
  char *base = PyBytes_AS_STRING(buffer);
  int64_t *out = reinterpret_cast<int64_t *>(base), *to = out + table;
  PyObject *result = PyTuple_New(1 + (table ? 1 : 0) + n - table);
  if (result == nullptr) {
    Py_DECREF(buffer);
    return nullptr;
  }
  PyTuple_SET_ITEM(result, 0, buffer);
  Py_ssize_t at = 1;
  if (table) PyTuple_SET_ITEM(result, at++, PyLong_FromVoidPtr(base));
  for (Py_ssize_t k = 0; k < n; ++k) {
    const int64_t here = tensors[k] ? (int64_t)reinterpret_cast<uintptr_t>(to) : 0;
    if (k < table) {
      out[k] = here;
    } else if (here) {
      PyTuple_SET_ITEM(result, at++, PyLong_FromLongLong(here));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(result, at++, Py_None);
    }
    if (!here) continue;
    // {allocated, aligned, offset, sizes, strides}: the storage's base, the
    // view's start in `offset`; an empty tensor has neither
    const at::Tensor &t = *tensors[k];
    const int64_t offset = t.numel() ? t.storage_offset() : 0;
    to[0] = to[1] = starts[k];
    to[2] = offset;
    const int64_t rank = t.dim();
    std::memcpy(to + 3, t.sizes().data(), rank * 8);
    std::memcpy(to + 3 + rank, t.strides().data(), rank * 8);
    to += 3 + 2 * rank;
  }
  if (PyErr_Occurred()) {
    Py_DECREF(result);
    return nullptr;
  }
  return result;
}

// torch throws for tensors without plain strides or storage (nested, wrapped)
PyObject *describe(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  try {
    return layout(args, nargs);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_TypeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"describe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(describe)), METH_FASTCALL,
     "describe(device, operands, table) -> (buffer, address, ...) or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", "Descriptors of a call's tensors.", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module_def); }
