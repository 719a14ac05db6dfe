// binding.cpp — the host side of a call from Python: makes the results that
// the caller did not give and lays out the descriptors of a call's tensors in
// one buffer.  In Python this costs a microsecond and more per tensor, more than
// the rest of a single-token call.
//
//   describe(device, operands, table) -> (buffer, results, address, ...) or None
//
// operands: a tuple of (name, tensor or None, rank), with a dtype as fourth
// field for other types than f32, and for a result, as fifth field, what it is
// made like where it was not given: a tensor whose shape it gets or a tuple of
// sizes (None: left out).  `results` holds the operands with five fields, given
// or made (contiguous and unset); their storage is asked for as what is written,
// so that one shared with a lazy clone becomes the result's own.  The buffer (bytes, to be kept until the call
// returns) holds a RemoraMemRefN for each tensor; its address follows in the
// tuple, None for None.  With table = k > 0 the first k addresses form an
// argument struct at the buffer's start, whose address stands for them.  None is
// returned when an operand is not a tensor of its type, rank and device, or a view
// whose values are the negatives of what its storage holds: the caller says which.
//
//   room(device, bytes) -> (uint8 tensor of that many unset bytes, its address)
//
//   written(tensor or None, ...): raises the version of what a call has written, by
//   which autograd notices that a value it kept is gone
#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

namespace {

constexpr Py_ssize_t kMaxOperands = 32;
constexpr int64_t kMaxRank = 10;

// of a negative device: in host memory
at::Tensor unset(at::IntArrayRef sizes, at::ScalarType type, long device) {
  const at::Device place = device < 0 ? at::Device(at::kCPU) : at::Device(at::kCUDA, (at::DeviceIndex)device);
  return at::empty(sizes, at::TensorOptions().dtype(type).device(place));
}

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
  at::Tensor results[kMaxOperands];
  const at::Tensor *tensors[kMaxOperands];
  int64_t starts[kMaxOperands];  // all that may throw is done before memory is taken
  int64_t words = table;
  for (Py_ssize_t k = 0; k < n; ++k) {
    PyObject *item = PyTuple_GET_ITEM(operands, k);
    const Py_ssize_t fields = PyTuple_Check(item) ? PyTuple_GET_SIZE(item) : 0;
    if (fields < 3 || fields > 5) {
      PyErr_SetString(PyExc_TypeError, "describe: an operand is (name, tensor, rank[, dtype[, shape]])");
      return nullptr;
    }
    PyObject *value = PyTuple_GET_ITEM(item, 1);
    tensors[k] = nullptr;
    PyObject *shape = fields == 5 ? PyTuple_GET_ITEM(item, 4) : Py_None;
    const bool make = value == Py_None && shape != Py_None;
    if (value == Py_None && !make) continue;
    if (!make && !THPVariable_Check(value)) Py_RETURN_NONE;
    const long rank = PyLong_AsLong(PyTuple_GET_ITEM(item, 2));
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type = at::kFloat;
    if (fields >= 4) {
      PyObject *d = PyTuple_GET_ITEM(item, 3);
      if (!THPDtype_Check(d)) {
        PyErr_SetString(PyExc_TypeError, "describe: the fourth field is a torch dtype");
        return nullptr;
      }
      type = reinterpret_cast<THPDtype *>(d)->scalar_type;
    }
    if (make) {
      int64_t sizes[kMaxRank] = {0};
      at::IntArrayRef of;
      if (THPVariable_Check(shape)) {
        of = THPVariable_Unpack(shape).sizes();
      } else if (PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) <= kMaxRank) {
        for (Py_ssize_t d = 0; d < PyTuple_GET_SIZE(shape); ++d) sizes[d] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
        if (PyErr_Occurred()) return nullptr;
        of = at::IntArrayRef(sizes, PyTuple_GET_SIZE(shape));
      } else {
        PyErr_SetString(PyExc_TypeError, "describe: the fifth field is a tensor or a tuple of at most 10 sizes");
        return nullptr;
      }
      results[k] = unset(of, type, device);
    }
    const at::Tensor &t = make ? results[k] : THPVariable_Unpack(value);
    if (t.scalar_type() != type || t.dim() != rank || rank > kMaxRank || t.get_device() != device ||
        !t.has_storage() || t.is_neg())
      Py_RETURN_NONE;
    tensors[k] = &t;
    t.strides();
    words += 3 + 2 * rank;
  }
  // results first: an operand may be the same tensor, or a view of it
  for (Py_ssize_t k = 0; k < n; ++k)
    if (tensors[k] && tensors[k]->numel() && PyTuple_GET_SIZE(PyTuple_GET_ITEM(operands, k)) == 5)
      tensors[k]->storage().mutable_data();
  for (Py_ssize_t k = 0; k < n; ++k)
    if (tensors[k])
      starts[k] = tensors[k]->numel() ? (int64_t)reinterpret_cast<uintptr_t>(tensors[k]->storage().data()) : 0;
  PyObject *buffer = PyBytes_FromStringAndSize(nullptr, words * 8);
  if (buffer == nullptr) return nullptr;
  char *base = PyBytes_AS_STRING(buffer);
  int64_t *out = reinterpret_cast<int64_t *>(base), *to = out + table;
  Py_ssize_t count = 0;
  for (Py_ssize_t k = 0; k < n; ++k) count += PyTuple_GET_SIZE(PyTuple_GET_ITEM(operands, k)) == 5;
  PyObject *made = PyTuple_New(count);
  PyObject *result = made ? PyTuple_New(2 + (table ? 1 : 0) + n - table) : nullptr;
  if (result == nullptr) {
    Py_XDECREF(made);
    Py_DECREF(buffer);
    return nullptr;
  }
  count = 0;
  for (Py_ssize_t k = 0; k < n; ++k) {
    PyObject *item = PyTuple_GET_ITEM(operands, k);
    if (PyTuple_GET_SIZE(item) != 5) continue;
    PyObject *out = PyTuple_GET_ITEM(item, 1);
    if (results[k].defined())
      out = THPVariable_Wrap(results[k]);
    else
      Py_INCREF(out);
    PyTuple_SET_ITEM(made, count++, out);
  }
  PyTuple_SET_ITEM(result, 0, buffer);
  PyTuple_SET_ITEM(result, 1, made);
  Py_ssize_t at = 2;
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

// torch throws without memory for a result, and for tensors without plain strides
// or storage (nested, wrapped)
PyObject *describe(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  return layout(args, nargs);
  END_HANDLE_TH_ERRORS
}

PyObject *room(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "room(device, bytes)");
    return nullptr;
  }
  const long device = PyLong_AsLong(args[0]);
  const int64_t bytes = PyLong_AsLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  HANDLE_TH_ERRORS
  const at::Tensor t = unset({bytes}, at::kByte, device);
  return Py_BuildValue("NN", THPVariable_Wrap(t), PyLong_FromVoidPtr(t.data_ptr()));
  END_HANDLE_TH_ERRORS
}

PyObject *written(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t k = 0; k < nargs; ++k) {
    if (args[k] == Py_None) continue;
    if (!THPVariable_Check(args[k])) {
      PyErr_SetString(PyExc_TypeError, "written(tensor or None, ...)");
      return nullptr;
    }
    const at::Tensor &t = THPVariable_Unpack(args[k]);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // an inference tensor has none
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"describe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(describe)), METH_FASTCALL,
     "describe(device, operands, table) -> (buffer, results, address, ...) or None"},
    {"room", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(room)), METH_FASTCALL,
     "room(device, bytes) -> (uint8 tensor, its address)"},
    {"written", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(written)), METH_FASTCALL,
     "written(tensor or None, ...): raises their versions"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", "Descriptors of a call's tensors.", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
  PyObject *module = PyModule_Create(&module_def);
  if (module && PyModule_AddStringConstant(module, "torch_release", REMORA_TORCH_RELEASE) < 0) Py_CLEAR(module);
  return module;
}
