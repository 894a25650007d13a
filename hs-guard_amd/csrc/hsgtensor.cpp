// What the operators' wrappers ask of their tensors, and their outputs, as Python functions (CPython extension
// hs_guard._hsgtensor, host code only): device, type, layout and length of every operand and its address in one call. Asked one
// by one from Python this is most of a small call: 13 operands 5.5 us, 0.3 here; a gated-delta step of one row 10.7 -> 6.6 us
// of host time, the attention 15.4 -> 10.9, the maps (five outputs) 8.7 -> 6.1.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/Functions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

namespace {

PyObject* refuse(const char* why) {
  PyErr_SetString(PyExc_AssertionError, why);
  return nullptr;
}

bool shape_is(const at::Tensor& t, int64_t n) { return t.dim() == 1 && t.size(0) == n; }

// Why a tensor is not of its kind, or NULL
const char* mismatch(char kind, const at::Tensor& t, int64_t rows, int64_t tokens) {
  const at::ScalarType type = t.scalar_type();
  switch (kind) {
    case 'p':
      return type == at::kBFloat16 ? nullptr : "bf16 tensors expected";
    case 'b':
      return type != at::kBFloat16 ? "bf16 tensors expected" : t.is_contiguous() ? nullptr : "tensors must be contiguous";
    case 's':
      return (type == at::kFloat || type == at::kHalf) && t.is_contiguous() ? nullptr
                                                                            : "state must be contiguous, float32 or float16";
    case 'u':
      return type == at::kByte && t.is_contiguous() ? nullptr : "workspace must be contiguous uint8";
    default:
      if (type != at::kLong || !t.is_contiguous()) return "index tensors must be contiguous int64";
      if (kind == 'n' && !shape_is(t, rows)) return "lens, offsets, commits, starts and slots must be [n]";
      if (kind == 't' && !shape_is(t, tokens)) return "parents and masks must be [T], one for each packed token";
      return nullptr;
  }
}

// operands(kinds, rows, tokens, *tensors) -> (device, address of each). One letter a tensor: p bf16 whose rows may lie apart, b
// contiguous bf16, s contiguous fp32 or fp16, u contiguous uint8, i contiguous int64, n such of [rows], t of [tokens]; None has
// no address. All are on one GPU.
PyObject* operands(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 4) return refuse("operands(kinds, rows, tokens, *tensors)");
  Py_ssize_t count;
  const char* kinds = PyUnicode_AsUTF8AndSize(args[0], &count);
  if (!kinds) return nullptr;
  const int64_t rows = PyLong_AsLongLong(args[1]), tokens = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  if (count != nargs - 3) return refuse("one kind for each tensor");
  PyObject* out = PyTuple_New(count + 1);
  if (!out) return nullptr;
  try {
    int64_t device = -1;
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* const o = args[3 + i];
      PyObject* address = nullptr;
      if (o == Py_None) {
        address = Py_None;
        Py_INCREF(address);
      } else {
        const char* why = THPVariable_Check(o) ? nullptr : "tensors expected";
        if (!why) {
          const at::Tensor& t = THPVariable_Unpack(o);
          if (!t.is_cuda()) why = "HS-Guard kernels take GPU tensors";
          else if (device >= 0 && t.get_device() != device) why = "tensors must be on one GPU";
          else why = mismatch(kinds[i], t, rows, tokens);
          if (!why) {
            device = t.get_device();
            address = PyLong_FromVoidPtr(t.data_ptr());
          }
        }
        if (why) refuse(why);
        if (!address) {
          Py_DECREF(out);
          return nullptr;
        }
      }
      PyTuple_SET_ITEM(out, i + 1, address);
    }
    PyObject* const index = PyLong_FromLongLong(device);
    if (!index) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, 0, index);
    return out;
  } catch (const std::exception& e) {
    Py_DECREF(out);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// row_stride(tensor, tokens, width) -> elements between its tokens, each of which holds `width` values next to one another
PyObject* row_stride(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3 || !THPVariable_Check(args[0])) return refuse("row_stride(tensor, tokens, width)");
  const int64_t tokens = PyLong_AsLongLong(args[1]), width = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor& t = THPVariable_Unpack(args[0]);
    if (t.dim() == 0 || t.size(0) != tokens || t.numel() != tokens * width)
      return refuse(("[" + std::to_string(tokens) + ", " + std::to_string(width) + "] values expected").c_str());
    if (t.is_contiguous()) return PyLong_FromLongLong(width);
    int64_t inner = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      if (t.size(d) != 1 && t.stride(d) != inner) return refuse("a token's values must be contiguous");
      inner *= t.size(d);
    }
    const int64_t stride = tokens > 1 ? t.stride(0) : width;
    if (stride < width) return refuse("tokens must not overlap");
    return PyLong_FromLongLong(stride);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// empties(like, *lengths) -> a tensor [length] of like's type and device for each, all in one allocation. (Tensors made of a
// storage and a size: a slice of a tensor costs as much as an allocation.)
PyObject* empties(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 2 || !THPVariable_Check(args[0])) return refuse("empties(like, *lengths)");
  int64_t total = 0;
  for (Py_ssize_t i = 1; i < nargs; ++i) {
    const int64_t n = PyLong_AsLongLong(args[i]);
    if (n < 0) return PyErr_Occurred() ? nullptr : refuse("lengths are not negative");
    total += n;
  }
  PyObject* out = PyTuple_New(nargs - 1);
  if (!out) return nullptr;
  try {
    const at::Tensor all = at::empty({total}, THPVariable_Unpack(args[0]).options());
    int64_t at = 0;
    for (Py_ssize_t i = 1; i < nargs; ++i) {
      const int64_t n = PyLong_AsLongLong(args[i]);
      at::Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
      part.unsafeGetTensorImpl()->set_storage_offset(at);
      part.unsafeGetTensorImpl()->set_sizes_contiguous({n});
      PyObject* const o = THPVariable_Wrap(part);
      if (!o) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i - 1, o);
      at += n;
    }
    return out;
  } catch (const std::exception& e) {
    Py_DECREF(out);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// empty_rows(like, rows, width) -> a tensor [rows, width] of like's type and device
PyObject* empty_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3 || !THPVariable_Check(args[0])) return refuse("empty_rows(like, rows, width)");
  const int64_t rows = PyLong_AsLongLong(args[1]), width = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  try {
    return THPVariable_Wrap(at::empty({rows, width}, THPVariable_Unpack(args[0]).options()));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"empty_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&empty_rows)), METH_FASTCALL, nullptr},
    {"empties", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&empties)), METH_FASTCALL, nullptr},
    {"operands", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&operands)), METH_FASTCALL, nullptr},
    {"row_stride", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&row_stride)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hsgtensor", "Checks of the operators' tensors", -1, methods, nullptr, nullptr,
                      nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hsgtensor(void) { return PyModule_Create(&module); }
