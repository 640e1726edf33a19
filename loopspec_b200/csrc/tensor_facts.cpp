// What the serving operators' Python wrappers ask of their tensor arguments, in
// one call each instead of five to eight attribute reads at 50-110 ns: a small
// call spent 4-5 of its 8-9 microseconds on them, more than its kernel runs.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

namespace {

// LS_BF16, LS_F16, LS_F32, then int32 and bytes; -1: another type
int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    case at::kInt: return 3;
    case at::kByte: return 4;
    default: return -1;
  }
}

const at::Tensor* as_tensor(PyObject* o) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  PyErr_Format(PyExc_TypeError, "expected a tensor, got %s", Py_TYPE(o)->tp_name);
  return nullptr;
}

bool on_gpu(const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided; }

// facts(t) -> (data pointer, device index, type code, *sizes, *strides), or None unless t is a CUDA tensor.
PyObject* facts(PyObject*, PyObject* arg) {
  try {
    const at::Tensor* t = as_tensor(arg);
    if (!t) return nullptr;
    if (!on_gpu(*t)) Py_RETURN_NONE;
    const int64_t dims = t->dim();
    PyObject* out = PyTuple_New(3 + 2 * dims);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, PyLong_FromUnsignedLongLong(reinterpret_cast<uintptr_t>(t->mutable_data_ptr())));
    PyTuple_SET_ITEM(out, 1, PyLong_FromLong(t->get_device()));
    PyTuple_SET_ITEM(out, 2, PyLong_FromLong(type_code(*t)));
    for (int64_t d = 0; d < dims; ++d) {
      PyTuple_SET_ITEM(out, 3 + d, PyLong_FromLongLong(t->size(d)));
      PyTuple_SET_ITEM(out, 3 + dims + d, PyLong_FromLongLong(t->stride(d)));
    }
    return out;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// pointers(device index, type code, t0, n0, t1, n1, ...) -> the data pointers (0
// for None), or None unless every tensor is a contiguous one on that GPU, of that
// type and with n elements (-1: any number).
PyObject* pointers(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  constexpr Py_ssize_t kMost = 16;
  const Py_ssize_t n = (n_args - 2) / 2;
  if (n_args < 2 || n_args % 2 != 0 || n > kMost) {
    PyErr_SetString(PyExc_TypeError, "expected a device index, a type code and up to 16 pairs of tensor and count");
    return nullptr;
  }
  try {
    const long device = PyLong_AsLong(args[0]), type = PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    uintptr_t found[kMost] = {};
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = args[2 + 2 * i];
      if (o == Py_None) continue;
      const at::Tensor* t = as_tensor(o);
      if (!t) return nullptr;
      const long long count = PyLong_AsLongLong(args[3 + 2 * i]);
      if (count == -1 && PyErr_Occurred()) return nullptr;
      if (!on_gpu(*t) || t->get_device() != device || type_code(*t) != type || !t->is_contiguous() ||
          (count >= 0 && t->numel() != count))
        Py_RETURN_NONE;
      found[i] = reinterpret_cast<uintptr_t>(t->mutable_data_ptr());
    }
    PyObject* out = PyTuple_New(n);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) PyTuple_SET_ITEM(out, i, PyLong_FromUnsignedLongLong(found[i]));
    return out;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"facts", facts, METH_O, "(data pointer, device index, type code, *sizes, *strides) of a CUDA tensor, else None"},
    {"pointers", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pointers)), METH_FASTCALL,
     "data pointers of contiguous tensors on one GPU, of one type, with the given element counts, else None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_facts", nullptr, -1, methods};

}  // namespace

// made_for: the torch and the Python that this module was compiled against
PyMODINIT_FUNC PyInit__tensor_facts() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddObject(m, "made_for", Py_BuildValue("(sii)", TORCH_VERSION, PY_MAJOR_VERSION, PY_MINOR_VERSION)) < 0)
    Py_CLEAR(m);
  return m;
}
