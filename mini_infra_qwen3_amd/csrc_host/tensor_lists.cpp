// Checks of per-layer tensor lists in one call: the data plane's entry points take a key and a value pool (and sources or
// outputs) of every layer, and asking Python for shape, type, layout, device and address of each took most of a small
// call's time.  56 pools of 28 layers: a block copy whose kernel takes 5 us took 21, and takes 7 with this; a gather over
// 112 tensors whose kernel takes 11 took 35, and takes 10 to 11.
//
// A CPython module beside the C ABI library, which knows no torch type.  It decides nothing: a list that is not uniform
// comes back as None, and the caller's own checks say what is wrong with it.
#include <Python.h>

#include <vector>

#include <torch/csrc/autograd/python_variable.h>

namespace {

// addresses(tensors, like, strided) -> bytes | None: the addresses (8 bytes each, native order) of GPU tensors that all have
// like's sizes, type and device, and are contiguous, or with `strided` have like's strides.
PyObject* addresses(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "addresses(tensors, like, strided)");
    return nullptr;
  }
  if (!THPVariable_Check(args[1]) || (!PyList_Check(args[0]) && !PyTuple_Check(args[0]))) Py_RETURN_NONE;
  const int strided = PyObject_IsTrue(args[2]);
  if (strided < 0) return nullptr;
  try {
    const at::Tensor& like = THPVariable_Unpack(args[1]);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(args[0]);
    std::vector<uint64_t> out(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* item = PySequence_Fast_GET_ITEM(args[0], i);
      if (!THPVariable_Check(item)) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(item);
      if (!t.is_cuda() || t.layout() != at::kStrided || t.device() != like.device() || t.scalar_type() != like.scalar_type() ||
          t.sizes() != like.sizes() || (strided ? t.strides() != like.strides() : !t.is_contiguous()))
        Py_RETURN_NONE;
      out[i] = reinterpret_cast<uint64_t>(t.data_ptr());
    }
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(out.data()), n * static_cast<Py_ssize_t>(sizeof(uint64_t)));
  } catch (...) {  // a tensor without storage, say: the caller's checks meet it again
    Py_RETURN_NONE;
  }
}

PyMethodDef methods[] = {{"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(addresses)), METH_FASTCALL,
                          "addresses(tensors, like, strided) -> bytes | None"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", "Checks of tensor lists.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() { return PyModule_Create(&module); }
