// tensors.cc - uninitialised tensors for the ops' results and workspaces, several in one call (module _tensors).
//
// Through torch's Python interface a tensor costs 1.4 to 2.1 us, here 0.5: of an op on small tensors that is most of its time on the host, beside a launch of some
// 3 us. new(like, spec, ...) returns a tuple with one contiguous tensor on like's device for each spec (dtype, size, ...), None for None.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

namespace {

PyObject* make(const at::Device device, PyObject* spec) {
    if (!PyTuple_Check(spec) || PyTuple_GET_SIZE(spec) < 1 || PyTuple_GET_SIZE(spec) > 9 || !THPDtype_Check(PyTuple_GET_ITEM(spec, 0))) {
        PyErr_SetString(PyExc_TypeError, "a tuple of a dtype and up to eight sizes is wanted");
        return nullptr;
    }
    const Py_ssize_t dims = PyTuple_GET_SIZE(spec) - 1;
    int64_t size[8];
    for (Py_ssize_t i = 0; i < dims; ++i) {
        size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(spec, i + 1));
        if (size[i] == -1 && PyErr_Occurred()) return nullptr;
        if (size[i] < 0) {
            PyErr_SetString(PyExc_ValueError, "a size is negative");
            return nullptr;
        }
    }
    const at::ScalarType type = reinterpret_cast<THPDtype*>(PyTuple_GET_ITEM(spec, 0))->scalar_type;
    return THPVariable_Wrap(at::Tensor(at::detail::empty_cuda(at::IntArrayRef(size, static_cast<size_t>(dims)), type, device, std::nullopt)));
}

PyObject* new_tensors(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n < 1 || !THPVariable_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "the first argument has to be a tensor");
        return nullptr;
    }
    // what torch throws (out of memory) becomes its Python exception
    HANDLE_TH_ERRORS
    const at::Device device = THPVariable_Unpack(args[0]).device();
    if (!device.is_cuda()) {
        PyErr_SetString(PyExc_ValueError, "a CUDA tensor is wanted");
        return nullptr;
    }
    THPObjectPtr out(PyTuple_New(n - 1));
    if (!out) return nullptr;
    for (Py_ssize_t i = 1; i < n; ++i) {
        PyObject* t = args[i] == Py_None ? Py_NewRef(Py_None) : make(device, args[i]);
        if (!t) return nullptr;
        PyTuple_SET_ITEM(out.get(), i - 1, t);
    }
    return out.release();
    END_HANDLE_TH_ERRORS
}

PyMethodDef functions[] = {
    {"new", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&new_tensors)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, functions, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
