// What a launch takes of its tensors, checked and read in one native call: type, device, shape and layout against what is expected,
// and the addresses.  us a call, checked in Python / here: adjusted logits of one row, 13 tensors, 10.4 / 7.2 (its kernel takes 4.0);
// rows of 64 requests, 10 tensors, 9.4 / 6.8 (5.0); pages of 64 requests 7.2 / 5.9 (3.2).  Called with the interpreter's lock held
// (ctypes.PyDLL).  The checks in ops/kernels.py (_at, _rows_of) are what these mean: they run where this says no, and give the
// reason, and where the library could not be built.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

// spec: (device, tensor, dtype, shape, tensor, dtype, shape, ...) with tuples of whole numbers as shapes; a tensor may be None.  out gets
// an address a tensor (0 for None).  0: all of them are contiguous tensors of that type and shape on that device; else which is not, from 1 on.
extern "C" long long kva_tensor_args(PyObject *spec, long long *out) {
    if (!PyTuple_Check(spec) || PyTuple_GET_SIZE(spec) % 3 != 1) return -1;
    const Py_ssize_t n = PyTuple_GET_SIZE(spec);
    const long device = PyLong_AsLong(PyTuple_GET_ITEM(spec, 0));
    if (device == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return -1;
    }
    try {
        for (Py_ssize_t i = 1, j = 0; i < n; i += 3, ++j) {
            PyObject *t = PyTuple_GET_ITEM(spec, i), *type = PyTuple_GET_ITEM(spec, i + 1), *shape = PyTuple_GET_ITEM(spec, i + 2);
            if (t == Py_None) {
                out[j] = 0;
                continue;
            }
            if (!THPVariable_Check(t) || !THPDtype_Check(type) || !PyTuple_Check(shape)) return j + 1;
            const at::Tensor &x = THPVariable_Unpack(t);
            if (!x.is_cuda() || x.layout() != at::kStrided || x.get_device() != device || x.scalar_type() != reinterpret_cast<THPDtype *>(type)->scalar_type ||
                x.dim() != PyTuple_GET_SIZE(shape) || !x.is_contiguous())
                return j + 1;
            for (int64_t d = 0; d < x.dim(); ++d) {
                const long long expected = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
                if (expected == -1 && PyErr_Occurred()) {
                    PyErr_Clear();
                    return j + 1;
                }
                if (expected != x.size(d)) return j + 1;
            }
            out[j] = (long long)(uintptr_t)x.data_ptr();
        }
    } catch (...) {
        return -1;
    }
    return 0;
}

// out: address, rows, columns, elements from a row to the next, type (0 fp32, 1 bf16), device.  0: a matrix on a GPU whose rows'
// elements lie next to each other and whose rows do not overlap.
extern "C" long long kva_tensor_rows(PyObject *t, long long *out) {
    if (!THPVariable_Check(t)) return 1;
    try {
        const at::Tensor &x = THPVariable_Unpack(t);
        if (!x.is_cuda() || x.layout() != at::kStrided || x.dim() != 2) return 1;
        const long long rows = x.size(0), cols = x.size(1);
        if ((cols > 1 && x.stride(1) != 1) || (rows > 1 && x.stride(0) < cols)) return 1;
        const bool f32 = x.scalar_type() == at::kFloat;
        if (!f32 && x.scalar_type() != at::kBFloat16) return 1;
        out[0] = (long long)(uintptr_t)x.data_ptr();
        out[1] = rows;
        out[2] = cols;
        out[3] = rows > 1 ? x.stride(0) : cols;
        out[4] = f32 ? 0 : 1;
        out[5] = x.get_device();
    } catch (...) {
        return 1;
    }
    return 0;
}
