// binding_args.cpp -- the part of the Python binding that runs once per tensor of a paged call: torch tensors into the descriptors of the C ABI (include/ggml_hip_cdna4.h).
// A paged call is a few microseconds of work on the device and takes up to eleven tensors; reading type, device, sizes, strides and address of one through Python costs 0.55 us, here 0.1.
// A CPython module over torch's own C++ tensors; no HIP, no kernels.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ops/empty.h>

#include <cstdint>
#include <cstring>
#include <exception>

namespace {
struct Desc { void *data; int32_t type; int64_t ne[4]; int64_t nb[4]; };          // cdna4_tensor
static_assert(sizeof(Desc) == 80, "cdna4_tensor");
PyObject *g_error = nullptr;          // Cdna4Error(code, message)

PyObject *refuse(const char *name, const char *what) {
    PyObject *msg = PyUnicode_FromFormat("%s: %s", name, what);
    if (!msg) return nullptr;
    PyObject *e = g_error ? PyObject_CallFunction(g_error, "iO", -2, msg) : nullptr;
    if (e) { PyErr_SetObject(g_error, e); Py_DECREF(e); } else if (!PyErr_Occurred()) PyErr_SetObject(PyExc_ValueError, msg);
    Py_DECREF(msg);
    return nullptr;
}
// enum ggml_type of a torch type, -1: none of the ABI's
int type_of(at::ScalarType t) {
    switch (t) { case at::kFloat: return 0; case at::kHalf: return 1; case at::kInt: return 26; case at::kBFloat16: return 30; default: return -1; }
}
// on device `index` (-1: host memory, for the functions that need no device)
bool is_on(const at::Tensor &x, long index) { return index < 0 ? x.is_cpu() : x.is_cuda() && x.get_device() == index; }

// a call into torch that throws (a tensor without memory of its own, for one) is a refusal and not the end of the process
#define GUARDED(...) try { __VA_ARGS__ } catch (const std::exception &) { return refuse(name, "a tensor with strided memory of its own"); }

// desc(tensor, name, device): the 80 bytes of a cdna4_tensor, sizes and byte strides from the innermost dimension out
PyObject *desc(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 3) { PyErr_SetString(PyExc_TypeError, "desc(tensor, name, device)"); return nullptr; }
    const char *name = PyUnicode_AsUTF8(a[1]); const long index = PyLong_AsLong(a[2]);
    if (!name || (index == -1 && PyErr_Occurred())) return nullptr;
    if (!THPVariable_Check(a[0])) return refuse(name, "a tensor");
    GUARDED(
    const at::Tensor &x = THPVariable_Unpack(a[0]);
    if (x.layout() != at::kStrided || x.is_neg() || !is_on(x, index)) return refuse(name, "a strided tensor on the backend's device");          // (is_neg: memory holds the negated values)
    const int type = type_of(x.scalar_type()); const int64_t dims = x.dim(), es = type == 0 || type == 26 ? 4 : 2;
    if (type < 0) return refuse(name, "float32, float16, bfloat16 or int32");
    if (dims < 2 || dims > 4) return refuse(name, "2 to 4 dimensions");
    Desc d; std::memset(&d, 0, sizeof(d));
    d.data = x.data_ptr(); d.type = type;
    if (!d.data && x.numel()) return refuse(name, "a tensor with memory of its own");
    const auto ne = x.sizes(), st = x.strides();
    for (int64_t i = 0; i < 4; ++i) { d.ne[i] = i < dims ? ne[dims - 1 - i] : 1; d.nb[i] = i < dims ? st[dims - 1 - i] * es : 0; }
    return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&d), sizeof(d));
    )
}
// vec(tensor or None, name, elements, type, device): the address of a dense vector, None for None
PyObject *vec(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "vec(tensor, name, elements, type, device)"); return nullptr; }
    if (a[0] == Py_None) Py_RETURN_NONE;
    const char *name = PyUnicode_AsUTF8(a[1]); const long count = PyLong_AsLong(a[2]), type = PyLong_AsLong(a[3]), index = PyLong_AsLong(a[4]);
    if (!name || PyErr_Occurred()) return nullptr;
    const char *what = type == 0 ? "a dense float32 vector of as many elements on the backend's device" : "a dense int32 vector of as many elements on the backend's device";
    if (!THPVariable_Check(a[0])) return refuse(name, what);
    GUARDED(
    const at::Tensor &x = THPVariable_Unpack(a[0]);
    if (x.layout() != at::kStrided || x.is_neg() || !is_on(x, index) || type_of(x.scalar_type()) != type || x.numel() != count || !x.is_contiguous()) return refuse(name, what);
    return PyLong_FromVoidPtr(x.data_ptr());
    )
}
// empty(tensor, type, size ...): a dense tensor of type 0 (float32) or 26 (int32) on the tensor's device
PyObject *empty(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS          // (out of memory stays what torch calls it)
    if (n < 3 || n > 6 || !THPVariable_Check(a[0])) { PyErr_SetString(PyExc_TypeError, "empty(tensor, type, size ...)"); return nullptr; }
    const long type = PyLong_AsLong(a[1]); int64_t size[4] = {0, 0, 0, 0};
    for (Py_ssize_t i = 2; i < n; ++i) size[i - 2] = PyLong_AsLongLong(a[i]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor &x = THPVariable_Unpack(a[0]);
    return THPVariable_Wrap(at::empty(at::IntArrayRef(size, (size_t)(n - 2)), at::TensorOptions().device(x.device()).dtype(type == 0 ? at::kFloat : at::kInt)));
    END_HANDLE_TH_ERRORS
}
PyObject *set_error(PyObject *, PyObject *cls) { Py_INCREF(cls); Py_XDECREF(g_error); g_error = cls; Py_RETURN_NONE; }

PyMethodDef methods[] = {{"desc", (PyCFunction)(void *)desc, METH_FASTCALL, "cdna4_tensor of a torch tensor"}, {"vec", (PyCFunction)(void *)vec, METH_FASTCALL, "address of a dense vector"},
                         {"empty", (PyCFunction)(void *)empty, METH_FASTCALL, "a new dense tensor beside another"},
                         {"set_error", set_error, METH_O, "the class of what is raised"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "cdna4_args", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}
PyMODINIT_FUNC PyInit_cdna4_args(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_with", BUILT_WITH) < 0) { Py_DECREF(m); return nullptr; }          // (the loader compares it with the torch that is there)
    return m;
}
