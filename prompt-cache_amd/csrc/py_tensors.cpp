// What the wrappers of the paged cache look at in a tensor before a launch, in one call from Python instead of five to ten: a step's kernels are shorter than those looks.
// Nothing is decided here: a tensor that does not qualify goes to the Python function of the same name, which says what is wrong with it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

namespace {

PyObject* slow[4];                                                    // flat, heads, table, pool in Python
enum { FLAT, HEADS, TABLE, POOL };

// the tensor behind an argument, null where there is none
const at::Tensor* tensor_of(PyObject* o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.layout() == at::kStrided ? &t : nullptr;
}
PyObject* address(const at::Tensor& t) { return PyLong_FromVoidPtr(t.data_ptr()); }
bool number(PyObject* o, long long& v) {
    v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
// contiguous, of a type, on a device, of at least n elements
bool whole(const at::Tensor* t, at::ScalarType type, long long n, long long dev) {
    return t && t->scalar_type() == type && t->get_device() == dev && t->is_contiguous() && t->numel() >= n;
}

template <typename F>
PyObject* guarded(int which, PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F&& f) {
    PyObject* r = nullptr;
    if (n == want) {
        try {
            r = f();
        } catch (...) {                                               // (a tensor without memory or strides)
            r = nullptr;
        }
    }
    if (r || PyErr_Occurred()) return r;
    if (!slow[which]) {
        PyErr_SetString(PyExc_RuntimeError, "behind(..) comes first");
        return nullptr;
    }
    return PyObject_Vectorcall(slow[which], args, (size_t)n, nullptr);
}

// flat(tensor or None, dtype, elements, device, what) -> address
PyObject* flat(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n == 5 && a[0] == Py_None) return PyLong_FromLong(0);
    return guarded(FLAT, a, n, 5, [&]() -> PyObject* {
        long long least, dev;
        if (!THPDtype_Check(a[1]) || !number(a[2], least) || !number(a[3], dev)) return nullptr;
        const at::Tensor* t = tensor_of(a[0]);
        return whole(t, reinterpret_cast<THPDtype*>(a[1])->scalar_type, least, dev) ? address(*t) : nullptr;
    });
}

// heads(tensor, heads, dim, device, what) -> (address, row stride, head stride)
PyObject* heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(HEADS, a, n, 5, [&]() -> PyObject* {
        long long h, dim, dev;
        const at::Tensor* t = tensor_of(a[0]);
        if (!t || !number(a[1], h) || !number(a[2], dim) || !number(a[3], dev) || t->dim() != 3) return nullptr;
        const auto size = t->sizes(), stride = t->strides();
        if (size[1] != h || size[2] != dim || (stride[2] != 1 && t->numel() > 0) || t->get_device() != dev) return nullptr;
        return Py_BuildValue("NLL", address(*t), (long long)(size[0] > 1 ? stride[0] : 0), (long long)(h > 1 ? stride[1] : 0));
    });
}

// table(tensor, rows, device, what) -> (address, row stride, pages)
PyObject* table(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(TABLE, a, n, 4, [&]() -> PyObject* {
        long long rows, dev;
        const at::Tensor* t = tensor_of(a[0]);
        if (!t || !number(a[1], rows) || !number(a[2], dev) || t->dim() != 2 || t->scalar_type() != at::kInt) return nullptr;
        const auto size = t->sizes(), stride = t->strides();
        if (size[0] < rows || (stride[1] != 1 && t->numel() > 0) || t->get_device() != dev) return nullptr;
        return Py_BuildValue("NLL", address(*t), (long long)(size[0] > 1 ? stride[0] : std::max(stride[0], size[1])), (long long)size[1]);
    });
}

// pool(key codes, key scales, value codes, value scales, device, what) -> (code, pages, P, Hkv, dim)
PyObject* pool(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(POOL, a, n, 6, [&]() -> PyObject* {
        long long dev;
        const at::Tensor *kc = tensor_of(a[0]), *ks = tensor_of(a[1]), *vc = tensor_of(a[2]), *vs = tensor_of(a[3]);
        if (!kc || !vc || !number(a[4], dev) || kc->dim() != 4 || vc->dim() != 4) return nullptr;
        const auto type = kc->scalar_type();
        const auto k = kc->sizes(), v = vc->sizes();
        if ((type != at::kFloat8_e4m3fn && type != at::kChar) || v[0] != k[0] || v[1] != k[1] || v[2] != k[3] || v[3] != k[2]) return nullptr;
        if (!whole(kc, type, 0, dev) || !whole(vc, type, 0, dev) || !whole(ks, at::kFloat, k[0] * k[1], dev) || !whole(vs, at::kFloat, k[0] * k[1], dev)) return nullptr;
        return Py_BuildValue("iLLLL", type == at::kChar ? 1 : 0, (long long)k[0], (long long)k[2], (long long)k[1], (long long)k[3]);
    });
}

// behind(flat, heads, table, pool): the Python functions that say what is wrong
PyObject* behind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "four functions");
        return nullptr;
    }
    for (int i = 0; i < 4; ++i) {
        Py_INCREF(a[i]);
        Py_XSETREF(slow[i], a[i]);
    }
    Py_RETURN_NONE;
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(flat), ENTRY(heads), ENTRY(table), ENTRY(pool), ENTRY(behind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
