// Host side of the many-tensor operators (Python module _fgs_host): reads gradients, addresses and sizes of tensor
// lists and checks them, at about 15 ns per tensor where the same through Python attributes takes about 75 ns for each
// of the five things that are checked. No compute and no CUDA calls; the lists are read anew at every call.
#include <Python.h>
#include <exception>
#include <torch/csrc/autograd/python_variable.h>

namespace {

const char* kTypeNames[] = {"float32", "bfloat16", "float16", "uint8"};

int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        case at::kByte: return 3;
        default: return -1;
    }
}

// live(params) -> [(type code, parameters, gradients), ...]: the parameters that have a gradient, by type
PyObject* live(PyObject*, PyObject* arg) {
    if (!PyList_Check(arg)) return PyErr_Format(PyExc_TypeError, "a list of parameters is needed");
    PyObject* lists[3][2] = {};
    PyObject* out = nullptr;
    try {
        const Py_ssize_t n = PyList_GET_SIZE(arg);
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject* o = PyList_GET_ITEM(arg, i);
            if (!THPVariable_Check(o)) {
                PyErr_SetString(PyExc_TypeError, "parameters must be tensors");
                goto done;
            }
            const at::Tensor& p = THPVariable_Unpack(o);
            const at::Tensor& g = p.grad();
            if (!g.defined()) continue;
            const int c = type_code(p);
            if (c < 0 || c > 2) {
                PyErr_SetString(PyExc_RuntimeError, "parameters must be float32, bfloat16 or float16 tensors");
                goto done;
            }
            for (int k = 0; k < 2; k++)
                if (!lists[c][k] && !(lists[c][k] = PyList_New(0))) goto done;
            PyObject* go = THPVariable_Wrap(g);
            if (!go) goto done;
            const bool bad = PyList_Append(lists[c][0], o) != 0 || PyList_Append(lists[c][1], go) != 0;
            Py_DECREF(go);
            if (bad) goto done;
        }
        out = PyList_New(0);
        for (int c = 0; out && c < 3; c++) {
            if (!lists[c][0]) continue;
            PyObject* t = Py_BuildValue("(iOO)", c, lists[c][0], lists[c][1]);
            if (!t || PyList_Append(out, t) != 0) Py_CLEAR(out);
            Py_XDECREF(t);
        }
    } catch (const std::exception& e) {
        Py_CLEAR(out);
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
done:
    for (auto& pair : lists)
        for (PyObject* l : pair) Py_XDECREF(l);
    return out;
}

// pack(tensors, name, type code, device index, counts address, per, addresses address): writes every tensor's data
// address; counts: int64 per tensor, written with its element count (per = 0), or checked: count elements (per = 1) or
// one per `per` of them. Returns the device index. Raises RuntimeError for a tensor of another type, device (device
// index -1: the first tensor's, which must be a CUDA one), size or layout.
PyObject* pack(PyObject*, PyObject* args) {
    PyObject* list;
    const char* name;
    int code, device;
    long long per;
    unsigned long long counts_at, addresses_at;
    if (!PyArg_ParseTuple(args, "O!siiKLK", &PyList_Type, &list, &name, &code, &device, &counts_at, &per, &addresses_at)) return nullptr;
    if (code < 0 || code > 3) return PyErr_Format(PyExc_ValueError, "unknown type code");
    auto* counts = reinterpret_cast<int64_t*>(counts_at);
    auto* addresses = reinterpret_cast<uint64_t*>(addresses_at);
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o)) return PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
            const at::Tensor& t = THPVariable_Unpack(o);
            if (t.layout() != at::kStrided || type_code(t) != code || !t.is_contiguous())
                return PyErr_Format(PyExc_RuntimeError, "%s must be a contiguous %s tensor", name, kTypeNames[code]);
            if (!t.is_cuda()) return PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor", name);
            if (device < 0) device = t.get_device();
            if (t.get_device() != device) return PyErr_Format(PyExc_RuntimeError, "%s must be on device cuda:%d like the others", name, device);
            const int64_t numel = t.numel();
            if (per == 0) counts[i] = numel;
            else if (numel != (counts[i] + per - 1) / per)
                return PyErr_Format(PyExc_RuntimeError, "%s has %lld elements, expected %lld", name, static_cast<long long>(numel),
                                    static_cast<long long>((counts[i] + per - 1) / per));
            addresses[i] = reinterpret_cast<uint64_t>(t.data_ptr());
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    return PyLong_FromLong(device);
}

PyMethodDef kMethods[] = {{"live", live, METH_O, "parameters with a gradient, by type"},
                          {"pack", pack, METH_VARARGS, "checked addresses of a list of tensors"},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fgs_host", "checked addresses of tensor lists", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fgs_host() { return PyModule_Create(&kModule); }
