// insmos_amd/csrc/host_tensors.cpp -- the host side of the optimiser step that touches every tensor: one pass in C++ over Python lists of
// tensors that checks them and writes the InsmosOptTensor table (include/insmos_hip.h).  From Python the same pass costs ten attribute
// reads per tensor (some 0.1 us each: 0.5 ms for 250 tensors, ten times what the GPU needs for them).  Built as the extension module
// insmos_amd._host; nothing here runs on the GPU.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <string>
#include <utility>
#include <vector>

#include "../../include/insmos_hip.h"

namespace {

struct Refused : std::exception {
    std::string text;
    explicit Refused(std::string t) : text(std::move(t)) {}
    const char* what() const noexcept override { return text.c_str(); }
};

// whether a tensor fills its memory without gaps or overlaps, in some order of its dimensions
bool dense(const at::Tensor& t) {
    if (t.is_contiguous()) return true;
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t want = 1;
    for (const auto& d : dims) {
        if (d.first != want) return false;
        want *= d.second;
    }
    return true;
}
bool same_order(const at::Tensor& a, const at::Tensor& b) { return a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()); }

const char* place(const at::Tensor& t, std::string& buf) {
    buf = std::string(c10::toString(t.scalar_type())) + " on " + t.device().str();
    return buf.c_str();
}
const at::Tensor& tensor_at(PyObject* list, Py_ssize_t i, const char* what, const char* kind) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) throw Refused(std::string(what) + ": " + kind + " " + std::to_string(i) + " is no tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != c10::kStrided) throw Refused(std::string(what) + ": " + kind + " " + std::to_string(i) + " is sparse");
    return t;
}
int dtype_code(c10::ScalarType t) {
    return t == c10::ScalarType::Float ? INSMOS_F32 : t == c10::ScalarType::BFloat16 ? INSMOS_BF16 : t == c10::ScalarType::Half ? INSMOS_F16 : -1;
}

// opt_table(what, params or None, grads, table, any_device) -> (entries, dtype code, length of the state buffers, gradients to reorder)
// params None: grads alone (the norm).  A gradient whose memory order is not its parameter's (or, alone, that is not dense) is named in the
// last list, by index: the caller puts a copy in its place and calls again.
PyObject* opt_table(PyObject*, PyObject* args) {
    const char* what;
    PyObject *params, *grads;
    Py_buffer out;
    int any_device;
    if (!PyArg_ParseTuple(args, "sOO!w*p", &what, &params, &PyList_Type, &grads, &out, &any_device)) return nullptr;
    PyObject* reorder = nullptr;
    PyObject* result = nullptr;
    try {
        const bool alone = params == Py_None;
        if (!alone && !PyList_Check(params)) throw Refused(std::string(what) + ": params is a list");
        const Py_ssize_t n = PyList_GET_SIZE(grads);
        if (!alone && PyList_GET_SIZE(params) != n)
            throw Refused(std::string(what) + ": " + std::to_string(PyList_GET_SIZE(params)) + " parameters and " + std::to_string(n) + " gradients");
        if (n == 0) throw Refused(std::string(what) + ": no " + (alone ? "gradients" : "parameters"));
        if (out.len < (Py_ssize_t)sizeof(InsmosOptTensor) * n) throw Refused(std::string(what) + ": the table is too short");
        reorder = PyList_New(0);
        if (!reorder) throw Refused("out of memory");
        InsmosOptTensor* table = (InsmosOptTensor*)out.buf;
        const char* kind = alone ? "tensor" : "parameter";
        const at::Tensor& first = tensor_at(alone ? grads : params, 0, what, kind);
        const int code = dtype_code(first.scalar_type());
        std::string a, b;
        if (code < 0) throw Refused(std::string(what) + ": float32, bfloat16 or float16, not " + place(first, a));
        if (!any_device && !first.is_cuda()) throw Refused(std::string(what) + ": tensors on the GPU, not on " + first.device().str());
        Py_ssize_t used = 0;
        int64_t off = 0;
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;
        for (Py_ssize_t i = 0; i < n; ++i) {
            const at::Tensor& p = tensor_at(alone ? grads : params, i, what, kind);
            if (p.scalar_type() != first.scalar_type() || p.device() != first.device())
                throw Refused(std::string(what) + ": " + kind + " " + std::to_string(i) + " is " + place(p, a) + ", the first one " + place(first, b));
            const int64_t count = p.numel();
            InsmosOptTensor e = {nullptr, nullptr, count, off};
            off += (count + 255) / 256 * 256;
            if (!alone) {
                if (!dense(p)) throw Refused(std::string(what) + ": parameter " + std::to_string(i) + " has gaps or overlaps in memory");
                e.param = p.data_ptr();
                if (count) spans.emplace_back((uintptr_t)e.param, (uintptr_t)e.param + (uintptr_t)count * p.element_size());
                if (PyList_GET_ITEM(grads, i) == Py_None) continue;
            }
            const at::Tensor& g = alone ? p : tensor_at(grads, i, what, "gradient");
            if (!alone) {
                if (g.scalar_type() != first.scalar_type() || g.device() != first.device())
                    throw Refused(std::string(what) + ": gradient " + std::to_string(i) + " is " + place(g, a) + ", its parameter " + place(p, b));
                if (g.sizes() != p.sizes()) throw Refused(std::string(what) + ": gradient " + std::to_string(i) + " is of another shape than its parameter");
            }
            if (alone ? !dense(g) : !same_order(g, p)) {
                PyObject* k = PyLong_FromSsize_t(i);
                if (!k || PyList_Append(reorder, k)) { Py_XDECREF(k); throw Refused("out of memory"); }
                Py_DECREF(k);
            }
            e.grad = g.data_ptr();
            table[used++] = e;
        }
        // a parameter that appears twice, or overlaps another, would be written by lanes of two workgroups
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].first < spans[i - 1].second) throw Refused(std::string(what) + ": two parameters share memory");
        result = Py_BuildValue("niLO", used, code, (long long)off, reorder);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "opt_table failed");
    }
    Py_XDECREF(reorder);
    PyBuffer_Release(&out);
    return result;
}

PyMethodDef kMethods[] = {{"opt_table", opt_table, METH_VARARGS, "checks lists of tensors and writes their InsmosOptTensor table"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
