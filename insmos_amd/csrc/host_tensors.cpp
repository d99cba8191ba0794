// insmos_amd/csrc/host_tensors.cpp -- host sides that Python is too slow for, over torch's tensors.  Built as the extension module
// insmos_amd._host; nothing here runs on the GPU.
//   opt_table: one pass over the optimiser step's lists that checks them and writes the InsmosOptTensor table (include/insmos_hip.h).  From
//     Python the same pass costs ten attribute reads per tensor (some 0.1 us each: 0.5 ms for 250 tensors, ten times what the GPU needs).
//   linear: the layer with its node on the autograd tape -- checks, allocations and the calls of insmos_linear(_backward) (20 us forward and
//     90 with a backward from Python, where the GPU needs 7 for one row).  linear_forward, linear_backward: the same without a node, for the
//     registered operator that linear() takes where a program is being traced.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <stdexcept>
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
struct Unsupported : Refused { using Refused::Refused; };   // NotImplementedError

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
    if (t.is_neg()) throw Refused(std::string(what) + ": " + kind + " " + std::to_string(i) + " is a negated view (resolve_neg() makes it a tensor)");
    return t;
}
int dtype_code(c10::ScalarType t) {
    return t == c10::ScalarType::Float ? INSMOS_F32 : t == c10::ScalarType::BFloat16 ? INSMOS_BF16 : t == c10::ScalarType::Half ? INSMOS_F16 : -1;
}

void add_order(uint64_t& h, const at::Tensor& t) {
    auto add = [&](int64_t v) { h = (h ^ (uint64_t)v) * 0x100000001B3u; };
    add(t.dim());
    for (int64_t d = 0; d < t.dim(); ++d) {
        add(t.size(d));
        add(t.stride(d));
    }
}
constexpr uint64_t kOrder = 0xCBF29CE484222325u;
// opt_order(params) -> a hash of the tensors' sizes and strides
PyObject* opt_order(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) { PyErr_SetString(PyExc_ValueError, "opt_order: params is a list"); return nullptr; }
    uint64_t h = kOrder;
    try {
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) add_order(h, tensor_at(list, i, "opt_order", "parameter"));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    return PyLong_FromUnsignedLongLong(h);
}
// opt_grads(params) -> (that hash, the parameters' gradients, how many have none)
PyObject* opt_grads(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) { PyErr_SetString(PyExc_ValueError, "opt_grads: params is a list"); return nullptr; }
    uint64_t h = kOrder;
    Py_ssize_t missing = 0;
    PyObject* grads = PyList_New(PyList_GET_SIZE(list));
    if (!grads) return nullptr;
    try {
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
            const at::Tensor& t = tensor_at(list, i, "opt_grads", "parameter");
            add_order(h, t);
            PyObject* o = PyList_GET_ITEM(list, i);
            PyObject* g = THPVariable_CheckExact(o) ? THPVariable_Wrap(t.grad()) : PyObject_GetAttrString(o, "grad");   // (a subclass may have its own)
            if (!g) { Py_DECREF(grads); return nullptr; }
            missing += g == Py_None;
            PyList_SET_ITEM(grads, i, g);
        }
    } catch (const std::exception& e) {
        Py_DECREF(grads);
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    return Py_BuildValue("KNn", (unsigned long long)h, grads, missing);
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
        if (!any_device && !first.is_cuda()) throw Refused(std::string(what) + ": tensors on the GPU, not on " + first.device().str());
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

// ---- linear -----------------------------------------------------------------------------------------------------------------
decltype(&insmos_linear) g_linear = nullptr;
decltype(&insmos_linear_ws_bytes_for) g_linear_ws = nullptr;
decltype(&insmos_linear_backward) g_backward = nullptr;
decltype(&insmos_linear_backward_ws_bytes_for) g_backward_ws = nullptr;

// bind_linear(addresses of insmos_linear, _ws_bytes_for, _backward, _backward_ws_bytes_for)
PyObject* bind_linear(PyObject*, PyObject* args) {
    unsigned long long f[4];
    if (!PyArg_ParseTuple(args, "KKKK", &f[0], &f[1], &f[2], &f[3])) return nullptr;
    g_linear = (decltype(g_linear))f[0];
    g_linear_ws = (decltype(g_linear_ws))f[1];
    g_backward = (decltype(g_backward))f[2];
    g_backward_ws = (decltype(g_backward_ws))f[3];
    Py_RETURN_NONE;
}
std::string shape(const at::Tensor& t) {
    std::string r = "(";
    for (int64_t d = 0; d < t.dim(); ++d) r += (d ? ", " : "") + std::to_string(t.size(d));
    return r + ")";
}
[[noreturn]] void refuse(const std::string& t) { throw Refused("linear: " + t); }
at::Tensor arg(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " is no tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != c10::kStrided) refuse(std::string(name) + " is sparse");
    if (t._fw_grad(0).defined()) throw Unsupported(std::string("linear: ") + name + " has a forward-mode tangent, and linear has no forward-mode derivative");
    return t.is_neg() ? t.resolve_neg() : t;   // (a view whose memory holds the values with the other sign)
}
// Whether something outside takes down which operators run (a tracer, a dispatch mode) or a tensor stands for another one (a fake one, a wrapper):
// the calls below would pass it by.
bool observed(std::initializer_list<const at::Tensor*> tensors) {
    if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        throw Unsupported("linear: no rules for torch.func's transforms (grad, vmap, jvp)");
    if (at::tracer::impl::is_dispatch_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return true;
    for (const at::Tensor* t : tensors)
        if (t->defined() && (t->is_meta() || t->key_set().has(c10::DispatchKey::Python) || t->key_set().has(c10::DispatchKey::Functionalize))) return true;
    return false;
}
constexpr int64_t kMost = 1 << 20;   // widths and pitches
// t as rows of `cols` whose values are contiguous and that do not overlap (shared: they may be one row), and their pitch; a copy only where t
// is not so
struct Rows { at::Tensor t; int64_t n, ld; };
Rows rows_of(const at::Tensor& t, int64_t cols, bool shared = false) {
    at::Tensor v = t.dim() == 2 ? t : t.reshape({-1, cols});
    const int64_t n = v.size(0);
    if ((cols != 1 && v.stride(1) != 1) || (n != 1 && !((v.stride(0) >= cols && v.stride(0) <= kMost) || (shared && v.stride(0) == 0)))) v = v.contiguous();
    return {v, n, n != 1 ? v.stride(0) : cols};
}
struct Weight { at::Tensor t; int64_t ld; int out_in; };
// whether w lies as (cout, cin) rows
bool out_in_of(const at::Tensor& w) {
    const auto rows = [&](int d, int64_t cols) { return w.stride(1 - d) == 1 && w.stride(d) >= cols && w.stride(d) <= kMost; };
    return !rows(0, w.size(1)) && rows(1, w.size(0));
}
Weight weight_of(const at::Tensor& w) {
    if (out_in_of(w)) return {w, w.stride(1), 1};
    const int64_t cout = w.size(1);
    if (w.stride(1) == 1 && w.stride(0) >= cout && w.stride(0) <= kMost) return {w, w.stride(0), 0};
    return {w.contiguous(), cout, 0};
}
void* at_ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
struct LibraryError : std::runtime_error { using std::runtime_error::runtime_error; };
void checked(int rc, const char* what) {
    if (rc != 0)
        throw LibraryError(std::string(what) + " failed: " + (rc == INSMOS_EINVAL ? "INSMOS_EINVAL (bad argument)" : rc == INSMOS_EHIP ? "INSMOS_EHIP (HIP runtime error)"
                                                              : rc == INSMOS_EWORKSPACE ? "INSMOS_EWORKSPACE" : std::to_string(rc)));
}
// an exception class by name
void raise(const char* module, const char* name, const char* text) {
    PyObject* m = PyImport_ImportModule(module);
    PyObject* kind = m ? PyObject_GetAttrString(m, name) : nullptr;
    if (kind) PyErr_SetString(kind, text);   // (else the import's own error stands)
    Py_XDECREF(kind);
    Py_XDECREF(m);
}
PyObject* wrap(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}
template <class F>
PyObject* guarded(F f) {   // no C++ exception leaves the module
    try {
        return f();
    } catch (const Unsupported& e) {
        PyErr_SetString(PyExc_NotImplementedError, e.what());
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const LibraryError& e) {
        raise("insmos_amd._lib", "InsmosHipError", e.what());
    } catch (python_error& e) {   // (a hook on saved tensors that raised: checkpoints stop their recomputation that way)
        e.restore();
    } catch (const c10::OutOfMemoryError& e) {
        raise("torch", "OutOfMemoryError", e.what_without_backtrace());   // as torch's own allocations do
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "linear failed");
    }
    return nullptr;
}
// rows of a buffer of the module's own start on 16 bytes
int64_t padded(int64_t cols, const at::Tensor& like) {
    const int64_t chunk = 16 / (int64_t)like.element_size();
    return (cols + chunk - 1) / chunk * chunk;
}

// What the backward pass is given of the activation.  relu: y > 0 says what z > 0 does, unless a residual was added behind it.  (y as rounded: a z
// below fp16's smallest number counts as shut, as it does to a relu of a rounded product.)
int slope_kind(int act, bool residual, bool first) {
    if (act == INSMOS_ACT_NONE) return INSMOS_SLOPE_NONE;
    return act != INSMOS_ACT_RELU ? INSMOS_SLOPE_STORED : residual && !first ? INSMOS_SLOPE_GATE : INSMOS_SLOPE_SIGN;
}

struct Layer { at::Tensor x, w, b, r; int act; bool first; };   // b, r: undefined where there is none

// (y, slopes for the backward pass where `keep`) of a layer whose arguments are checked here
std::pair<at::Tensor, at::Tensor> forward_of(const Layer& l, bool keep) {
    const at::Tensor &x = l.x, &w = l.w;
    const int dt = dtype_code(x.scalar_type());
    std::string buf;
    if (dt < 0) refuse(std::string("float32, bfloat16 or float16, not ") + place(x, buf));
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(0)) refuse("x (..., cin) and weight (cin, cout), not " + shape(x) + " and " + shape(w));
    const int64_t cin = w.size(0), cout = w.size(1);
    if (cin < 1 || cin > kMost || cout > kMost) refuse("widths from 1 to 2^20, not " + std::to_string(cin) + " -> " + std::to_string(cout));
    auto same = [&](const at::Tensor& t, const char* name) {
        std::string b1, b2;
        if (t.scalar_type() != x.scalar_type() || t.device() != x.device())
            refuse(std::string(name) + " is " + place(t, b1) + ", x " + place(x, b2));
    };
    same(w, "weight");
    std::vector<int64_t> out(x.sizes().begin(), x.sizes().end());
    out.back() = cout;
    at::Tensor b;
    if (l.b.defined()) {
        same(l.b, "bias");
        if (l.b.dim() != 1 || l.b.size(0) != cout) refuse("bias (" + std::to_string(cout) + ",), not " + shape(l.b));
        b = l.b.contiguous();
    }
    if (l.r.defined()) {
        same(l.r, "residual");
        if (l.r.sizes() != at::IntArrayRef(out)) refuse("residual of the output's shape, not " + shape(l.r));
    }
    if (x.numel() / cin > 0x7FFFFF00) refuse("at most " + std::to_string(0x7FFFFF00) + " rows");
    if (!x.is_cuda()) refuse("tensors on the GPU, not on " + x.device().str());
    c10::DeviceGuard guard(x.device());
    const auto opt = x.options().requires_grad(false);
    at::Tensor y = at::empty(out, opt), slope;
    const int64_t n = x.numel() / cin, ld = padded(cout, x);
    if (keep) slope = at::empty({n, ld}, opt.dtype(dt == INSMOS_F32 ? at::kFloat : at::kShort));
    if (n && cout) {
        const Rows xr = rows_of(x, cin);
        const Weight wt = weight_of(w);
        Rows rr{};
        if (l.r.defined()) rr = rows_of(l.r, cout, true);
        const size_t need = g_linear_ws(xr.t.data_ptr(), xr.ld, wt.t.data_ptr(), wt.ld, wt.out_in, n, (int)cin, (int)cout, dt);
        const at::Tensor ws = need ? at::empty({(int64_t)need}, opt.dtype(at::kByte)) : at::Tensor();
        checked(g_linear(xr.t.data_ptr(), xr.ld, wt.t.data_ptr(), wt.ld, wt.out_in, at_ptr(b), at_ptr(rr.t), rr.ld, l.first, l.act, n, (int)cin, (int)cout, dt,
                         y.data_ptr(), cout, at_ptr(slope), ld, at_ptr(ws), need, stream_of(x)), "insmos_linear");
    }
    return {y, slope};
}
struct Grads { at::Tensor x, w, b, z; };
// The gradients that are asked for (z: that of the value before the activation).  x is read for w's gradient alone and w for x's; out_in: the layout
// that w's gradient is given in.  kind: INSMOS_SLOPE_*
Grads backward_of(const at::Tensor& dy, const at::Tensor& slope, const at::Tensor& x, const at::Tensor& w, int64_t cin, bool out_in, int kind, bool need_x, bool need_w,
                  bool need_b, bool need_z) {
    const int dt = dtype_code(dy.scalar_type());
    const int64_t cout = dy.size(-1), n = cout ? dy.numel() / cout : 0, ld = padded(cout, dy);
    for (const at::Tensor* t : {&x, &w})
        if (t->defined() && (dy.scalar_type() != t->scalar_type() || dy.device() != t->device())) refuse("the gradient is of another type or device than the output");
    c10::DeviceGuard guard(dy.device());
    const auto opt = dy.options().requires_grad(false);
    std::vector<int64_t> in(dy.sizes().begin(), dy.sizes().end());
    in.back() = cin;
    Grads g;
    if (need_x) g.x = at::empty(in, opt);
    if (need_w) g.w = out_in ? at::empty({cout, cin}, opt) : at::empty({cin, cout}, opt);
    if (need_b) g.b = at::empty({cout}, opt);
    if (need_z) g.z = n && cout ? at::empty({n, ld}, opt) : at::empty(dy.sizes(), opt);
    if (n && cout) {
        if (need_x || need_w || need_b || need_z) {
            const Rows d = rows_of(dy, cout);
            Rows xr{at::Tensor(), n, cin};
            if (need_w) xr = rows_of(x, cin);
            Weight wt{at::Tensor(), out_in ? cin : cout, out_in};
            if (need_x) wt = weight_of(w);
            const size_t need = g_backward_ws(d.t.data_ptr(), d.ld, kind, at_ptr(xr.t), xr.ld, at_ptr(wt.t), wt.ld, out_in, n, (int)cin, (int)cout, dt,
                                              need_x, need_w, need_b, need_z);
            const at::Tensor ws = need ? at::empty({(int64_t)need}, opt.dtype(at::kByte)) : at::Tensor();
            checked(g_backward(d.t.data_ptr(), d.ld, at_ptr(slope), kind >= INSMOS_SLOPE_STORED ? ld : cout, kind, at_ptr(xr.t), xr.ld, at_ptr(wt.t), wt.ld, out_in,
                               n, (int)cin, (int)cout, dt, at_ptr(g.x), cin, at_ptr(g.w), out_in ? cin : cout, at_ptr(g.b), at_ptr(g.z), ld, at_ptr(ws), need,
                               stream_of(dy)), "insmos_linear_backward");
        }
        if (need_z) g.z = g.z.narrow(1, 0, cout).reshape(dy.sizes());
    } else {
        for (at::Tensor* t : {&g.x, &g.w, &g.b})
            if (t->defined()) t->zero_();
    }
    if (need_w && out_in) g.w = g.w.t();
    return g;
}
// A backward pass that is captured into a graph must not reach a node that was recorded on the default stream (a leaf's, kept alive by an eager
// graph): the tape would make that stream wait for the captured one, which cannot be captured and ends the process.
void refuse_default_stream() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (const auto& edge : node->next_edges()) {
        const auto stream = edge.function ? edge.function->stream() : std::nullopt;
        if (stream && stream->id() == 0)
            refuse("a backward pass is being captured, but a graph on the default stream shares its inputs and is alive (drop that graph's outputs before the capture)");
    }
}
// The node keeps x where W needs a gradient, W where x does, and the activation's slopes (16 bits each with 16-bit types; y itself for a relu without a residual behind it).
struct LinearNode : torch::autograd::Function<LinearNode> {
    enum : int64_t { kFirst = 4, kBias = 8, kResidual = 16, kOutIn = 32, kCin = 8 };   // beside the two bits of INSMOS_SLOPE_*; cin from bit 8 on
    using Maybe = std::optional<at::Tensor>;
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const Maybe& b, const Maybe& r, int64_t act,
                              bool first) {
        const int kind = slope_kind((int)act, r.has_value(), first);
        const auto out = forward_of({x, w, b.value_or(at::Tensor()), r.value_or(at::Tensor()), (int)act, first}, kind >= INSMOS_SLOPE_STORED);
        ctx->save_for_backward({w.requires_grad() ? x : at::Tensor(), x.requires_grad() ? w : at::Tensor(), kind == INSMOS_SLOPE_SIGN ? out.first : out.second});
        ctx->saved_data["meta"] = kind + (first ? kFirst : 0) + (b ? kBias : 0) + (r ? kResidual : 0) + (out_in_of(w) ? kOutIn : 0) + (w.size(0) << kCin);
        return out.first;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dys) {
        const bool again = at::GradMode::is_enabled();   // create_graph
        torch::autograd::variable_list out(6);
        try {
            at::AutoGradMode off(false);
            refuse_default_stream();
            const auto saved = ctx->get_saved_variables();
            const int64_t meta = ctx->saved_data["meta"].toInt();
            const int kind = (int)(meta & 3);
            // an input that is not there has no edge
            const bool need_b = meta & kBias && ctx->needs_input_grad(2), need_r = meta & kResidual && ctx->needs_input_grad(meta & kBias ? 3 : 2);
            const bool z = need_r && meta & kFirst && kind != INSMOS_SLOPE_NONE;
            const at::Tensor dy = dys[0].resolve_neg();
            const Grads g = backward_of(dy, saved[2], saved[0], saved[1], meta >> kCin, meta & kOutIn, kind, ctx->needs_input_grad(0), ctx->needs_input_grad(1), need_b, z);
            out[0] = g.x;
            out[1] = g.w;
            out[2] = g.b;
            if (need_r) out[3] = z ? g.z : dy;
        } catch (const LibraryError& e) {   // the tape hands a Python error on as it is
            PyGILState_STATE gil = PyGILState_Ensure();
            raise("insmos_amd._lib", "InsmosHipError", e.what());
            python_error error;
            error.persist();
            PyGILState_Release(gil);
            throw error;
        }
        if (again) {   // a second derivative raises, and is not taken for zero
            for (auto& t : out)
                if (t.defined()) t = t.detach().requires_grad_(true);
            const auto error = std::make_shared<torch::autograd::DelayedError>("linear is differentiable once: its gradients have none", (int64_t)out.size());
            out = (*error)(std::move(out));
        }
        return out;
    }
};
Layer layer_of(PyObject* const* a) {
    return {arg(a[0], "x"), arg(a[1], "weight"), a[2] == Py_None ? at::Tensor() : arg(a[2], "bias"), a[3] == Py_None ? at::Tensor() : arg(a[3], "residual"),
            (int)PyLong_AsLong(a[4]), PyObject_IsTrue(a[5]) == 1};
}
// linear_forward(x, weight, bias or None, residual or None, act, residual_first) -> (y, slopes or None)
PyObject* linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 6 || !g_linear) refuse("internal call");
        const Layer l = layer_of(a);
        const auto out = forward_of(l, slope_kind(l.act, l.r.defined(), l.first) >= INSMOS_SLOPE_STORED);
        return Py_BuildValue("NN", wrap(out.first), wrap(out.second));
    });
}
// linear_backward(dy, slopes or y or None, x, weight, act, residual behind the activation, need_x, need_w, need_b, need_z) -> (dx, dw, db, dz), None
// where not needed
PyObject* linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 10 || !g_linear) refuse("internal call");
        refuse_default_stream();
        bool is[5];
        for (int i = 0; i < 5; ++i) is[i] = PyObject_IsTrue(a[5 + i]) == 1;
        const int kind = slope_kind((int)PyLong_AsLong(a[4]), is[0], !is[0]);
        const at::Tensor w = arg(a[3], "weight");
        const Grads g = backward_of(arg(a[0], "the gradient"), a[1] == Py_None ? at::Tensor() : arg(a[1], "slope"), arg(a[2], "x"), w, w.size(0), out_in_of(w), kind,
                                    is[1], is[2], is[3], is[4]);
        return Py_BuildValue("NNNN", wrap(g.x), wrap(g.w), wrap(g.b), wrap(g.z));
    });
}
// linear(x, weight, bias or None, residual or None, act, residual_first) -> y, or NotImplemented where the registered operator has to be called
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 6 || !g_linear) refuse("internal call");
        const Layer l = layer_of(a);
        if (observed({&l.x, &l.w, &l.b, &l.r})) Py_RETURN_NOTIMPLEMENTED;
        bool tape = false;
        if (at::GradMode::is_enabled())
            for (const at::Tensor* t : {&l.x, &l.w, &l.b, &l.r}) tape = tape || (t->defined() && t->requires_grad());
        if (tape) {
            auto maybe = [](const at::Tensor& t) { return t.defined() ? LinearNode::Maybe(t) : std::nullopt; };
            return wrap(LinearNode::apply(l.x, l.w, maybe(l.b), maybe(l.r), (int64_t)l.act, l.first));
        }
        return wrap(forward_of(l, false).first);
    });
}

PyMethodDef kMethods[] = {{"opt_order", opt_order, METH_O, "a hash of sizes and strides"},
                          {"opt_grads", opt_grads, METH_O, "that hash and the parameters' gradients"},
                          {"opt_table", opt_table, METH_VARARGS, "checks lists of tensors and writes their InsmosOptTensor table"},
                          {"bind_linear", bind_linear, METH_VARARGS, "addresses of the library's functions"},
                          {"linear", (PyCFunction)(void (*)())linear, METH_FASTCALL, "the layer, on the autograd tape"},
                          {"linear_forward", (PyCFunction)(void (*)())linear_forward, METH_FASTCALL, "the layer and its slopes"},
                          {"linear_backward", (PyCFunction)(void (*)())linear_backward, METH_FASTCALL, "its gradients"},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
