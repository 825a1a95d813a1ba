// The calls of the sequence operators from Python (functional.py) and their gradients' nodes: outputs and workspaces are allocated and the C ABI
// (include/mv2.h) is called on the current stream of the tensors' device, in one native call each and without the interpreter's lock.  What the
// arguments' shapes, strides and types lead to is in a plan: functional.py checks them and makes it.  Where the host is what a call takes, the
// same from Python (ctypes, torch.empty, a Function of Python's) is dearer: a single token 9.1 us against 6.4, norms of 32 rows 11.9 and 7.2,
// norms of 4097 x 501 fp32 and their six gradients 165 and 101 (native calls under a Function of Python's 122; torch's engine takes some 80).
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <mutex>
#include <string>
#include <vector>
#include "../../include/mv2.h"

namespace {

PyObject* error_class = nullptr;       // Mv2Error

struct LoopPlan {
    mv2_gateloop_desc d;
    int fused, device;
    std::vector<int64_t> part, y, h, states, stride;      // shapes (states is empty where none are kept), a part's strides
    int64_t ws_forward, ws_backward;
};
struct NormPlan {
    mv2_block_norm_desc d;
    int branch, normed, keeps, device;
    std::vector<int64_t> shape, stride[3];                // strides of x, branch and gate; empty: dense
    int64_t ws_backward;
};
const char LOOP[] = "mv2.loop_plan", NORM[] = "mv2.norm_plan";

// a capsule holds a shared plan: the nodes of a graph keep theirs
template <typename P> void drop(PyObject* o) { delete static_cast<std::shared_ptr<const P>*>(PyCapsule_GetPointer(o, PyCapsule_GetName(o))); }

bool read_shape(PyObject* o, std::vector<int64_t>& v) {
    PyObject* t = PySequence_Tuple(o);
    if (!t) return false;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(t); ++i) v.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(t, i)));
    Py_DECREF(t);
    return !PyErr_Occurred();
}
template <typename D> bool read_desc(const Py_buffer& b, D& d) {
    if (b.len != (Py_ssize_t)sizeof(D)) { PyErr_SetString(PyExc_ValueError, "descriptor of another size"); return false; }
    memcpy(&d, b.buf, sizeof(D));
    return true;
}

struct Unlocked {                     // torch's allocator may wait for memory
    PyThreadState* held = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(held); }
};
struct Device {
    c10::DeviceIndex index;
    c10::DeviceGuard guard;
    explicit Device(int i) : index((c10::DeviceIndex)i), guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)i)) {}
    at::Tensor empty(at::IntArrayRef shape, at::ScalarType t) const { return at::empty(shape, at::TensorOptions(t).device(c10::kCUDA, index)); }
    at::Tensor workspace(int64_t bytes) const { return bytes ? empty({bytes}, at::kByte) : at::Tensor(); }
    void* stream() const { return c10::hip::getCurrentHIPStream(index).stream(); }
};

const at::Tensor& tensor(PyObject* o) {           // None: undefined
    static const at::Tensor none;
    return o == Py_None ? none : THPVariable_Unpack(o);
}
template <typename T = void> T* ptr(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
// what a hook on saved tensors gave back must still be what was saved, but for the layout of rows
void still(const at::Tensor& t, int device, at::ScalarType type, at::IntArrayRef shape, bool whole) {
    TORCH_CHECK(!t.defined() || (t.device() == c10::Device(c10::kCUDA, (c10::DeviceIndex)device) && t.scalar_type() == type && t.sizes() == shape &&
                                 !t.is_neg() && (!whole || t.is_contiguous())), "a tensor saved for the backward pass came back with another type, size, layout or device");
}
at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }      // (a gradient may be negated lazily)

PyObject* wrapped(std::initializer_list<at::Tensor> ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) {
        PyObject* o = Py_None;
        if (t.defined()) o = THPVariable_Wrap(t);
        else Py_INCREF(o);
        if (!r || !o) { Py_XDECREF(r); Py_XDECREF(o); return nullptr; }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}
// a refusal or a launch's error, as Mv2Error, from a thread with or without the interpreter's lock
void check(const char* what, int rc) {
    if (rc == 0) return;
    pybind11::gil_scoped_acquire held;
    PyErr_Format(error_class ? error_class : PyExc_RuntimeError, "%s failed with code %d", what, rc);
    python_error e;
    e.persist();
    throw e;
}

// q, kv, a: the thirds of one tensor, or three tensors
struct Parts {
    char *q, *kv, *a;
    Parts(const LoopPlan& p, const at::Tensor& x, const at::Tensor& y, const at::Tensor& z) {
        q = ptr<char>(x);
        const int64_t third = (int64_t)p.d.C * (p.d.dtype == MV2_BF16 ? 2 : 4);
        kv = p.fused ? q + third : ptr<char>(y);
        a = p.fused ? q + 2 * third : ptr<char>(z);
    }
};
at::ScalarType row_type(int dtype) { return dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat; }

// the nodes end here: gradients of gradients are refused where they are asked for
torch::autograd::variable_list first_order(torch::autograd::variable_list g, const char* what) {
    if (!at::GradMode::is_enabled()) return g;
    for (at::Tensor& t : g) if (t.defined()) t = t.detach().requires_grad_(true);
    auto end = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has gradients of first order only", (int64_t)g.size());
    return end->apply(std::move(g));
}
// whether or not the inputs require gradients: a dual tensor need not, and its tangent would be left out in silence
void no_tangents(std::initializer_list<const at::Tensor*> ts, const char* what) {
    for (const at::Tensor* t : ts) TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

struct LoopNode : torch::autograd::Node {
    std::shared_ptr<const LoopPlan> plan;
    torch::autograd::SavedVariable state, lengths, resets, states, parts[3];
    std::string name() const override { return "GateLoopBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto* v : {&state, &lengths, &resets, &states, parts, parts + 1, parts + 2}) v->reset_data();
    }
    // gradients of y and the last state -> of the first state and the parts
    torch::autograd::variable_list apply(torch::autograd::variable_list&& up) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const LoopPlan& p = *plan;
        const int np = p.fused ? 1 : 3;
        const at::ScalarType type = row_type(p.d.dtype);
        torch::autograd::variable_list g(1 + np);
        at::Tensor h0 = state.unpack(), n = lengths.unpack(), cuts = resets.unpack(), kept = states.unpack(), x[3];
        for (int i = 0; i < np; ++i) x[i] = parts[i].unpack();
        if (!up[0].defined() && !up[1].defined()) return g;
        no_tangents({&up[0], &up[1]}, "gate_loop");
        const int64_t rows = (int64_t)p.d.B * p.d.P * p.d.C;
        mv2_gateloop_desc d = p.d;
        bool same = true;
        for (int i = 0; i < np; ++i) {
            still(x[i], p.device, type, p.part, false);
            same = same && x[i].strides() == at::IntArrayRef(p.stride);
        }
        if (!same) {                                      // hooks on saved tensors may lay them out anew
            for (int i = 0; i < np; ++i) x[i] = x[i].contiguous();
            d.in_p = (int64_t)d.C * (p.fused ? 3 : 1);
            d.in_t = d.P * d.in_p;
            d.in_b = d.T * d.in_t;
        }
        still(h0, p.device, at::kFloat, p.h, true);
        still(kept, p.device, at::kFloat, p.states, true);
        still(n, p.device, at::kInt, {p.d.B}, true);
        if (cuts.defined()) still(cuts, p.device, cuts.scalar_type() == at::kBool ? at::kBool : at::kByte, {p.d.B, p.d.T}, true);
        const Device at(p.device);
        const at::Tensor dy = up[0].defined() ? dense(up[0]) : at.empty(p.y, type).zero_(), dh = dense(up[1]);
        for (int i = 0; i < np; ++i) g[1 + i] = at.empty(p.part, type);
        if (task_should_compute_output(0)) g[0] = at.empty(p.h, at::kFloat);
        const at::Tensor ws = at.workspace(p.ws_backward);
        const Parts in(p, x[0], x[1], x[2]), out(p, g[1], g[np > 1 ? 2 : 1], g[np > 1 ? 3 : 1]);
        check("mv2_gateloop_backward", mv2_gateloop_backward(&d, in.q, in.kv, in.a, ptr<float>(h0), ptr<int32_t>(n), ptr<unsigned char>(cuts), ptr<float>(kept),
                                                             ptr(dy), ptr<float>(dh), out.q, out.kv, out.a, ptr<float>(g[0]), ptr(ws), (size_t)p.ws_backward,
                                                             at.stream()));
        return first_order(std::move(g), "gate_loop");
    }
};

struct NormNode : torch::autograd::Node {
    std::shared_ptr<const NormPlan> plan;
    torch::autograd::SavedVariable saved[7];              // x, branch, gate, post_gamma, scale, pre_gamma, norms
    std::string name() const override { return "BlockNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : saved) v.reset_data();
    }
    // gradients of out and normed -> of x, branch, gate, post_gamma, scale, pre_gamma
    torch::autograd::variable_list apply(torch::autograd::variable_list&& up) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const NormPlan& p = *plan;
        const at::ScalarType type = row_type(p.d.dtype);
        torch::autograd::variable_list g(6);
        at::Tensor t[7];
        for (int i = 0; i < 7; ++i) t[i] = saved[i].unpack();
        if (!up[0].defined() && !up[1].defined()) return g;
        no_tangents({&up[0], &up[1]}, "block_norm");
        mv2_block_norm_desc d = p.d;
        bool same = true;
        for (int i = 0; i < 3; ++i) {
            still(t[i], p.device, type, p.shape, false);
            same = same && (!t[i].defined() || (p.stride[i].empty() ? t[i].is_contiguous() : t[i].strides() == at::IntArrayRef(p.stride[i])));
        }
        if (!same) {                                      // hooks on saved tensors may lay them out anew
            for (int i = 0; i < 3; ++i) t[i] = dense(t[i]);
            d.x_stride = d.branch_stride = d.gate_stride = d.C;
        }
        for (int i = 3; i < 6; ++i) still(t[i], p.device, at::kFloat, {p.d.C}, true);
        still(t[6], p.device, at::kFloat, {2, p.d.rows}, true);
        const Device at(p.device);
        const at::Tensor dout = dense(up[0]), dn = dense(up[1]);
        for (int i = 0; i < 6; ++i)
            if (task_should_compute_output(i)) g[i] = i < 3 ? at.empty(p.shape, type) : at.empty({p.d.C}, at::kFloat);
        const int64_t bytes = g[3].defined() || g[4].defined() || g[5].defined() ? p.ws_backward : 0;
        const at::Tensor ws = at.workspace(bytes);
        check("mv2_block_norm_backward", mv2_block_norm_backward(&d, ptr(t[0]), ptr(t[1]), ptr(t[2]), ptr<float>(t[3]), ptr<float>(t[4]), ptr<float>(t[5]),
                                                                 ptr<float>(t[6]), ptr(dout), ptr(dn), ptr(g[0]), ptr(g[1]), ptr(g[2]), ptr<float>(g[3]),
                                                                 ptr<float>(g[4]), ptr<float>(g[5]), ptr(ws), (size_t)bytes, at.stream()));
        return first_order(std::move(g), "block_norm");
    }
};

#define PLAN(P, name) const auto* held = static_cast<const std::shared_ptr<const P>*>(PyCapsule_GetPointer(args[0], name)); if (!held) return nullptr; const P* p = held->get()
#define ARGS(n) if (nargs != n) { PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", n, nargs); return nullptr; }

// (plan, (qkva,) or (q, kv, a), state, lengths, resets, state_out, want) -> (y, last state); want: 1 the last state, 2 and gradients
PyObject* loop_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(7)
    PLAN(LoopPlan, LOOP);
    const int np = p->fused ? 1 : 3;
    if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != np) { PyErr_SetString(PyExc_TypeError, "expected (qkva,) or (q, kv, a)"); return nullptr; }
    at::Tensor x[3];
    for (int i = 0; i < np; ++i) x[i] = tensor(PyTuple_GET_ITEM(args[1], i));
    const at::Tensor &state = tensor(args[2]), &lengths = tensor(args[3]), &resets = tensor(args[4]);
    at::Tensor h = tensor(args[5]), y;
    no_tangents({&state, &h, x, x + 1, x + 2}, "gate_loop");
    const bool own = !h.defined();
    const long want = PyLong_AsLong(args[6]);
    {
        const Unlocked unlocked;
        const Device at(p->device);
        at::Tensor states;
        {
            y = at.empty(p->y, row_type(p->d.dtype));
            if (own && want >= 1) h = at.empty(p->h, at::kFloat);
            if (want >= 2 && !p->states.empty()) states = at.empty(p->states, at::kFloat);
            const at::Tensor ws = at.workspace(p->ws_forward);
            const Parts in(*p, x[0], x[1], x[2]);
            check("mv2_gateloop_forward", mv2_gateloop_forward(&p->d, in.q, in.kv, in.a, ptr<float>(state), ptr<int32_t>(lengths), ptr<unsigned char>(resets),
                                                               ptr(y), ptr<float>(h), ptr<float>(states), ptr(ws), (size_t)p->ws_forward, at.stream()));
        }
        if (want >= 2) {
            auto node = std::shared_ptr<LoopNode>(new LoopNode(), torch::autograd::deleteNode);
            if (p->fused) node->set_next_edges(torch::autograd::collect_next_edges(state, x[0]));
            else node->set_next_edges(torch::autograd::collect_next_edges(state, x[0], x[1], x[2]));
            node->plan = *held;
            node->state = torch::autograd::SavedVariable(state, false);
            node->lengths = torch::autograd::SavedVariable(lengths, false);
            node->resets = torch::autograd::SavedVariable(resets, false);
            node->states = torch::autograd::SavedVariable(states, false);
            for (int i = 0; i < np; ++i) node->parts[i] = torch::autograd::SavedVariable(x[i], false);
            torch::autograd::set_history(y, node);
            torch::autograd::set_history(h, node);
        }
    }
    return wrapped({y, own ? h : at::Tensor()});
    END_HANDLE_TH_ERRORS
}

// (plan, x, branch, gate, post_gamma, scale, pre_gamma, gradients?) -> (out, normed)
PyObject* norm_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(8)
    PLAN(NormPlan, NORM);
    at::Tensor t[7], out, normed;
    for (int i = 0; i < 6; ++i) t[i] = tensor(args[1 + i]);
    no_tangents({t, t + 1, t + 2, t + 3, t + 4, t + 5}, "block_norm");
    const bool train = args[7] == Py_True;
    {
        const Unlocked unlocked;
        const Device at(p->device);
        {
            const at::ScalarType type = row_type(p->d.dtype);
            if (p->branch) out = at.empty(p->shape, type);
            if (p->normed) normed = at.empty(p->shape, type);
            if (train && p->keeps) t[6] = at.empty({2, p->d.rows}, at::kFloat);
            check("mv2_block_norm_forward", mv2_block_norm_forward(&p->d, ptr(t[0]), ptr(t[1]), ptr(t[2]), ptr<float>(t[3]), ptr<float>(t[4]), ptr<float>(t[5]),
                                                                   ptr(out), ptr(normed), ptr<float>(t[6]), at.stream()));
        }
        if (train) {
            auto node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(t[0], t[1], t[2], t[3], t[4], t[5]));
            node->plan = *held;
            for (int i = 0; i < 7; ++i) node->saved[i] = torch::autograd::SavedVariable(t[i], false);
            for (at::Tensor* o : {&out, &normed}) {
                if (o->defined()) torch::autograd::set_history(*o, node);
                else node->add_input_metadata(torch::autograd::Node::undefined_input());
            }
        }
    }
    return wrapped({out, normed});
    END_HANDLE_TH_ERRORS
}

// (descriptor, fused, device, shape of a part, of y, of the state, of the kept states or (), a part's strides, workspace bytes forward, backward)
PyObject* loop_plan(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    Py_buffer desc;
    PyObject *part, *y, *h, *states, *stride;
    auto p = std::make_shared<LoopPlan>();
    long long wf, wb;
    if (!PyArg_ParseTuple(args, "y*piOOOOOLL", &desc, &p->fused, &p->device, &part, &y, &h, &states, &stride, &wf, &wb)) return nullptr;
    const bool ok = read_desc(desc, p->d);
    PyBuffer_Release(&desc);
    if (!ok || !read_shape(part, p->part) || !read_shape(y, p->y) || !read_shape(h, p->h) || !read_shape(states, p->states) ||
        !read_shape(stride, p->stride)) return nullptr;
    p->ws_forward = wf; p->ws_backward = wb;
    return PyCapsule_New(new std::shared_ptr<const LoopPlan>(std::move(p)), LOOP, drop<LoopPlan>);
    END_HANDLE_TH_ERRORS
}

// (descriptor, device, shape, branch?, second norm?, norms to keep?, the strides of x, branch and gate or (): dense, workspace bytes backward)
PyObject* norm_plan(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    Py_buffer desc;
    PyObject *shape, *stride[3];
    auto p = std::make_shared<NormPlan>();
    long long wb;
    if (!PyArg_ParseTuple(args, "y*iOpppOOOL", &desc, &p->device, &shape, &p->branch, &p->normed, &p->keeps, stride, stride + 1, stride + 2, &wb)) return nullptr;
    const bool ok = read_desc(desc, p->d);
    PyBuffer_Release(&desc);
    if (!ok || !read_shape(shape, p->shape)) return nullptr;
    for (int i = 0; i < 3; ++i) if (!read_shape(stride[i], p->stride[i])) return nullptr;
    p->ws_backward = wb;
    return PyCapsule_New(new std::shared_ptr<const NormPlan>(std::move(p)), NORM, drop<NormPlan>);
    END_HANDLE_TH_ERRORS
}

// what a plan depends on of its arguments, as bytes: of a tensor shape, strides, type, device and whether it is negated lazily, of a tuple or list of tensors those of each, of a
// text itself, of None that it is None.  None is returned for anything else (functional.py then says what is wrong with it).
bool add_key(std::string& k, PyObject* o, int depth) {
    const auto put = [&](int64_t v) { k.append(reinterpret_cast<const char*>(&v), sizeof v); };
    if (o == Py_None) put(-1);
    else if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided) return false;
        put(t.dim());
        for (int64_t v : t.sizes()) put(v);
        for (int64_t v : t.strides()) put(v);
        put((int64_t)t.is_neg() << 40 | (int64_t)t.scalar_type() << 32 | (int64_t)(uint8_t)t.device().type() << 16 | (uint16_t)t.device().index());
    } else if (PyUnicode_Check(o)) {
        Py_ssize_t n;
        const char* c = PyUnicode_AsUTF8AndSize(o, &n);
        if (!c) { PyErr_Clear(); return false; }
        put(-2 - n);
        k.append(c, n);
    } else if ((PyTuple_Check(o) || PyList_Check(o)) && depth == 0) {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
        put(INT64_MIN + n);
        for (Py_ssize_t i = 0; i < n; ++i) if (!add_key(k, PySequence_Fast_GET_ITEM(o, i), 1)) return false;
    } else return false;
    return true;
}
PyObject* key(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    std::string k;
    k.reserve(512);
    for (Py_ssize_t i = 0; i < nargs; ++i) if (!add_key(k, args[i], 0)) Py_RETURN_NONE;
    return PyBytes_FromStringAndSize(k.data(), (Py_ssize_t)k.size());
    END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    Py_XSETREF(error_class, cls);
    Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(loop_forward), FAST(norm_forward), FAST(key),
                         {"loop_plan", loop_plan, METH_VARARGS, nullptr}, {"norm_plan", norm_plan, METH_VARARGS, nullptr},
                         {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", MV2_BUILT_FOR) < 0) Py_CLEAR(m);      // ops_hip.py compares it with what is running
    return m;
}
