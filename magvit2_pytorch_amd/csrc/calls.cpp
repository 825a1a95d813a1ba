// The calls of the sequence operators from Python (functional.py): outputs and workspaces are allocated and the C ABI (include/mv2.h) is called
// on the current stream of the tensors' device, in one native call each.  What the arguments' shapes, strides and types lead to is in a plan
// (functional.py checks them and makes it); nothing is checked or kept here.  The same from Python, over ctypes and torch.empty, is dearer where the host
// is what a call takes: a single token 9.1 us against 7.2, norms of 32 rows 11.9 and 8.8, norms of 4097 rows and their gradients 165 and 122.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <vector>
#include "../../include/mv2.h"

namespace {

PyObject* error_class = nullptr;       // Mv2Error

struct LoopPlan {
    mv2_gateloop_desc d;
    int fused, device;
    std::vector<int64_t> part, y, h, states;      // shapes; states is empty where none are kept
    int64_t ws_forward, ws_backward;
};
struct NormPlan {
    mv2_block_norm_desc d;
    int branch, normed, keeps, device;
    std::vector<int64_t> shape;
    int64_t ws_backward;
};
const char LOOP[] = "mv2.loop_plan", NORM[] = "mv2.norm_plan";

template <typename P> void drop(PyObject* o) { delete static_cast<P*>(PyCapsule_GetPointer(o, PyCapsule_GetName(o))); }

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

// allocations and launches of one call, without the interpreter's lock (torch's allocator may wait for memory)
struct Unlocked {
    PyThreadState* held = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(held); }
};
struct Launch {
    Unlocked unlocked;
    int device;
    c10::DeviceGuard guard;
    explicit Launch(int dev) : device(dev), guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)dev)) {}
    at::Tensor empty(at::IntArrayRef shape, at::ScalarType t) const { return at::empty(shape, at::TensorOptions(t).device(c10::kCUDA, (c10::DeviceIndex)device)); }
    at::Tensor workspace(int64_t bytes) const { return bytes ? empty({bytes}, at::kByte) : at::Tensor(); }
    void* stream() const { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
};

const at::Tensor& tensor(PyObject* o) {           // None: undefined
    static const at::Tensor none;
    return o == Py_None ? none : THPVariable_Unpack(o);
}
template <typename T = void> T* ptr(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
// what a hook on saved tensors gave back must still be what was saved (its layout of rows is functional.py's to look at)
void still(const at::Tensor& t, int device, at::ScalarType type, int64_t n, bool whole) {
    TORCH_CHECK(!t.defined() || (t.device() == c10::Device(c10::kCUDA, (c10::DeviceIndex)device) && t.scalar_type() == type && t.numel() == n &&
                                 (!whole || t.is_contiguous())), "a tensor saved for the backward pass came back with another type, size, layout or device");
}
at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.contiguous() : t; }

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
PyObject* failed(const char* what, int rc) { return PyErr_Format(error_class ? error_class : PyExc_RuntimeError, "%s failed with code %d", what, rc); }

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
#define PLAN(P, name) const auto* p = static_cast<const P*>(PyCapsule_GetPointer(args[0], name)); if (!p) return nullptr
#define ARGS(n) if (nargs != n) { PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", n, nargs); return nullptr; }
#define PARTS() if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != (p->fused ? 1 : 3)) { PyErr_SetString(PyExc_TypeError, "expected (qkva,) or (q, kv, a)"); return nullptr; }
#define PART(i) tensor(PyTuple_GET_ITEM(args[1], p->fused ? 0 : i))

// (plan, (qkva,) or (q, kv, a), state, lengths, resets, state_out, want) -> (y, last state, kept states); want: 1 the last state, 2 both
PyObject* loop_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(7)
    PLAN(LoopPlan, LOOP);
    PARTS()
    const Parts in(*p, PART(0), PART(1), PART(2));
    const at::Tensor &state = tensor(args[2]), &lengths = tensor(args[3]), &resets = tensor(args[4]);
    at::Tensor h = tensor(args[5]), y, states;
    const bool own = !h.defined();
    const long want = PyLong_AsLong(args[6]);
    const at::ScalarType type = p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat;
    int rc;
    {
        Launch at(p->device);
        y = at.empty(p->y, type);
        if (own && want >= 1) h = at.empty(p->h, at::kFloat);
        if (want >= 2 && !p->states.empty()) states = at.empty(p->states, at::kFloat);
        const at::Tensor ws = at.workspace(p->ws_forward);
        rc = mv2_gateloop_forward(&p->d, in.q, in.kv, in.a, ptr<float>(state), ptr<int32_t>(lengths), ptr<unsigned char>(resets), ptr(y), ptr<float>(h),
                                  ptr<float>(states), ptr(ws), (size_t)p->ws_forward, at.stream());
    }
    if (rc) return failed("mv2_gateloop_forward", rc);
    return wrapped({y, own ? h : at::Tensor(), states});
    END_HANDLE_TH_ERRORS
}

// (plan, parts, state, lengths, resets, kept states, dy, dh, state's gradient wanted?) -> (its gradient, the parts' gradients ...)
PyObject* loop_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(9)
    PLAN(LoopPlan, LOOP);
    PARTS()
    const Parts in(*p, PART(0), PART(1), PART(2));
    const at::Tensor &state = tensor(args[2]), &lengths = tensor(args[3]), &resets = tensor(args[4]), &states = tensor(args[5]);
    const int64_t rows = (int64_t)p->d.B * p->d.P * p->d.C;
    for (int i = 0; i < (p->fused ? 1 : 3); ++i)
        still(PART(i), p->device, p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat, rows * p->d.T * (p->fused ? 3 : 1), false);
    still(state, p->device, at::kFloat, rows, true);
    still(states, p->device, at::kFloat, p->states.empty() ? 0 : rows * p->states[1], true);
    still(lengths, p->device, at::kInt, p->d.B, true);
    if (resets.defined()) still(resets, p->device, resets.scalar_type() == at::kBool ? at::kBool : at::kByte, (int64_t)p->d.B * p->d.T, true);
    at::Tensor dy = tensor(args[6]), dh = tensor(args[7]), g[3], dstate;
    const bool wanted = args[8] == Py_True;
    const at::ScalarType type = p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat;
    int rc;
    {
        Launch at(p->device);
        dy = dy.defined() ? dy.contiguous() : at.empty(p->y, type).zero_();
        dh = dense(dh);
        for (int i = 0; i < (p->fused ? 1 : 3); ++i) g[i] = at.empty(p->part, type);
        if (wanted) dstate = at.empty(p->h, at::kFloat);
        const Parts out(*p, g[0], g[1], g[2]);
        const at::Tensor ws = at.workspace(p->ws_backward);
        rc = mv2_gateloop_backward(&p->d, in.q, in.kv, in.a, ptr<float>(state), ptr<int32_t>(lengths), ptr<unsigned char>(resets), ptr<float>(states), ptr(dy),
                                   ptr<float>(dh), out.q, out.kv, out.a, ptr<float>(dstate), ptr(ws), (size_t)p->ws_backward, at.stream());
    }
    if (rc) return failed("mv2_gateloop_backward", rc);
    return p->fused ? wrapped({dstate, g[0]}) : wrapped({dstate, g[0], g[1], g[2]});
    END_HANDLE_TH_ERRORS
}

// (plan, x, branch, gate, post_gamma, scale, pre_gamma, keep the norms?) -> (out, normed, norms)
PyObject* norm_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(8)
    PLAN(NormPlan, NORM);
    const at::Tensor &x = tensor(args[1]), &branch = tensor(args[2]), &gate = tensor(args[3]), &post = tensor(args[4]), &scale = tensor(args[5]),
                     &pre = tensor(args[6]);
    const bool keep = args[7] == Py_True && p->keeps;
    const at::ScalarType type = p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat;
    at::Tensor out, normed, rstd;
    int rc;
    {
        Launch at(p->device);
        if (p->branch) out = at.empty(p->shape, type);
        if (p->normed) normed = at.empty(p->shape, type);
        if (keep) rstd = at.empty({2, p->d.rows}, at::kFloat);
        rc = mv2_block_norm_forward(&p->d, ptr(x), ptr(branch), ptr(gate), ptr<float>(post), ptr<float>(scale), ptr<float>(pre), ptr(out), ptr(normed),
                                    ptr<float>(rstd), at.stream());
    }
    if (rc) return failed("mv2_block_norm_forward", rc);
    return wrapped({out, normed, rstd});
    END_HANDLE_TH_ERRORS
}

// (plan, x, branch, gate, post_gamma, scale, pre_gamma, norms, dout, dn, which of the six gradients are wanted) -> the six
PyObject* norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    ARGS(11)
    PLAN(NormPlan, NORM);
    const at::Tensor &x = tensor(args[1]), &branch = tensor(args[2]), &gate = tensor(args[3]), &post = tensor(args[4]), &scale = tensor(args[5]),
                     &pre = tensor(args[6]), &rstd = tensor(args[7]);
    for (const at::Tensor* t : {&x, &branch, &gate}) still(*t, p->device, p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat, p->d.rows * p->d.C, false);
    for (const at::Tensor* t : {&post, &scale, &pre}) still(*t, p->device, at::kFloat, p->d.C, true);
    still(rstd, p->device, at::kFloat, 2 * p->d.rows, true);
    at::Tensor dout = tensor(args[8]), dn = tensor(args[9]), g[6];
    bool want[6];
    for (int i = 0; i < 6; ++i) want[i] = PyTuple_GET_ITEM(args[10], i) == Py_True;
    const at::ScalarType type = p->d.dtype == MV2_BF16 ? at::kBFloat16 : at::kFloat;
    int rc;
    {
        Launch at(p->device);
        dout = dense(dout); dn = dense(dn);
        for (int i = 0; i < 3; ++i) if (want[i]) g[i] = at.empty(p->shape, type);
        for (int i = 3; i < 6; ++i) if (want[i]) g[i] = at.empty({p->d.C}, at::kFloat);
        const int64_t bytes = want[3] || want[4] || want[5] ? p->ws_backward : 0;
        const at::Tensor ws = at.workspace(bytes);
        rc = mv2_block_norm_backward(&p->d, ptr(x), ptr(branch), ptr(gate), ptr<float>(post), ptr<float>(scale), ptr<float>(pre), ptr<float>(rstd), ptr(dout),
                                     ptr(dn), ptr(g[0]), ptr(g[1]), ptr(g[2]), ptr<float>(g[3]), ptr<float>(g[4]), ptr<float>(g[5]), ptr(ws), (size_t)bytes,
                                     at.stream());
    }
    if (rc) return failed("mv2_block_norm_backward", rc);
    return wrapped({g[0], g[1], g[2], g[3], g[4], g[5]});
    END_HANDLE_TH_ERRORS
}

// (descriptor, fused, device, shape of a part, of y, of the state, of the kept states or (), workspace bytes forward, backward)
PyObject* loop_plan(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    Py_buffer desc;
    PyObject *part, *y, *h, *states;
    auto p = std::make_unique<LoopPlan>();
    long long wf, wb;
    if (!PyArg_ParseTuple(args, "y*piOOOOLL", &desc, &p->fused, &p->device, &part, &y, &h, &states, &wf, &wb)) return nullptr;
    const bool ok = read_desc(desc, p->d);
    PyBuffer_Release(&desc);
    if (!ok || !read_shape(part, p->part) || !read_shape(y, p->y) || !read_shape(h, p->h) || !read_shape(states, p->states)) return nullptr;
    p->ws_forward = wf; p->ws_backward = wb;
    return PyCapsule_New(p.release(), LOOP, drop<LoopPlan>);
    END_HANDLE_TH_ERRORS
}

// (descriptor, device, shape, branch?, second norm?, norms to keep?, workspace bytes backward)
PyObject* norm_plan(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    Py_buffer desc;
    PyObject* shape;
    auto p = std::make_unique<NormPlan>();
    long long wb;
    if (!PyArg_ParseTuple(args, "y*iOpppL", &desc, &p->device, &shape, &p->branch, &p->normed, &p->keeps, &wb)) return nullptr;
    const bool ok = read_desc(desc, p->d);
    PyBuffer_Release(&desc);
    if (!ok || !read_shape(shape, p->shape)) return nullptr;
    p->ws_backward = wb;
    return PyCapsule_New(p.release(), NORM, drop<NormPlan>);
    END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    Py_XSETREF(error_class, cls);
    Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(loop_forward), FAST(loop_backward), FAST(norm_forward), FAST(norm_backward),
                         {"loop_plan", loop_plan, METH_VARARGS, nullptr}, {"norm_plan", norm_plan, METH_VARARGS, nullptr},
                         {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() { return PyModule_Create(&module); }
