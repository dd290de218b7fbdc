// asca_b200._torch_ops: the entry points of a training step around the blocks on torch tensors, for asca_b200.ops. Checks, outputs and
// scratch of a call are made here rather than in Python and ctypes, where they took two to four times as long as launching the
// kernels does (11 us of host time for a scaled embedding lookup, 4 here). Outputs and scratch come from torch's allocator on
// torch's current stream, which has to be the context's.
//
// Every function takes (context address, device, stream the context is bound to, ...) and its own arguments, all positional;
// asca_b200.ops gives them their names, defaults and documentation.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <string>
#include <vector>

#include "../../include/asca_b200.h"

namespace {

struct Raised {};   // a Python error is set

struct Ref {   // a reference of our own
    PyObject* p;
    ~Ref() { Py_XDECREF(p); }
};

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    PyErr_SetString(type, buf);
    throw Raised{};
}

std::string shape_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + (s[i] < 0 ? std::string("any") : std::to_string(s[i]));
    return t + (s.size() == 1 ? ",)" : ")");
}

using T = at::Tensor;
constexpr auto F32 = at::kFloat, BF16 = at::kBFloat16, I32 = at::kInt;

// The arguments of one call, read in order.
struct Call {
    PyObject* const* arg;
    Py_ssize_t n, i = 0;
    asca_ctx* ctx;
    int device;
    Call(PyObject* const* a, Py_ssize_t count, Py_ssize_t want) : arg(a), n(count) {
        if (n != want + 3) raise(PyExc_TypeError, "expected %zd arguments, got %zd", want + 3, n);
        ctx = (asca_ctx*)PyLong_AsVoidPtr(arg[i++]);
        device = (int)integer();
        if (!ctx) raise(PyExc_ValueError, "the context is closed");
        const auto bound = integer();
        const auto now = (int64_t)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        if (bound != (now ? now : 1)) raise(PyExc_RuntimeError, "the context is not on torch's current stream: call gpu.use_torch_stream()");
    }
    PyObject* next() { return arg[i++]; }
    int64_t integer() {
        const int64_t v = PyLong_AsLongLong(next());
        if (v == -1 && PyErr_Occurred()) throw Raised{};
        return v;
    }
    float number() {
        const double v = PyFloat_AsDouble(next());
        if (v == -1.0 && PyErr_Occurred()) throw Raised{};
        return (float)v;
    }
    bool truth() {
        const int v = PyObject_IsTrue(next());
        if (v < 0) throw Raised{};
        return v != 0;
    }
    // a tensor on the context's device, contiguous; the caller checks dtype and shape. Null for None where that is allowed.
    const T* tensor(const char* name, bool or_none = false) { return as_tensor(next(), name, or_none); }
    const T* as_tensor(PyObject* o, const char* name, bool or_none = false) const {
        if (o == Py_None && or_none) return nullptr;
        if (!THPVariable_Check(o)) raise(PyExc_ValueError, "%s: expected a tensor on cuda:%d", name, device);
        const T* t = &THPVariable_Unpack(o);
        if (!t->is_cuda() || t->get_device() != device) raise(PyExc_ValueError, "%s: expected a tensor on cuda:%d", name, device);
        return t;
    }
    bool none() {
        if (arg[i] != Py_None) return false;
        ++i;
        return true;
    }
    at::ScalarType dtype(const char* name, at::ScalarType other) {   // None: other
        PyObject* o = next();
        if (o == Py_None) return other;
        if (!THPDtype_Check(o)) raise(PyExc_TypeError, "%s: expected a torch dtype", name);
        return reinterpret_cast<THPDtype*>(o)->scalar_type;
    }
    T make(at::IntArrayRef shape, at::ScalarType type) const { return T(at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), c10::nullopt)); }
    // scratch of torch's allocator, back in its hands at the end of the call (negative: sizes that the entry point will refuse)
    struct Scratch {
        c10::DataPtr at;
        size_t bytes = 0;
        void* p() const { return at.get(); }
        size_t n() const { return bytes; }
    };
    Scratch scratch(int64_t bytes) const {
        if (bytes <= 0) return {};
        const c10::cuda::CUDAGuard on((c10::DeviceIndex)device);
        return {c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes), (size_t)bytes};
    }
    void ok(int rc) const {
        if (rc == ASCA_OK) return;
        PyObject* m = PyImport_ImportModule("asca_b200");
        PyObject* type = m ? PyObject_GetAttrString(m, "AscaError") : nullptr;
        PyObject* e = type ? PyObject_CallFunction(type, "is", rc, asca_last_error(ctx)) : nullptr;
        if (e) PyErr_SetObject(type, e);
        Py_XDECREF(e);
        Py_XDECREF(type);
        Py_XDECREF(m);
        throw Raised{};
    }
};

const char* name_of(at::ScalarType t) { return t == F32 ? "torch.float32" : t == BF16 ? "torch.bfloat16" : t == I32 ? "torch.int32" : c10::toString(t); }

void contiguous(const T& t, const char* name) {
    if (!t.is_contiguous()) raise(PyExc_ValueError, "%s: expected a contiguous tensor", name);
}
void shaped(const T& t, const char* name, at::IntArrayRef shape) {   // -1: any extent
    bool same = t.dim() == (int64_t)shape.size();
    for (size_t i = 0; same && i < shape.size(); ++i) same = shape[i] < 0 || shape[i] == t.size(i);
    if (!same) raise(PyExc_ValueError, "%s: expected the shape %s, got %s", name, shape_text(shape).c_str(), shape_text(t.sizes()).c_str());
}
int floating(const T& t, const char* name) {
    if (t.scalar_type() == F32) return ASCA_F32;
    if (t.scalar_type() == BF16) return ASCA_BF16;
    raise(PyExc_TypeError, "%s: expected float32 or bfloat16, got %s", name, name_of(t.scalar_type()));
}
int floating(at::ScalarType t, const char* name) {
    if (t != F32 && t != BF16) raise(PyExc_TypeError, "%s: expected float32 or bfloat16, got %s", name, name_of(t));
    return t == F32 ? ASCA_F32 : ASCA_BF16;
}
void typed(const T& t, const char* name, at::ScalarType type) {
    if (t.scalar_type() != type) raise(PyExc_TypeError, "%s: expected %s, got %s", name, name_of(type), name_of(t.scalar_type()));
}
template <typename P>
P* ptr(const T* t) { return t ? static_cast<P*>(t->data_ptr()) : nullptr; }

// A contiguous tensor of this dtype and shape, or None.
const T* given(Call& c, const char* name, at::ScalarType type, at::IntArrayRef shape, bool or_none = true) {
    const T* t = c.tensor(name, or_none);
    if (t) {
        typed(*t, name, type);
        shaped(*t, name, shape);
        contiguous(*t, name);
    }
    return t;
}
// The output that the caller gave, or a new one.
T output(Call& c, const char* name, at::ScalarType type, at::IntArrayRef shape) {
    const T* t = given(c, name, type, shape);
    return t ? *t : c.make(shape, type);
}
const uint32_t* token_ids(const T& t) {
    if (t.scalar_type() != I32 && t.scalar_type() != at::kUInt32) raise(PyExc_TypeError, "ids: expected torch.int32 or torch.uint32, got %s", name_of(t.scalar_type()));
    contiguous(t, "ids");
    return static_cast<const uint32_t*>(t.data_ptr());
}
PyObject* wrap(const T& t) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) throw Raised{};
    return o;
}
PyObject* tuple(std::initializer_list<PyObject*> items) {
    PyObject* t = PyTuple_New((Py_ssize_t)items.size());
    if (!t) throw Raised{};
    Py_ssize_t i = 0;
    for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
    return t;
}
PyObject* none() { return Py_NewRef(Py_None); }

// Small outputs of one call share an allocation: a tensor of its own on a part of it. It saves the host 1.1 us of the 10.9 that a gated
// residual's gradient takes and 0.9 of a routing's 5.5. Not above 256 KiB: a part that is kept holds on to all of it.
constexpr int64_t SHARED = 1 << 16;   // elements
T part(const T& whole, int64_t offset, at::IntArrayRef shape) {
    T t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
}

// ------------------------------------------------------------------ embedding
PyObject* embed_fwd(Call& c) {   // table, ids, scale, out_dtype, out
    const T &table = *c.tensor("table"), &ids = *c.tensor("ids");
    const int table_type = floating(table, "table");
    shaped(table, "table", {-1, -1});
    contiguous(table, "table");
    const uint32_t* id = token_ids(ids);
    const float scale = c.number();
    const bool any = c.arg[c.i] == Py_None;   // no dtype asked for: the given output's, else the table's
    auto type = c.dtype("out_dtype", table.scalar_type());
    if (any && c.arg[c.i] != Py_None) type = c.as_tensor(c.arg[c.i], "out")->scalar_type();
    const int out_type = floating(type, "out");
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(table.size(1));
    const T out = output(c, "out", type, shape);
    c.ok(asca_embed_scaled_fwd(c.ctx, table.data_ptr(), id, ids.numel(), table.size(1), table.size(0), scale, table_type, out_type, out.data_ptr()));
    return wrap(out);
}

PyObject* embed_bwd(Call& c) {   // dx, ids, vocab, scale, d_table, accumulate
    const T &dx = *c.tensor("dx"), &ids = *c.tensor("ids");
    const int type = floating(dx, "dx");
    const uint32_t* id = token_ids(ids);
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(-1);
    shaped(dx, "dx", shape);
    contiguous(dx, "dx");
    const int64_t vocab = c.integer(), d = dx.size(-1), n = ids.numel();
    const float scale = c.number();
    if (vocab <= 0 || d <= 0) raise(PyExc_ValueError, "embed_bwd: the table has no rows or no columns");
    const int64_t bytes = asca_embed_scaled_bwd_ws(n, d, vocab);
    if (bytes < 0) c.ok(asca_embed_scaled_bwd(c.ctx, dx.data_ptr(), id, n, d, vocab, scale, type, 0, nullptr, nullptr, 0));   // refused before a table is made
    const bool fresh = c.arg[c.i] == Py_None;
    const T d_table = output(c, "d_table", F32, {vocab, d});
    const bool accumulate = c.truth();
    if (accumulate && fresh) raise(PyExc_ValueError, "embed_bwd: accumulate needs the d_table to add to");
    const auto ws = c.scratch(bytes);
    c.ok(asca_embed_scaled_bwd(c.ctx, dx.data_ptr(), id, n, d, vocab, scale, type, accumulate, ptr<float>(&d_table), ws.p(), ws.n()));
    return wrap(d_table);
}

// ------------------------------------------------------------------ gated residual with its norms
struct JoinArgs {
    const T *gate, *w_post, *w_pre;
    int64_t gate_rows, rows, cols;
    bool post;
    float skip, branch, eps;
    int type;
    JoinArgs(Call& c, const T& y) {   // gate, gate_rows, w_post, w_pre, post_norm, skip_scale, branch_scale, eps
        type = floating(y, "y");
        shaped(y, "y", {-1, -1});
        contiguous(y, "y");
        rows = y.size(0), cols = y.size(1);
        gate = c.tensor("gate", true);
        gate_rows = c.none() ? (rows > 0 ? rows : 1) : c.integer();
        if (gate_rows <= 0) raise(PyExc_ValueError, "gate_rows: expected a positive number of rows");
        gate_rows = std::min(gate_rows, std::max<int64_t>(rows, 1));   // (one gate for all of them)
        if (gate) {
            typed(*gate, "gate", F32);
            shaped(*gate, "gate", {(rows + gate_rows - 1) / gate_rows, cols});
            contiguous(*gate, "gate");
        }
        w_post = given(c, "w_post", F32, {cols});
        w_pre = given(c, "w_pre", F32, {cols});
        post = c.truth();
        if (w_post && !post) raise(PyExc_ValueError, "w_post belongs to the norm after the block: post_norm is False");
        skip = c.number(), branch = c.number(), eps = c.number();
    }
};

PyObject* join_fwd(Call& c) {   // y, x, (join), want_norm, x_out
    const T &y = *c.tensor("y"), &x = *c.tensor("x");
    const JoinArgs a(c, y);
    typed(x, "x", F32);
    shaped(x, "x", {a.rows, a.cols});
    contiguous(x, "x");
    const bool want = c.truth();
    const T x_out = output(c, "x_out", F32, {a.rows, a.cols});
    T xn;
    if (want) xn = c.make({a.rows, a.cols}, y.scalar_type());
    c.ok(asca_gated_residual_rmsnorm_fwd(c.ctx, y.data_ptr(), ptr<float>(&x), ptr<float>(a.w_post), ptr<float>(a.gate), a.gate_rows, ptr<float>(a.w_pre), a.post,
                                         a.skip, a.branch, a.eps, a.rows, a.cols, a.type, ptr<float>(&x_out), want ? xn.data_ptr() : nullptr));
    return tuple({wrap(x_out), want ? wrap(xn) : none()});
}

PyObject* join_bwd(Call& c) {   // y, x_out, d_xn, d_out, (join), grads
    const T &y = *c.tensor("y"), &x_out = *c.tensor("x_out");
    const T *d_xn = c.tensor("d_xn", true), *d_out = c.tensor("d_out", true);
    const JoinArgs a(c, y);
    for (const auto& [t, name, type] : {std::tuple(&x_out, "x_out", F32), std::tuple(d_xn, "d_xn", y.scalar_type()), std::tuple(d_out, "d_out", F32)}) {
        if (!t) continue;
        typed(*t, name, type);
        shaped(*t, name, {a.rows, a.cols});
        contiguous(*t, name);
    }
    if (!d_xn && !d_out) raise(PyExc_ValueError, "gated_residual_rmsnorm_bwd: needs d_xn or d_out");
    PyObject* grads = c.next();
    const char* names[3] = {"d_w_post", "d_gate", "d_w_pre"};
    const T* of[3] = {a.w_post, a.gate, a.w_pre};
    T sums[3], together;
    int64_t offset = 0, all = 0;
    for (const T* t : of) all += t ? (t->numel() + 63) / 64 * 64 : 0;
    if (grads == Py_None && all > 0 && all <= SHARED) together = c.make({all}, F32);
    for (int i = 0; i < 3; ++i) {
        if (!of[i]) continue;
        if (grads == Py_None) {
            sums[i] = together.defined() ? part(together, offset, of[i]->sizes()) : c.make(of[i]->sizes(), F32);
            offset += (of[i]->numel() + 63) / 64 * 64;
            continue;
        }
        const Ref o{PyMapping_GetItemString(grads, names[i])};
        if (!o.p) throw Raised{};
        sums[i] = *c.as_tensor(o.p, names[i]);
        typed(sums[i], names[i], F32);
        shaped(sums[i], names[i], of[i]->sizes());
        contiguous(sums[i], names[i]);
    }
    const T d_x = c.make({a.rows, a.cols}, F32), d_y = c.make({a.rows, a.cols}, y.scalar_type());
    const auto ws = c.scratch(asca_gated_residual_rmsnorm_bwd_ws(c.ctx, a.rows, a.cols));
    auto sum = [&](int i) { return of[i] ? ptr<float>(&sums[i]) : nullptr; };
    c.ok(asca_gated_residual_rmsnorm_bwd(c.ctx, y.data_ptr(), ptr<float>(&x_out), ptr<void>(d_xn), ptr<float>(d_out), ptr<float>(a.w_post), ptr<float>(a.gate),
                                         a.gate_rows, ptr<float>(a.w_pre), a.post, a.skip, a.branch, a.eps, a.rows, a.cols, a.type, grads != Py_None,
                                         ptr<float>(&d_x), d_y.data_ptr(), sum(0), sum(1), sum(2), ws.p(), ws.n()));
    PyObject* d = PyDict_New();
    if (!d) throw Raised{};
    auto put = [&](const char* name, const T& t) {
        PyObject* o = wrap(t);
        PyDict_SetItemString(d, name, o);
        Py_DECREF(o);
    };
    put("d_x", d_x);
    put("d_y", d_y);
    for (int i = 0; i < 3; ++i)
        if (of[i]) put(names[i], sums[i]);
    return d;
}

// ------------------------------------------------------------------ rows by expert
PyObject* moe_dispatch(Call& c) {   // experts, E
    const T& experts = *c.tensor("experts");
    typed(experts, "experts", I32);
    shaped(experts, "experts", {-1, -1});
    contiguous(experts, "experts");
    const int64_t e = c.integer(), n = experts.size(0), k = experts.size(1);
    const int64_t bytes = asca_moe_topk_dispatch_ws(n, k, e);
    if (bytes < 0) c.ok(asca_moe_topk_dispatch(c.ctx, ptr<int32_t>(&experts), n, k, e, nullptr, nullptr, nullptr, nullptr, 0));   // refused before an output is made
    const int64_t bins = e + 1, list = (n * k + 63) / 64 * 64;
    T perm, offsets, slot;
    if (2 * list + bins <= SHARED) {
        const T all = c.make({2 * list + bins}, I32);
        perm = part(all, 0, {n * k}), slot = part(all, list, {n, k}), offsets = part(all, 2 * list, {bins});
    } else perm = c.make({n * k}, I32), offsets = c.make({bins}, I32), slot = c.make({n, k}, I32);
    const auto ws = c.scratch(bytes);
    c.ok(asca_moe_topk_dispatch(c.ctx, ptr<int32_t>(&experts), n, k, e, ptr<int32_t>(&perm), ptr<int32_t>(&offsets), ptr<int32_t>(&slot), ws.p(), ws.n()));
    return tuple({wrap(perm), wrap(offsets), wrap(slot)});
}

const T& slots(Call& c, int64_t n) {   // (n, any) int32; n = -1: any
    const T& slot = *c.tensor("slot");
    typed(slot, "slot", I32);
    shaped(slot, "slot", {n, -1});
    contiguous(slot, "slot");
    return slot;
}

PyObject* moe_sort(Call& c) {   // x, slot, out_dtype, out
    const T& x = *c.tensor("x");
    const int x_type = floating(x, "x");
    shaped(x, "x", {-1, -1});
    contiguous(x, "x");
    const T& slot = slots(c, x.size(0));
    const int64_t n = x.size(0), d = x.size(1), k = slot.size(1);
    const bool any = c.arg[c.i] == Py_None;
    auto type = c.dtype("out_dtype", x.scalar_type());
    if (any && c.arg[c.i] != Py_None) type = c.as_tensor(c.arg[c.i], "out")->scalar_type();
    const int out_type = floating(type, "out");
    const T out = output(c, "out", type, {n * k, d});
    c.ok(asca_moe_sort_rows(c.ctx, x.data_ptr(), ptr<int32_t>(&slot), n, k, d, x_type, out_type, out.data_ptr()));
    return wrap(out);
}

PyObject* moe_unsort(Call& c) {   // ys, slot, weights, out_dtype, out
    const T& ys = *c.tensor("ys");
    const T& slot = slots(c, -1);
    const int64_t n = slot.size(0), k = slot.size(1);
    const int y_type = floating(ys, "ys");
    shaped(ys, "ys", {n * k, -1});
    contiguous(ys, "ys");
    const int64_t d = ys.size(1);
    const T* weights = given(c, "weights", F32, {n, k});
    auto type = c.dtype("out_dtype", F32);
    if (c.arg[c.i] != Py_None) type = c.as_tensor(c.arg[c.i], "out")->scalar_type();
    const int out_type = floating(type, "out");
    const T out = output(c, "out", type, {n, d});
    c.ok(asca_moe_unsort_rows(c.ctx, ys.data_ptr(), ptr<int32_t>(&slot), ptr<float>(weights), n, k, d, y_type, out_type, out.data_ptr()));
    return wrap(out);
}

PyObject* moe_unsort_bwd(Call& c) {   // d_out, ys, slot, weights, d_ys
    const T &d_out = *c.tensor("d_out"), &ys = *c.tensor("ys");
    const T& slot = slots(c, -1);
    const int64_t n = slot.size(0), k = slot.size(1);
    const int g_type = floating(d_out, "d_out"), y_type = floating(ys, "ys");
    shaped(ys, "ys", {n * k, -1});
    contiguous(ys, "ys");
    const int64_t d = ys.size(1);
    shaped(d_out, "d_out", {n, d});
    contiguous(d_out, "d_out");
    const T* weights = given(c, "weights", F32, {n, k});
    const T d_ys = output(c, "d_ys", ys.scalar_type(), {n * k, d});
    T d_w;
    if (weights) d_w = c.make({n, k}, F32);
    c.ok(asca_moe_unsort_rows_bwd(c.ctx, d_out.data_ptr(), weights ? ys.data_ptr() : nullptr, ptr<int32_t>(&slot), ptr<float>(weights), n, k, d, g_type, y_type,
                                  d_ys.data_ptr(), weights ? ptr<float>(&d_w) : nullptr));
    return tuple({wrap(d_ys), weights ? wrap(d_w) : none()});
}

// ------------------------------------------------------------------ gradient norm, clipping, AdamW
struct List {
    const Ref seq;   // (kept to the end of the call: tensors that only an iterator made live as long)
    std::vector<void*> p;
    std::vector<int64_t> n;
    std::vector<int> dtype;
    explicit List(Call& c) : seq{PySequence_Fast(c.next(), "grads: expected a sequence of tensors")} {
        if (!seq.p) throw Raised{};
        const Py_ssize_t count = PySequence_Fast_GET_SIZE(seq.p);
        p.reserve(count), n.reserve(count), dtype.reserve(count);
        for (Py_ssize_t i = 0; i < count; ++i) {
            const T& t = *c.as_tensor(PySequence_Fast_GET_ITEM(seq.p, i), "grads");
            dtype.push_back(floating(t, "grads"));
            contiguous(t, "grads");
            p.push_back(t.data_ptr());
            n.push_back(t.numel());
        }
    }
    int count() const { return (int)p.size(); }
};

PyObject* grad_norm(Call& c) {   // grads, out
    const List l(c);
    const T out = output(c, "out", F32, {1});
    const auto ws = c.scratch(asca_grad_norm_ws(c.ctx, l.count()));
    c.ok(asca_grad_norm(c.ctx, l.p.data(), l.n.data(), l.dtype.data(), l.count(), ptr<float>(&out), ws.p(), ws.n()));
    return wrap(out);
}

PyObject* clip_grads(Call& c) {   // grads, max_norm, norm
    const List l(c);
    const float most = c.number();
    const T* norm = given(c, "norm", F32, {1}, false);
    c.ok(asca_clip_grads(c.ctx, l.p.data(), l.n.data(), l.dtype.data(), l.count(), ptr<float>(norm), most));
    return none();
}

struct Buffer {   // a C-contiguous host array
    Py_buffer b{};
    Buffer(PyObject* o, const char* name, Py_ssize_t itemsize, Py_ssize_t count) {
        if (PyObject_GetBuffer(o, &b, PyBUF_C_CONTIGUOUS) != 0) throw Raised{};
        if (b.itemsize != itemsize || (count >= 0 && b.len != count * itemsize)) {
            PyBuffer_Release(&b);
            raise(PyExc_ValueError, "%s: a host array of another length or item size", name);
        }
    }
    ~Buffer() { PyBuffer_Release(&b); }
};

PyObject* adamw_clip(Call& c) {   // p, g, m, v, seg_off, lr_t, eps_t, beta1, beta2, wd_eff, norm, max_norm
    const T* t[4];
    const char* names[4] = {"p", "g", "m", "v"};
    for (int i = 0; i < 4; ++i) t[i] = c.tensor(names[i]);
    for (int i = 0; i < 4; ++i) {
        typed(*t[i], names[i], F32);
        contiguous(*t[i], names[i]);
        if (t[i]->numel() != t[0]->numel()) raise(PyExc_ValueError, "%s: expected as many elements as p has", names[i]);
    }
    const Buffer off(c.next(), "seg_off", 8, -1);
    const Py_ssize_t segs = off.b.len / 8 - 1;
    if (segs < 1 || static_cast<const int64_t*>(off.b.buf)[segs] > t[0]->numel()) raise(PyExc_ValueError, "seg_off: no tensors, or more elements than p has");
    const Buffer lr(c.next(), "lr_t", 4, segs), eps(c.next(), "eps_t", 4, segs);
    const float b1 = c.number(), b2 = c.number(), wd = c.number();
    const T* norm = given(c, "norm", F32, {1}, false);
    const float most = c.number();
    c.ok(asca_adamw_segmented_clip(c.ctx, ptr<float>(t[0]), ptr<float>(t[1]), ptr<float>(t[2]), ptr<float>(t[3]), static_cast<const int64_t*>(off.b.buf),
                                   static_cast<const float*>(lr.b.buf), static_cast<const float*>(eps.b.buf), (int)segs, b1, b2, wd, nullptr, ptr<float>(norm), most));
    return none();
}

template <PyObject* (*F)(Call&), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS   // (torch's own: an allocation that failed, say)
    try {
        Call c(args, n, N);
        return F(c);
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
#define ASCA_ENTRY(name, fn, n) {name, (PyCFunction)(void (*)(void))entry<fn, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ASCA_ENTRY("embed_fwd", embed_fwd, 5), ASCA_ENTRY("embed_bwd", embed_bwd, 6), ASCA_ENTRY("join_fwd", join_fwd, 12),
                         ASCA_ENTRY("join_bwd", join_bwd, 13), ASCA_ENTRY("moe_dispatch", moe_dispatch, 2), ASCA_ENTRY("moe_sort", moe_sort, 4),
                         ASCA_ENTRY("moe_unsort", moe_unsort, 5), ASCA_ENTRY("moe_unsort_bwd", moe_unsort_bwd, 5), ASCA_ENTRY("grad_norm", grad_norm, 2),
                         ASCA_ENTRY("clip_grads", clip_grads, 3), ASCA_ENTRY("adamw_clip", adamw_clip, 12), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", "Tensor checks, outputs and scratch of asca_b200.ops", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", ASCA_BUILT_FOR) != 0) {   // (the torch and the interpreter: asca_b200/build.py)
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
