// Python module _attn_bind: the calls of adaptivepnp_sci_amd/attention.py from torch tensors to the C ABI (include/scipnp.h).
//
// A decoding step is five launches of a few microseconds each; forty attribute reads of tensors and a packed argument block cost 7 to 10 us
// a call in Python and hold them up (a call of head_norm_rotate: 12.3 us then, 6.4 now).  Here a call checks its arguments, allocates its
// results and its workspace from torch, fills the argument block and makes the one C call.  Nothing is kept from a call but the entry
// points, which attention.py hands over once (the library that ctypes has loaded: there is one of it in the process).
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/version.h>
#include <cmath>
#include <string>
#include "../../include/scipnp.h"

namespace {

using at::Tensor;

decltype(&scipnp_head_norm_rotate) head_norm;
decltype(&scipnp_head_norm_rotate_backward) head_norm_bwd;
decltype(&scipnp_head_norm_rotate_backward_workspace_bytes) head_norm_bwd_bytes;
decltype(&scipnp_block_summary) summary_fn;
decltype(&scipnp_select_blocks) select_fn;
decltype(&scipnp_block_attn_workspace_bytes) attn_bytes;
decltype(&scipnp_block_attn) attn_fn;
decltype(&scipnp_block_attn_backward) attn_bwd;
PyObject *check_fn, *no_gpu_error, *device_fn, *stream_fn;            // _lib.check, ScipnpError, the current device, its current stream

struct Raised {};                                                     // a Python exception is set
template <typename... A>
[[noreturn]] void refuse(PyObject* type, const char* format, A... a) {
    PyErr_Format(type, format, a...);
    throw Raised{};
}

std::string show(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}
const char* show(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return at::toString(t);
    }
}

int whole(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    if (v != (int)v) refuse(PyExc_ValueError, "%s is %lld: does not fit 32 bits", name, v);
    return (int)v;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return (float)v;
}
int truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v;
}

// every tensor of a call is on the current device: its stream is the one the call goes to
struct Call {
    int dev = -1;
    void on_device(const Tensor& t, const char* name) {
        if (!t.is_cuda()) refuse(no_gpu_error, "%s must be a CUDA/ROCm tensor (the hot path has no CPU fallback)", name);
        if (dev < 0) {
            PyObject* const d = PyObject_CallNoArgs(device_fn);
            if (!d) throw Raised{};
            dev = (int)PyLong_AsLong(d);
            Py_DECREF(d);
        }
        if (t.get_device() != dev) refuse(PyExc_ValueError, "%s is on cuda:%d, the current device is cuda:%d", name, (int)t.get_device(), dev);
    }
    scipnp_stream_t stream() {
        PyObject* const d = PyLong_FromLong(dev);
        PyObject* const s = PyObject_CallOneArg(stream_fn, d);
        Py_DECREF(d);
        if (!s) throw Raised{};
        void* const p = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        return (scipnp_stream_t)p;
    }
};

void done(int rc, const char* name) {
    if (rc == 0) return;
    PyObject* const r = PyObject_CallFunction(check_fn, "is", rc, name);      // raises
    Py_XDECREF(r);
    if (r) PyErr_Format(PyExc_RuntimeError, "%s: code %d", name, rc);
    throw Raised{};
}

const Tensor* given(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) refuse(PyExc_ValueError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
    return &THPVariable_Unpack(o);
}
const Tensor& shape4(PyObject* o, const char* name) {
    if (!THPVariable_Check(o) || THPVariable_Unpack(o).dim() != 4) refuse(PyExc_ValueError, "%s must be a (B, L, H, D) tensor", name);
    const Tensor& t = THPVariable_Unpack(o);
    if (t.numel() == 0) refuse(PyExc_ValueError, "%s has an empty dimension: %s", name, show(t.sizes()).c_str());
    for (const int64_t d : t.sizes())
        if (d > INT_MAX) refuse(PyExc_ValueError, "%s has a dimension past 32 bits: %s", name, show(t.sizes()).c_str());
    return t;
}

// pointer and element strides (batch, token, head) of a (B, L, H, D) tensor
struct Tokens {
    void* p;
    int64_t s[3];
    void to(const void*& q, int64_t* stride) const { q = p, put(stride); }
    void to(void*& q, int64_t* stride) const { q = p, put(stride); }
    void put(int64_t* stride) const {
        for (int i = 0; i < 3; ++i) stride[i] = s[i];
    }
};
Tokens tokens(const Tensor& t, const char* name, at::IntArrayRef shape = {}, at::ScalarType dtype = at::ScalarType::Undefined) {
    if (t.dim() != 4) refuse(PyExc_ValueError, "%s must be a (B, L, H, D) tensor", name);
    const at::ScalarType d = t.scalar_type();
    if (dtype == at::ScalarType::Undefined ? d != at::kFloat && d != at::kBFloat16 : d != dtype)
        refuse(PyExc_ValueError, "%s is %s: expected %s", name, show(d), dtype == at::ScalarType::Undefined ? "float32 or bfloat16" : show(dtype));
    if (shape.size() && t.sizes() != shape) refuse(PyExc_ValueError, "%s has shape %s, expected %s", name, show(t.sizes()).c_str(), show(shape).c_str());
    const auto n = t.sizes(), s = t.strides();
    if (s[3] != 1 && n[3] != 1) refuse(PyExc_ValueError, "%s: the last dimension must be contiguous", name);
    return {t.data_ptr(), {n[0] > 1 ? s[0] : 0, n[1] > 1 ? s[1] : 0, n[2] > 1 ? s[2] : 0}};
}
void* array(const Tensor* t, const char* name, at::IntArrayRef shape, at::ScalarType dtype) {
    if (!t) return nullptr;
    if (t->scalar_type() != dtype || t->sizes() != shape || !t->is_contiguous())
        refuse(PyExc_ValueError, "%s must be a contiguous %s tensor of shape %s, got %s %s%s", name, show(dtype), show(shape).c_str(), show(t->scalar_type()),
               show(t->sizes()).c_str(), t->is_contiguous() ? "" : ", not contiguous");
    return t->data_ptr();
}
// a null pointer here is an argument that the call cannot do without
const Tensor& needed(PyObject* o, const char* name) {
    const Tensor* const t = given(o, name);
    if (!t) refuse(PyExc_ValueError, "%s is missing", name);
    return *t;
}
// A given result must not have places that are one in memory, nor share memory with what the call reads or writes elsewhere: rows are read and
// written in any order.  (Views that interleave are told apart by nobody cheaply: only overlaps that are certain are refused.)
bool in_place(const Tensor& a, const Tensor& b) { return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides(); }
void apart(const Tensor* out, const char* name, const Tensor* other, const char* other_name) {
    if (!out || !other || !out->numel() || !other->numel()) return;
    const auto s = at::get_overlap_status(*out, *other);
    if (out->data_ptr() == other->data_ptr() || s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial)
        refuse(PyExc_ValueError, "%s shares memory with %s", name, other_name);
}
void single(const Tensor* out, const char* name) {
    if (out && at::has_internal_overlap(*out) == at::MemOverlap::Yes) refuse(PyExc_ValueError, "%s has several places in one memory location (an expanded tensor)", name);
}
// a given result was written: autograd notices where it had saved what was there
void written(const Tensor* out) {
    if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}
int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? SCIPNP_F32 : SCIPNP_BF16; }
Tensor new_bytes(const Tensor& like, size_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* back(PyObject* o) { return Py_INCREF(o), o; }

#define ENTER(count)                                                                                              \
    HANDLE_TH_ERRORS                                                                                              \
    if (n != count) { PyErr_Format(PyExc_TypeError, "%d arguments, got %zd", count, n); return nullptr; }         \
    try {                                                                                                         \
        at::AutoDispatchBelowADInplaceOrView below;                                                               \
        Call call;
#define LEAVE                                                                                                     \
    } catch (const Raised&) {                                                                                     \
        return nullptr;                                                                                           \
    }                                                                                                             \
    END_HANDLE_TH_ERRORS
#define WITHOUT_GIL(expr) [&] { int rc_; Py_BEGIN_ALLOW_THREADS rc_ = (expr); Py_END_ALLOW_THREADS return rc_; }()

// ---- norm and rotation: what both directions share
struct Norm {
    scipnp_head_norm_args a = {};
    at::ScalarType dt;
    Norm(Call& call, const Tensor& q, const Tensor* k, PyObject* wq, PyObject* wk, PyObject* turns_, PyObject* positions_, PyObject* first, PyObject* eps) {
        dt = q.scalar_type();
        const auto s = q.sizes();
        tokens(q, "q").to(a.q, a.q_stride);
        const Tensor *w = &needed(wq, "wq"), *turns = given(turns_, "turns"), *positions = given(positions_, "positions");
        a.struct_size = sizeof(a);
        a.dtype = type_of(q), a.B = (int)s[0], a.L = (int)s[1], a.Hq = (int)s[2], a.D = (int)s[3];
        a.rot = turns ? 2 * (int)turns->numel() : 0, a.first = whole(first, "first"), a.eps = real(eps);
        a.wq = (const float*)array(w, "wq", {s[3]}, at::kFloat);
        call.on_device(q, "q"), call.on_device(*w, "wq");
        if (k) {
            a.Hk = (int)k->size(2);
            tokens(*k, "k", {s[0], s[1], a.Hk, s[3]}, dt).to(a.k, a.k_stride);
            w = &needed(wk, "wk");
            a.wk = (const float*)array(w, "wk", {s[3]}, at::kFloat);
            call.on_device(*k, "k"), call.on_device(*w, "wk");
        }
        a.turns = (const double*)array(turns, "turns", {a.rot / 2}, at::kDouble);
        a.positions = (const int32_t*)array(positions, "positions", {s[0], s[1]}, at::kInt);
        if (turns) call.on_device(*turns, "turns");
        if (positions) call.on_device(*positions, "positions");
    }
};

// (q, k, wq, wk, turns, positions, first, eps, out_q, out_k, v, out_v, slots)
PyObject* head_norm_rotate(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(13)
    const Tensor& q = shape4(o[0], "q");
    const Tensor* const k = o[1] == Py_None ? nullptr : &shape4(o[1], "k");
    if (!k && (o[9] != Py_None || o[10] != Py_None || o[12] != Py_None)) refuse(PyExc_ValueError, "out_k, v and slots need k");
    const Tensor *out_q = given(o[8], "out_q"), *out_k = given(o[9], "out_k"), *v = given(o[10], "v"), *out_v = given(o[11], "out_v"), *slots = given(o[12], "slots");
    if (slots && !out_k) refuse(PyExc_ValueError, "slots need out_k (a cache)");
    if (v && !out_v) refuse(PyExc_ValueError, "v needs out_v");
    const struct { const Tensor *out, *in; const char *name, *in_name; } own[] = {{out_q, &q, "out_q", "q"}, {out_k, k, "out_k", "k"}, {v ? out_v : nullptr, v, "out_v", "v"}};
    for (int i = 0; i < 3; ++i) {
        single(own[i].out, own[i].name);
        for (int j = 0; j < 3; ++j) {
            if (i != j) apart(own[i].out, own[i].name, own[j].in, own[j].in_name);
            else if (own[i].out && own[i].in && !(i && slots) && !in_place(*own[i].out, *own[i].in)) apart(own[i].out, own[i].name, own[i].in, own[i].in_name);
            if (j < i) apart(own[i].out, own[i].name, own[j].out, own[j].name);
        }
    }
    Norm c(call, q, k, o[2], o[3], o[4], o[5], o[6], o[7]);
    scipnp_head_norm_args& a = c.a;
    Tensor new_q, new_k;
    if (out_q) call.on_device(*out_q, "out_q");
    else new_q = at::empty_like(q), out_q = &new_q;
    tokens(*out_q, "out_q", q.sizes(), c.dt).to(a.out_q, a.out_q_stride);
    if (k) {
        if (out_k) call.on_device(*out_k, "out_k");
        else new_k = at::empty_like(*k), out_k = &new_k;
        const int64_t rows = slots ? (shape4(o[9], "out_k"), out_k->size(1)) : a.L;
        const int64_t out[4] = {a.B, rows, a.Hk, a.D};
        tokens(*out_k, "out_k", out, c.dt).to(a.out_k, a.out_k_stride);
        if (v) {
            call.on_device(*v, "v"), call.on_device(*out_v, "out_v");
            tokens(*v, "v", k->sizes(), c.dt).to(a.v, a.v_stride);
            tokens(*out_v, "out_v", out, c.dt).to(a.out_v, a.out_v_stride);
        }
        if (slots) {
            call.on_device(*slots, "slots");
            a.slots = (const int32_t*)array(slots, "slots", {a.B, a.L}, at::kInt);
            if (rows > INT_MAX) refuse(PyExc_ValueError, "out_k has too many rows");
            a.Lout = (int)rows;
        }
    }
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(head_norm(&a, st)), "scipnp_head_norm_rotate");
    written(out_q), written(out_k), written(v ? out_v : nullptr);
    return Py_BuildValue("NN", o[8] == Py_None ? wrap(new_q) : back(o[8]), !k ? back(Py_None) : o[9] == Py_None ? wrap(new_k) : back(o[9]));
    LEAVE
}

// (g_q, g_k, q, k, wq, wk, turns, positions, first, eps)
PyObject* head_norm_rotate_backward(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(10)
    const Tensor& q = shape4(o[2], "q");
    const Tensor* const k = o[3] == Py_None ? nullptr : &shape4(o[3], "k");
    Norm c(call, q, k, o[4], o[5], o[6], o[7], o[8], o[9]);
    scipnp_head_norm_args& a = c.a;
    const Tensor& gq = needed(o[0], "g_q");
    tokens(gq, "g_q", q.sizes(), c.dt).to(a.g_q, a.g_q_stride);
    call.on_device(gq, "g_q");
    const Tensor dq = at::empty(q.sizes(), q.options()), dwq = at::empty({a.D}, q.options().dtype(at::kFloat));
    Tensor dk, dwk;
    tokens(dq, "dq").to(a.out_q, a.out_q_stride);
    a.dwq = dwq.data_ptr<float>();
    if (k) {
        const Tensor& gk = needed(o[1], "g_k");
        tokens(gk, "g_k", k->sizes(), c.dt).to(a.g_k, a.g_k_stride);
        call.on_device(gk, "g_k");
        dk = at::empty(k->sizes(), q.options()), dwk = at::empty_like(dwq);
        tokens(dk, "dk").to(a.out_k, a.out_k_stride);
        a.dwk = dwk.data_ptr<float>();
    }
    a.workspace_bytes = head_norm_bwd_bytes(&a);
    const Tensor ws = new_bytes(q, a.workspace_bytes);
    a.workspace = ws.data_ptr();
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(head_norm_bwd(&a, st)), "scipnp_head_norm_rotate_backward");
    return Py_BuildValue("NNNN", wrap(dq), k ? wrap(dk) : back(Py_None), wrap(dwq), k ? wrap(dwk) : back(Py_None));
    LEAVE
}

// (k, block, klen, newest, out)
PyObject* block_summary(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(5)
    const Tensor& k = shape4(o[0], "k");
    const int block = whole(o[1], "block"), newest = whole(o[3], "newest");
    if (block < 1 || newest < 0) refuse(PyExc_ValueError, "block %d must be positive, newest %d not negative", block, newest);
    const Tensor *klen = given(o[2], "klen"), *out = given(o[4], "out");
    if (newest && !out) refuse(PyExc_ValueError, "newest needs out");
    apart(out, "out", &k, "k");
    const Tokens t = tokens(k, "k");
    const int64_t shape[4] = {k.size(0), (k.size(1) + block - 1) / block, k.size(2), k.size(3)};
    const int32_t* const kl = (const int32_t*)array(klen, "klen", {k.size(0)}, at::kInt);
    call.on_device(k, "k");
    if (klen) call.on_device(*klen, "klen");
    Tensor made;
    if (out) call.on_device(*out, "out");
    else made = at::empty(shape, k.options().dtype(at::kFloat)), out = &made;
    float* const p = (float*)array(out, "out", shape, at::kFloat);
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(summary_fn(t.p, t.s, type_of(k), kl, p, (int)k.size(0), (int)k.size(1), (int)k.size(2), (int)k.size(3), block, newest, st)), "scipnp_block_summary");
    written(out);
    return o[4] == Py_None ? wrap(made) : back(o[4]);
    LEAVE
}

// (q, summary, n_sel, block, query_block, keys, causal, qlen, klen, sink, local)
PyObject* select_blocks(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(11)
    const Tensor& q = shape4(o[0], "q");
    const Tensor& su = needed(o[1], "summary");
    const auto s = q.sizes();
    if (su.dim() != 4 || su.size(0) != s[0] || su.size(3) != s[3] || su.size(2) < 1 || s[2] % su.size(2))
        refuse(PyExc_ValueError, "summary must be (B, blocks, Hk, D) of q %s, got %s", show(s).c_str(), show(su.sizes()).c_str());
    scipnp_select_args a = {};
    a.struct_size = sizeof(a);
    a.n_sel = whole(o[2], "n_sel"), a.block = whole(o[3], "block"), a.query_block = whole(o[4], "query_block");
    if (a.block < 1 || a.query_block < 1 || a.n_sel < 1) refuse(PyExc_ValueError, "block %d, query_block %d and n_sel %d must be positive", a.block, a.query_block, a.n_sel);
    const int64_t nb = su.size(1), keys = o[5] == Py_None ? nb * a.block : whole(o[5], "keys");
    if (keys < 1 || (keys + a.block - 1) / a.block != nb)
        refuse(PyExc_ValueError, "%lld keys in blocks of %d are not the %lld blocks of the summary", (long long)keys, a.block, (long long)nb);
    if (keys > INT_MAX) refuse(PyExc_ValueError, "too many keys");
    a.dtype = type_of(q), a.B = (int)s[0], a.Lq = (int)s[1], a.Lk = (int)keys, a.Hq = (int)s[2], a.Hk = (int)su.size(2), a.D = (int)s[3];
    a.causal = truth(o[6]), a.sink = whole(o[9], "sink"), a.local = whole(o[10], "local");
    tokens(q, "q").to(a.q, a.q_stride);
    const Tensor *qlen = given(o[7], "qlen"), *klen = given(o[8], "klen");
    a.summary = (const float*)array(&su, "summary", su.sizes(), at::kFloat);
    a.qlen = (const int32_t*)array(qlen, "qlen", {s[0]}, at::kInt), a.klen = (const int32_t*)array(klen, "klen", {s[0]}, at::kInt);
    call.on_device(q, "q"), call.on_device(su, "summary");
    if (qlen) call.on_device(*qlen, "qlen");
    if (klen) call.on_device(*klen, "klen");
    const Tensor sel = at::empty({s[0], a.Hk, (s[1] + a.query_block - 1) / a.query_block, a.n_sel}, q.options().dtype(at::kInt));
    a.sel = sel.data_ptr<int32_t>();
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(select_fn(&a, st)), "scipnp_select_blocks");
    return wrap(sel);
    LEAVE
}

// ---- attention: what both directions share.  o: q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos
struct Attention {
    scipnp_block_attn_args a = {};
    const Tensor &q, &k;
    const Tensor *v, *bias;
    Attention(Call& call, PyObject* const* o) : q(shape4(o[0], "q")), k(shape4(o[1], "k")) {
        const auto s = q.sizes(), r = k.sizes();
        if (r[0] != s[0] || r[3] != s[3] || s[2] % r[2])
            refuse(PyExc_ValueError, "q %s and k %s: same batch and head size, query heads a multiple of key heads", show(s).c_str(), show(r).c_str());
        a.struct_size = sizeof(a);
        a.block = whole(o[4], "block"), a.query_block = whole(o[5], "query_block");
        if (a.block < 1 || a.query_block < 1) refuse(PyExc_ValueError, "block %d and query_block %d must be positive", a.block, a.query_block);
        const int64_t groups = (s[1] + a.query_block - 1) / a.query_block;
        const Tensor* const sel = given(o[3], "sel");
        if (!sel || sel->dim() != 4)
            refuse(PyExc_ValueError, "sel must be (B, Hk, groups, n) = (%lld, %lld, %lld, n)", (long long)s[0], (long long)r[2], (long long)groups);
        const at::ScalarType dt = q.scalar_type();
        a.dtype = type_of(q), a.B = (int)s[0], a.Lq = (int)s[1], a.Lk = (int)r[1], a.Hq = (int)s[2], a.Hk = (int)r[2], a.D = (int)s[3], a.n_sel = (int)sel->size(3);
        a.scale = o[6] == Py_None ? (float)(1.0 / std::sqrt((double)a.D)) : real(o[6]), a.causal = truth(o[7]);
        tokens(q, "q").to(a.q, a.q_stride);
        tokens(k, "k", {}, dt).to(a.k, a.k_stride);
        v = &needed(o[2], "v");
        tokens(*v, "v", r, dt).to(a.v, a.v_stride);
        a.sel = (const int32_t*)array(sel, "sel", {s[0], r[2], groups, sel->size(3)}, at::kInt);
        const Tensor *qlen = given(o[8], "qlen"), *klen = given(o[9], "klen"), *bucket_of = given(o[10], "bucket_of"), *q_pos = given(o[12], "q_pos"),
                     *k_pos = given(o[13], "k_pos");
        bias = given(o[11], "bias");
        a.qlen = (const int32_t*)array(qlen, "qlen", {s[0]}, at::kInt), a.klen = (const int32_t*)array(klen, "klen", {s[0]}, at::kInt);
        if (!bias != !bucket_of) refuse(PyExc_ValueError, "bias and bucket_of belong together");
        if (bias) {
            if (bias->dim() != 2 || bucket_of->dim() != 1 || bucket_of->size(0) % 2 == 0)
                refuse(PyExc_ValueError, "bias must be (buckets, Hq), bucket_of (2 * max_distance + 1,)");
            if (bias->size(0) < 1 || bias->size(0) > INT_MAX || bucket_of->size(0) > INT_MAX) refuse(PyExc_ValueError, "bias without buckets, or too many");
            a.num_buckets = (int)bias->size(0), a.max_distance = (int)(bucket_of->size(0) / 2);
            a.bias = (const float*)array(bias, "bias", {a.num_buckets, s[2]}, at::kFloat);
            a.bucket_of = (const int32_t*)array(bucket_of, "bucket_of", {bucket_of->size(0)}, at::kInt);
            a.q_pos = (const int32_t*)array(q_pos, "q_pos", {s[0], s[1]}, at::kInt), a.k_pos = (const int32_t*)array(k_pos, "k_pos", {s[0], r[1]}, at::kInt);
        } else if (q_pos || k_pos) {
            refuse(PyExc_ValueError, "q_pos and k_pos are positions for the bias");
        }
        const struct { const Tensor* t; const char* name; } all[] = {{&q, "q"}, {&k, "k"}, {v, "v"}, {sel, "sel"}, {qlen, "qlen"}, {klen, "klen"}, {bias, "bias"},
                                                                    {bucket_of, "bucket_of"}, {q_pos, "q_pos"}, {k_pos, "k_pos"}};
        for (const auto& x : all)
            if (x.t) call.on_device(*x.t, x.name);
    }
    Tensor workspace(int backward) {
        a.workspace_bytes = attn_bytes(&a, backward);
        if (!a.workspace_bytes) return {};
        const Tensor ws = new_bytes(q, a.workspace_bytes);
        a.workspace = ws.data_ptr();
        return ws;
    }
};

// (the fourteen of Attention, out, save)
PyObject* block_attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(16)
    const Tensor* out = given(o[14], "out");
    single(out, "out");
    apart(out, "out", given(o[1], "k"), "k");
    apart(out, "out", given(o[2], "v"), "v");
    if (const Tensor* const q = given(o[0], "q"); q && out && !in_place(*out, *q)) apart(out, "out", q, "q");
    Attention c(call, o);
    Tensor made, lse, rest, out32;
    if (out) call.on_device(*out, "out");
    else made = at::empty_like(c.q), out = &made, c.a.zero_rest = 1;
    tokens(*out, "out", c.q.sizes(), c.q.scalar_type()).to(c.a.out, c.a.out_stride);
    const bool save = truth(o[15]);
    if (save) {
        lse = at::empty({c.a.B, c.a.Hq, c.a.Lq}, c.q.options().dtype(at::kFloat)), rest = at::empty_like(lse), out32 = at::empty(c.q.sizes(), c.q.options().dtype(at::kFloat));
        c.a.lse = lse.data_ptr<float>(), c.a.lse_rest = rest.data_ptr<float>(), c.a.out32 = out32.data_ptr<float>();
    }
    const Tensor ws = c.workspace(0);
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(attn_fn(&c.a, st)), "scipnp_block_attn");
    written(out);
    PyObject* const r = o[14] == Py_None ? wrap(made) : back(o[14]);
    return save ? Py_BuildValue("N(NNN)", r, wrap(lse), wrap(out32), wrap(rest)) : r;
    LEAVE
}

// (the fourteen of Attention, dout, lse, out32, lse_rest)
PyObject* block_attention_backward(PyObject*, PyObject* const* o, Py_ssize_t n) {
    ENTER(18)
    Attention c(call, o);
    scipnp_block_attn_args& a = c.a;
    const Tensor &dout = needed(o[14], "dout"), &lse = needed(o[15], "saved[0]"), &out32 = needed(o[16], "saved[1]"), &rest = needed(o[17], "saved[2]");
    tokens(dout, "dout", c.q.sizes(), c.q.scalar_type()).to(a.dout, a.dout_stride);
    a.lse = (float*)array(&lse, "saved[0]", {a.B, a.Hq, a.Lq}, at::kFloat), a.out32 = (float*)array(&out32, "saved[1]", c.q.sizes(), at::kFloat);
    a.lse_rest = (float*)array(&rest, "saved[2]", {a.B, a.Hq, a.Lq}, at::kFloat);
    call.on_device(dout, "dout"), call.on_device(lse, "saved[0]"), call.on_device(out32, "saved[1]"), call.on_device(rest, "saved[2]");
    const Tensor dq = at::empty(c.q.sizes(), c.q.options()), dk = at::empty(c.k.sizes(), c.k.options()), dv = at::empty(c.k.sizes(), c.k.options());
    Tensor dbias;
    a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr();
    if (c.bias) dbias = at::empty(c.bias->sizes(), c.bias->options()), a.dbias = dbias.data_ptr<float>();
    const Tensor ws = c.workspace(1);
    const scipnp_stream_t st = call.stream();
    done(WITHOUT_GIL(attn_bwd(&a, st)), "scipnp_block_attn_backward");
    return Py_BuildValue("NNNN", wrap(dq), wrap(dk), wrap(dv), c.bias ? wrap(dbias) : back(Py_None));
    LEAVE
}

// the addresses of the entries above in their order, then _lib.check, ScipnpError, the current device's function and its stream's
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    void** const to[] = {(void**)&head_norm, (void**)&head_norm_bwd, (void**)&head_norm_bwd_bytes, (void**)&summary_fn, (void**)&select_fn, (void**)&attn_bytes,
                         (void**)&attn_fn, (void**)&attn_bwd};
    PyObject** const kept[] = {&check_fn, &no_gpu_error, &device_fn, &stream_fn};
    if (n != 12) return PyErr_Format(PyExc_TypeError, "12 arguments, got %zd", n);
    for (int i = 0; i < 8; ++i) {
        *to[i] = PyLong_AsVoidPtr(o[i]);
        if (!*to[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "entry %d is null", i);
    }
    for (int i = 0; i < 4; ++i) *kept[i] = back(o[8 + i]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
    FAST(bind), FAST(head_norm_rotate), FAST(head_norm_rotate_backward), FAST(block_summary), FAST(select_blocks), FAST(block_attention), FAST(block_attention_backward),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attn_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (built_for: a tensor's layout in memory is that of the torch whose headers this saw)
PyMODINIT_FUNC PyInit__attn_bind(void) {
    PyObject* const m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
