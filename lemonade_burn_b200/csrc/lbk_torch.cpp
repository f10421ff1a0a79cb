// The calls around drafted tokens (lemonade_burn_b200/ops.py) on torch tensors: checks of arguments, results, the current stream, the call into the library.
// In Python these were most of a small call's time: us a call on the host, before / so: attn_tree 13.0 / 5.2, rope_kv_append_tree 7.8 / 2.5, tree_accept 10.7 /
// 4.1, kv_keep_path 6.3 / 2.3, token_logprobs 15.8 / 4.5.
//
// The library itself knows nothing of torch: its functions are handed over by address (bind), so that this file works with whatever library the process has
// loaded. No exception leaves an entry point: torch's become RuntimeError, a status that is not 0 becomes LbkError.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/ScalarTypeToTypeMeta.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <exception>
#include <type_traits>

#include "lbk.h"

namespace {

struct Library {
    decltype(&lbk_rope_kv_append_tree) append = nullptr;
    decltype(&lbk_attn_tree_scratch) scratch = nullptr;
    decltype(&lbk_attn_tree) attn = nullptr;
    decltype(&lbk_tree_accept) accept = nullptr;
    decltype(&lbk_kv_keep_path) keep = nullptr;
    decltype(&lbk_advance_pos_by) advance = nullptr;
    decltype(&lbk_token_logprobs) logprobs = nullptr;
    decltype(&lbk_advance_pos_path) advance_path = nullptr;
} lib;
PyObject *g_check = nullptr, *g_context = nullptr;  // raises for a status; the default context
PyObject *g_handle = nullptr, *g_value = nullptr, *g_device = nullptr;  // attribute names

// A refusal on its way to Python, whose error is set.
struct Refused {};
[[noreturn]] __attribute__((format(printf, 2, 3))) void refuse(PyObject *kind, const char *format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(kind, format, args);
    va_end(args);
    throw Refused();
}

// A function that the loaded library has (one family's part of it: _lib.use).
template <class F>
F have(F f, const char *name) {
    if (!f) refuse(PyExc_RuntimeError, "the library that is loaded has no %s", name);
    return f;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s is a tensor", name);
    return THPVariable_Unpack(o);
}
// None is a tensor that is not defined.
at::Tensor maybe(PyObject *o, const char *name) { return o == Py_None ? at::Tensor() : tensor(o, name); }
const void *data(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
template <class T>
T *data(const at::Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}
const int32_t *ints(const at::Tensor &t) { return data<int32_t>(t); }
bool is(const at::Tensor &t, at::ScalarType type) { return t.scalar_type() == type; }

struct Context {
    lbk_ctx *handle;
    int device;
    explicit Context(PyObject *o) {
        PyObject *ctx = o == Py_None ? PyObject_CallNoArgs(g_context) : Py_NewRef(o);
        if (!ctx) throw Refused();
        PyObject *h = PyObject_GetAttr(ctx, g_handle), *v = h ? PyObject_GetAttr(h, g_value) : nullptr, *d = PyObject_GetAttr(ctx, g_device);
        Py_XDECREF(h);
        Py_DECREF(ctx);
        handle = v && v != Py_None ? static_cast<lbk_ctx *>(PyLong_AsVoidPtr(v)) : nullptr;
        device = d ? static_cast<int>(PyLong_AsLong(d)) : -1;
        Py_XDECREF(v);
        Py_XDECREF(d);
        if (PyErr_Occurred()) throw Refused();
        if (!handle) refuse(PyExc_ValueError, "the context is closed");
    }
    void lives_here(const at::Tensor &t) const {
        if (t.defined() && (!t.is_cuda() || t.get_device() != device)) refuse(PyExc_ValueError, "every tensor must live on cuda:%d", device);
    }
    // the tensors lie on this GPU without gaps
    template <class... Tensors>
    void *stream(const Tensors &...tensors) const {
        const at::Tensor *all[] = {&tensors...};
        for (const at::Tensor *t : all) {
            lives_here(*t);
            if (t->defined() && !t->is_contiguous()) refuse(PyExc_ValueError, "tensors must be contiguous");
        }
        return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    }
};
void done(int status) {
    if (!status) return;
    PyObject *r = PyObject_CallFunction(g_check, "i", status);
    Py_XDECREF(r);
    throw Refused();
}

struct Tree {
    int64_t b, t;
};
// A batch of trees, or of paths through them
Tree tree(const at::Tensor &parents, const at::Tensor &counts, const at::Tensor &pos) {
    if (parents.dim() != 2) refuse(PyExc_ValueError, "the trees are [sequences, nodes]");
    const Tree s{parents.size(0), parents.size(1)};
    if (s.t < 1 || s.t > LBK_TREE_NODES) refuse(PyExc_ValueError, "a tree has 1 to %d nodes (got %lld)", LBK_TREE_NODES, static_cast<long long>(s.t));
    if (!is(parents, at::kInt)) refuse(PyExc_TypeError, "the trees are int32");
    for (const at::Tensor *v : {&counts, &pos})
        if (v->defined() && (!is(*v, at::kInt) || v->dim() != 1 || v->size(0) != s.b)) refuse(PyExc_ValueError, "positions and counts are int32, one for each of the %lld sequences", static_cast<long long>(s.b));
    return s;
}
struct Cache {
    int64_t layers, kv_heads, cap, hd;
};
Cache caches(const at::Tensor &k, const at::Tensor &v, int64_t b, int64_t dims) {
    if (!is(k, at::kBFloat16) || !is(v, at::kBFloat16)) refuse(PyExc_TypeError, "caches are bf16");
    if (k.dim() != dims || !k.sizes().equals(v.sizes()) || k.size(dims - 4) != b)
        refuse(PyExc_ValueError, "caches are [%s%lld, kv_heads, capacity, head_dim], keys like values", dims == 5 ? "layers, " : "", static_cast<long long>(b));
    return {dims == 5 ? k.size(0) : 1, k.size(dims - 3), k.size(dims - 2), k.size(dims - 1)};
}
at::Tensor like(const at::Tensor &t, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, t.options().dtype(type)); }

// Results of one call that share an allocation: four of their own are 4 us. Of 32-bit values, each from a 16-byte boundary on.
class Results {
    c10::Storage storage_;
    int64_t at_ = 0;

public:
    static int64_t room(int64_t values) { return (values + 3) / 4 * 4; }
    Results(const at::Tensor &beside, int64_t values) : storage_(like(beside, {values}, at::kFloat).storage()) {}
    at::Tensor take(at::IntArrayRef shape, at::ScalarType type) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage_), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_storage_offset(at_);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        at_ += room(t.numel());
        return t;
    }
};

// The body of an entry point: `n` arguments, no exception to Python's side.
template <class Body>
PyObject *entry(Py_ssize_t given, Py_ssize_t wanted, Body &&body) {
    try {
        if (given != wanted) refuse(PyExc_TypeError, "%zd arguments, not %zd", wanted, given);
        return body();
    } catch (const Refused &) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the call was refused");
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

// q, k, v, cos, sin, pos, parents, kcache, vcache, counts, ctx
PyObject *rope_kv_append_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 11, [&] {
        const auto call = have(lib.append, "lbk_rope_kv_append_tree");
        const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &cos = tensor(a[3], "cos"), &sin = tensor(a[4], "sin"), &pos = tensor(a[5], "pos"),
                         &parents = tensor(a[6], "parents"), &kc = tensor(a[7], "kcache"), &vc = tensor(a[8], "vcache");
        const at::Tensor counts = maybe(a[9], "counts");
        const Tree s = tree(parents, counts, pos);
        const Cache c = caches(kc, vc, s.b, 4);
        for (const at::Tensor *t : {&q, &k, &v, &cos, &sin})
            if (!is(*t, at::kFloat)) refuse(PyExc_TypeError, "queries, keys, values and rotation tables are f32");
        const int64_t row = s.b * s.t * c.hd, heads = row ? q.numel() / row : 0;
        if (q.numel() != heads * row || k.numel() != c.kv_heads * row || v.numel() != k.numel())
            refuse(PyExc_ValueError, "q, k and v are rows of heads of %lld for %lld x %lld nodes", static_cast<long long>(c.hd), static_cast<long long>(s.b), static_cast<long long>(s.t));
        if (cos.dim() != 2 || cos.size(0) < c.cap || cos.size(1) != c.hd || !sin.sizes().equals(cos.sizes())) refuse(PyExc_ValueError, "the rotation tables have a row for every place of the cache");
        const Context ctx(a[10]);
        void *st = ctx.stream(q, k, v, cos, sin, pos, parents, kc, vc, counts);
        done(call(ctx.handle, data<float>(q), data<float>(k), data<float>(v), data<float>(cos), data<float>(sin), ints(pos), ints(parents), ints(counts), s.b, s.t, heads, c.kv_heads, c.hd,
                        c.cap, data<uint16_t>(kc), data<uint16_t>(vc), st));
        Py_RETURN_NONE;
    });
}

// Values from one node's row to the next in [b, t, heads, head_dim]
int64_t node_pitch(const at::Tensor &x, const Tree &s, int64_t heads, int64_t hd) {
    if (x.is_contiguous()) return heads * hd;
    const int64_t pitch = s.t > 1 ? x.stride(1) : s.b > 1 ? x.stride(0) : heads * hd;
    if (x.stride(3) != 1 || (heads > 1 && x.stride(2) != hd) || (s.b > 1 && x.stride(0) != s.t * pitch) || pitch < heads * hd)
        refuse(PyExc_ValueError, "the heads of a node lie side by side, nodes and sequences at one distance");
    return pitch;
}

// q, kcache, vcache, pos, parents, counts, scale, out, ctx
PyObject *attn_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 9, [&] {
        const auto call = have(lib.attn, "lbk_attn_tree");
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "kcache"), &vc = tensor(a[2], "vcache"), &pos = tensor(a[3], "pos"), &parents = tensor(a[4], "parents");
        const at::Tensor counts = maybe(a[5], "counts");
        at::Tensor out = maybe(a[7], "out");
        const Tree s = tree(parents, counts, pos);
        const Cache c = caches(kc, vc, s.b, 4);
        const bool f32 = is(q, at::kFloat);
        if (!f32 && !is(q, at::kBFloat16)) refuse(PyExc_TypeError, "queries are f32 or bf16");
        if (q.dim() != 4 || q.size(0) != s.b || q.size(1) != s.t || q.size(3) != c.hd)
            refuse(PyExc_ValueError, "queries are [%lld, %lld, heads, %lld]", static_cast<long long>(s.b), static_cast<long long>(s.t), static_cast<long long>(c.hd));
        const int64_t heads = q.size(2);
        if (c.hd != 128 || !heads || !c.kv_heads || heads % c.kv_heads)
            refuse(PyExc_ValueError, "heads of 128, a multiple of the KV heads (got %lld and %lld heads of %lld)", static_cast<long long>(heads), static_cast<long long>(c.kv_heads),
                   static_cast<long long>(c.hd));
        const double scale = a[6] == Py_None ? 0.08838834764831845 : PyFloat_AsDouble(a[6]);  // 128^-0.5
        if (PyErr_Occurred()) throw Refused();
        if (out.defined() && (out.scalar_type() != q.scalar_type() || !out.sizes().equals(q.sizes()))) refuse(PyExc_ValueError, "out is like q");
        const int64_t q_pitch = node_pitch(q, s, heads, c.hd), out_pitch = out.defined() ? node_pitch(out, s, heads, c.hd) : heads * c.hd;
        const Context ctx(a[8]);
        void *st = ctx.stream(kc, vc, pos, parents, counts);
        ctx.lives_here(q);
        ctx.lives_here(out);
        if (!out.defined()) out = like(q, q.sizes(), q.scalar_type());
        const at::Tensor scratch = like(q, {static_cast<int64_t>(lib.scratch(ctx.handle, s.t, heads, c.kv_heads))}, at::kFloat);
        done(call(ctx.handle, f32 ? LBK_COMPUTE_F32 : LBK_COMPUTE_BF16, data(q), q_pitch, data<uint16_t>(kc), data<uint16_t>(vc), ints(pos), ints(parents), ints(counts), s.b, s.t, heads,
                      c.kv_heads, c.hd, c.cap, static_cast<float>(scale), data<float>(scratch), data<void>(out), out_pitch, st));
        return a[7] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[7]);
    });
}

PyObject *wrap(std::initializer_list<at::Tensor> tensors) {
    PyObject *tuple = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    if (!tuple) throw Refused();
    Py_ssize_t i = 0;
    for (const at::Tensor &t : tensors) {
        PyObject *o = THPVariable_Wrap(t);
        if (!o) {
            Py_DECREF(tuple);
            throw Refused();
        }
        PyTuple_SET_ITEM(tuple, i++, o);
    }
    return tuple;
}

// tokens, parents, best, counts, ctx
PyObject *tree_accept(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 5, [&] {
        const auto call = have(lib.accept, "lbk_tree_accept");
        const at::Tensor &tokens = tensor(a[0], "tokens"), &parents = tensor(a[1], "parents"), &best = tensor(a[2], "best");
        const at::Tensor counts = maybe(a[3], "counts");
        const Tree s = tree(parents, counts, at::Tensor());
        if (!is(tokens, at::kInt) || !is(best, at::kInt)) refuse(PyExc_TypeError, "tokens and best are int32");
        if (!tokens.sizes().equals(parents.sizes()) || !best.sizes().equals(parents.sizes()))
            refuse(PyExc_ValueError, "tokens and best are [%lld, %lld], as parents", static_cast<long long>(s.b), static_cast<long long>(s.t));
        const Context ctx(a[4]);
        void *st = ctx.stream(tokens, parents, best, counts);
        Results r(parents, Results::room(s.b * s.t) + 2 * Results::room(s.b));
        const at::Tensor path = r.take({s.b, s.t}, at::kInt), count = r.take({s.b}, at::kInt), after = r.take({s.b}, at::kInt);
        done(call(ctx.handle, ints(tokens), ints(parents), ints(best), ints(counts), s.b, s.t, data<int32_t>(path), data<int32_t>(count), data<int32_t>(after), st));
        return wrap({path, count, after});
    });
}

// k, v, pos, path, count, ctx, advance
PyObject *kv_keep_path(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 7, [&] {
        const auto call = have(lib.keep, "lbk_kv_keep_path");
        const auto move = have(lib.advance_path, "lbk_advance_pos_path");
        const int advance = PyObject_IsTrue(a[6]);
        if (advance < 0) throw Refused();
        const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &pos = tensor(a[2], "pos"), &path = tensor(a[3], "path"), &count = tensor(a[4], "count");
        const Tree s = tree(path, count, pos);
        const Cache c = caches(k, v, s.b, 5);
        const Context ctx(a[5]);
        void *st = ctx.stream(k, v, pos, path, count);
        done(call(ctx.handle, data<uint16_t>(k), data<uint16_t>(v), c.layers, s.b * c.kv_heads * c.cap * c.hd, s.b, c.kv_heads, c.hd, c.cap, ints(pos), ints(path), ints(count), s.t, st));
        if (advance) done(move(ctx.handle, data<int32_t>(pos), ints(path), ints(count), s.b, s.t, c.cap, st));
        Py_RETURN_NONE;
    });
}

// pos, count, ctx
PyObject *advance_pos_by(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 3, [&] {
        const auto call = have(lib.advance, "lbk_advance_pos_by");
        const at::Tensor &pos = tensor(a[0], "pos"), &count = tensor(a[1], "count");
        if (!is(pos, at::kInt) || !is(count, at::kInt) || pos.dim() != 1 || !pos.sizes().equals(count.sizes()))
            refuse(PyExc_ValueError, "pos and count are int32, one number for each sequence");
        const Context ctx(a[2]);
        void *st = ctx.stream(pos, count);
        done(call(ctx.handle, data<int32_t>(pos), ints(count), pos.size(0), st));
        Py_RETURN_NONE;
    });
}

// logits, tokens, top, scale, ctx
PyObject *token_logprobs(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 5, [&] {
        const auto call = have(lib.logprobs, "lbk_token_logprobs");
        const at::Tensor &logits = tensor(a[0], "logits");
        const at::Tensor tokens = maybe(a[1], "tokens");
        const long long top = PyLong_AsLongLong(a[2]);
        const double scale = PyFloat_AsDouble(a[3]);
        if (PyErr_Occurred()) throw Refused();
        const bool f32 = is(logits, at::kFloat);
        if (!f32 && !is(logits, at::kBFloat16)) refuse(PyExc_TypeError, "logits are f32 or bf16");
        if (logits.dim() != 2 || logits.size(1) < 1) refuse(PyExc_ValueError, "logits are [rows, vocab]");
        const int64_t rows = logits.size(0), vocab = logits.size(1), pitch = rows > 1 ? logits.stride(0) : vocab;
        if ((vocab > 1 && logits.stride(1) != 1) || pitch < vocab) refuse(PyExc_ValueError, "the values of a row lie side by side, rows do not overlap");
        if (top < 0 || top > vocab || top > LBK_LOGPROBS_TOP) refuse(PyExc_ValueError, "%lld alternatives of %lld: at most %d", top, static_cast<long long>(vocab), LBK_LOGPROBS_TOP);
        int64_t given = 0;
        if (tokens.defined()) {
            if (!is(tokens, at::kInt)) refuse(PyExc_TypeError, "tokens are int32");
            if ((tokens.dim() != 1 && tokens.dim() != 2) || tokens.size(0) != rows) refuse(PyExc_ValueError, "tokens are [rows] or [rows, given]");
            given = tokens.dim() == 1 ? 1 : tokens.size(1);
        }
        const Context ctx(a[4]);
        void *st = ctx.stream(tokens);
        ctx.lives_here(logits);
        Results r(logits, Results::room(rows * given) + Results::room(rows) + 2 * Results::room(rows * top));
        const at::Tensor lp = r.take({rows, given}, at::kFloat), entropy = r.take({rows}, at::kFloat), ids = r.take({rows, static_cast<int64_t>(top)}, at::kInt),
                         best = r.take({rows, static_cast<int64_t>(top)}, at::kFloat);
        done(call(ctx.handle, f32 ? LBK_DTYPE_F32 : LBK_DTYPE_BF16, data(logits), pitch, rows, vocab, given ? ints(tokens) : nullptr, given, static_cast<float>(scale), top,
                          data<float>(lp), data<float>(entropy), data<int32_t>(ids), data<float>(best), st));
        return wrap({lp, entropy, ids, best});
    });
}

// the library's functions by address, what raises for a status, what gives the default context
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return entry(n, 10, [&] {
        void *at[8];
        for (int i = 0; i < 8; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) throw Refused();
        lib = {reinterpret_cast<decltype(lib.append)>(at[0]), reinterpret_cast<decltype(lib.scratch)>(at[1]), reinterpret_cast<decltype(lib.attn)>(at[2]),
               reinterpret_cast<decltype(lib.accept)>(at[3]), reinterpret_cast<decltype(lib.keep)>(at[4]), reinterpret_cast<decltype(lib.advance)>(at[5]),
               reinterpret_cast<decltype(lib.logprobs)>(at[6]), reinterpret_cast<decltype(lib.advance_path)>(at[7])};
        Py_XSETREF(g_check, Py_NewRef(a[8]));
        Py_XSETREF(g_context, Py_NewRef(a[9]));
        Py_RETURN_NONE;
    });
}

template <class F>
PyCFunction fast(F *f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},
                         {"rope_kv_append_tree", fast(rope_kv_append_tree), METH_FASTCALL, nullptr},
                         {"attn_tree", fast(attn_tree), METH_FASTCALL, nullptr},
                         {"tree_accept", fast(tree_accept), METH_FASTCALL, nullptr},
                         {"kv_keep_path", fast(kv_keep_path), METH_FASTCALL, nullptr},
                         {"advance_pos_by", fast(advance_pos_by), METH_FASTCALL, nullptr},
                         {"token_logprobs", fast(token_logprobs), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

// What this was compiled against (build.torch_ops_target): build.py looks for it in the file, ops.py in the module.
#ifndef LBK_TORCH_TARGET
#error "LBK_TORCH_TARGET says what this is compiled against"
#endif
const char target[] = LBK_TORCH_TARGET;

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() {
    g_handle = PyUnicode_InternFromString("handle");
    g_value = PyUnicode_InternFromString("value");
    g_device = PyUnicode_InternFromString("device");
    if (!g_handle || !g_value || !g_device) return nullptr;
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "target", target) < 0) Py_CLEAR(m);
    return m;
}
