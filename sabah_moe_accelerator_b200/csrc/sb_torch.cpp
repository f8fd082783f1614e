// The torch side of the operators around the experts: argument checks, outputs
// and the current stream, then one call of the C ABI. A call of these operators
// on few tokens takes the GPU a few microseconds, and checking a dozen tensors
// from Python takes longer than that (17-25 us a call, measured); from here it
// takes about one. Nothing is computed and nothing is kept between calls. The
// entry points come from the loaded libsabah_rt.so as addresses (bind), so the
// library itself stays free of torch.
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DispatchKeySet.h>

#include "../../include/sabah_rt.h"

namespace {

decltype(&sabah_qk_norm_rope) g_norm_rope;
decltype(&sabah_attend_paged) g_attend;
decltype(&sabah_attend_paged_workspace) g_workspace;
decltype(&sabah_route_topk) g_route;
decltype(&sabah_rt_last_error) g_last_error;
PyObject* g_error;   // rt.SabahCudaError

#define NEED(ok, what)                                \
    do {                                              \
        if (!(ok)) {                                  \
            PyErr_SetString(PyExc_ValueError, what);  \
            return nullptr;                           \
        }                                             \
    } while (0)

// A tensor that stands for others, or for one laid out otherwise. A mode that is
// active around the call (a counter of operations, say) does not make it one.
bool wrapper(const at::Tensor& t) {
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                        c10::DispatchKey::Batched});
    return t.key_set().has_any(keys) || t.layout() != at::kStrided || t.is_nested();
}

// The tensor behind an argument, which the caller holds during the call; an
// undefined one for None, null with the error for anything else. A wrapper (of
// vmap, a functional transform, a dispatching subclass) has no memory of its own;
// a tensor with the negative bit, a lazy zero or a freed storage has no memory that
// holds its values. Nothing here has a derivative, so whatever would lose one is
// refused too, a norm's weight or an output no less than the queries.
const at::Tensor* tensor(PyObject* o, const char* name, bool optional) {
    static const at::Tensor none;
    if (o == Py_None && optional) return &none;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s: a tensor%s, not %.100s", name, optional ? " or None" : "", Py_TYPE(o)->tp_name);
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (wrapper(t)) {
        PyErr_Format(PyExc_ValueError, "%s: a plain tensor (not inside vmap or another transform, no dispatching subclass)",
                     name);
        return nullptr;
    }
    if (t.is_neg() || t._is_zerotensor() || (t.numel() && t.is_cuda() && !t.data_ptr())) {
        PyErr_Format(PyExc_ValueError, "%s: its memory does not hold its values (a negative view, a lazy zero, a freed storage)", name);
        return nullptr;
    }
    if (t.requires_grad() && at::GradMode::is_enabled()) {
        PyErr_Format(PyExc_ValueError, "%s: this operator has no gradient (use torch.no_grad or detach)", name);
        return nullptr;
    }
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
        PyErr_Format(PyExc_ValueError, "%s: this operator has no forward gradient (unpack the dual tensor)", name);
        return nullptr;
    }
    return &t;
}
#define TENSOR(t, o, optional)                             \
    const at::Tensor* t##_arg = tensor(o, #t, optional);   \
    if (!t##_arg) return nullptr;                          \
    const at::Tensor& t = *t##_arg
// the same for an output, to be filled in where it is None
#define OUTPUT(t, o)                                   \
    const at::Tensor* t##_arg = tensor(o, #t, true);   \
    if (!t##_arg) return nullptr;                      \
    at::Tensor t = *t##_arg

int act_type(const at::Tensor& t) {   // ggml's codes
    switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 30;
    default: return -1;
    }
}
bool dense(const at::Tensor& t, at::ScalarType type, at::IntArrayRef sizes, const at::Tensor& like) {
    return t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous() && t.device() == like.device();
}
bool last_dense(const at::Tensor& t) { return t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1; }
bool here(const at::Tensor& t) { return t.is_cuda() && t.device().index() == c10::cuda::current_device(); }
// the current stream; the ABI reads 0 as its own stream, so the default one is passed as cudaStreamLegacy
void* stream() {
    void* s = c10::cuda::getCurrentCUDAStream().stream();
    return s ? s : (void*)1;
}
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);   // torch.empty without its dispatch
}
// The ABI's call without the lock. Its arguments are values, read before the lock
// is given up: reading a tensor may throw, and throws into Python.
template <class F, class... A>
int unlocked(F f, A... a) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(a...);
    Py_END_ALLOW_THREADS
    return rc;
}
bool failed(int rc, const char* what) {
    if (rc == 0) return false;
    PyErr_Format(g_error, "%s failed: %s", what, g_last_error());
    return true;
}

// byte strides of pages, rows and heads of a cache [pages, page_size, kv_heads, head_dim]
struct Cache {
    size_t page, row, head;
    explicit Cache(const at::Tensor& t)
        : page(t.size(0) > 1 ? 2 * t.stride(0) : 0), row(t.size(1) > 1 ? 2 * t.stride(1) : 0), head(t.size(2) > 1 ? 2 * t.stride(2) : 0) {}
};
const char* cache_fault(const at::Tensor& k, const at::Tensor& v, const at::Tensor& like) {
    if (k.dim() != 4 || k.sizes() != v.sizes()) return "caches: two of [pages, page_size, kv_heads, head_dim]";
    if (k.scalar_type() != v.scalar_type() || (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16))
        return "caches: f16 or bf16";
    if (k.device() != like.device() || v.device() != like.device()) return "caches: on the device of the other tensors";
    if (!last_dense(k) || !last_dense(v)) return "caches: head_dim must be dense";
    for (int i = 0; i < 4; ++i)
        if (k.size(i) > 0x7fffffff) return "caches: a dimension is too large";
    return nullptr;
}

// (q, k, v, q_weight, k_weight, table, positions, eps, pairs, pair_axis, k_cache, v_cache, slots, q_out, k_out)
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NEED(n == 15, "qk_norm_rope: 15 arguments");
    TENSOR(q, a[0], false);
    TENSOR(k, a[1], false);
    TENSOR(v, a[2], true);
    TENSOR(q_weight, a[3], true);
    TENSOR(k_weight, a[4], true);
    TENSOR(table, a[5], true);
    TENSOR(positions, a[6], true);
    const double eps = PyFloat_AsDouble(a[7]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const int pairs = PyObject_IsTrue(a[8]);
    if (pairs < 0) return nullptr;
    TENSOR(pair_axis, a[9], true);
    TENSOR(k_cache, a[10], true);
    TENSOR(v_cache, a[11], true);
    TENSOR(slots, a[12], true);
    OUTPUT(q_out, a[13]);
    OUTPUT(k_out, a[14]);
    const bool cache = a[12] != Py_None;

    NEED(q.dim() == 3 && k.dim() == 3, "q, k: [tokens, heads, head_dim]");
    const int64_t T = q.size(0), n_q = q.size(1), D = q.size(2), n_kv = k.size(1);
    NEED(k.size(0) == T && k.size(2) == D, "k: [tokens, kv_heads, head_dim] beside q");
    NEED(T <= 0x7fffffff && n_q <= 65536 && n_kv <= 65536 && D <= 65536, "q, k: a dimension is too large");
    const int act = act_type(q);
    NEED(act >= 0 && k.scalar_type() == q.scalar_type(), "q and k: both f32, f16 or bf16");
    NEED(here(q) && k.device() == q.device(), "q and k: on the current CUDA device");
    NEED(last_dense(q) && last_dense(k), "q and k: head_dim must be dense");
    const int64_t row[] = {D};
    NEED(!q_weight.defined() || dense(q_weight, at::kFloat, row, q), "q_weight: dense float32 [head_dim] or None");
    NEED(!k_weight.defined() || dense(k_weight, at::kFloat, row, q), "k_weight: dense float32 [head_dim] or None");
    int64_t n_pos = 0, rope = 0, axes = 0;
    if (table.defined()) {
        NEED(table.dim() == 3 && table.size(2) == 2 && table.size(0) <= 0x7fffffff && table.size(1) <= 65536 &&
             dense(table, at::kFloat, table.sizes(), q), "table: dense float32 [positions, rope_dim / 2, 2]");
        n_pos = table.size(0), rope = 2 * table.size(1);
        NEED(positions.defined() && (positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == T &&
             dense(positions, at::kInt, positions.sizes(), q), "positions: dense int32 [tokens] or [axes, tokens]");
        axes = positions.dim() == 2 ? positions.size(0) : 1;
        NEED(axes <= 65536, "positions: too many axes");
        const int64_t half[] = {rope / 2};
        NEED(!pair_axis.defined() || dense(pair_axis, at::kByte, half, q), "pair_axis: dense uint8 [rope_dim / 2] or None");
    }
    size_t eb = q.element_size(), vs[2] = {0, 0};
    Cache kc_at(q), vc_at(q);   // placeholders where there is no cache
    if (cache) {
        NEED(k_cache.defined() && v_cache.defined(), "cache: (k_cache, v_cache, slots)");
        if (const char* f = cache_fault(k_cache, v_cache, q)) {
            PyErr_SetString(PyExc_ValueError, f);
            return nullptr;
        }
        NEED(k_cache.size(2) == n_kv && k_cache.size(3) == D, "caches: kv_heads and head_dim as k's");
        NEED(v.defined() && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device() &&
             last_dense(v), "v: as k");
        const int64_t tokens[] = {T};
        NEED(dense(slots, at::kLong, tokens, q), "slots: dense int64 [tokens]");
        kc_at = Cache(k_cache), vc_at = Cache(v_cache);
        vs[0] = eb * v.stride(0), vs[1] = eb * v.stride(1);
    } else if (!k_out.defined()) {
        k_out = empty(k.sizes(), k.scalar_type(), k);
    }
    if (!q_out.defined()) q_out = empty(q.sizes(), q.scalar_type(), q);
    NEED(dense(q_out, q.scalar_type(), q.sizes(), q), "q_out: dense, as q");
    NEED(!k_out.defined() || dense(k_out, k.scalar_type(), k.sizes(), k), "k_out: dense, as k");
    auto ptr = [](const at::Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
    void* st = stream();
    const int rc = unlocked(
        g_norm_rope, ptr(q), eb * q.stride(0), eb * q.stride(1), (int)n_q, ptr(k), eb * k.stride(0), eb * k.stride(1),
        cache ? ptr(v) : nullptr, vs[0], vs[1], (int)n_kv, (int)T, (int)D, act, (const float*)ptr(q_weight),
        (const float*)ptr(k_weight), (float)eps, (const float*)ptr(table), (int)n_pos, (int)rope, pairs,
        table.defined() ? (const int32_t*)ptr(positions) : nullptr, (int)axes,
        table.defined() ? (const uint8_t*)ptr(pair_axis) : nullptr, ptr(q_out), ptr(k_out),
        cache ? ptr(k_cache) : nullptr, kc_at.page, kc_at.row, kc_at.head, cache ? ptr(v_cache) : nullptr,
        vc_at.page, vc_at.row, vc_at.head, cache ? (int)k_cache.size(0) : 0, cache ? (int)k_cache.size(1) : 0,
        cache ? act_type(k_cache) : 0, cache ? (const int64_t*)ptr(slots) : nullptr, st);
    if (failed(rc, "sabah_qk_norm_rope")) return nullptr;
    if (cache) return THPVariable_Wrap(q_out);
    PyObject *x = THPVariable_Wrap(q_out), *y = THPVariable_Wrap(k_out);
    PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
    END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, block_table, lens, scale or None, window, out, lse, workspace)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NEED(n == 10, "attend_paged: 10 arguments");
    TENSOR(q, a[0], false);
    TENSOR(k_cache, a[1], false);
    TENSOR(v_cache, a[2], false);
    TENSOR(block_table, a[3], false);
    TENSOR(lens, a[4], false);
    OUTPUT(out, a[7]);
    TENSOR(lse, a[8], true);
    OUTPUT(workspace, a[9]);
    const long window = PyLong_AsLong(a[6]);
    if (window == -1 && PyErr_Occurred()) return nullptr;

    NEED(q.dim() == 3, "q: [sequences, q_heads, head_dim]");
    const int64_t B = q.size(0), H = q.size(1), D = q.size(2);
    if (const char* f = cache_fault(k_cache, v_cache, q)) {
        PyErr_SetString(PyExc_ValueError, f);
        return nullptr;
    }
    const int64_t n_kv = k_cache.size(2);
    const int act = act_type(q);
    NEED(act == 0 || (act > 0 && q.scalar_type() == k_cache.scalar_type()), "q: f32 or the cache's type");
    NEED(k_cache.size(3) == D && n_kv > 0 && H % n_kv == 0, "q heads: a multiple of the cache's, of one head_dim");
    NEED(B <= 0x7fffffff && H <= 65536 && D <= 65536, "q: a dimension is too large");
    NEED(here(q), "q: on the current CUDA device");
    NEED(last_dense(q), "q: head_dim must be dense");
    NEED(block_table.dim() == 2 && block_table.size(0) == B && block_table.size(1) <= 0x7fffffff &&
         block_table.scalar_type() == at::kInt && last_dense(block_table) && block_table.device() == q.device(),
         "block_table: int32 [sequences, pages per sequence]");
    const int64_t seqs[] = {B}, rows[] = {B, H};
    NEED(dense(lens, at::kInt, seqs, q), "lens: dense int32 [sequences]");
    NEED(window >= 0 && window <= 0x7fffffff, "window: 0 (all keys) or a number of keys");
    double scale = 1.0 / std::sqrt((double)(D ? D : 1));
    if (a[5] != Py_None) {
        scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    }
    if (out.defined())
        NEED(dense(out, q.scalar_type(), q.sizes(), q), "out: dense, as q");
    else
        out = empty(q.sizes(), q.scalar_type(), q);
    NEED(!lse.defined() || dense(lse, at::kFloat, rows, q), "lse: dense float32 [sequences, q_heads]");
    if (workspace.defined())
        NEED(workspace.is_contiguous() && workspace.device() == q.device(), "workspace: dense, on q's device");
    else
        workspace = empty({(int64_t)g_workspace((int)H, (int)n_kv, (int)D)}, at::kByte, q);
    const Cache kc(k_cache), vc(v_cache);
    const size_t eb = q.element_size();
    void* st = stream();
    const int rc = unlocked(
        g_attend, q.data_ptr(), eb * q.stride(0), eb * q.stride(1), act, k_cache.data_ptr(), kc.page, kc.row, kc.head,
        v_cache.data_ptr(), vc.page, vc.row, vc.head, act_type(k_cache), (int)k_cache.size(0), (int)k_cache.size(1),
        (const int32_t*)block_table.data_ptr(), 4 * (size_t)block_table.stride(0), (int)block_table.size(1),
        (const int32_t*)lens.data_ptr(), (int)B, (int)H, (int)n_kv, (int)D, (float)scale, (int)window,
        out.data_ptr(), lse.defined() ? (float*)lse.data_ptr() : nullptr, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), st);
    if (failed(rc, "sabah_attend_paged")) return nullptr;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// (logits, n_used, renorm, scale, ids, w)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NEED(n == 6, "route_topk: 6 arguments");
    TENSOR(logits, a[0], false);
    const long used = PyLong_AsLong(a[1]);
    if (used == -1 && PyErr_Occurred()) return nullptr;
    const int renorm = PyObject_IsTrue(a[2]);
    if (renorm < 0) return nullptr;
    const double scale = PyFloat_AsDouble(a[3]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    OUTPUT(ids, a[4]);
    OUTPUT(w, a[5]);
    NEED(logits.dim() == 2, "logits: [tokens, experts]");
    const int64_t T = logits.size(0), E = logits.size(1), rows[] = {T, used};
    const int act = act_type(logits);
    NEED(act >= 0 && here(logits), "logits: f32, f16 or bf16 on the current CUDA device");
    NEED(last_dense(logits), "logits: experts must be dense");
    NEED(T <= 0x7fffffff && E <= 0x7fffffff && used > 0 && used <= E, "n_used: from 1 to the number of experts");
    if (!ids.defined()) ids = empty(rows, at::kInt, logits);
    if (!w.defined()) w = empty(rows, at::kFloat, logits);
    NEED(dense(ids, at::kInt, rows, logits) && dense(w, at::kFloat, rows, logits),
         "ids and w: dense int32 and float32 [tokens, n_used]");
    void* st = stream();
    const int rc = unlocked(g_route, logits.data_ptr(), logits.element_size() * logits.stride(0), act, (int)T, (int)E,
                            (int)used, renorm, (float)scale, (int32_t*)ids.data_ptr(), (float*)w.data_ptr(), st);
    if (failed(rc, "sabah_route_topk")) return nullptr;
    PyObject *x = THPVariable_Wrap(ids), *y = THPVariable_Wrap(w);
    PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
    END_HANDLE_TH_ERRORS
}

// (norm_rope, attend, workspace, route, last_error) addresses, error class
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long f[5];
    PyObject* error;
    if (!PyArg_ParseTuple(args, "KKKKKO", f, f + 1, f + 2, f + 3, f + 4, &error)) return nullptr;
    g_norm_rope = (decltype(g_norm_rope))f[0];
    g_attend = (decltype(g_attend))f[1];
    g_workspace = (decltype(g_workspace))f[2];
    g_route = (decltype(g_route))f[3];
    g_last_error = (decltype(g_last_error))f[4];
    Py_INCREF(error);
    Py_XDECREF(g_error);
    g_error = error;
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"bind", bind, METH_VARARGS, nullptr},
                          {"norm_rope", (PyCFunction)(void*)norm_rope, METH_FASTCALL, nullptr},
                          {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, nullptr},
                          {"route", (PyCFunction)(void*)route, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__torch_ops() { return PyModule_Create(&kModule); }
