// vox_ops_call.cpp — the calls of voxtral_c_amd/ops.py on torch tensors, compiled: a short kernel's call is bound by the host, and most of that was the
// interpreter (a call of a few tensors: attribute lookups, shape comparisons, argument conversions).  Measured, by ctypes / here: plan + accept + commit 31 / 16 us, scores
// of one row 18.8 / 12.3, linear_i8 1 x 1280 x 6144 9.7 / 5.8, attention of 2 nodes 17 / 14.4 (now its kernels').  Bound by the launches, 3.2 us each.
//
// Each function takes the arguments of its namesake in ops.py, checks that they are what it takes without further ado, allocates results
// and scratch memory from torch's allocator and calls the C entry (include/vox_hip_ops.h).  Anything else (a wrong shape, a table that is not contiguous, a tensor
// that needs gradients or has a tangent, an error of the C entry) gives None: ops.py then does the same call itself and says what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "../../include/vox_hip_ops.h"

namespace {

// The C entries' addresses, in the library that the package has loaded, and torch's function from a device to its current stream.
struct Entries {
    decltype(&vox_hip_tree_plan) tree_plan;
    decltype(&vox_hip_tree_attention_workspace) attention_workspace;
    decltype(&vox_hip_tree_attention) attention;
    decltype(&vox_hip_tree_accept) tree_accept;
    decltype(&vox_hip_tree_commit) tree_commit;
    decltype(&vox_hip_token_scores_workspace) scores_workspace;
    decltype(&vox_hip_token_scores) scores;
    decltype(&vox_hip_quantize_rows_i8) quantize;
    decltype(&vox_hip_linear_i8_workspace) i8_workspace;
    decltype(&vox_hip_linear_i8) i8;
} entry;
PyObject *current_stream = nullptr;

typedef const at::Tensor &Arg;
bool is_tensor(PyObject *o) { return THPVariable_CheckExact(o); }
Arg tensor(PyObject *o) { return THPVariable_Unpack(o); }
bool all_tensors(PyObject *const *args, int n) {
    for (int i = 0; i < n; i++)
        if (!is_tensor(args[i])) return false;
    return true;
}

// What one call's tensors have in common: a GPU, and the floating type of those that have one.
struct Call {
    int device = -1, dtype = -1;
    at::ScalarType type = at::ScalarType::Undefined;
    const bool grad = c10::AutogradState::get_tls_state().get_grad_mode(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    bool ok = true;
    bool plain(Arg t) const { return !(grad && t.requires_grad()) && !(forward && t._fw_grad(0).defined()); }      // no derivative is wanted
    bool here(Arg t) {
        if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg()) return ok = false;
        if (device < 0) device = t.get_device();
        return ok = ok && t.get_device() == device;
    }
    void table(Arg t, at::IntArrayRef shape, at::ScalarType want = at::kInt) {
        ok = ok && here(t) && t.scalar_type() == want && t.sizes() == shape && t.is_contiguous() && plain(t);
    }
    void floats(Arg t, at::IntArrayRef shape) {
        if (!ok || !here(t)) return;
        const at::ScalarType s = t.scalar_type();
        if (dtype < 0) {
            type = s;
            dtype = s == at::kFloat ? VOX_F32 : s == at::kBFloat16 ? VOX_BF16 : VOX_F16;
            ok = s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
        }
        ok = ok && s == type && t.sizes() == shape && (t.stride(-1) == 1 || t.size(-1) <= 1) && plain(t);
    }
    void *stream() {
        PyObject *d = PyLong_FromLong(device);
        PyObject *s = d ? PyObject_CallOneArg(current_stream, d) : nullptr;
        Py_XDECREF(d);
        if (!s) throw python_error();
        void *p = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        if (!p && PyErr_Occurred()) throw python_error();
        return p;
    }
    at::Tensor make(at::IntArrayRef shape, at::ScalarType t) const { return at::empty(shape, at::TensorOptions().dtype(t).device(at::kCUDA, (c10::DeviceIndex)device)); }
};
at::Tensor scratch(const Call &c, int64_t bytes) { return bytes > 0 ? c.make({bytes}, at::kByte) : at::Tensor(); }
void *ptr(Arg t) { return t.defined() ? t.data_ptr() : nullptr; }
int32_t *ints(Arg t) { return (int32_t *)ptr(t); }
float *f32s(Arg t) { return (float *)ptr(t); }
PyObject *tuple(std::initializer_list<at::Tensor> list) {
    PyObject *r = PyTuple_New((Py_ssize_t)list.size());
    if (!r) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor &t : list) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    return r;
}
// A whole number of `lo` to `hi`; Python's own int only.
bool whole(PyObject *o, int64_t lo, int64_t hi, int64_t *v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &over);
    return !over && *v >= lo && *v <= hi;
}

#define BEGIN(n, tensors) HANDLE_TH_ERRORS if (!current_stream || count != (n) || !all_tensors(args, tensors)) Py_RETURN_NONE; Call c;
#define END END_HANDLE_TH_ERRORS
#define OR_NONE(cond) do { if (!(cond)) Py_RETURN_NONE; } while (0)

// parents, n_nodes or None
PyObject *tree_plan(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(2, 1)
    Arg parents = tensor(args[0]);
    OR_NONE(parents.dim() == 2 && parents.size(1) <= VOX_TREE_MAX_NODES && parents.size(0) <= INT_MAX);
    const int64_t B = parents.size(0), T = parents.size(1);
    c.table(parents, {B, T});
    const int32_t *n = nullptr;
    if (args[1] != Py_None) {
        OR_NONE(is_tensor(args[1]));
        c.table(tensor(args[1]), {B});
        n = c.ok ? ints(tensor(args[1])) : nullptr;
    }
    OR_NONE(c.ok);
    at::Tensor ancestors = c.make({B, T, (T + 63) / 64}, at::kLong), depth = c.make({B, T}, at::kInt);
    OR_NONE(entry.tree_plan(ints(parents), n, (int)B, (int)T, (uint64_t *)ptr(ancestors), ints(depth), c.device, c.stream()) == 0);
    return tuple({ancestors, depth});
    END
}

// q, k, v, k_cache, v_cache, cache_len, ancestors, depth, scale or None, window, return_lse
PyObject *tree_attention(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(11, 8)
    Arg q = tensor(args[0]), k = tensor(args[1]), v = tensor(args[2]), kc = tensor(args[3]), vc = tensor(args[4]);
    int64_t window;
    OR_NONE(q.dim() == 4 && k.dim() == 4 && kc.dim() == 4 && whole(args[9], INT_MIN, INT_MAX, &window) && PyBool_Check(args[10]));
    OR_NONE(args[8] == Py_None || PyFloat_CheckExact(args[8]));
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), cap = kc.size(1), Hk = k.size(2);
    OR_NONE(T <= VOX_TREE_MAX_NODES && Hk >= 1 && H <= 4096 && D >= 1 && D <= 256 && cap >= 1 && cap <= INT_MAX && B <= 65535 && H % Hk == 0);
    c.floats(q, {B, T, H, D});
    c.floats(k, {B, T, Hk, D});
    c.floats(v, {B, T, Hk, D});
    c.floats(kc, {B, cap, Hk, D});
    c.floats(vc, {B, cap, Hk, D});
    c.table(tensor(args[5]), {B});
    c.table(tensor(args[6]), {B, T, (T + 63) / 64}, at::kLong);
    c.table(tensor(args[7]), {B, T});
    OR_NONE(c.ok);
    const double scale = args[8] == Py_None ? std::pow((double)D, -0.5) : PyFloat_AS_DOUBLE(args[8]);
    OR_NONE(std::fabs(scale) <= 3e38);
    at::Tensor out = c.make({B, T, H, D}, c.type), lse;
    if (args[10] == Py_True) lse = c.make({B, T, H}, at::kFloat);
    vox_hip_tree_attn_t a{ptr(q), ptr(k), ptr(v), ptr(kc), ptr(vc), ints(tensor(args[5])), (const uint64_t *)ptr(tensor(args[6])), ints(tensor(args[7])), ptr(out), f32s(lse)};
    int64_t *st = &a.q_sb;
    for (const at::Tensor *t : {&q, &k, &v, &kc, &vc, (const at::Tensor *)&out})
        for (int i = 0; i < 3; i++) *st++ = t->stride(i);
    a.dtype = c.dtype; a.batch = (int)B; a.nodes = (int)T; a.heads = (int)H; a.kv_heads = (int)Hk; a.head_dim = (int)D; a.cap = (int)cap;
    a.window = (int)std::max<int64_t>(window, -1);
    a.scale = (float)scale;
    a.reserved = 0;
    const int64_t need = entry.attention_workspace(&a);
    OR_NONE(need >= 0);
    const at::Tensor ws = scratch(c, need);
    OR_NONE(entry.attention(&a, ptr(ws), (size_t)need, c.device, c.stream()) == 0);
    if (!lse.defined()) return THPVariable_Wrap(out);
    return tuple({out, lse});
    END
}

// tokens, choices, root_choice, parents, ancestors, depth, cache_len
PyObject *tree_accept(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(7, 7)
    Arg tokens = tensor(args[0]);
    OR_NONE(tokens.dim() == 2 && tokens.size(1) >= 1 && tokens.size(1) <= VOX_TREE_MAX_NODES && tokens.size(0) <= INT_MAX);
    const int64_t B = tokens.size(0), T = tokens.size(1);
    for (int i : {0, 1, 3, 5}) c.table(tensor(args[i]), {B, T});
    for (int i : {2, 6}) c.table(tensor(args[i]), {B});
    c.table(tensor(args[4]), {B, T, (T + 63) / 64}, at::kLong);
    OR_NONE(c.ok);
    at::Tensor path = c.make({B, T}, at::kInt), n = c.make({B}, at::kInt), after = c.make({B}, at::kInt), length = c.make({B}, at::kInt);
    OR_NONE(entry.tree_accept(ints(tokens), ints(tensor(args[1])), ints(tensor(args[2])), ints(tensor(args[3])), (const uint64_t *)ptr(tensor(args[4])),
                              ints(tensor(args[5])), ints(tensor(args[6])), (int)B, (int)T, ints(path), ints(n), ints(after), ints(length), c.device, c.stream()) == 0);
    return tuple({path, n, after, length});
    END
}

// k, v, k_cache, v_cache (all with layers), path, n_accepted, cache_len -> True
PyObject *tree_commit(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(7, 7)
    Arg k = tensor(args[0]), kc = tensor(args[2]);
    OR_NONE(k.dim() == 5 && kc.dim() == 5);
    const int64_t L = k.size(0), B = k.size(1), T = k.size(2), Hk = k.size(3), D = k.size(4), cap = kc.size(2);
    OR_NONE(L <= INT_MAX && B <= INT_MAX && T <= VOX_TREE_MAX_NODES && Hk <= INT_MAX && D <= INT_MAX && cap >= T && cap <= INT_MAX);
    int64_t st[4][4];
    for (int i = 0; i < 4; i++) {
        Arg t = tensor(args[i]);
        if (i < 2) c.floats(t, {L, B, T, Hk, D});
        else c.floats(t, {L, B, cap, Hk, D});
        OR_NONE(c.ok);
        for (int j = 0; j < 5; j++) OR_NONE(i < 2 || t.size(j) <= 1 || t.stride(j) != 0);
        for (int j = 0; j < 4; j++) st[i][j] = t.stride(j);
    }
    c.table(tensor(args[4]), {B, T});
    c.table(tensor(args[5]), {B});
    c.table(tensor(args[6]), {B});
    OR_NONE(c.ok);
    OR_NONE(entry.tree_commit(c.dtype, (int)L, (int)B, (int)T, (int)Hk, (int)D, (int)cap, ptr(k), st[0], ptr(tensor(args[1])), st[1], ptr(kc), st[2], ptr(tensor(args[3])), st[3],
                              ints(tensor(args[4])), ints(tensor(args[5])), ints(tensor(args[6])), c.device, c.stream()) == 0);
    for (int i : {2, 3})                                     // what autograd has saved of them is theirs no longer
        if (!tensor(args[i]).is_inference()) tensor(args[i]).unsafeGetTensorImpl()->bump_version();
    Py_RETURN_TRUE;
    END
}

// logits, tokens or None, top
PyObject *token_scores(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(3, 1)
    Arg logits = tensor(args[0]);
    int64_t top, given = 0;
    OR_NONE(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= INT_MAX);
    const int64_t R = logits.size(0), V = logits.size(1);
    OR_NONE(whole(args[2], 0, std::min<int64_t>(VOX_SCORES_MAX_TOP, V), &top));
    c.floats(logits, {R, V});
    const int32_t *tokens = nullptr;
    bool flat = false;
    if (args[1] != Py_None) {
        OR_NONE(is_tensor(args[1]));
        Arg t = tensor(args[1]);
        flat = t.dim() == 1;
        OR_NONE(flat || t.dim() == 2);
        given = flat ? 1 : t.size(1);
        if (flat) c.table(t, {R});
        else c.table(t, {R, given});
        OR_NONE(c.ok && given <= INT_MAX);
        tokens = ints(t);
    }
    OR_NONE(c.ok);
    const int64_t need = entry.scores_workspace(c.dtype, R, (int)V, (int)top);
    OR_NONE(need >= 0);
    at::Tensor logprob = flat ? c.make({R}, at::kFloat) : c.make({R, given}, at::kFloat), entropy = c.make({R}, at::kFloat), lse = c.make({R}, at::kFloat);
    at::Tensor index = c.make({R, top}, at::kInt), best = c.make({R, top}, at::kFloat);
    const at::Tensor ws = scratch(c, need);
    OR_NONE(entry.scores(c.dtype, ptr(logits), logits.stride(0), R, (int)V, tokens, (int)given, (int)top, f32s(logprob), f32s(entropy), f32s(lse), ints(index), f32s(best),
                         ptr(ws), (size_t)need, c.device, c.stream()) == 0);
    return tuple({logprob, entropy, lse, index, best});
    END
}

// x
PyObject *quantize_rows_i8(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(1, 1)
    Arg x = tensor(args[0]);
    OR_NONE(x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= VOX_I8_MAX_K);
    const int64_t M = x.size(0), K = x.size(1);
    c.floats(x, {M, K});
    OR_NONE(c.ok);
    at::Tensor q = c.make({M, K}, at::kChar), scale = c.make({M}, at::kFloat);
    OR_NONE(entry.quantize(c.dtype, ptr(x), x.stride(0), M, (int)K, (int8_t *)ptr(q), f32s(scale), c.device, c.stream()) == 0);
    return tuple({q, scale});
    END
}

// x, w, w_scale, bias or None
PyObject *linear_i8(PyObject *, PyObject *const *args, Py_ssize_t count) {
    BEGIN(4, 3)
    Arg x = tensor(args[0]), w = tensor(args[1]);
    OR_NONE(x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= VOX_I8_MAX_K && w.dim() == 2 && w.size(0) <= INT_MAX);
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    c.floats(x, {M, K});
    OR_NONE(c.ok && c.here(w) && w.scalar_type() == at::kChar && w.size(1) == K && (w.stride(1) == 1 || K == 1));
    c.table(tensor(args[2]), {N}, at::kFloat);
    const void *bias = nullptr;
    if (args[3] != Py_None) {
        OR_NONE(is_tensor(args[3]) && tensor(args[3]).dim() == 1);
        c.floats(tensor(args[3]), {N});
        bias = c.ok ? ptr(tensor(args[3])) : nullptr;
    }
    OR_NONE(c.ok);
    const int8_t *wp = (const int8_t *)ptr(w);
    const int64_t need = entry.i8_workspace(c.dtype, M, (int)K, (int)N, wp, w.stride(0));
    OR_NONE(need >= 0);
    at::Tensor y = c.make({M, N}, c.type);
    const at::Tensor ws = scratch(c, need);
    OR_NONE(entry.i8(c.dtype, ptr(x), x.stride(0), M, (int)K, (int)N, wp, w.stride(0), f32s(tensor(args[2])), bias, ptr(y), N, ptr(ws), (size_t)need, c.device, c.stream()) == 0);
    return THPVariable_Wrap(y);
    END
}

// current stream function, then the addresses in the order of Entries
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t count) {
    constexpr int N = sizeof(Entries) / sizeof(void *);
    if (count != N + 1) return PyErr_Format(PyExc_TypeError, "bind: %d arguments are needed", N + 1);
    void *p[N];
    for (int i = 0; i < N; i++) {
        p[i] = PyLong_AsVoidPtr(args[i + 1]);
        if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "bind: no address");
    }
    memcpy(&entry, p, sizeof entry);
    Py_INCREF(args[0]);
    Py_XDECREF(current_stream);
    current_stream = args[0];
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(tree_plan), METHOD(tree_attention), METHOD(tree_accept), METHOD(tree_commit), METHOD(token_scores), METHOD(quantize_rows_i8),
                         METHOD(linear_i8), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_call(void) { return PyModule_Create(&module); }
