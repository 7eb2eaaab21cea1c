// python_calls.cpp -- the Python side of the C ABI as native functions: tensors in, device pointers and torch's current
// stream out.
//
// What bounds a small call is the host: a decoded token's attention step is 48 launches, and a ctypes call that checks
// five tensors and asks torch for the stream costs 6 - 8 us of interpreter work before the launch (2 us) begins.  Here
// the checks and the stream are a few loads each (0.3 us).
//
// The library itself is not linked: bind() takes the addresses that the loaded library exports, so that one build of
// this module serves any build of the library.
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/bonsai_b200_ext.h"

namespace {

constexpr int64_t PAGE_ROW = 256;           // values of a paged cache's row

// Kinds of argument beside plain numbers: device memory (a CUDA tensor or None), a handle (an integer or an object with
// an integer `value`, as ctypes makes them), a truth value.
struct Mem { void *p; };
// Device memory of the current device, of values of a type (Undefined: bytes, of whatever type the tensor is), and how many there are (-1: None, or an object that does not say).
template <at::ScalarType T> struct Dev { void *p; int64_t n; };
template <at::ScalarType T> struct Strided { void *p; int64_t n; };     // ... whose strides are arguments of the call, so that it need not be contiguous
using Floats = Dev<at::kFloat>;
using Doubles = Dev<at::kDouble>;
using Int32s = Dev<at::kInt>;
using Bytes = Dev<at::ScalarType::Undefined>;
struct Ints { const void *p; int64_t n; };      // host memory: an int32 tensor
struct Handle { void *p; };
struct Truth { int v; };

// An object that is no torch tensor but has a tensor's is_cuda, is_contiguous() and data_ptr().
bool get_like_tensor(PyObject *o, const char *name, Mem &out) {
    auto truth = [](PyObject *v) {
        const int t = v ? PyObject_IsTrue(v) : -1;
        Py_XDECREF(v);
        return t;
    };
    const int cuda = truth(PyObject_GetAttrString(o, "is_cuda"));
    if (cuda < 0) return false;
    if (!cuda) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor: this library has no CPU path", name);
        return false;
    }
    const int contiguous = truth(PyObject_CallMethod(o, "is_contiguous", nullptr));
    if (contiguous < 0) return false;
    if (!contiguous) {
        PyErr_Format(PyExc_RuntimeError, "%s must be contiguous", name);
        return false;
    }
    PyObject *p = PyObject_CallMethod(o, "data_ptr", nullptr);
    if (!p) return false;
    out.p = PyLong_AsVoidPtr(p);
    Py_DECREF(p);
    return !PyErr_Occurred();
}

bool get(PyObject *o, const char *name, Mem &out) {
    if (o == Py_None) {
        out.p = nullptr;
        return true;
    }
    if (!THPVariable_Check(o)) return get_like_tensor(o, name, out);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor: this library has no CPU path", name);
        return false;
    }
    if (!t.is_contiguous()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be contiguous", name);
        return false;
    }
    out.p = t.mutable_data_ptr();           // outputs are written: a tensor that shares its memory until then gets its own, as by data_ptr()
    return true;
}
bool here(PyObject *o, const char *name) {
    if (o == Py_None || !THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) return true;
    const int at = (int)THPVariable_Unpack(o).get_device(), now = (int)c10::cuda::current_device();
    if (at != now) PyErr_Format(PyExc_RuntimeError, "%s is on device %d, the current device is %d", name, at, now);
    return at == now;
}
// A tensor's type is the one that the call reads it as.  (An object like a tensor says nothing of it.)
bool of_type(PyObject *o, const char *name, at::ScalarType type) {
    if (type == at::ScalarType::Undefined || !THPVariable_Check(o) || THPVariable_Unpack(o).scalar_type() == type) return true;
    PyErr_Format(PyExc_RuntimeError, "%s must be a tensor of %s, not of %s", name, c10::toString(type), c10::toString(THPVariable_Unpack(o).scalar_type()));
    return false;
}
template <at::ScalarType T> bool get(PyObject *o, const char *name, Dev<T> &out) {
    Mem m{};
    if (!of_type(o, name, T) || !here(o, name) || !get(o, name, m)) return false;
    out.p = m.p;
    out.n = !THPVariable_Check(o) ? -1 : T == at::ScalarType::Undefined ? (int64_t)THPVariable_Unpack(o).nbytes() : THPVariable_Unpack(o).numel();
    return true;
}
template <at::ScalarType T> bool get(PyObject *o, const char *name, Strided<T> &out) {
    if (!THPVariable_Check(o)) {
        Mem m{};
        if (!get(o, name, m)) return false;
        out.p = m.p;
        out.n = -1;
        return true;
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!of_type(o, name, T)) return false;
    if (!t.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor: this library has no CPU path", name);
        return false;
    }
    if (!here(o, name)) return false;
    out.p = t.mutable_data_ptr();
    out.n = (int64_t)(t.storage().nbytes() / t.element_size()) - t.storage_offset();       // to the end of its memory
    return true;
}
bool get(PyObject *o, const char *name, Ints &out) {
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cpu() || THPVariable_Unpack(o).scalar_type() != at::kInt || !THPVariable_Unpack(o).is_contiguous()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a contiguous int32 tensor in host memory", name);
        return false;
    }
    out.p = THPVariable_Unpack(o).data_ptr();
    out.n = THPVariable_Unpack(o).numel();
    return true;
}
bool get(PyObject *o, const char *, Handle &out) {
    if (o == Py_None) {
        out.p = nullptr;
        return true;
    }
    if (PyLong_Check(o)) {
        out.p = PyLong_AsVoidPtr(o);
        return !PyErr_Occurred();
    }
    PyObject *v = PyObject_GetAttrString(o, "value");
    if (!v) return false;
    out.p = v == Py_None ? nullptr : PyLong_AsVoidPtr(v);
    Py_DECREF(v);
    return !PyErr_Occurred();
}
bool get(PyObject *o, const char *, Truth &out) {
    out.v = PyObject_IsTrue(o);
    return out.v >= 0;
}
bool get(PyObject *o, const char *, int64_t &out) {
    out = PyLong_AsLongLong(o);
    return !(out == -1 && PyErr_Occurred());
}
bool get(PyObject *o, const char *name, int &out) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v != (long)(int)v) {
        PyErr_Format(PyExc_OverflowError, "%s does not fit an int", name);
        return false;
    }
    out = (int)v;
    return true;
}
bool get(PyObject *o, const char *, float &out) {
    const double v = PyFloat_AsDouble(o);
    out = (float)v;
    return !(v == -1.0 && PyErr_Occurred());
}

void *raw(Mem m) { return m.p; }
template <at::ScalarType T> void *raw(Dev<T> m) { return m.p; }
template <at::ScalarType T> void *raw(Strided<T> m) { return m.p; }
const void *raw(Ints m) { return m.p; }
void *raw(Handle h) { return h.p; }
int raw(Truth t) { return t.v; }
template <typename T> T raw(T v) { return v; }
template <typename T> using Raw = decltype(raw(std::declval<T>()));

constexpr int MAX_ARGS = 20;

// Host lists are as long as the call's last argument says.
template <typename T> bool long_enough(const T &, int64_t) { return true; }
inline bool long_enough(const Ints &v, int64_t n) { return v.n >= n; }

// Whether there are as many values as the sizes beside them say: the product of them.  Sizes that are no sizes are the library's to refuse.
template <typename M> bool holds(const M &m, std::initializer_list<int64_t> sizes) {
    unsigned __int128 all = 1;
    for (int64_t x : sizes) {
        if (x <= 0) return true;
        all *= (unsigned __int128)x;
        if (all > (unsigned __int128)INT64_MAX) all = (unsigned __int128)INT64_MAX + 1;         // (no tensor has them)
    }
    return m.n < 0 || all <= (unsigned __int128)m.n;
}

// One exported function: its address, filled in by bind(), the names of its arguments, and where the call has sizes what finds the tensor that is too small for them (its place, -1: none).
template <typename... A>
struct Call {
    using Fn = int (*)(Raw<A>..., void *);
    static constexpr int N = sizeof...(A);
    const char *name;
    const char *args[N];
    int (*small)(const std::tuple<A...> &) = nullptr;
    Fn fn = nullptr;

    template <size_t... I>
    PyObject *go(PyObject *const *v, std::index_sequence<I...>) {
        std::tuple<A...> a{};
        if (!(get(v[I], args[I], std::get<I>(a)) && ...)) return nullptr;
        if constexpr ((std::is_same_v<A, Ints> || ...)) {
            if (!(long_enough(std::get<I>(a), std::get<N - 1>(a)) && ...)) {
                PyErr_Format(PyExc_RuntimeError, "%s: a list is shorter than %s", name, args[N - 1]);
                return nullptr;
            }
        }
        if (const int at = small ? small(a) : -1; at >= 0) {
            PyErr_Format(PyExc_RuntimeError, "%s: %s is smaller than the sizes beside it say", name, args[at]);
            return nullptr;
        }
        void *stream = c10::cuda::getCurrentCUDAStream().stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = fn(raw(std::get<I>(a))..., stream);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(rc);
    }

    PyObject *call(PyObject *const *v, Py_ssize_t n, PyObject *kw) {
        static_assert(N <= MAX_ARGS, "");
        PyObject *all[MAX_ARGS];
        if (!fn) {
            PyErr_Format(PyExc_RuntimeError, "%s is not bound to a library", name);
            return nullptr;
        }
        if (kw || n != N) {          // named arguments: put them in their places
            const Py_ssize_t nk = kw ? PyTuple_GET_SIZE(kw) : 0;
            if (n + nk != N) {
                PyErr_Format(PyExc_TypeError, "%s() takes %d arguments, got %zd", name, N, n + nk);
                return nullptr;
            }
            for (int i = 0; i < N; ++i) all[i] = i < n ? v[i] : nullptr;
            for (Py_ssize_t k = 0; k < nk; ++k) {
                const char *s = PyUnicode_AsUTF8(PyTuple_GET_ITEM(kw, k));
                if (!s) return nullptr;
                int at = 0;
                while (at < N && std::strcmp(s, args[at])) ++at;
                if (at == N || all[at]) {
                    PyErr_Format(PyExc_TypeError, "%s() got an unexpected or repeated argument '%s'", name, s);
                    return nullptr;
                }
                all[at] = v[n + k];
            }
            v = all;
        }
        try {
            return go(v, std::make_index_sequence<N>{});
        } catch (const std::exception &e) {
            PyErr_SetString(PyExc_RuntimeError, e.what());
            return nullptr;
        }
    }
};

// include/bonsai_p40.h
Call<Mem, Mem, Mem, int64_t, int64_t> gemv{"gemv", {"W", "xq", "y", "n_out", "n_in"}};
Call<Mem, Mem, int64_t> quant_activations{"quant_activations", {"x", "out", "n"}};
Call<Mem, Mem, Mem, int64_t, int64_t, int64_t> gemm{"gemm", {"W", "Xq", "Y", "n_out", "n_in", "n_tok"}};
Call<Mem, Mem, int64_t, int64_t> repack{"repack", {"src", "dst", "n_out", "n_in"}};
Call<Mem, Mem, Mem, int64_t, int64_t> gemv_repack{"gemv_repack", {"W", "x", "y", "n_out", "n_in"}};
Call<Mem, Mem, int64_t> fwht{"fwht", {"x", "signs", "n"}};
Call<Mem, Mem, Mem, int64_t, int64_t, float> rmsnorm{"rmsnorm", {"x", "w", "y", "n_rows", "n", "eps"}};
Call<Mem, Mem, Mem, Mem, Mem, Mem, Mem, int, int, int, int> gdn_step{
    "gdn_step", {"state", "q", "k", "v", "g", "beta", "out", "n_k_heads", "n_v_heads", "K", "V"}};
Call<Mem, Mem, Mem, Mem, int, int, int, int, float> attn{
    "attn", {"q", "k", "v", "out", "n_tok", "n_head", "n_head_kv", "head_dim", "scale"}};
// include/bonsai_b200_ext.h
Call<Mem, Mem, Mem, Mem, int64_t> fwht_quant{"fwht_quant", {"x", "signs", "xq", "x_rot", "n"}};
Call<Mem, Mem, Mem, int64_t> swiglu{"swiglu", {"gate", "up", "y", "n"}};
Call<Mem, Mem, Mem, int64_t, int64_t, Truth> quant_batch{"quant_batch", {"X", "signs", "Xq", "n_in", "n_tok", "rotate"}};
Call<Mem, Mem, Mem, Mem, Mem, int64_t, int64_t> linear{"linear", {"W", "x", "signs", "y", "xq_scratch", "n_out", "n_in"}};
Call<Mem, Mem, Mem, Mem, int64_t, int64_t> linear_static{"linear_static", {"W", "x", "signs", "y", "n_out", "n_in"}};
Call<Handle> chain_run{"chain_run", {"chain"}};
Call<Strided<at::kFloat>, Strided<at::kFloat>, Floats, Floats, Int32s, Doubles, Floats, Floats, int64_t, int, int, int, int, int64_t, int64_t, int64_t, int64_t, float> qk_norm_rope{
    "qk_norm_rope", {"q", "k", "q_weight", "k_weight", "pos", "freq", "q_out", "k_out", "n_tok", "n_head", "n_head_kv", "head_dim", "n_rot", "q_tok_stride",
                     "q_head_stride", "k_tok_stride", "k_head_stride", "eps"},
    [](const auto &a) {
        const auto &[q, k, q_weight, k_weight, pos, freq, q_out, k_out, n_tok, n_head, n_head_kv, head_dim, n_rot, qt, qh, kt, kh, eps] = a;
        // from the first row's begin to the last one's end; a stride of one row is not used
        auto spans = [&](const auto &x, int64_t heads, int64_t tok_stride, int64_t head_stride) {
            const __int128 last = (__int128)(n_tok - 1) * (n_tok > 1 ? tok_stride : 0) + (__int128)(heads - 1) * (heads > 1 ? head_stride : 0) + head_dim;
            return n_tok <= 0 || heads <= 0 || head_dim <= 0 || x.n < 0 || last <= x.n;
        };
        if (n_tok <= 0 || (n_head <= 0 && n_head_kv <= 0)) return -1;
        if (!spans(q, n_head, qt, qh)) return 0;
        if (!spans(k, n_head_kv, kt, kh)) return 1;
        if (n_head > 0 && !holds(q_weight, {head_dim})) return 2;
        if (n_head_kv > 0 && !holds(k_weight, {head_dim})) return 3;
        if (n_rot > 0 && !holds(pos, {n_tok})) return 4;
        if (!holds(freq, {n_rot / 2})) return 5;
        if (!holds(q_out, {n_tok, n_head, head_dim})) return 6;
        return holds(k_out, {n_tok, n_head_kv, head_dim}) ? -1 : 7;
    }};
// (the struct's own memory is Pages.__init__'s to look at)
Call<Handle, int, Floats, Floats> pages_append{"pages_append", {"pages", "layer", "k", "v"}, [](const auto &a) {
        const auto &[pages, layer, k, v] = a;
        const auto *p = static_cast<const bonsai_b200_pages *>(pages.p);
        if (!p || p->n_seq <= 0) return -1;
        if (!holds(k, {p->n_tok, p->n_head_kv, PAGE_ROW})) return 2;
        return holds(v, {p->n_tok, p->n_head_kv, PAGE_ROW}) ? -1 : 3;
    }};
Call<Handle, int, Floats, Floats, int, int, Bytes, int64_t, float> pages_attn{
    "pages_attn", {"pages", "layer", "q", "out", "n_head", "max_len", "workspace", "workspace_bytes", "scale"},
    [](const auto &a) {
        const auto &[pages, layer, q, out, n_head, max_len, workspace, workspace_bytes, scale] = a;
        const auto *p = static_cast<const bonsai_b200_pages *>(pages.p);
        if (!p || p->n_seq <= 0) return -1;
        if (!holds(q, {p->n_tok, n_head, PAGE_ROW})) return 2;
        if (!holds(out, {p->n_tok, n_head, PAGE_ROW})) return 3;
        return holds(workspace, {workspace_bytes}) ? -1 : 6;
    }};
Call<Bytes, int64_t, int, Ints, Ints, int> pages_copy{"pages_copy", {"pool", "page_bytes", "n_pages", "src", "dst", "n"}, [](const auto &a) {
        return std::get<5>(a) <= 0 || holds(std::get<0>(a), {std::get<1>(a), std::get<2>(a)}) ? -1 : 0;
    }};
Call<Floats, Floats, Floats, Floats, Floats, Floats, Floats, Int32s, Int32s, Bytes, int64_t, int, int, int, int, int, int, int> gdn_seqs{
    "gdn_seqs", {"state", "q", "k", "v", "g", "beta", "out", "start", "slot", "workspace", "workspace_bytes", "n_seq", "n_slots", "n_tok", "n_k_heads",
                 "n_v_heads", "K", "V"},
    [](const auto &a) {
        const auto &[state, q, k, v, g, beta, out, start, slot, workspace, workspace_bytes, n_seq, n_slots, n_tok, n_k_heads, n_v_heads, K, V] = a;
        if (n_seq <= 0 || n_tok <= 0) return -1;
        if (!holds(state, {n_slots, n_v_heads, K, V})) return 0;
        if (!holds(q, {n_tok, n_k_heads, K})) return 1;
        if (!holds(k, {n_tok, n_k_heads, K})) return 2;
        if (!holds(v, {n_tok, n_v_heads, V})) return 3;
        if (!holds(g, {n_tok, n_v_heads})) return 4;
        if (!holds(beta, {n_tok, n_v_heads})) return 5;
        if (!holds(out, {n_tok, n_v_heads, V})) return 6;
        if (!holds(start, {(int64_t)n_seq + 1})) return 7;
        if (!holds(slot, {n_seq})) return 8;
        return holds(workspace, {workspace_bytes}) ? -1 : 9;
    }};
// include/bonsai_kv.h
Call<Handle, int, int, Mem, Mem> kv_append{"kv_append", {"kv", "layer", "pos", "k", "v"}};
Call<Handle, int, int, int, Mem, Mem> kv_append_batch{"kv_append_batch", {"kv", "layer", "pos0", "n_tok", "k", "v"}};
Call<Handle, int, int, Mem, Mem> kv_attn_decode{"kv_attn_decode", {"kv", "layer", "pos", "q", "out"}};

#define EACH_CALL(X)                                                                                                  \
    X(gemv) X(quant_activations) X(gemm) X(repack) X(gemv_repack) X(fwht) X(rmsnorm) X(gdn_step) X(attn)                \
    X(fwht_quant) X(swiglu) X(quant_batch) X(linear) X(linear_static) X(chain_run) X(kv_append) X(kv_append_batch)      \
    X(kv_attn_decode) X(qk_norm_rope) X(pages_append) X(pages_attn) X(pages_copy) X(gdn_seqs)

#define WRAPPER(f)                                                                                                    \
    PyObject *py_##f(PyObject *, PyObject *const *v, Py_ssize_t n, PyObject *kw) { return f.call(v, n, kw); }
EACH_CALL(WRAPPER)

// bind({name: address}): every function of this module needs an address.
PyObject *bind(PyObject *, PyObject *addresses) {
    if (!PyDict_Check(addresses)) {
        PyErr_SetString(PyExc_TypeError, "bind() takes a dict of addresses");
        return nullptr;
    }
#define BIND(f)                                                                                                       \
    {                                                                                                                 \
        PyObject *a = PyDict_GetItemString(addresses, #f);                                                              \
        void *p = a ? PyLong_AsVoidPtr(a) : nullptr;                                                                    \
        if (!p) {                                                                                                     \
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #f);                                                 \
            return nullptr;                                                                                           \
        }                                                                                                             \
        f.fn = reinterpret_cast<decltype(f)::Fn>(p);                                                                    \
    }
    EACH_CALL(BIND)
    Py_RETURN_NONE;
}

#define ENTRY(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(py_##f)), METH_FASTCALL | METH_KEYWORDS, nullptr},
PyMethodDef methods[] = {EACH_CALL(ENTRY){"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
