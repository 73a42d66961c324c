// p8_cache_py.cpp -- the Python side of the key/value cache operators (module _cache_calls): checks the tensors, fills the
// C ABI's argument structures and calls it. A decode step makes several of these calls per layer, each a few
// microseconds on the GPU; the same checks in Python take longer than that (6 to 9 us a call measured, here under 1).
//
// The module does not link against the library: bind() is given the entry points' addresses by the package, which has
// the library loaded. Every function returns the p8_status; what is refused before the call raises ValueError.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "pingala8.h"

namespace {

using at::Tensor;

struct Entries {
    decltype(&p8_kv_append) append;
    decltype(&p8_tree_attn_workspace) attn_workspace;
    decltype(&p8_tree_attn) attn;
    decltype(&p8_attn_mass) mass;
    decltype(&p8_kv_evict) evict;
    decltype(&p8_tree_accept) accept;
} g_p8;

struct Refused {
    std::string what;
};
[[noreturn]] void refuse(std::string what) { throw Refused{std::move(what)}; }

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const char *type_name(at::ScalarType t) { return t == at::kInt ? "int32" : t == at::kLong ? "int64" : t == at::kFloat ? "float32" : "the cache's type"; }
std::string shape_name(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

// a cache [batch, kv heads, slots, width], with a leading layer dimension where `layers`; v may be absent
struct Cache {
    p8_kv c;
    at::ScalarType type;
    int64_t dev;
};
Cache cache(const Tensor &k, const Tensor *v, bool layers) {
    Cache r;
    r.type = k.scalar_type();
    if (!k.is_cuda() || (r.type != at::kFloat && r.type != at::kHalf && r.type != at::kBFloat16)) refuse("the cache must be float32, float16 or bfloat16 CUDA tensors");
    const int64_t nd = k.dim();
    if (nd != 4 && !(layers && nd == 5))
        refuse(std::string("the cache must be [batch, kv heads, slots, width]") + (layers ? " or [layers, batch, kv heads, slots, width]" : "") + ", not " + shape_name(k.sizes()));
    if (v && (v->sizes() != k.sizes() || v->scalar_type() != r.type || v->device() != k.device())) refuse("keys and values must have one shape, type and device");
    const auto s = k.sizes(), ks = k.strides(), vs = v ? v->strides() : k.strides();
    if (ks[nd - 1] != 1 || vs[nd - 1] != 1) refuse("the cache's last dimension must have unit stride");
    const int64_t o = nd - 4;
    r.dev = k.get_device();
    r.c.k = k.data_ptr();
    r.c.v = v ? v->data_ptr() : nullptr;
    r.c.type = r.type == at::kFloat ? P8_KV_F32 : r.type == at::kHalf ? P8_KV_F16 : P8_KV_BF16;
    r.c.layers = o ? s[0] : 1;
    r.c.batch = s[o];
    r.c.heads = s[o + 1];
    r.c.slots = s[o + 2];
    r.c.width = s[o + 3];
    r.c.k_stride[0] = o ? ks[0] : 0;
    r.c.v_stride[0] = o ? vs[0] : 0;
    for (int i = 0; i < 3; ++i) {
        r.c.k_stride[1 + i] = ks[o + i];
        r.c.v_stride[1 + i] = vs[o + i];
    }
    return r;
}

// a contiguous tensor of exactly this shape, or NULL for None
template <typename T>
T *flat(PyObject *o, const char *name, at::ScalarType type, at::IntArrayRef shape, const Cache &c, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    const Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != c.dev || !t.is_contiguous())
        refuse(std::string(name) + " must be contiguous " + type_name(type) + " " + shape_name(shape) + " on the cache's device");
    return static_cast<T *>(t.data_ptr());
}
// [batch, tokens, heads, width]: address and outer strides
template <typename T>
T *rows(PyObject *o, const char *name, at::ScalarType type, at::IntArrayRef shape, const Cache &c, int64_t (&st)[3]) {
    const Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != c.dev || t.stride(3) != 1)
        refuse(std::string(name) + " must be " + type_name(type) + " " + shape_name(shape) + " with unit stride in its last dimension, on the cache's device");
    for (int i = 0; i < 3; ++i) st[i] = t.stride(i);
    return static_cast<T *>(t.data_ptr());
}
struct Query {
    int64_t tokens, heads;
};
Query query(const Tensor &q, const Cache &c, int64_t most) {
    if (q.dim() != 4) refuse("q must be [batch, tokens, heads, width]");
    const Query r{q.size(1), q.size(2)};
    if (r.tokens < (most ? 1 : 0) || (most && r.tokens > most) || r.heads < 1 || c.c.heads < 1 || r.heads % c.c.heads)
        refuse(most ? "1 to 64 tokens, and query heads in whole groups" : "query heads must come in whole groups");
    return r;
}
// float32 [.., kv heads, slots] of the cache's first dimensions; the strides of layer, sequence and head
float *masses(PyObject *o, const char *name, const Cache &c, int64_t dims, int64_t slots, int64_t (&st)[3]) {
    const Tensor &t = tensor(o, name);
    const auto &k = c.c;
    const bool four = dims == 5;
    if (t.scalar_type() != at::kFloat || !t.is_cuda() || t.get_device() != c.dev || t.dim() != dims - 1 || (four && t.size(0) != k.layers) || t.size(four) != k.batch ||
        t.size(four + 1) != k.heads || t.size(four + 2) != slots || t.stride(four + 2) != 1)
        refuse(std::string(name) + " must be float32 [.., kv heads, slots] of the cache with unit slot stride, on its device");
    st[0] = four ? t.stride(0) : 0;
    st[1] = t.stride(four);
    st[2] = t.stride(four + 1);
    return static_cast<float *>(t.data_ptr());
}

double number(PyObject *o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw nullptr;
    return x;
}
int64_t integer(PyObject *o) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw nullptr;
    return x;
}

// The tensors' device current for the launch, and its current stream.
struct On {
    std::optional<c10::DeviceGuard> guard;
    void *stream;
    explicit On(const Cache &c) {
        const c10::Device d(c10::kCUDA, (c10::DeviceIndex)c.dev);
        guard.emplace(d);
        stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
    }
};

#define ENTRY(name, count)                                                                  \
    PyObject *name(PyObject *, PyObject *const *a, Py_ssize_t n) {                          \
        try {                                                                               \
            if (n != (count)) refuse(#name " takes " #count " arguments");                  \
            if (!g_p8.append) refuse("bind() comes first");                                 \
            return PyLong_FromLong(name##_(a));                                             \
        } catch (const Refused &r) {                                                        \
            PyErr_SetString(PyExc_ValueError, r.what.c_str());                              \
        } catch (const std::exception &e) {                                                 \
            PyErr_SetString(PyExc_RuntimeError, e.what());                                  \
        } catch (std::nullptr_t) { /* the Python error is set */                            \
        }                                                                                   \
        return nullptr;                                                                     \
    }

// q k v k_cache v_cache lens pos cos sin q_norm k_norm eps counts q_out
p8_status kv_append_(PyObject *const *a) {
    const Tensor &k = tensor(a[3], "k_cache"), &v = tensor(a[4], "v_cache"), &q = tensor(a[0], "q"), &cs = tensor(a[7], "cos");
    const Cache c = cache(k, &v, false);
    const Query t = query(q, c, 0);
    if (cs.dim() != 2) refuse("cos must be [positions, width / 2]");
    const int64_t B = c.c.batch, T = t.tokens, hk = c.c.heads, D = c.c.width, P = cs.size(0);
    p8_kv_append_args x;
    x.q = rows<float>(a[0], "q", at::kFloat, {B, T, t.heads, D}, c, x.q_stride);
    x.k = rows<float>(a[1], "k", at::kFloat, {B, T, hk, D}, c, x.k_stride);
    x.v = rows<float>(a[2], "v", at::kFloat, {B, T, hk, D}, c, x.v_stride);
    x.tokens = T;
    x.heads = t.heads;
    x.lens = flat<int32_t>(a[5], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[12], "counts", at::kInt, {B}, c, true);
    x.pos = flat<int32_t>(a[6], "pos", at::kInt, {B, T}, c);
    x.cos = flat<float>(a[7], "cos", at::kFloat, {P, D / 2}, c);
    x.sin = flat<float>(a[8], "sin", at::kFloat, {P, D / 2}, c);
    x.positions = P;
    x.q_norm = flat<float>(a[9], "q_norm", at::kFloat, {D}, c, true);
    x.k_norm = flat<float>(a[10], "k_norm", at::kFloat, {D}, c, true);
    x.eps = number(a[11]);
    x.q_out = rows<void>(a[13], "q_out", c.type, {B, T, t.heads, D}, c, x.q_out_stride);
    const On on(c);
    return g_p8.append(&c.c, &x, on.stream);
}
ENTRY(kv_append, 14)

// q k_cache v_cache lens mask counts scale out lse workspace
p8_status tree_attention_(PyObject *const *a) {
    const Tensor &k = tensor(a[1], "k_cache"), &v = tensor(a[2], "v_cache"), &q = tensor(a[0], "q");
    const Cache c = cache(k, &v, false);
    const Query t = query(q, c, P8_TREE_MAX);
    const int64_t B = c.c.batch, T = t.tokens, D = c.c.width;
    p8_tree_attn_args x;
    x.q = rows<void>(a[0], "q", c.type, {B, T, t.heads, D}, c, x.q_stride);
    x.tokens = T;
    x.heads = t.heads;
    x.lens = flat<int32_t>(a[3], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[5], "counts", at::kInt, {B}, c, true);
    x.mask = nullptr;
    x.mask_stride = 0;
    if (a[4] != Py_None) {
        const bool per = tensor(a[4], "mask").dim() == 2;
        x.mask = per ? flat<uint64_t>(a[4], "mask", at::kLong, {B, T}, c) : flat<uint64_t>(a[4], "mask", at::kLong, {T}, c);
        x.mask_stride = per ? T : 0;
    }
    x.scale = a[6] == Py_None ? 1.0 / std::sqrt((double)D) : number(a[6]);
    x.out = rows<void>(a[7], "out", c.type, {B, T, t.heads, D}, c, x.out_stride);
    x.lse = flat<float>(a[8], "lse", at::kFloat, {B, T, t.heads}, c);
    const On on(c);
    Tensor ws;
    if (a[9] == Py_None) {
        ws = at::empty({(int64_t)g_p8.attn_workspace(&c.c, T, t.heads)}, k.options().dtype(at::kByte));
    } else {
        ws = tensor(a[9], "workspace");
        if (!ws.is_cuda() || ws.get_device() != c.dev || !ws.is_contiguous()) refuse("workspace must be contiguous on the cache's device");
    }
    return g_p8.attn(&c.c, &x, ws.data_ptr(), ws.nbytes(), on.stream);
}
ENTRY(tree_attention, 10)

// q lse k_cache lens mass rows counts scale out
p8_status attention_mass_(PyObject *const *a) {
    const Tensor &k = tensor(a[2], "k_cache"), &q = tensor(a[0], "q");
    const Cache c = cache(k, nullptr, false);
    const Query t = query(q, c, P8_TREE_MAX);
    const int64_t B = c.c.batch, T = t.tokens;
    p8_attn_mass_args x;
    x.q = rows<void>(a[0], "q", c.type, {B, T, t.heads, c.c.width}, c, x.q_stride);
    x.tokens = T;
    x.heads = t.heads;
    x.lse = flat<float>(a[1], "lse", at::kFloat, {B, T, t.heads}, c);
    x.lens = flat<int32_t>(a[3], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[6], "counts", at::kInt, {B}, c, true);
    x.rows = flat<int32_t>(a[5], "rows", at::kInt, {B, T}, c, true);
    x.scale = a[7] == Py_None ? 1.0 / std::sqrt((double)c.c.width) : number(a[7]);
    int64_t st[3];
    x.mass = masses(a[4], "mass", c, 4, c.c.slots, st);
    for (int i = 0; i < 2; ++i) x.mass_stride[i] = st[1 + i];
    x.out = masses(a[8], "out", c, 4, c.c.slots, st);
    for (int i = 0; i < 2; ++i) x.out_stride[i] = st[1 + i];
    const On on(c);
    return g_p8.mass(&c.c, &x, on.stream);
}
ENTRY(attention_mass, 9)

// k_cache v_cache mass lens budget sinks recent k_out v_out mass_out new_lens kept
p8_status kv_evict_(PyObject *const *a) {
    const Tensor &k = tensor(a[0], "k_cache"), &v = tensor(a[1], "v_cache"), &ko = tensor(a[7], "k_out"), &vo = tensor(a[8], "v_out");
    const Cache c = cache(k, &v, true), d = cache(ko, &vo, true);
    if (ko.dim() != k.dim() || d.type != c.type || d.dev != c.dev || d.c.layers != c.c.layers || d.c.batch != c.c.batch || d.c.heads != c.c.heads || d.c.width != c.c.width)
        refuse("k_out must have the cache's shape but for its slots, its type and its device");
    p8_kv_evict_args x;
    x.budget = integer(a[4]);
    x.sinks = integer(a[5]);
    x.recent = integer(a[6]);
    x.mass = masses(a[2], "mass", c, k.dim(), c.c.slots, x.mass_stride);
    x.mass_out = masses(a[9], "mass_out", c, k.dim(), d.c.slots, x.mass_out_stride);
    x.lens = flat<int32_t>(a[3], "lens", at::kInt, {c.c.batch}, c);
    x.new_lens = flat<int32_t>(a[10], "new_lens", at::kInt, {c.c.batch}, c);
    if (k.dim() == 5) x.kept = flat<int32_t>(a[11], "kept", at::kInt, {c.c.layers, c.c.batch, c.c.heads, x.budget}, c);
    else x.kept = flat<int32_t>(a[11], "kept", at::kInt, {c.c.batch, c.c.heads, x.budget}, c);
    const On on(c);
    return g_p8.evict(&c.c, &d.c, &x, on.stream);
}
ENTRY(kv_evict, 12)

// tokens parents target k_cache v_cache lens counts path accepted next_token new_lens
p8_status tree_accept_(PyObject *const *a) {
    const Tensor &k = tensor(a[3], "k_cache"), &v = tensor(a[4], "v_cache"), &tok = tensor(a[0], "tokens");
    const Cache c = cache(k, &v, true);
    if (tok.dim() != 2 || tok.size(1) < 1 || tok.size(1) > P8_TREE_MAX) refuse("tokens must be [batch, 1 to 64]");
    const int64_t B = c.c.batch, T = tok.size(1);
    p8_tree_accept_args x;
    x.tokens = flat<int64_t>(a[0], "tokens", at::kLong, {B, T}, c);
    x.target = flat<int64_t>(a[2], "target", at::kLong, {B, T}, c);
    x.parents = flat<int32_t>(a[1], "parents", at::kInt, {B, T}, c);
    x.ntokens = T;
    x.lens = flat<int32_t>(a[5], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[6], "counts", at::kInt, {B}, c, true);
    x.path = flat<int32_t>(a[7], "path", at::kInt, {B, T}, c);
    x.accepted = flat<int32_t>(a[8], "accepted", at::kInt, {B}, c);
    x.next_token = flat<int64_t>(a[9], "next_token", at::kLong, {B}, c);
    x.new_lens = flat<int32_t>(a[10], "new_lens", at::kInt, {B}, c);
    const On on(c);
    return g_p8.accept(&c.c, &x, on.stream);
}
ENTRY(tree_accept, 11)

PyObject *workspace_(PyObject *const *a, Py_ssize_t n) {
    if (n != 3) refuse("attention_workspace takes 3 arguments");
    const Tensor &k = tensor(a[0], "k_cache");
    const Cache c = cache(k, &k, false);
    const On on(c);  // the size goes by the device's SMs
    return PyLong_FromSize_t(g_p8.attn_workspace(&c.c, integer(a[1]), integer(a[2])));
}
PyObject *attention_workspace(PyObject *, PyObject *const *a, Py_ssize_t n) {
    try {
        if (!g_p8.append) refuse("bind() comes first");
        return workspace_(a, n);
    } catch (const Refused &r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (std::nullptr_t) {
    }
    return nullptr;
}

// the addresses of p8_kv_append, p8_tree_attn_workspace, p8_tree_attn, p8_attn_mass, p8_kv_evict, p8_tree_accept
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    void *p[6];
    if (n != 6) {
        PyErr_SetString(PyExc_ValueError, "bind takes six addresses");
        return nullptr;
    }
    for (int i = 0; i < 6; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: no address");
            return nullptr;
        }
    }
    g_p8 = {(decltype(&p8_kv_append))p[0], (decltype(&p8_tree_attn_workspace))p[1], (decltype(&p8_tree_attn))p[2],
            (decltype(&p8_attn_mass))p[3], (decltype(&p8_kv_evict))p[4], (decltype(&p8_tree_accept))p[5]};
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, (PyCFunction)(void *)f, METH_FASTCALL, ""}
PyMethodDef g_methods[] = {METHOD(bind), METHOD(kv_append), METHOD(tree_attention), METHOD(attention_mass), METHOD(kv_evict), METHOD(tree_accept),
                           METHOD(attention_workspace), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_cache_calls", "calls of the key/value cache operators (see pingala8_llm_b200.cache)", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cache_calls() { return PyModule_Create(&g_module); }
