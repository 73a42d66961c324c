// p8_paged_py.cpp -- the Python side of the paged cache and beam search operators (module _paged_calls): checks the tensors, fills the
// C ABI's argument structures and calls it, as p8_cache_py.cpp does for the contiguous cache. bind() is given the entry
// points' addresses by the package. Every call returns the p8_status; what is refused before it raises ValueError.
#include "p8_py.h"

#include <c10/cuda/CUDACachingAllocator.h>

namespace {

struct Entries {
    decltype(&p8_paged_append) append;
    decltype(&p8_paged_attn_workspace) attn_workspace;
    decltype(&p8_paged_attn) attn;
    decltype(&p8_beam_select_workspace) select_workspace;
    decltype(&p8_beam_select) select;
    decltype(&p8_beam_reorder) reorder;
} g_p8;

// pages [pages, kv heads, page slots, width], with a leading layer dimension where `layers`, and their tables [rows, columns]
struct Pages {
    p8_paged c;
    at::ScalarType type;
    int64_t dev;
};
Pages pages(const Tensor &k, const Tensor &v, const Tensor &tables, bool layers) {
    Pages r;
    r.type = k.scalar_type();
    if (!k.is_cuda() || (r.type != at::kFloat && r.type != at::kHalf && r.type != at::kBFloat16)) refuse("the pages must be float32, float16 or bfloat16 CUDA tensors");
    const int64_t nd = k.dim();
    if (nd != 4 && !(layers && nd == 5))
        refuse(std::string("the pages must be [pages, kv heads, page slots, width]") + (layers ? " or [layers, pages, kv heads, page slots, width]" : "") + ", not " + shape_name(k.sizes()));
    if (v.sizes() != k.sizes() || v.scalar_type() != r.type || v.device() != k.device()) refuse("keys and values must have one shape, type and device");
    const auto s = k.sizes(), ks = k.strides(), vs = v.strides();
    if (ks[nd - 1] != 1 || vs[nd - 1] != 1) refuse("the pages' last dimension must have unit stride");
    const int64_t o = nd - 4;
    r.dev = k.get_device();
    r.c.k = k.data_ptr();
    r.c.v = v.data_ptr();
    r.c.type = r.type == at::kFloat ? P8_KV_F32 : r.type == at::kHalf ? P8_KV_F16 : P8_KV_BF16;
    r.c.layers = o ? s[0] : 1;
    r.c.pages = s[o];
    r.c.heads = s[o + 1];
    r.c.page = s[o + 2];
    r.c.width = s[o + 3];
    r.c.k_stride[0] = o ? ks[0] : 0;
    r.c.v_stride[0] = o ? vs[0] : 0;
    for (int i = 0; i < 3; ++i) {
        r.c.k_stride[1 + i] = ks[o + i];
        r.c.v_stride[1 + i] = vs[o + i];
    }
    if (tables.scalar_type() != at::kInt || tables.dim() != 2 || !tables.is_cuda() || tables.get_device() != r.dev || (tables.size(1) > 1 && tables.stride(1) != 1))
        refuse("tables must be int32 [rows, columns] with unit column stride, on the pages' device");
    r.c.tables = static_cast<int32_t *>(tables.data_ptr());
    r.c.rows = tables.size(0);
    r.c.columns = tables.size(1);
    r.c.table_stride = tables.stride(0);
    return r;
}

// q k v k_pages v_pages tables lens pos cos sin interleaved q_norm k_norm eps counts q_out
p8_status paged_append_(PyObject *const *a) {
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[3], "k_pages"), &v = tensor(a[4], "v_pages"), &cs = tensor(a[8], "cos");
    const Pages c = pages(k, v, tensor(a[5], "tables"), false);
    if (q.dim() != 4 || c.c.heads < 1 || q.size(2) < 1 || q.size(2) % c.c.heads) refuse("q must be [batch, tokens, heads, width], its heads in whole groups");
    if (cs.dim() != 2) refuse("cos must be [positions, turned elements / 2]");
    const int64_t B = c.c.rows, T = q.size(1), H = q.size(2), hk = c.c.heads, D = c.c.width, P = cs.size(0);
    p8_paged_append_args x;
    x.q = rows<float>(a[0], "q", at::kFloat, {B, T, H, D}, c, x.q_stride);
    x.k = rows<float>(a[1], "k", at::kFloat, {B, T, hk, D}, c, x.k_stride);
    x.v = rows<float>(a[2], "v", at::kFloat, {B, T, hk, D}, c, x.v_stride);
    x.tokens = T;
    x.heads = H;
    x.lens = flat<int32_t>(a[6], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[14], "counts", at::kInt, {B}, c, true);
    x.pos = flat<int32_t>(a[7], "pos", at::kInt, {B, T}, c);
    x.cos = flat<float>(a[8], "cos", at::kFloat, {P, cs.size(1)}, c);
    x.sin = flat<float>(a[9], "sin", at::kFloat, {P, cs.size(1)}, c);
    x.positions = P;
    x.rotary = 2 * cs.size(1);
    x.interleaved = PyObject_IsTrue(a[10]);
    if (x.interleaved < 0) throw nullptr;
    x.q_norm = flat<float>(a[11], "q_norm", at::kFloat, {D}, c, true);
    x.k_norm = flat<float>(a[12], "k_norm", at::kFloat, {D}, c, true);
    x.eps = number(a[13]);
    x.q_out = rows<void>(a[15], "q_out", c.type, {B, T, H, D}, c, x.q_out_stride);
    const On on(c);
    return g_p8.append(&c.c, &x, on.stream);
}
ENTRY(paged_append, 16)

// the caller's workspace, or one of torch's allocator for this call (which goes back in the stream's order)
struct Scratch {
    c10::DataPtr own;
    void *at = nullptr;
    size_t bytes = 0;
    Scratch(PyObject *o, size_t need, int64_t dev) {
        if (o != Py_None) {
            const Tensor &ws = tensor(o, "workspace");
            if (!ws.is_cuda() || ws.get_device() != dev || !ws.is_contiguous()) refuse("workspace must be contiguous on the call's device");
            at = ws.data_ptr();
            bytes = ws.nbytes();
        } else if (need) {
            own = c10::cuda::CUDACachingAllocator::get()->allocate(need);
            at = own.get();
            bytes = need;
        }
    }
};

// q k_pages v_pages tables lens counts scale out lse workspace
p8_status paged_attention_(PyObject *const *a) {
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
    const Pages c = pages(k, v, tensor(a[3], "tables"), false);
    if (q.dim() != 3 || c.c.heads < 1 || q.size(1) < 1 || q.size(1) % c.c.heads) refuse("q must be [batch, heads, width], its heads in whole groups");
    const int64_t B = c.c.rows, H = q.size(1), D = c.c.width;
    p8_paged_attn_args x;
    x.q = rows<void>(a[0], "q", c.type, {B, H, D}, c, x.q_stride);
    x.heads = H;
    x.lens = flat<int32_t>(a[4], "lens", at::kInt, {B}, c);
    x.counts = flat<int32_t>(a[5], "counts", at::kInt, {B}, c, true);
    x.scale = a[6] == Py_None ? 1.0 / std::sqrt((double)D) : number(a[6]);
    x.out = rows<void>(a[7], "out", c.type, {B, H, D}, c, x.out_stride);
    x.lse = flat<float>(a[8], "lse", at::kFloat, {B, H}, c);
    const On on(c);
    const Scratch ws(a[9], a[9] == Py_None ? g_p8.attn_workspace(&c.c, H) : 0, c.dev);
    return g_p8.attn(&c.c, &x, ws.at, ws.bytes, on.stream);
}
ENTRY(paged_attention, 10)

// logits scores done end candidates out_scores parents tokens out_done workspace
p8_status beam_select_(PyObject *const *a) {
    const Tensor &l = tensor(a[0], "logits");
    struct { int64_t dev; } c;
    const at::ScalarType type = l.scalar_type();
    if (!l.is_cuda() || (type != at::kFloat && type != at::kHalf && type != at::kBFloat16)) refuse("logits must be a float32, float16 or bfloat16 CUDA tensor");
    if (l.dim() != 3 || (l.size(2) > 1 && l.stride(2) != 1)) refuse("logits must be [batch, beams, vocabulary] with unit stride in its last dimension, not " + shape_name(l.sizes()));
    c.dev = l.get_device();
    p8_beam_select_args x;
    const int64_t B = l.size(0), W = l.size(1), n = integer(a[4]);
    x.logits = l.data_ptr();
    x.type = type == at::kFloat ? P8_KV_F32 : type == at::kHalf ? P8_KV_F16 : P8_KV_BF16;
    x.batch = B;
    x.beams = W;
    x.vocab = l.size(2);
    x.stride[0] = l.stride(0);
    x.stride[1] = l.stride(1);
    x.scores = flat<float>(a[1], "scores", at::kFloat, {B, W}, c);
    x.done = flat<uint8_t>(a[2], "done", at::kBool, {B, W}, c, true);
    x.end = a[3] == Py_None ? -1 : integer(a[3]);
    if (a[3] != Py_None && x.end < 0) refuse("end must be a token");
    if (x.done && x.end < 0) refuse("beams that have ended need the end token");
    x.candidates = n;
    x.out_scores = flat<float>(a[5], "out_scores", at::kFloat, {B, n}, c);
    x.parents = flat<int32_t>(a[6], "parents", at::kInt, {B, n}, c);
    x.tokens = flat<int64_t>(a[7], "tokens", at::kLong, {B, n}, c);
    x.out_done = flat<uint8_t>(a[8], "out_done", at::kBool, {B, n}, c);
    const On on(c);
    const Scratch ws(a[9], a[9] == Py_None ? g_p8.select_workspace(B, W, x.vocab, n) : 0, c.dev);
    return g_p8.select(&x, ws.at, ws.bytes, on.stream);
}
ENTRY(beam_select, 10)

// parents k_pages v_pages tables lens
p8_status beam_reorder_(PyObject *const *a) {
    const Tensor &p = tensor(a[0], "parents"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
    const Pages c = pages(k, v, tensor(a[3], "tables"), true);
    if (p.dim() != 2 || p.size(0) < 1 || p.size(1) < 1 || p.size(0) * p.size(1) != c.c.rows) refuse("parents must be int32 [batch, beams], and the tables have batch x beams rows");
    const int64_t B = p.size(0), W = p.size(1);
    const int32_t *parents = flat<int32_t>(a[0], "parents", at::kInt, {B, W}, c), *lens = flat<int32_t>(a[4], "lens", at::kInt, {B * W}, c);
    const On on(c);
    return g_p8.reorder(&c.c, parents, lens, B, W, on.stream);
}
ENTRY(beam_reorder, 5)

// k_pages v_pages tables heads
PyObject *attention_workspace(PyObject *, PyObject *const *a, Py_ssize_t n) {
    try {
        if (n != 4) refuse("attention_workspace takes 4 arguments");
        if (!g_bound) refuse("bind() comes first");
        const Pages c = pages(tensor(a[0], "k_pages"), tensor(a[1], "v_pages"), tensor(a[2], "tables"), false);
        const On on(c);  // the size goes by the device's SMs
        return PyLong_FromSize_t(g_p8.attn_workspace(&c.c, integer(a[3])));
    } catch (const Refused &r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (std::nullptr_t) {
    }
    return nullptr;
}
// logits candidates
PyObject *select_workspace(PyObject *, PyObject *const *a, Py_ssize_t n) {
    try {
        if (n != 2) refuse("select_workspace takes 2 arguments");
        if (!g_bound) refuse("bind() comes first");
        const Tensor &l = tensor(a[0], "logits");
        if (!l.is_cuda() || l.dim() != 3) refuse("logits must be a CUDA tensor [batch, beams, vocabulary]");
        struct { int64_t dev; } c = {l.get_device()};
        const On on(c);
        return PyLong_FromSize_t(g_p8.select_workspace(l.size(0), l.size(1), l.size(2), integer(a[1])));
    } catch (const Refused &r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (std::nullptr_t) {
    }
    return nullptr;
}

// the addresses of p8_paged_append, p8_paged_attn_workspace, p8_paged_attn, p8_beam_select_workspace, p8_beam_select, p8_beam_reorder
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
    g_p8 = {(decltype(&p8_paged_append))p[0], (decltype(&p8_paged_attn_workspace))p[1], (decltype(&p8_paged_attn))p[2],
            (decltype(&p8_beam_select_workspace))p[3], (decltype(&p8_beam_select))p[4], (decltype(&p8_beam_reorder))p[5]};
    g_bound = true;
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, (PyCFunction)(void *)f, METH_FASTCALL, ""}
PyMethodDef g_methods[] = {METHOD(bind), METHOD(paged_append), METHOD(paged_attention), METHOD(beam_select), METHOD(beam_reorder), METHOD(attention_workspace), METHOD(select_workspace),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged_calls", "calls of the paged cache and beam search operators (see pingala8_llm_b200.paged)", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_calls() { return PyModule_Create(&g_module); }
