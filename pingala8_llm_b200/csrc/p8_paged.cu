// p8_paged.cu -- operators on a paged key/value cache: append (norm, rotation, write through the tables) and the C ABI entry
// points of attention, beam selection and beam reordering (p8_paged_attn.cuh, p8_beam.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "p8_cache_common.cuh"
#include "p8_device.cuh"
#include "p8_internal.h"
#include "p8_paged_index.h"

namespace p8 {

unsigned int cache_wait_ns();  // p8_cache_wait_limit

__device__ unsigned int g_paged_error = 0;  // bits 64 and 128 of p8_device_error

unsigned int read_and_clear_paged_error() {
    unsigned int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_paged_error, sizeof(v));
    cudaMemcpyToSymbol(g_paged_error, &z, sizeof(z));
    return v;
}

namespace {

__device__ __forceinline__ void out_of_range() { atomicOr(&g_paged_error, kErrRange); }

int sm_count() {
    static std::atomic<int> n[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int v = n[dev].load(std::memory_order_relaxed);
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
        n[dev].store(v, std::memory_order_relaxed);
    }
    return v;
}

// Raises a kernel's limit of dynamic shared memory, once on each device; `slot` says which kernel it is.
template <typename K>
bool allow_shared(K *kernel, int64_t slot, int bytes) {
    static std::atomic<unsigned long long> done_on[64];
    int dev = 0;
    const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && slot < 64;
    if (known && (done_on[dev].load(std::memory_order_acquire) >> slot & 1)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    if (known) done_on[dev].fetch_or(1ull << slot, std::memory_order_release);
    return true;
}

// ----------------------------------------------------------------------------------------------------------------
// append: y = rotate(norm(x)) for each head of a token, keys and values to the page that the table names. D / 8 lanes
// hold one head's row, eight values each: the elements 4l.. and half + 4l.. of the two halves, or 8l.. where pairs are
// neighbours; so a pair is in one lane, and lanes from rotary / 8 on hold what does not turn. The table's entry is looked up while the
// row itself is on its way. Bound by memory on a prompt (4,099 tokens x 48 heads of 128, 151 MB: 27.4 us, 5.5 TB/s), by its one launch on a
// token (eight sequences 2.2 us).
struct PagedAppendArgs {
    const float *x[3];          // q, k, v
    long long xs[3][3];
    void *q_out;
    long long qs[3];
    void *kv[2];
    long long ps[2][3];         // page, head, slot
    const int *tables, *lens, *counts, *pos;
    long long ts;
    const float *cos, *sin, *qn, *kn;
    long long positions, slots;
    PageDiv div;
    int tokens, heads, kvh, batch, pages, half;
    float eps;
};

// four values, rounded to the type, that make room in the L2 for others first
__device__ __forceinline__ void stream4(float *p, const float (&v)[4]) { __stcs(reinterpret_cast<float4 *>(p), make_float4(v[0], v[1], v[2], v[3])); }
template <typename T>
__device__ __forceinline__ void stream4(T *p, const float (&v)[4]) {
    union { T t[4]; uint2 u; } r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.t[i] = from_f<T>(v[i]);
    __stcs(reinterpret_cast<uint2 *>(p), r.u);
}

template <typename T, int D, bool kPairs, int kRows>
__global__ void __launch_bounds__(128) k_paged_append(const __grid_constant__ PagedAppendArgs a) {
    constexpr int L = D / 8, RPB = 128 / L;
    after_prior();
    const unsigned int rows = a.heads + 2 * a.kvh, per = (rows + kRows - 1) / kRows, id = blockIdx.x * RPB + threadIdx.x / L;
    const int l = threadIdx.x % L;
    const unsigned int tok = id / per;
    if (tok >= (unsigned int)a.batch * a.tokens) return;  // a whole group of lanes leaves
    const int r0 = (int)(id - tok * per) * kRows, b = (int)(tok / (unsigned int)a.tokens), t = (int)(tok - (unsigned int)b * a.tokens);
    const int turned = a.half / 4, past = l - turned;  // lanes that turn; this lane among the others
    const int e0 = kPairs ? 8 * l : past < 0 ? 4 * l : 2 * a.half + 4 * past, e1 = kPairs ? 8 * l + 4 : past < 0 ? a.half + 4 * l : a.half + D / 2 + 4 * past;
    float u[kRows][4], w[kRows][4];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i, which = r < a.heads ? 0 : r < a.heads + a.kvh ? 1 : 2, h = which == 0 ? r : which == 1 ? r - a.heads : r - a.heads - a.kvh;
        if (r >= (int)rows) break;
        const float *x = a.x[which] + b * a.xs[which][0] + t * a.xs[which][1] + h * a.xs[which][2];
        *reinterpret_cast<float4 *>(u[i]) = __ldcs(reinterpret_cast<const float4 *>(x + e0));
        *reinterpret_cast<float4 *>(w[i]) = __ldcs(reinterpret_cast<const float4 *>(x + e1));
    }
    const int p = a.pos[tok], len = a.lens[b], n = a.counts ? a.counts[b] : a.tokens;
    if (len < 0 || n < 0 || n > a.tokens || (long long)len + n > a.slots) {
        if (t == 0 && r0 == 0 && l == 0) out_of_range();
        return;
    }
    if (t >= n) return;
    if (p < 0 || p >= a.positions) {
        if (r0 == 0 && l == 0) out_of_range();
        return;
    }
    unsigned int in = 0;
    int at = 0;
    if (r0 + kRows > a.heads) {  // keys or values among the rows
        const unsigned int page = page_of(a.div, len + t);
        in = len + t - page * a.div.size;
        at = a.tables[b * a.ts + page];
    }
    float c[4], s[4];
    if (past < 0 && r0 < a.heads + a.kvh) {
        *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(a.cos + (long long)p * a.half + 4 * l);
        *reinterpret_cast<float4 *>(s) = *reinterpret_cast<const float4 *>(a.sin + (long long)p * a.half + 4 * l);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = r0 + i, which = r < a.heads ? 0 : r < a.heads + a.kvh ? 1 : 2, h = which == 0 ? r : which == 1 ? r - a.heads : r - a.heads - a.kvh;
        if (r >= (int)rows) break;
        if (which < 2) {
            const float *g = which == 0 ? a.qn : a.kn;
            if (g) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) ss += u[i][j] * u[i][j] + w[i][j] * w[i][j];
                const unsigned int group = (L == 32 ? 0xffffffffu : (1u << L) - 1u) << (threadIdx.x % 32 / L * L);
#pragma unroll
                for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(group, ss, m);
                const float rs = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[i][j] = u[i][j] * rs * g[e0 + j];
                    w[i][j] = w[i][j] * rs * g[e1 + j];
                }
            }
            if (past < 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float &x0 = kPairs ? (j < 2 ? u[i][2 * j] : w[i][2 * j - 4]) : u[i][j], &x1 = kPairs ? (j < 2 ? u[i][2 * j + 1] : w[i][2 * j - 3]) : w[i][j];
                    const float y0 = x0 * c[j] - x1 * s[j], y1 = x1 * c[j] + x0 * s[j];
                    x0 = y0;
                    x1 = y1;
                }
            }
        }
        T *y;
        if (which == 0) {
            y = static_cast<T *>(a.q_out) + b * a.qs[0] + t * a.qs[1] + h * a.qs[2];
        } else {
            if ((unsigned int)at >= (unsigned int)a.pages) {
                if (h == 0 && l == 0) out_of_range();
                continue;
            }
            const int z = which - 1;
            y = static_cast<T *>(a.kv[z]) + at * a.ps[z][0] + h * a.ps[z][1] + in * a.ps[z][2];
        }
        if (kRows > 1) {
            stream4(y + e0, u[i]);
            stream4(y + e1, w[i]);
        } else {
            store4(y + e0, u[i]);
            store4(y + e1, w[i]);
        }
    }
}

#include "p8_paged_attn.cuh"
#include "p8_beam.cuh"

// ----------------------------------------------------------------------------------------------------------------
// host side: argument checks (nothing below them touches the device before they pass) and launches
bool paged_ok(const p8_paged *c) {
    if (!c || !c->k || !c->v || !c->tables || !al16(c->k) || !al16(c->v) || ((uintptr_t)c->tables & 3)) return false;
    if (c->type != P8_KV_F32 && c->type != P8_KV_F16 && c->type != P8_KV_BF16) return false;
    if (c->width != 64 && c->width != 128) return false;
    if (c->layers < 1 || c->layers > 32767 || c->pages < 1 || c->pages > INT32_MAX || c->heads < 1 || c->heads > 65535 || c->page < 1 || c->page > P8_PAGE_MAX) return false;
    if (c->rows < 1 || c->rows > (int64_t)P8_BATCH_MAX * P8_BEAMS_MAX || c->columns < 1 || c->columns > P8_SLOTS_MAX || c->columns * c->page > P8_SLOTS_MAX) return false;
    if (c->table_stride < 0 || (c->rows > 1 && c->table_stride > 0 && c->table_stride < c->columns)) return false;
    const int64_t dims[4] = {c->layers, c->pages, c->heads, c->page};
    const int es = elem_size(c->type);
    return strides_ok(c->k_stride, dims, 4, es) && strides_ok(c->v_stride, dims, 4, es);
}
bool group_ok(const p8_paged *c, int64_t heads) { return heads >= c->heads && heads % c->heads == 0 && heads <= 65535; }
View pages_view(const p8_paged *c, bool values) {
    const int64_t dims[4] = {c->layers, c->pages, c->heads, c->page};
    return View(values ? c->v : c->k, values ? c->v_stride : c->k_stride, dims, 4, elem_size(c->type), c->width);
}
View tables_view(const p8_paged *c) { return View(c->tables, &c->table_stride, &c->rows, 1, 4, c->columns); }

template <typename T, int D, bool kPairs>
cudaError_t run_paged_append(const PagedAppendArgs &a, cudaStream_t st) {
    const long long rows = a.heads + 2 * a.kvh, tokens = (long long)a.batch * a.tokens, per = 128 / (D / 8);
    const auto blocks = [&](int n) { return (tokens * ((rows + n - 1) / n) + per - 1) / per; };
    // Two rows a lane, asked for together, and what is written not kept for long (prompt of 4,099 tokens 27.1 us; 33.3 with one row and blocks of 256), where there is work for the whole GPU all the same; else one, which is done sooner.
    const int n = blocks(2) >= 8 * sm_count() ? 2 : 1;
    return launch_after(n == 2 ? k_paged_append<T, D, kPairs, 2> : k_paged_append<T, D, kPairs, 1>, dim3((unsigned int)blocks(n)), dim3(128), 0, st, a);
}
template <typename T>
cudaError_t run_paged_append(const p8_paged *c, const PagedAppendArgs &a, bool pairs, cudaStream_t st) {
    if (c->width == 128) return pairs ? run_paged_append<T, 128, true>(a, st) : run_paged_append<T, 128, false>(a, st);
    return pairs ? run_paged_append<T, 64, true>(a, st) : run_paged_append<T, 64, false>(a, st);
}

}  // namespace
}  // namespace p8

using namespace p8;

extern "C" {

p8_status p8_paged_append(const p8_paged *c, const p8_paged_append_args *a, void *stream) {
    if (!paged_ok(c) || !a || c->layers != 1 || c->rows > P8_BATCH_MAX || !group_ok(c, a->heads)) return P8_ERR_ARG;
    if (a->tokens < 0) return P8_ERR_ARG;
    if (a->tokens == 0) return P8_OK;  // buffers of nothing may have no address
    if (!a->q || !a->k || !a->v || !a->q_out || !a->lens || !a->pos || !a->cos || !a->sin || a->positions < 1) return P8_ERR_ARG;
    if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->q_out) || !al16(a->cos) || !al16(a->sin) || !(a->eps >= 0.0)) return P8_ERR_ARG;
    if (a->rotary < 8 || a->rotary > c->width || a->rotary % 8) return P8_ERR_ARG;
    if (a->tokens > c->columns * c->page || c->rows * a->tokens * (a->heads + 2 * c->heads) > (int64_t(1) << 31) - 64) return P8_ERR_ARG;
    const int es = elem_size(c->type);
    const int64_t B = c->rows, dq[3] = {B, a->tokens, a->heads}, dk[3] = {B, a->tokens, c->heads};
    if (!strides_ok(a->q_stride, dq, 3, 4) || !strides_ok(a->k_stride, dk, 3, 4) || !strides_ok(a->v_stride, dk, 3, 4) || !strides_ok(a->q_out_stride, dq, 3, es)) return P8_ERR_ARG;
    // in place: every lane writes what it has read
    const bool same = c->type == P8_KV_F32 && (const void *)a->q == a->q_out && same_strides(a->q_stride, a->q_out_stride, dq, 3);
    const int64_t table = a->positions * (a->rotary / 2) * 4;
    if (clash({View(a->q_out, a->q_out_stride, dq, 3, es, c->width), pages_view(c, false), pages_view(c, true)},
              {View(same ? nullptr : a->q, a->q_stride, dq, 3, 4, c->width), View(a->k, a->k_stride, dk, 3, 4, c->width), View(a->v, a->v_stride, dk, 3, 4, c->width), View(a->lens, 4 * B),
               View(a->counts, 4 * B), View(a->pos, 4 * B * a->tokens), View(a->cos, table), View(a->sin, table), View(a->q_norm, 4 * c->width), View(a->k_norm, 4 * c->width), tables_view(c)}))
        return P8_ERR_ARG;
    PagedAppendArgs k;
    const float *x[3] = {a->q, a->k, a->v};
    const int64_t *xs[3] = {a->q_stride, a->k_stride, a->v_stride}, *ps[2] = {c->k_stride, c->v_stride};
    for (int i = 0; i < 3; ++i) {
        k.x[i] = x[i];
        k.qs[i] = a->q_out_stride[i];
        for (int j = 0; j < 3; ++j) k.xs[i][j] = xs[i][j];
        for (int z = 0; z < 2; ++z) k.ps[z][i] = ps[z][1 + i];
    }
    k.q_out = a->q_out; k.kv[0] = c->k; k.kv[1] = c->v;
    k.tables = c->tables; k.ts = c->table_stride; k.lens = a->lens; k.counts = a->counts; k.pos = a->pos;
    k.cos = a->cos; k.sin = a->sin; k.qn = a->q_norm; k.kn = a->k_norm;
    k.positions = a->positions; k.slots = c->columns * c->page; k.div = page_div((uint32_t)c->page);
    k.tokens = (int)a->tokens; k.heads = (int)a->heads; k.kvh = (int)c->heads; k.batch = (int)B; k.pages = (int)c->pages; k.half = (int)a->rotary / 2;
    k.eps = (float)a->eps;
    const bool pairs = a->interleaved != 0;
    cudaStream_t st = (cudaStream_t)stream;
    return done(c->type == P8_KV_F32 ? run_paged_append<float>(c, k, pairs, st) : c->type == P8_KV_F16 ? run_paged_append<__half>(c, k, pairs, st) : run_paged_append<__nv_bfloat16>(c, k, pairs, st));
}

size_t p8_paged_attn_workspace(const p8_paged *c, int64_t heads) {
    if (!paged_ok(c) || c->layers != 1 || c->rows > P8_BATCH_MAX || !group_ok(c, heads)) return 0;
    return paged_attn_workspace(c, heads);
}

p8_status p8_paged_attn(const p8_paged *c, const p8_paged_attn_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    if (!paged_ok(c) || !a || c->layers != 1 || c->rows > P8_BATCH_MAX || !group_ok(c, a->heads)) return P8_ERR_ARG;
    if (!a->q || !a->out || !a->lens || !al16(a->q) || !al16(a->out) || !isfinite((float)a->scale * 1.4426950408889634f)) return P8_ERR_ARG;
    const int es = elem_size(c->type);
    const int64_t B = c->rows, dq[2] = {B, a->heads};
    if (!strides_ok(a->q_stride, dq, 2, es) || !strides_ok(a->out_stride, dq, 2, es)) return P8_ERR_ARG;
    const size_t need = paged_attn_workspace(c, a->heads);
    if (clash({View(a->out, a->out_stride, dq, 2, es, c->width), View(a->lse, 4 * B * a->heads), View(need && workspace_bytes >= need ? workspace : nullptr, (int64_t)need)},
              {View(a->q, a->q_stride, dq, 2, es, c->width), pages_view(c, false), pages_view(c, true), tables_view(c), View(a->lens, 4 * B), View(a->counts, 4 * B)}))
        return P8_ERR_ARG;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return P8_ERR_WORKSPACE;
    return launch_paged_attn(c, a, workspace, (cudaStream_t)stream);
}

size_t p8_beam_select_workspace(int64_t batch, int64_t beams, int64_t vocab, int64_t candidates) {
    if (!select_sizes_ok(batch, beams, vocab, candidates)) return 0;
    return select_workspace(batch, beams, vocab, candidates);
}

p8_status p8_beam_select(const p8_beam_select_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a || !select_sizes_ok(a->batch, a->beams, a->vocab, a->candidates) || !a->logits || !a->scores || !a->out_scores || !a->parents || !a->tokens) return P8_ERR_ARG;
    if (a->type != P8_KV_F32 && a->type != P8_KV_F16 && a->type != P8_KV_BF16) return P8_ERR_ARG;
    const int es = elem_size(a->type);
    if (((uintptr_t)a->logits & (es - 1)) || a->stride[0] < 0 || a->stride[1] < 0 || a->end >= a->vocab || (a->done && a->end < 0)) return P8_ERR_ARG;
    const size_t need = select_workspace(a->batch, a->beams, a->vocab, a->candidates);
    const int64_t BW = a->batch * a->beams, BN = a->batch * a->candidates, dims[2] = {a->batch, a->beams};
    if (clash({View(a->out_scores, 4 * BN), View(a->parents, 4 * BN), View(a->tokens, 8 * BN), View(a->out_done, BN), View(workspace_bytes >= need ? workspace : nullptr, (int64_t)need)},
              {View(a->logits, a->stride, dims, 2, es, a->vocab), View(a->scores, 4 * BW), View(a->done, BW)}))
        return P8_ERR_ARG;
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)) return P8_ERR_WORKSPACE;
    return launch_beam_select(a, workspace, (cudaStream_t)stream);
}

p8_status p8_beam_reorder(const p8_paged *c, const int32_t *parents, const int32_t *lens, int64_t batch, int64_t beams, void *stream) {
    if (!paged_ok(c) || !parents || !lens || batch < 1 || batch > P8_BATCH_MAX || beams < 1 || beams > P8_BEAMS_MAX || batch * beams != c->rows) return P8_ERR_ARG;
    if (c->rows > 1 && c->table_stride < c->columns) return P8_ERR_ARG;
    if (clash({tables_view(c), pages_view(c, false), pages_view(c, true)}, {View(parents, 4 * c->rows), View(lens, 4 * c->rows)})) return P8_ERR_ARG;
    return launch_beam_reorder(c, parents, lens, batch, beams, (cudaStream_t)stream);
}

}  // extern "C"
