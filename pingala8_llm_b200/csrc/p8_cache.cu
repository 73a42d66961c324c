// p8_cache.cu -- key/value cache operators: append (norm, rotation, write), eviction, tree acceptance, and the C ABI
// entry points of all five (the attention and mass kernels are in p8_tree_attn.cuh).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "p8_device.cuh"
#include "p8_internal.h"

namespace p8 {

// The operators' own error word (bits 64 and 128 of p8_device_error).
__device__ unsigned int g_cache_error = 0;
constexpr unsigned int kErrRange = 64u, kErrWait = 128u;

unsigned int read_and_clear_cache_error() {
    unsigned int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_cache_error, sizeof(v));
    cudaMemcpyToSymbol(g_cache_error, &z, sizeof(z));
    return v;
}

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Length of sequence b and its tokens in this call; false where they are out of range.
__device__ __forceinline__ bool seq_range(const int *lens, const int *counts, int b, int tokens, int64_t slots, int &len, int &n) {
    len = lens[b];
    n = counts ? counts[b] : tokens;
    return len >= 0 && n >= 0 && n <= tokens && (int64_t)len + n <= slots;
}

// four consecutive values, rounded to the cache's type
__device__ __forceinline__ void store4(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4]) {
    union { T t[4]; uint2 u; } r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.t[i] = from_f<T>(v[i]);
    *reinterpret_cast<uint2 *>(p) = r.u;
}

// Every launch here is one whose blocks may start while the launch before it in the stream ends (or, where that allows it
// early, still runs); before they read or write anything but their arguments they wait for all of it (after_prior). It
// saves the gap between dependent launches, 0.5 to 1 us of calls that take 2 to 10.
__device__ __forceinline__ void after_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ----------------------------------------------------------------------------------------------------------------
// append: y = rotate(norm(x)) per head of a token. A group of D / 8 lanes holds one head's row, lane l the values
// 4l..4l+3 of both halves, so a rotation pair is in one lane, the sum of squares is a butterfly over the group, and
// every access is 8 or 16 bytes wide. Bound by memory on a prompt (4,099 tokens x 48 heads of 128, 153 MB: 31 us, 4.9
// TB/s; 34.5 with the rows asked for only after the lengths and positions), by its one launch on a token (2.0 us).
struct AppendArgs {
    const float *x[3];          // q, k, v
    long long xs[3][3];
    void *y[3];                 // q_out, cache k, cache v
    long long ys[3][3];         // sequence, token (slot for the cache), head
    const int *lens, *counts, *pos;
    const float *cos, *sin, *qn, *kn;
    long long positions, slots;
    int tokens, heads, kvh, batch;
    float eps;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv_append(const AppendArgs a) {
    constexpr int L = D / 8, RPB = 256 / L;
    after_prior();
    const unsigned int rows = a.heads + 2 * a.kvh, id = blockIdx.x * RPB + threadIdx.x / L;
    const int l = threadIdx.x % L;
    const unsigned int tok = id / rows;
    if (tok >= (unsigned int)a.batch * a.tokens) return;  // a whole group of lanes leaves
    const int r = (int)(id - tok * rows), b = (int)(tok / (unsigned int)a.tokens), t = (int)(tok - (unsigned int)b * a.tokens);
    const int which = r < a.heads ? 0 : r < a.heads + a.kvh ? 1 : 2;
    const int h = which == 0 ? r : which == 1 ? r - a.heads : r - a.heads - a.kvh;
    // the row, the length and the position are asked for together: one round of latency before the table's
    const float *x = a.x[which] + b * a.xs[which][0] + t * a.xs[which][1] + h * a.xs[which][2] + 4 * l;
    float u[4], w[4];
    *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(x);
    *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(x + D / 2);
    const int p = a.pos[tok];
    int len, n;
    if (!seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n)) {
        if (t == 0 && r == 0 && l == 0) atomicOr(&g_cache_error, kErrRange);
        return;
    }
    if (t >= n) return;
    if (p < 0 || p >= a.positions) {
        if (r == 0 && l == 0) atomicOr(&g_cache_error, kErrRange);
        return;
    }
    if (which < 2) {
        float c[4], s[4];
        *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(a.cos + (long long)p * (D / 2) + 4 * l);
        *reinterpret_cast<float4 *>(s) = *reinterpret_cast<const float4 *>(a.sin + (long long)p * (D / 2) + 4 * l);
        const float *g = which == 0 ? a.qn : a.kn;
        if (g) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += u[i] * u[i] + w[i] * w[i];
            const unsigned int group = (L == 32 ? 0xffffffffu : (1u << L) - 1u) << (threadIdx.x % 32 / L * L);
#pragma unroll
            for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(group, ss, m);
            const float rs = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = u[i] * rs * g[4 * l + i];
                w[i] = w[i] * rs * g[4 * l + i + D / 2];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = u[i], x1 = w[i];
            u[i] = x0 * c[i] - x1 * s[i];
            w[i] = x1 * c[i] + x0 * s[i];
        }
    }
    T *y = static_cast<T *>(a.y[which]) + b * a.ys[which][0] + (which == 0 ? t : len + t) * a.ys[which][1] + h * a.ys[which][2] + 4 * l;
    store4(y, u);
    store4(y + D / 2, w);
}

// ----------------------------------------------------------------------------------------------------------------
// eviction, step 1: the kept slots of one (layer, sequence, head). A radix select on an order-preserving 32-bit key, in
// digits of 11, 11 and 10 bits, finds the smallest kept key; as soon as at most 1024 keys share its digits (after the
// first one, for most masses) only they are looked at. Then ballots and one scan over their counts give every kept slot
// its place, so that they come out in order and, among equal keys, the lowest slots win. Keys of up to 16384 slots stay in
// shared memory (two blocks an SM), longer middles are read again for each step. Bound by its dependent steps, and with
// many rows by the histogram's additions (two copies, for even and odd lanes, meet less often), not by the 4 bytes a slot.
struct EvictArgs {
    const float *mass;
    float *mass_out;
    long long ms[3], mos[3];
    const int *lens;
    int *new_lens, *kept;
    const char *src[2];
    char *dst[2];
    long long ss[2][4], ds[2][4];  // bytes: layer, sequence, head, slot
    long long slots;
    int batch, heads, budget, sinks, recent, row_bytes;
    int per_row;  // step 2: blocks of a row (all rows' blocks in one dimension of the grid: there may be more than 65,535 rows)
};

__device__ __forceinline__ uint32_t mass_key(float m) {  // larger mass, larger key; NaN as -infinity, -0 as +0
    if (isnan(m)) m = -INFINITY;
    m += 0.0f;
    const uint32_t u = __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelPiece = 16384, kSelFew = 1024, kSelBins = 2048, kSelCopy = kSelBins + 16;

__global__ void __launch_bounds__(1024, 2) k_evict_select(const EvictArgs a) {
    extern __shared__ uint32_t s_key[];  // kSelPiece
    __shared__ int hist[2 * kSelCopy];   // in the last step: ballots and counts
    __shared__ uint32_t few[kSelFew];
    __shared__ int wsum[32];
    __shared__ int s_digit, s_above, s_share, s_few, s_all;
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int h = row % a.heads, b = row / a.heads % a.batch, layer = row / a.heads / a.batch;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) s_few = 0;
    after_prior();
    const int len = a.lens[b];
    if (len < 0 || len > a.slots) {
        if (tid == 0) atomicOr(&g_cache_error, kErrRange);
        return;
    }
    if (layer == 0 && h == 0 && tid == 0) a.new_lens[b] = min(len, a.budget);
    int *kept = a.kept + (long long)row * a.budget;
    if (len <= a.budget) {
        for (int i = tid; i < a.budget; i += 1024) kept[i] = i < len ? i : -1;
        return;
    }
    const int need = a.budget - a.sinks - a.recent, lo = a.sinks, hi = len - a.recent, n = hi - lo;
    const float *m = a.mass + layer * a.ms[0] + b * a.ms[1] + h * a.ms[2] + lo;
    for (int i = tid; i < a.sinks; i += 1024) kept[i] = i;
    for (int i = tid; i < a.recent; i += 1024) kept[a.budget - a.recent + i] = hi + i;
    if (need == 0) return;
    const bool held = n <= kSelPiece;
    if (held) {
#pragma unroll 8
        for (int i = tid; i < n; i += 1024) s_key[i] = mass_key(m[i]);
    }
    uint32_t prefix = 0, fixed = 0;  // the threshold key's known bits, and which they are
    int left = need;                 // kept among the keys that share them
    bool in_few = false;             // those keys are in `few`
    int share = n;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : kSelBins;
        for (int i = tid; i < 2 * kSelCopy; i += 1024) hist[i] = 0;
        __syncthreads();
        int *mine = hist + (lane & 1) * kSelCopy;
        auto add = [&](uint32_t k) {
            if ((k & fixed) == prefix) atomicAdd(&mine[(k >> shift) & (bins - 1)], 1);
        };
        if (in_few) {
            if (tid < share) add(few[tid]);
        } else if (held) {
#pragma unroll 4
            for (int i = tid; i < n; i += 1024) add(s_key[i]);
        } else {
#pragma unroll 8
            for (int i = tid; i < n; i += 1024) add(mass_key(m[i]));
        }
        __syncthreads();
        // thread t holds two bins, counted from the top; a scan over them finds the digit where `left` falls
        const int hi_bin = bins - 1 - 2 * tid, lo_bin = hi_bin - 1;
        const int c0 = hi_bin > 0 ? hist[hi_bin] + hist[kSelCopy + hi_bin] : 0, c1 = hi_bin > 0 ? hist[lo_bin] + hist[kSelCopy + lo_bin] : 0;
        int sum = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) wsum[warp] = sum;
        __syncthreads();
        const int before = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0) + sum - c0 - c1;
        if (before < left && left <= before + c0) { s_digit = hi_bin; s_above = before; s_share = c0; }
        if (before + c0 < left && left <= before + c0 + c1) { s_digit = lo_bin; s_above = before + c0; s_share = c1; }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        fixed |= (uint32_t)(bins - 1) << shift;
        left -= s_above;
        if (!in_few) {
            share = s_share;
            if (pass < 2 && share <= kSelFew) {  // (in any order: only their values count from here on)
#pragma unroll 4
                for (int i = tid; i < n; i += 1024) {
                    const uint32_t k = held ? s_key[i] : mass_key(m[i]);
                    if ((k & fixed) == prefix) few[atomicAdd(&s_few, 1)] = k;
                }
                in_few = true;
            }
        }
    }
    // keys above `prefix` are kept, and the first `left` of those equal to it
    uint32_t *above = reinterpret_cast<uint32_t *>(hist), *equal = above + 512;  // ballots of 32 slots each
    int *count = hist + 1024;                                                    // their bits, above + 65536 equal; then the sums before them
    int gt0 = 0, eq0 = 0;                                                        // in the pieces before
    for (int piece = 0; piece < n; piece += kSelPiece) {
        const int groups = min(512, (n - piece + 31) / 32);
        __syncthreads();
#pragma unroll 4
        for (int w = warp; w < groups; w += 32) {
            const int i = piece + 32 * w + lane;
            const uint32_t k = i < n ? (held ? s_key[i] : mass_key(m[i])) : 0u;
            const unsigned int g = __ballot_sync(0xffffffffu, i < n && k > prefix), e = __ballot_sync(0xffffffffu, i < n && k == prefix);
            if (lane == 0) {
                above[w] = g;
                equal[w] = e;
                count[w] = __popc(g) | __popc(e) << 16;  // (at most 16384 each)
            }
        }
        __syncthreads();
        int own = 0, upto = 0;
        if (tid < 512) {
            own = upto = tid < groups ? count[tid] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            if (lane == 31) wsum[warp] = upto;
        }
        __syncthreads();
        if (tid < 512) {
            upto += __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0);
            count[tid] = upto - own;
            if (tid == 511) s_all = upto;
        }
        __syncthreads();
#pragma unroll 4
        for (int w = warp; w < groups; w += 32) {
            const uint32_t g = above[w], e = equal[w], below = (1u << lane) - 1u;
            const int c = count[w], eqs = eq0 + (c >> 16) + __popc(e & below);  // equal keys before this slot
            if ((g >> lane & 1) || ((e >> lane & 1) && eqs < left)) kept[a.sinks + gt0 + (c & 0xFFFF) + __popc(g & below) + min(eqs, left)] = lo + piece + 32 * w + lane;
        }
        gt0 += s_all & 0xFFFF;
        eq0 += s_all >> 16;
    }
}

// step 2, into other buffers: every row moves on its own, 16 bytes a thread. Bound by HBM (288 rows x 2,048 kept of 16,384
// slots, 604 MB: 105 to 110 us of the call's 136, 5.6 TB/s).
__global__ void __launch_bounds__(256) k_evict_copy(const EvictArgs a) {
    const int row = blockIdx.x / a.per_row, block = blockIdx.x - row * a.per_row, h = row % a.heads, b = row / a.heads % a.batch, layer = row / a.heads / a.batch;
    after_prior();  // every block: what follows in the stream waits for this launch alone
    const int len = a.lens[b];
    if (len < 0 || len > a.slots) return;
    const int keep = min(len, a.budget), per = a.row_bytes / 16, rows = 256 / per;
    const int *kept = a.kept + (long long)row * a.budget;
    const char *s0 = a.src[0] + layer * a.ss[0][0] + b * a.ss[0][1] + h * a.ss[0][2], *s1 = a.src[1] + layer * a.ss[1][0] + b * a.ss[1][1] + h * a.ss[1][2];
    char *d0 = a.dst[0] + layer * a.ds[0][0] + b * a.ds[0][1] + h * a.ds[0][2], *d1 = a.dst[1] + layer * a.ds[1][0] + b * a.ds[1][1] + h * a.ds[1][2];
    const int unit = 16 * (threadIdx.x % per);
    const int first = block * rows * 4 + threadIdx.x / per;
    uint4 x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = first + j * rows;
        if (i < keep) {
            const long long s = kept[i];
            x[j] = *reinterpret_cast<const uint4 *>(s0 + s * a.ss[0][3] + unit);
            y[j] = *reinterpret_cast<const uint4 *>(s1 + s * a.ss[1][3] + unit);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = first + j * rows;
        if (i < keep) {
            *reinterpret_cast<uint4 *>(d0 + i * a.ds[0][3] + unit) = x[j];
            *reinterpret_cast<uint4 *>(d1 + i * a.ds[1][3] + unit) = y[j];
        }
    }
    for (int i = block * rows * 4 + threadIdx.x; i < min(keep, (block + 1) * rows * 4); i += 256)
        a.mass_out[layer * a.mos[0] + b * a.mos[1] + h * a.mos[2] + i] = a.mass[layer * a.ms[0] + b * a.ms[1] + h * a.ms[2] + kept[i]];
}

// step 2 in place: kept[i] >= i, so a block that goes up through a range of the row's bytes (64 of them: its columns
// belong to no other block), reads a chunk of sources before it writes their destinations, and reads the next chunk
// (sources at or behind every destination written so far) meanwhile, loses nothing. blockIdx.y 0 / 1: keys / values,
// 2: the masses. Bound by its rounds of latency, eight for 2,048 kept rows of 256 bytes: one layer of 2,112 slots x 8 heads takes 17
// us, 36 layers of 16,384 slots 151, with the select before it.
template <typename U>
__device__ __forceinline__ void evict_slide(const char *base, long long stride, int per, int keep, const int *kept) {
    constexpr int kRows = 4;
    const int lanes = 256 / per, unit = threadIdx.x % per, r0 = threadIdx.x / per;
    char *p = const_cast<char *>(base) + (long long)unit * sizeof(U);
    U cur[kRows];
    int src[kRows], nxt[kRows];
    U ahead[kRows];
    const int step = lanes * kRows;
    auto fetch = [&](int i0, U (&v)[kRows], int (&s)[kRows]) {
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int i = i0 + j * lanes + r0;
            s[j] = i < keep ? kept[i] : -1;
            if (s[j] > i) v[j] = *reinterpret_cast<const U *>(p + s[j] * stride);
        }
    };
    fetch(0, cur, src);
    for (int i0 = 0; i0 < keep; i0 += step) {
        fetch(i0 + step, ahead, nxt);
        __syncthreads();  // every thread has read this chunk and the next
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int i = i0 + j * lanes + r0;
            if (src[j] > i) *reinterpret_cast<U *>(p + i * stride) = cur[j];
            cur[j] = ahead[j];
            src[j] = nxt[j];
        }
    }
}

__global__ void __launch_bounds__(256) k_evict_slide(const EvictArgs a) {
    const int row = blockIdx.x / a.per_row, block = blockIdx.x - row * a.per_row, h = row % a.heads, b = row / a.heads % a.batch, layer = row / a.heads / a.batch;
    after_prior();
    const int len = a.lens[b];
    if (len <= a.budget || len > a.slots) return;
    const int *kept = a.kept + (long long)row * a.budget;
    const int z = blockIdx.y;
    if (z == 2) {
        if (block == 0)
            evict_slide<float>(reinterpret_cast<const char *>(a.mass + layer * a.ms[0] + b * a.ms[1] + h * a.ms[2]), 4, 1, a.budget, kept);
        return;
    }
    evict_slide<uint4>(a.src[z] + layer * a.ss[z][0] + b * a.ss[z][1] + h * a.ss[z][2] + 64 * block, a.ss[z][3], 4, a.budget, kept);
}

// ----------------------------------------------------------------------------------------------------------------
// acceptance: one block per (layer, sequence, keys or values). Each finds the path on its own (the first warp, two
// nodes a lane, one ballot per step: cheaper than a launch between the walk and the moves), then moves the rows of all
// heads in chunks, reading a chunk before writing it: path[i] >= i and the chunks go up, so no source is lost. Bound by two
// rounds of latency and the launch: 2.4 us for 36 layers and 8 drafted tokens, 6.8 us for 32 layers x 16 sequences.
struct AcceptArgs {
    const long long *tokens, *target;
    const int *parents, *lens, *counts;
    int *path, *accepted, *new_lens;
    long long *next;
    char *kv[2];
    long long st[2][4];  // bytes
    long long slots;
    int T, batch, heads, row_bytes;
};

__global__ void __launch_bounds__(256) k_tree_accept(const AcceptArgs a) {
    __shared__ int path[P8_TREE_MAX];
    __shared__ int s_n;
    const int b = blockIdx.x % a.batch, z = blockIdx.x / a.batch % 2, layer = blockIdx.x / a.batch / 2;
    const int tid = threadIdx.x;
    const bool report = layer == 0 && z == 0;
    after_prior();
    int len, n;
    const bool ok = seq_range(a.lens, a.counts, b, a.T, a.slots, len, n);
    if (tid < 32) {
        const long long at = (long long)b * a.T;
        int par[2];
        bool fits[2];
        long long tok[2], tgt[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // the whole tree at once; a parent's target comes from its lane
            const int c = tid + 32 * k;
            par[k] = c < a.T ? a.parents[at + c] : -1;
            tok[k] = c < a.T ? a.tokens[at + c] : 0;
            tgt[k] = c < a.T ? a.target[at + c] : 0;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = tid + 32 * k;
            const long long t0 = __shfl_sync(0xffffffffu, tgt[0], par[k] & 31), t1 = __shfl_sync(0xffffffffu, tgt[1], par[k] & 31);
            fits[k] = ok && c < n && par[k] >= 0 && par[k] < c && tok[k] == (par[k] < 32 ? t0 : t1);
        }
        int cur = 0, cnt = ok && n > 0 ? 1 : 0;
        if (tid == 0) path[0] = 0;
        while (cnt) {
            const unsigned int m0 = __ballot_sync(0xffffffffu, fits[0] && par[0] == cur);
            const unsigned int m1 = __ballot_sync(0xffffffffu, fits[1] && par[1] == cur);
            if (!(m0 | m1)) break;
            cur = m0 ? __ffs(m0) - 1 : 31 + __ffs(m1);  // parents come first, so cur grows and the walk ends
            if (tid == 0) path[cnt] = cur;
            ++cnt;
        }
        __syncwarp();
        if (tid == 0) s_n = cnt;
        if (report) {
            for (int t = tid; t < a.T; t += 32) a.path[at + t] = t < cnt ? path[t] : -1;
            if (tid == 0) {
                a.accepted[b] = cnt;
                a.new_lens[b] = len + cnt;
                a.next[b] = cnt ? a.target[at + cur] : -1;
                if (!ok) atomicOr(&g_cache_error, kErrRange);
            }
        }
    }
    __syncthreads();
    const int cnt = s_n, per = a.row_bytes / 16, items = (cnt - 1) * a.heads * per;
    char *base = a.kv[z] + layer * a.st[z][0] + b * a.st[z][1] + len * a.st[z][3];
    for (int i0 = 0; i0 < items; i0 += 1024) {
        uint4 v[4];
        char *to[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * 256 + tid;
            to[j] = nullptr;
            if (i < items) {
                const int unit = i % per, h = i / per % a.heads, r = i / per / a.heads + 1;
                char *p = base + h * a.st[z][2] + 16 * unit;
                if (path[r] != r) {
                    v[j] = *reinterpret_cast<const uint4 *>(p + path[r] * a.st[z][3]);
                    to[j] = p + r * a.st[z][3];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (to[j]) *reinterpret_cast<uint4 *>(to[j]) = v[j];
    }
}

#include "p8_tree_attn.cuh"

// ----------------------------------------------------------------------------------------------------------------
// host side: argument checks (nothing below them touches the device before they pass) and launches
int elem_size(int64_t type) { return type == P8_KV_F32 ? 4 : 2; }
bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }
// strides (elements) of the dimensions that are used, as multiples of 16 bytes
bool strides_ok(const int64_t *st, const int64_t *dims, int n, int es) {
    for (int i = 0; i < n; ++i)
        if (dims[i] > 1 && (st[i] <= 0 || (st[i] * es) % 16)) return false;
    return true;
}

bool kv_ok(const p8_kv *c, bool values = true) {
    if (!c || !c->k || (values && !c->v) || !al16(c->k) || !al16(c->v)) return false;
    if (c->type != P8_KV_F32 && c->type != P8_KV_F16 && c->type != P8_KV_BF16) return false;
    if (c->width != 64 && c->width != 128) return false;
    if (c->layers < 1 || c->batch < 1 || c->batch > P8_BATCH_MAX || c->heads < 1 || c->slots < 1 || c->slots > P8_SLOTS_MAX) return false;
    if (c->heads > 65535 || c->layers > 65535 || c->layers * c->batch * c->heads > (int64_t(1) << 30)) return false;
    const int64_t dims[4] = {c->layers, c->batch, c->heads, c->slots};
    const int es = elem_size(c->type);
    return strides_ok(c->k_stride, dims, 4, es) && (!values || strides_ok(c->v_stride, dims, 4, es));
}
bool heads_ok(const p8_kv *c, int64_t heads) { return heads >= c->heads && heads % c->heads == 0 && heads <= 65535; }

bool scale_ok(double scale) { return isfinite((float)scale * 1.4426950408889634f); }  // in base 2, in the kernels' 32 bits

p8_status done(cudaError_t e) { return e == cudaSuccess ? P8_OK : P8_ERR_CUDA; }

template <typename T>
cudaError_t run_append(const p8_kv *c, const AppendArgs &a, cudaStream_t st) {
    const long long rows = (long long)a.batch * a.tokens * (a.heads + 2 * a.kvh), per = 256 / (c->width / 8);
    const dim3 grid((unsigned int)((rows + per - 1) / per));
    return launch_after(c->width == 128 ? k_kv_append<T, 128> : k_kv_append<T, 64>, grid, dim3(256), 0, st, a);
}

// A buffer as a call uses it: rows of `last` bytes at at + sum of i_k st[k], 0 <= i_k < dims[k].
// One whose address is NULL is not there.
struct View {
    uintptr_t at, lo, hi;  // [lo, hi): from the first of its bytes to the last
    int n;
    int64_t dims[4], st[4], last;
    View(const void *p, int64_t bytes) : at((uintptr_t)p), lo(at), hi(at + (uintptr_t)(p ? bytes : 0)), n(0), last(bytes) {}
    View(const void *p, const int64_t *strides, const int64_t *counts, int dimensions, int es, int64_t elements) : View(p, elements * es) {
        n = dimensions;
        for (int i = 0; i < n; ++i) {
            dims[i] = counts[i];
            st[i] = strides[i] * es;
            if (p) (st[i] < 0 ? lo : hi) += (uintptr_t)(st[i] * (dims[i] - 1));
        }
    }
    // Whether its rows may share bytes: each used stride has to step over all that the smaller ones reach, as the strides of every
    // slice and every order of a dense array's dimensions do.
    bool folds() const {
        int64_t reach = last;
        bool seen[4] = {};
        for (int k = 0; k < n; ++k) {
            int least = -1;
            for (int i = 0; i < n; ++i)
                if (!seen[i] && dims[i] > 1 && (least < 0 || std::abs(st[i]) < std::abs(st[least]))) least = i;
            if (least < 0) break;
            if (std::abs(st[least]) < reach) return true;
            seen[least] = true;
            reach += std::abs(st[least]) * (dims[least] - 1);
        }
        return false;
    }
};
// Terms c s with lo <= c <= hi, of which one sum between `least` and `most` is looked for, the largest strides first. Views
// cut from one buffer have strides that nest, which leaves one or two values for each; where there are more than `looks` in all the answer is yes.
struct Term { int64_t s, lo, hi; };
bool reaches(const Term *t, int n, int64_t least, int64_t most, int &looks) {
    if (n == 0) return least <= 0 && 0 <= most;
    int64_t lo = 0, hi = 0;  // what the others can come to
    for (int i = 1; i < n; ++i) { lo += t[i].lo * t[i].s; hi += t[i].hi * t[i].s; }
    const int64_t s = t->s;
    const auto down = [s](int64_t a) { return a / s - (a % s < 0); };
    const int64_t from = std::max(t->lo, -down(hi - least)), to = std::min(t->hi, down(most - lo));
    for (int64_t c = from; c <= to; ++c) {
        if (--looks < 0 || reaches(t + 1, n - 1, least - c * s, most - c * s, looks)) return true;
    }
    return false;
}
// whether two views share bytes; what lies between the rows of one may belong to the other
bool overlap(const View &x, const View &y) {
    if (x.lo >= y.hi || y.lo >= x.hi) return false;
    Term t[8] = {};  // by strides, the largest first
    int n = 0;
    const auto add = [&](int64_t st, int64_t most, int sign) {
        if (st == 0 || most == 0) return;
        const int64_t s = st < 0 ? -st : st;
        if (st < 0) sign = -sign;
        int i = 0;
        while (i < n && t[i].s > s) ++i;
        if (i == n || t[i].s != s) {
            for (int j = n++; j > i; --j) t[j] = t[j - 1];
            t[i] = {s, 0, 0};
        }
        (sign > 0 ? t[i].hi : t[i].lo) += sign * most;
    };
    for (int i = 0; i < x.n; ++i) add(x.st[i], x.dims[i] - 1, 1);
    for (int i = 0; i < y.n; ++i) add(y.st[i], y.dims[i] - 1, -1);
    const int64_t off = (int64_t)(y.at - x.at);  // a row of x and one of y share bytes where the rows' difference is within (off - x.last, off + y.last)
    int looks = 1000;
    return reaches(t, n, off - x.last + 1, off + y.last - 1, looks);
}
// whether a call would write to what it reads or to one place twice
bool clash(std::initializer_list<View> out, std::initializer_list<View> in) {
    for (const View *x = out.begin(); x != out.end(); ++x) {
        if (x->at && x->folds()) return true;
        for (const View *y = x + 1; y != out.end(); ++y)
            if (overlap(*x, *y)) return true;
        for (const View &y : in)
            if (overlap(*x, y)) return true;
    }
    return false;
}
// whether two views of the same sizes are one: a dimension of one has no stride to speak of
bool same_strides(const int64_t *a, const int64_t *b, const int64_t *dims, int n) {
    for (int i = 0; i < n; ++i)
        if (dims[i] > 1 && a[i] != b[i]) return false;
    return true;
}
}  // namespace
}  // namespace p8

using namespace p8;

extern "C" {

p8_status p8_cache_wait_limit(int64_t ns) {
    if (ns < 0 || ns > UINT32_MAX) return P8_ERR_ARG;
    g_wait_ns.store((unsigned int)ns, std::memory_order_relaxed);
    return P8_OK;
}

p8_status p8_kv_append(const p8_kv *c, const p8_kv_append_args *a, void *stream) {
    if (!kv_ok(c) || !a || c->layers != 1 || !heads_ok(c, a->heads)) return P8_ERR_ARG;
    if (a->tokens < 0) return P8_ERR_ARG;
    if (a->tokens == 0) return P8_OK;  // buffers of nothing may have no address
    if (!a->q || !a->k || !a->v || !a->q_out || !a->lens || !a->pos || !a->cos || !a->sin || a->positions < 1) return P8_ERR_ARG;
    if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->q_out) || !al16(a->cos) || !al16(a->sin) || !(a->eps >= 0.0)) return P8_ERR_ARG;
    if (a->tokens > c->slots || c->batch * a->tokens * (a->heads + 2 * c->heads) > (int64_t(1) << 31) - 64) return P8_ERR_ARG;
    const int es = elem_size(c->type);
    const int64_t dq[3] = {c->batch, a->tokens, a->heads}, dk[3] = {c->batch, a->tokens, c->heads};
    if (!strides_ok(a->q_stride, dq, 3, 4) || !strides_ok(a->k_stride, dk, 3, 4) || !strides_ok(a->v_stride, dk, 3, 4) ||
        !strides_ok(a->q_out_stride, dq, 3, es))
        return P8_ERR_ARG;
    // in place: every lane writes what it has read
    const bool same = c->type == P8_KV_F32 && (const void *)a->q == a->q_out && same_strides(a->q_stride, a->q_out_stride, dq, 3);
    const int64_t dkv[3] = {c->batch, c->heads, c->slots}, B = c->batch, table = a->positions * (c->width / 2) * 4;
    const View q(same ? nullptr : a->q, a->q_stride, dq, 3, 4, c->width);
    if (clash({View(a->q_out, a->q_out_stride, dq, 3, es, c->width), View(c->k, c->k_stride + 1, dkv, 3, es, c->width), View(c->v, c->v_stride + 1, dkv, 3, es, c->width)},
              {q, View(a->k, a->k_stride, dk, 3, 4, c->width), View(a->v, a->v_stride, dk, 3, 4, c->width), View(a->lens, 4 * B), View(a->counts, 4 * B),
               View(a->pos, 4 * B * a->tokens), View(a->cos, table), View(a->sin, table), View(a->q_norm, 4 * c->width), View(a->k_norm, 4 * c->width)}))
        return P8_ERR_ARG;
    AppendArgs k;
    const float *x[3] = {a->q, a->k, a->v};
    const int64_t *xs[3] = {a->q_stride, a->k_stride, a->v_stride};
    for (int i = 0; i < 3; ++i) {
        k.x[i] = x[i];
        for (int j = 0; j < 3; ++j) k.xs[i][j] = xs[i][j];
    }
    k.y[0] = a->q_out; k.y[1] = c->k; k.y[2] = c->v;
    for (int j = 0; j < 3; ++j) k.ys[0][j] = a->q_out_stride[j];
    const int64_t *cs[2] = {c->k_stride, c->v_stride};
    for (int i = 0; i < 2; ++i) { k.ys[1 + i][0] = cs[i][1]; k.ys[1 + i][1] = cs[i][3]; k.ys[1 + i][2] = cs[i][2]; }
    k.lens = a->lens; k.counts = a->counts; k.pos = a->pos;
    k.cos = a->cos; k.sin = a->sin; k.qn = a->q_norm; k.kn = a->k_norm;
    k.positions = a->positions; k.slots = c->slots;
    k.tokens = (int)a->tokens; k.heads = (int)a->heads; k.kvh = (int)c->heads; k.batch = (int)c->batch;
    k.eps = (float)a->eps;
    cudaStream_t st = (cudaStream_t)stream;
    return done(c->type == P8_KV_F32 ? run_append<float>(c, k, st) : c->type == P8_KV_F16 ? run_append<__half>(c, k, st) : run_append<__nv_bfloat16>(c, k, st));
}

size_t p8_tree_attn_workspace(const p8_kv *c, int64_t tokens, int64_t heads) {
    if (!kv_ok(c) || c->layers != 1 || tokens < 1 || tokens > P8_TREE_MAX || !heads_ok(c, heads)) return 0;
    return tree_attn_workspace(c, tokens, heads);
}

p8_status p8_tree_attn(const p8_kv *c, const p8_tree_attn_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    if (!kv_ok(c) || !a || c->layers != 1 || !heads_ok(c, a->heads)) return P8_ERR_ARG;
    if (!a->q || !a->out || !a->lens || a->tokens < 1 || a->tokens > P8_TREE_MAX || !al16(a->q) || !al16(a->out)) return P8_ERR_ARG;
    if (!scale_ok(a->scale) || (a->mask && a->mask_stride != 0 && a->mask_stride != a->tokens)) return P8_ERR_ARG;
    const int es = elem_size(c->type);
    const int64_t dq[3] = {c->batch, a->tokens, a->heads};
    if (!strides_ok(a->q_stride, dq, 3, es) || !strides_ok(a->out_stride, dq, 3, es)) return P8_ERR_ARG;
    const int64_t dkv[3] = {c->batch, c->heads, c->slots};
    const size_t need = tree_attn_workspace(c, a->tokens, a->heads);
    const int64_t B = c->batch, T = a->tokens;
    if (clash({View(a->out, a->out_stride, dq, 3, es, c->width), View(a->lse, 4 * B * T * a->heads), View(need && workspace_bytes >= need ? workspace : nullptr, (int64_t)need)},
              {View(a->q, a->q_stride, dq, 3, es, c->width), View(c->k, c->k_stride + 1, dkv, 3, es, c->width), View(c->v, c->v_stride + 1, dkv, 3, es, c->width),
               View(a->lens, 4 * B), View(a->counts, 4 * B), View(a->mask, 8 * T * (a->mask_stride ? B : 1))}))
        return P8_ERR_ARG;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return P8_ERR_WORKSPACE;
    return launch_tree_attn(c, a, workspace, (cudaStream_t)stream);
}

p8_status p8_attn_mass(const p8_kv *c, const p8_attn_mass_args *a, void *stream) {
    if (!kv_ok(c, false) || !a || c->layers != 1 || !heads_ok(c, a->heads)) return P8_ERR_ARG;
    if (!a->q || !a->lse || !a->lens || !a->mass || !a->out || a->tokens < 1 || a->tokens > P8_TREE_MAX || !al16(a->q)) return P8_ERR_ARG;
    if (!scale_ok(a->scale)) return P8_ERR_ARG;
    const int64_t dq[3] = {c->batch, a->tokens, a->heads};
    if (!strides_ok(a->q_stride, dq, 3, elem_size(c->type))) return P8_ERR_ARG;
    const int64_t dm[3] = {c->batch, c->heads, c->slots}, m3[2] = {a->mass_stride[0], a->mass_stride[1]}, o3[2] = {a->out_stride[0], a->out_stride[1]};
    const bool same = a->mass == a->out && same_strides(m3, o3, dm, 2);
    const int64_t B = c->batch, T = a->tokens;
    if (clash({View(a->out, o3, dm, 2, 4, c->slots)},
              {View(same ? nullptr : a->mass, m3, dm, 2, 4, c->slots), View(a->q, a->q_stride, dq, 3, elem_size(c->type), c->width), View(a->lse, 4 * B * T * a->heads),
               View(c->k, c->k_stride + 1, dm, 3, elem_size(c->type), c->width), View(a->lens, 4 * B), View(a->counts, 4 * B), View(a->rows, 4 * B * T)}))
        return P8_ERR_ARG;
    return launch_attn_mass(c, a, (cudaStream_t)stream);
}

p8_status p8_kv_evict(const p8_kv *s, const p8_kv *d, const p8_kv_evict_args *a, void *stream) {
    if (!kv_ok(s) || !kv_ok(d) || !a || !a->mass || !a->mass_out || !a->lens || !a->new_lens || !a->kept) return P8_ERR_ARG;
    if (s->type != d->type || s->width != d->width || s->layers != d->layers || s->batch != d->batch || s->heads != d->heads) return P8_ERR_ARG;
    if (a->budget < 1 || a->sinks < 0 || a->recent < 0 || a->sinks > a->budget || a->recent > a->budget - a->sinks || a->budget > d->slots ||
        a->budget > s->slots)
        return P8_ERR_ARG;
    const int es = elem_size(s->type);
    const int64_t dims[4] = {s->layers, s->batch, s->heads, s->slots}, ddims[4] = {s->layers, s->batch, s->heads, a->budget};
    // in place: all three buffers and their strides the same; else no overlap at all
    const bool same = s->k == d->k && s->v == d->v && a->mass == a->mass_out && same_strides(s->k_stride, d->k_stride, dims, 4) &&
                      same_strides(s->v_stride, d->v_stride, dims, 4) && same_strides(a->mass_stride, a->mass_out_stride, dims, 3);
    const int64_t B = s->batch;
    const View sk(s->k, s->k_stride, dims, 4, es, s->width), sv(s->v, s->v_stride, dims, 4, es, s->width), sm(a->mass, a->mass_stride, dims, 3, 4, s->slots);
    const View dk(d->k, d->k_stride, ddims, 4, es, s->width), dv(d->v, d->v_stride, ddims, 4, es, s->width), dm(a->mass_out, a->mass_out_stride, dims, 3, 4, a->budget);
    const View lens(a->lens, 4 * B), new_lens(a->new_lens, 4 * B), kept(a->kept, 4 * s->layers * B * s->heads * a->budget);
    if (same ? clash({new_lens, kept, sk, sv, sm}, {lens}) : clash({new_lens, kept, dk, dv, dm}, {lens, sk, sv, sm})) return P8_ERR_ARG;
    EvictArgs k;
    k.mass = a->mass; k.mass_out = a->mass_out;
    for (int i = 0; i < 3; ++i) { k.ms[i] = a->mass_stride[i]; k.mos[i] = a->mass_out_stride[i]; }
    k.lens = a->lens; k.new_lens = a->new_lens; k.kept = a->kept;
    k.src[0] = (const char *)s->k; k.src[1] = (const char *)s->v; k.dst[0] = (char *)d->k; k.dst[1] = (char *)d->v;
    for (int i = 0; i < 4; ++i) {
        k.ss[0][i] = s->k_stride[i] * es; k.ss[1][i] = s->v_stride[i] * es;
        k.ds[0][i] = d->k_stride[i] * es; k.ds[1][i] = d->v_stride[i] * es;
    }
    k.slots = s->slots; k.batch = (int)s->batch; k.heads = (int)s->heads;
    k.budget = (int)a->budget; k.sinks = (int)a->sinks; k.recent = (int)a->recent; k.row_bytes = (int)s->width * es;
    const int64_t rows = s->layers * s->batch * s->heads;
    const int chunk = 4 * (256 / (k.row_bytes / 16));
    k.per_row = same ? k.row_bytes / 64 : (int)((a->budget + chunk - 1) / chunk);
    if (rows * k.per_row > INT32_MAX) return P8_ERR_UNSUPPORTED;
    cudaStream_t st = (cudaStream_t)stream;
    // Keys go to shared memory as far as a middle can be long. Beside the kernel's own 22 KB, more than 24 KB needs the limit
    // raised; on every call, since it is the device's.
    const int64_t most = s->slots - a->sinks - a->recent;
    const int smem = (int)std::min<int64_t>(std::max<int64_t>(most, 0), kSelPiece) * 4;
    if (smem > 24 * 1024 && cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelPiece * 4) != cudaSuccess) return P8_ERR_CUDA;
    if (launch_after(k_evict_select, dim3((unsigned int)rows), dim3(1024), (size_t)smem, st, k) != cudaSuccess) return P8_ERR_CUDA;
    return done(launch_after(same ? k_evict_slide : k_evict_copy, dim3((unsigned int)(rows * k.per_row), same ? 3 : 1), dim3(256), 0, st, k));
}

p8_status p8_tree_accept(const p8_kv *c, const p8_tree_accept_args *a, void *stream) {
    if (!kv_ok(c) || !a || !a->tokens || !a->target || !a->parents || !a->lens || !a->path || !a->accepted || !a->new_lens || !a->next_token)
        return P8_ERR_ARG;
    if (a->ntokens < 1 || a->ntokens > P8_TREE_MAX) return P8_ERR_ARG;
    const int es = elem_size(c->type);
    // every block reads the tree, and one writes the results: no order is between them
    const int64_t dims[4] = {c->layers, c->batch, c->heads, c->slots}, B = c->batch, BT = B * a->ntokens;
    if (clash({View(a->path, 4 * BT), View(a->accepted, 4 * B), View(a->new_lens, 4 * B), View(a->next_token, 8 * B), View(c->k, c->k_stride, dims, 4, es, c->width),
               View(c->v, c->v_stride, dims, 4, es, c->width)},
              {View(a->tokens, 8 * BT), View(a->target, 8 * BT), View(a->parents, 4 * BT), View(a->lens, 4 * B), View(a->counts, 4 * B)}))
        return P8_ERR_ARG;
    AcceptArgs k;
    k.tokens = (const long long *)a->tokens; k.target = (const long long *)a->target; k.next = (long long *)a->next_token;
    k.parents = a->parents; k.lens = a->lens; k.counts = a->counts;
    k.path = a->path; k.accepted = a->accepted; k.new_lens = a->new_lens;
    k.kv[0] = (char *)c->k; k.kv[1] = (char *)c->v;
    for (int i = 0; i < 4; ++i) { k.st[0][i] = c->k_stride[i] * es; k.st[1][i] = c->v_stride[i] * es; }
    k.slots = c->slots; k.T = (int)a->ntokens; k.batch = (int)c->batch; k.heads = (int)c->heads; k.row_bytes = (int)c->width * es;
    return done(launch_after(k_tree_accept, dim3((unsigned int)(c->layers * c->batch * 2)), dim3(256), 0, (cudaStream_t)stream, k));
}

}  // extern "C"
