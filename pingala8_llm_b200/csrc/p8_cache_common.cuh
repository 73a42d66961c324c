// p8_cache_common.cuh -- what the cache operators' files share: conversions, dependent launches, and the host's checks of buffers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <algorithm>
#include <initializer_list>

#include "pingala8.h"

namespace p8 {
constexpr unsigned int kErrRange = 64u, kErrWait = 128u;  // of p8_device_error

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

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
// host side
int elem_size(int64_t type) { return type == P8_KV_F32 ? 4 : 2; }
bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }
// strides (elements) of the dimensions that are used, as multiples of 16 bytes
bool strides_ok(const int64_t *st, const int64_t *dims, int n, int es) {
    for (int i = 0; i < n; ++i)
        if (dims[i] > 1 && (st[i] <= 0 || (st[i] * es) % 16)) return false;
    return true;
}

p8_status done(cudaError_t e) { return e == cudaSuccess ? P8_OK : P8_ERR_CUDA; }

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
