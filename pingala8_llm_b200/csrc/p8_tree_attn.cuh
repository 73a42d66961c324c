// p8_tree_attn.cuh -- attention of a tree of drafted tokens over a cache, and the attention mass per slot (included by
// p8_cache.cu).
#pragma once

struct AttnArgs {
    const void *q, *k, *v;
    long long qs[3], ks[3], vs[3], os[3];  // q, out: sequence, token, head; k, v: sequence, head, slot
    const int *lens, *counts, *rows;
    const unsigned long long *mask;
    long long mask_stride, slots;
    void *out;
    float *lse;
    const float *lse_in, *mass;
    float *mass_out;
    long long ms[2], mos[2];
    int batch, tokens, heads, kvh, group;
    float scale;
};

// One block per (sequence, cache head, eight query rows): a running maximum and sum over tiles of 32 slots, products on
// the CUDA cores. Simple, and right for every type.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_tree_attn_plain(const AttnArgs a) {
    constexpr int R = 8, KT = 32;
    __shared__ float sq[R][D], sk[KT][D + 1], sp[R][KT], sv[KT][D];
    __shared__ float s_m[R], s_l[R], s_c[R];
    const int b = blockIdx.z, h = blockIdx.y, r0 = blockIdx.x * R, tid = threadIdx.x;
    int len, n;
    if (!seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n)) {
        if (r0 == 0 && h == 0 && tid == 0) atomicOr(&g_cache_error, kErrRange);
        return;
    }
    const int rows = n * a.group;
    if (r0 >= rows) return;
    for (int i = tid; i < R * D; i += 128) {
        const int r = r0 + i / D;
        sq[i / D][i % D] = r < rows ? to_f(static_cast<const T *>(a.q)[b * a.qs[0] + r / a.group * a.qs[1] + (h * a.group + r % a.group) * a.qs[2] + i % D]) : 0.f;
    }
    if (tid < R) { s_m[tid] = -INFINITY; s_l[tid] = 0.f; }
    float acc[R] = {};
    const int end = len + n;
    const T *K = static_cast<const T *>(a.k) + b * a.ks[0] + h * a.ks[1], *V = static_cast<const T *>(a.v) + b * a.vs[0] + h * a.vs[1];
    for (int j0 = 0; j0 < end; j0 += KT) {
        __syncthreads();
        for (int i = tid; i < KT * D; i += 128) {
            const int j = j0 + i / D;
            sk[i / D][i % D] = j < end ? to_f(K[j * a.ks[2] + i % D]) : 0.f;
            sv[i / D][i % D] = j < end ? to_f(V[j * a.vs[2] + i % D]) : 0.f;
        }
        __syncthreads();
        const int j = j0 + tid % KT;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const int r = tid / KT * 2 + rr, t = (r0 + r) / a.group;
            float s = 0.f;
            for (int d = 0; d < D; ++d) s += sq[r][d] * sk[tid % KT][d];
            bool see = r0 + r < rows && j < end;
            if (see && j >= len) see = a.mask ? (a.mask[b * a.mask_stride + t] >> (j - len)) & 1 : j - len <= t;
            s = see ? s * a.scale : -INFINITY;
            float top = s;
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            const float m0 = s_m[r], m1 = fmaxf(m0, top);
            const float p = see ? expf(s - m1) : -1.f;
            float sum = see ? p : 0.f;
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            __syncwarp();
            sp[r][tid % KT] = p;
            if (tid % KT == 0) {
                s_c[r] = m1 == -INFINITY ? 1.f : expf(m0 - m1);
                s_l[r] = s_l[r] * s_c[r] + sum;
                s_m[r] = m1;
            }
        }
        __syncthreads();
        for (int r = 0; r < R; ++r) {
            if (tid < D) {
                float x = acc[r] * s_c[r];
                for (int i = 0; i < KT; ++i)
                    if (sp[r][i] >= 0.f || isnan(sp[r][i])) x += sp[r][i] * sv[i][tid];
                acc[r] = x;
            }
        }
    }
    __syncthreads();
    for (int r = 0; r < R && r0 + r < rows; ++r) {
        const int t = (r0 + r) / a.group, i = h * a.group + (r0 + r) % a.group;
        if (tid < D) static_cast<T *>(a.out)[b * a.os[0] + t * a.os[1] + i * a.os[2] + tid] = from_f<T>(s_m[r] == -INFINITY ? 0.f : acc[r] / s_l[r]);
        if (a.lse && tid == 0) a.lse[((long long)b * a.tokens + t) * a.heads + i] = s_m[r] == -INFINITY ? -INFINITY : s_m[r] + logf(s_l[r]);
    }
}

// One thread per slot: the query rows pass through shared memory, the slot's key stays in registers as it was read.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_attn_mass_plain(const AttnArgs a) {
    __shared__ float sq[8][D], sl[8];
    __shared__ int st[8];
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    int len, n;
    if (!seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n)) {
        if (blockIdx.x == 0 && h == 0 && tid == 0) atomicOr(&g_cache_error, kErrRange);
        return;
    }
    const int end = len + n;
    const T *K = static_cast<const T *>(a.k) + b * a.ks[0] + h * a.ks[1];
    for (int j0 = blockIdx.x * 128; j0 < end; j0 += gridDim.x * 128) {
        const int j = j0 + tid;
        float w = 0.f;
        for (int r0 = 0; r0 < n * a.group; r0 += 8) {
            __syncthreads();
            for (int i = tid; i < 8 * D; i += 128) {
                const int r = r0 + i / D, t = r / a.group;
                int src = -1;
                if (r < n * a.group) src = a.rows ? a.rows[b * a.tokens + t] : t;
                if (src < -1 || src >= a.tokens || (src < 0 && r < n * a.group)) { atomicOr(&g_cache_error, kErrRange); src = -1; }
                const int hq = h * a.group + r % a.group;
                sq[i / D][i % D] = src >= 0 ? to_f(static_cast<const T *>(a.q)[b * a.qs[0] + src * a.qs[1] + hq * a.qs[2] + i % D]) : 0.f;
                if (i % D == 0) {
                    sl[i / D] = src >= 0 ? a.lse_in[((long long)b * a.tokens + src) * a.heads + hq] : -INFINITY;
                    st[i / D] = t;
                }
            }
            __syncthreads();
            if (j < end)
                for (int r = 0; r < 8; ++r) {
                    if (sl[r] == -INFINITY || j > len + st[r]) continue;
                    float s = 0.f;
                    for (int d = 0; d < D; ++d) s += sq[r][d] * to_f(K[j * a.ks[2] + d]);
                    w += expf(s * a.scale - sl[r]);
                }
        }
        if (j < end) a.mass_out[b * a.mos[0] + h * a.mos[1] + j] = (j < len ? a.mass[b * a.ms[0] + h * a.ms[1] + j] : 0.f) + w;
    }
}

size_t tree_attn_workspace(const p8_kv *, int64_t, int64_t) { return 0; }

template <typename T>
void run_attn(const p8_kv *c, const AttnArgs &a, bool mass, cudaStream_t st) {
    const int blocks = (a.tokens * a.group + 7) / 8;
    if (mass) {
        const dim3 g(512, a.kvh, a.batch);
        if (c->width == 128) k_attn_mass_plain<T, 128><<<g, 128, 0, st>>>(a);
        else k_attn_mass_plain<T, 64><<<g, 128, 0, st>>>(a);
    } else {
        const dim3 g(blocks, a.kvh, a.batch);
        if (c->width == 128) k_tree_attn_plain<T, 128><<<g, 128, 0, st>>>(a);
        else k_tree_attn_plain<T, 64><<<g, 128, 0, st>>>(a);
    }
}

void base_args(AttnArgs &x, const p8_kv *c, const void *q, const int64_t *qs, int64_t tokens, int64_t heads) {
    memset(&x, 0, sizeof(x));
    x.q = q; x.k = c->k; x.v = c->v;
    for (int i = 0; i < 3; ++i) { x.qs[i] = qs[i]; x.ks[i] = c->k_stride[1 + i]; x.vs[i] = c->v_stride[1 + i]; }
    x.slots = c->slots; x.batch = (int)c->batch; x.tokens = (int)tokens; x.heads = (int)heads; x.kvh = (int)c->heads;
    x.group = (int)(heads / c->heads);
}

p8_status launch_attn(const p8_kv *c, const AttnArgs &x, bool mass, cudaStream_t st) {
    if (c->type == P8_KV_F32) run_attn<float>(c, x, mass, st);
    else if (c->type == P8_KV_F16) run_attn<__half>(c, x, mass, st);
    else run_attn<__nv_bfloat16>(c, x, mass, st);
    return cudaGetLastError() == cudaSuccess ? P8_OK : P8_ERR_CUDA;
}

p8_status launch_tree_attn(const p8_kv *c, const p8_tree_attn_args *a, void *, cudaStream_t st) {
    AttnArgs x;
    base_args(x, c, a->q, a->q_stride, a->tokens, a->heads);
    x.lens = a->lens; x.counts = a->counts; x.mask = (const unsigned long long *)a->mask; x.mask_stride = a->mask_stride;
    x.scale = (float)a->scale; x.out = a->out; x.lse = a->lse;
    for (int i = 0; i < 3; ++i) x.os[i] = a->out_stride[i];
    return launch_attn(c, x, false, st);
}

p8_status launch_attn_mass(const p8_kv *c, const p8_attn_mass_args *a, cudaStream_t st) {
    AttnArgs x;
    base_args(x, c, a->q, a->q_stride, a->tokens, a->heads);
    x.lens = a->lens; x.counts = a->counts; x.rows = a->rows; x.lse_in = a->lse; x.scale = (float)a->scale;
    x.mass = a->mass; x.mass_out = a->out;
    for (int i = 0; i < 2; ++i) { x.ms[i] = a->mass_stride[i]; x.mos[i] = a->out_stride[i]; }
    return launch_attn(c, x, true, st);
}
