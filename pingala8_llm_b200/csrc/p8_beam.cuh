// p8_beam.cuh -- beam search: the best continuations of a group of beams, and the paged cache going on from their parents;
// included by p8_paged.cu.

// ----------------------------------------------------------------------------------------------------------------
// selection, step 1: every row of logits in equal pieces, one block each, read once. A lane keeps the sum of exp(x - m) for the
// largest x it has seen. What may be among the row's best goes to a list of
// its warp: whatever is at least the warp's bar, which rises to the n-th best of the list whenever that is full, and begins as
// the n-th largest of the lanes' first maxima. So nearly all logits cost one comparison for sixteen of them.
struct SelectArgs {
    const void *logits;
    long long ls[2];
    const float *scores;
    const unsigned char *done;
    float *out_scores;
    int *parents;
    long long *tokens;
    unsigned char *out_done;
    unsigned long long *best;  // [rows][splits][n], the best first, 0 behind them
    float2 *sums;              // [rows][splits]: the largest logit m, the sum of exp(x - m)
    long long end;
    int batch, beams, vocab, n, splits, chunk;
};

constexpr int kListSize = 128;  // of a warp
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ void unpack(const uint4 &v, float *x);
template <> __device__ __forceinline__ void unpack<float>(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 y = unpack2<__half>(w[i]); x[2 * i] = y.x; x[2 * i + 1] = y.y; }
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 y = unpack2<__nv_bfloat16>(w[i]); x[2 * i] = y.x; x[2 * i + 1] = y.y; }
}

// A continuation of a row as one number: larger where its logit is, or where those are equal the token lower. Never 0.
__device__ __forceinline__ unsigned long long continuation(float x, int token) {
    return (unsigned long long)order_key(__float_as_uint(x + 0.0f)) << 32 | (0xffffffffu - (unsigned int)token);
}

// the 128 entries of a warp's list (0 where there is none) in order, the largest first: entry 4 lane + i in x[i]
__device__ __forceinline__ void sort128(unsigned long long (&x)[4], int lane) {
#pragma unroll
    for (int size = 2; size <= 128; size *= 2) {
#pragma unroll
        for (int step = size / 2; step >= 1; step /= 2) {
            if (step >= 4) {
                const bool keep_max = ((4 * lane & size) == 0) == ((4 * lane & step) == 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned long long y = __shfl_xor_sync(0xffffffffu, x[i], step / 4);
                    x[i] = (x[i] > y) == keep_max ? x[i] : y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = i ^ step;
                    if (j > i) {
                        const bool down = ((4 * lane + i) & size) == 0;
                        const bool swap = down ? x[i] < x[j] : x[i] > x[j];
                        const unsigned long long a = swap ? x[j] : x[i], b = swap ? x[i] : x[j];
                        x[i] = a;
                        x[j] = b;
                    }
                }
            }
        }
    }
}

// keeps the n best of a warp's list, in order, and fills what is behind them with 0; returns the n-th
__device__ __forceinline__ unsigned long long prune(unsigned long long *list, int count, int n, int lane) {
    unsigned long long x[4];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 4 * lane + i < count ? list[4 * lane + i] : 0;
    sort128(x, lane);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) list[4 * lane + i] = 4 * lane + i < n ? x[i] : 0;
    __syncwarp();
    return list[n - 1];
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) k_beam_scan(const __grid_constant__ SelectArgs a) {
    constexpr int kW = kVec ? 16 / (int)sizeof(T) : 1, kE = 16, kU = kE / kW;  // a load's logits; a lane's in a round; its loads
    __shared__ unsigned long long s_list[8][kListSize];
    __shared__ unsigned long long s_bar;
    __shared__ float s_m[8], s_s[8];
    __shared__ int s_count[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    after_prior();
    const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits, b = row / a.beams, w = row - b * a.beams;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if ((a.done && a.done[row]) || !isfinite(a.scores[row])) return;  // the whole block
    const T *x0 = static_cast<const T *>(a.logits) + b * a.ls[0] + w * a.ls[1];
    const int begin = split * a.chunk, end = min(a.vocab, begin + a.chunk);
    if (threadIdx.x == 0) s_bar = 0;
    __syncthreads();
    unsigned long long *list = s_list[warp];
    unsigned long long bar = 0;  // what is below it is not among the best; 0: not known yet
    int count = 0;
    float m = -INFINITY, sum = 0.f;
    for (int at = begin + warp * 32 * kE; at < end; at += 256 * kE) {
        float x[kE];
        // (a lane's logits: kU groups of kW, a warp's groups side by side)
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = at + u * 32 * kW + lane * kW;
            if (kVec) {
                if (i + kW <= end) {
                    unpack<T>(ld_once(reinterpret_cast<const char *>(x0 + i)), x + u * kW);
                } else {
#pragma unroll
                    for (int e = 0; e < kW; ++e) x[u * kW + e] = i + e < end ? to_f<T>(x0[i + e]) : -INFINITY;
                }
            } else {
                x[u] = i < end ? to_f<T>(x0[i]) : -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < kE; ++e) top = fmaxf(top, x[e]);
        if (!(top > -INFINITY)) top = -INFINITY;  // (NaN alone)
        if (top > m) {
            sum *= ex2((m - top) * kLog2e);
            m = top;
        }
        const float from = m == -INFINITY ? 0.f : m;
        float more = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e) more += ex2((x[e] - from) * kLog2e);
        if (more != more) {  // NaN counts as -infinity
            more = 0.f;
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                if (x[e] != x[e]) x[e] = -INFINITY;
                more += ex2((x[e] - from) * kLog2e);
            }
        }
        sum += more;
        // candidates
        const unsigned long long others = *reinterpret_cast<volatile unsigned long long *>(&s_bar);
        bar = others > bar ? others : bar;
        if (bar == 0 && a.n <= 32) {  // n lanes have a logit at least as large as the n-th largest of their maxima
            const uint32_t key = order_key(__float_as_uint(top + 0.0f));
            int rank = 0;
#pragma unroll
            for (int o = 0; o < 32; ++o) {
                const uint32_t y = __shfl_sync(0xffffffffu, key, o);
                rank += y > key || (y == key && o < lane);
            }
            const unsigned int who = __ballot_sync(0xffffffffu, rank == a.n - 1 && top > -INFINITY);
            if (who) {
                bar = (unsigned long long)__shfl_sync(0xffffffffu, key, __ffs(who) - 1) << 32;
                if (lane == 0) atomicMax(&s_bar, bar);
            }
        }
        const float at_least = bar == 0 ? -INFINITY : __uint_as_float(order_bits((uint32_t)(bar >> 32)));
        if (__any_sync(0xffffffffu, top >= at_least && top > -INFINITY)) {
unsigned int reach = 0;  // those of this lane that reach it
#pragma unroll
            for (int e = 0; e < kE; ++e) reach |= (x[e] >= at_least && x[e] > -INFINITY) << e;
            while (__any_sync(0xffffffffu, reach)) {  // one of every lane at a time
                const int e = __ffs(reach) - 1;
                float y = x[0];
#pragma unroll
                for (int f = 1; f < kE; ++f) y = e == f ? x[f] : y;
                const unsigned long long c = continuation(y, at + e / kW * 32 * kW + lane * kW + e % kW);
                const bool in = reach && c > bar;
                reach &= reach - 1;
                const unsigned int who = __ballot_sync(0xffffffffu, in);
                if (in) list[count + __popc(who & ((1u << lane) - 1))] = c;
                count += __popc(who);
                if (count > kListSize - 32) {
                    const unsigned long long nth = prune(list, count, a.n, lane);
                    if (nth > bar) {
                        bar = nth;
                        if (lane == 0) atomicMax(&s_bar, bar);
                    }
                    count = a.n;
                }
            }
        }
    }
    // this block's best, and its sum
    prune(list, count, a.n, lane);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float pm = __shfl_xor_sync(0xffffffffu, m, o), ps = __shfl_xor_sync(0xffffffffu, sum, o), now = fmaxf(m, pm);
        sum = (m == now ? sum : sum * ex2((m - now) * kLog2e)) + (pm == now ? ps : ps * ex2((pm - now) * kLog2e));
        m = now;
    }
    if (lane == 0) { s_m[warp] = m; s_s[warp] = sum; s_count[warp] = min(count, a.n); }
    __syncthreads();
    const long long piece = (long long)row * a.splits + split;
    for (int i = threadIdx.x; i < 8 * a.n; i += 256) {
        const int v = i / a.n, k = i - v * a.n;
        const unsigned long long c = s_list[v][k];
        int rank = c ? k : a.n;
#pragma unroll
        for (int o = 0; o < 8; ++o) {
            if (o == v) continue;
            int lo = 0, hi = a.n;  // how many of that list are above it
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (s_list[o][mid] > c) lo = mid + 1; else hi = mid;
            }
            rank += lo;
        }
        if (rank < a.n) a.best[piece * a.n + rank] = c;
    }
    int have = 0;
    for (int o = 0; o < 8; ++o) have += s_count[o];
    for (int i = have + threadIdx.x; i < a.n; i += 256) a.best[piece * a.n + i] = 0;
    if (threadIdx.x == 0) {
        float M = s_m[0], S = 0.f;
        for (int o = 1; o < 8; ++o) M = fmaxf(M, s_m[o]);
        for (int o = 0; o < 8; ++o) S += s_m[o] == M ? s_s[o] : s_s[o] * ex2((s_m[o] - M) * kLog2e);
        a.sums[piece] = make_float2(M, S);
    }
}

// step 2, one block a group: the rows' log sums in 64 bits, then the best of all pieces' lists. Each list is in order, so
// the n-th largest of their first entries is a bar that all of the group's n best reach; what reaches it is counted out against one another.
__device__ __forceinline__ unsigned long long total_key(double t) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(t + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
constexpr int kMaxLists = 256, kPicked = 1024;

__global__ void __launch_bounds__(256) k_beam_join(const __grid_constant__ SelectArgs a) {
    __shared__ double s_shift[P8_BEAMS_MAX];  // score - log sum
    __shared__ int s_kind[P8_BEAMS_MAX];      // 0: no continuation, 1: from its logits, 2: ended
    __shared__ unsigned long long s_head[kMaxLists], s_total[kPicked], s_which[kPicked];
    __shared__ int s_count;
    __shared__ unsigned long long s_bar;
    after_prior();
    const int b = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32, lists = a.beams * a.splits;
    if (threadIdx.x == 0) { s_count = 0; s_bar = 0; }
    for (int w = warp; w < a.beams; w += 8) {
        const long long row = (long long)b * a.beams + w;
        const float score = a.scores[row];
        const bool ended = a.done && a.done[row];
        int kind = !isfinite(score) ? 0 : ended ? 2 : 1;
        double shift = score;
        if (kind == 1) {
            float top = -INFINITY;
            for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, a.sums[row * a.splits + i].x);
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            double sum = 0.0;
            for (int i = lane; i < a.splits; i += 32) {
                const float2 p = a.sums[row * a.splits + i];
                if (p.x > -INFINITY) sum += (double)p.y * exp((double)(p.x - top));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (!isfinite(top) || !(sum > 0.0)) kind = 0;
            else shift -= (double)top + log(sum);
        }
        if (lane == 0) { s_shift[w] = shift; s_kind[w] = kind; }
    }
    __syncthreads();
    const auto logit = [&](unsigned long long c) { return (double)__uint_as_float(order_bits((uint32_t)(c >> 32))); };
    for (int l = threadIdx.x; l < lists; l += 256) {
        const int w = l / a.splits;
        unsigned long long key = 0;
        if (s_kind[w] == 1) {
            const unsigned long long c = a.best[((long long)b * lists + l) * a.n];
            if (c) key = total_key(s_shift[w] + logit(c));
        } else if (s_kind[w] == 2 && l == w * a.splits) {
            key = total_key(s_shift[w]);
        }
        s_head[l] = key;
    }
    __syncthreads();
    for (int l = threadIdx.x; l < lists; l += 256) {
        const unsigned long long key = s_head[l];
        int rank = 0;
        for (int o = 0; o < lists; ++o) rank += s_head[o] > key || (s_head[o] == key && o < l);
        if (rank == a.n - 1) s_bar = key;
    }
    __syncthreads();
    const unsigned long long bar = s_bar;
    // Those that reach the bar, in rounds of what the list takes: only the n best so far stay from one to the next.
    for (int l0 = 0; l0 < lists; l0 += 256) {
        const int l = l0 + threadIdx.x, w = l < lists ? l / a.splits : 0;
        const bool any = l < lists && s_head[l] && s_head[l] >= bar;
        for (int i0 = 0; i0 < a.n; i0 += 2) {
            // two entries of every list at most 512 a round; before the next one, the list is cut to its n best
            bool live = false;
            if (any) {
                for (int i = i0; i < min(a.n, i0 + 2); ++i) {
                    unsigned long long key = 0, which = 0;
                    if (s_kind[w] == 2) {
                        if (i == 0) { key = total_key(s_shift[w]); which = (unsigned long long)w << 32 | (unsigned int)a.end; }
                    } else {
                        const unsigned long long c = a.best[((long long)b * lists + l) * a.n + i];
                        if (c) { key = total_key(s_shift[w] + logit(c)); which = (unsigned long long)w << 32 | (0xffffffffu - (unsigned int)c); }
                    }
                    if (key && key >= bar) {
                        const int k = atomicAdd(&s_count, 1);
                        s_total[k] = key;
                        s_which[k] = which;
                        live = true;
                    }
                }
            }
            const bool go_on = __syncthreads_or(live);
            const int have = s_count;
            if (have > kPicked - 512 || !go_on || (l0 + 256 >= lists && i0 + 2 >= a.n)) {
                // count out: entry k stays at the place that is the number of entries before it
                unsigned long long key[4], which[4];
                int rank[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = threadIdx.x + 256 * j;
                    rank[j] = INT_MAX;
                    if (k < have) {
                        key[j] = s_total[k];
                        which[j] = s_which[k];
                        int r = 0;
                        for (int o = 0; o < have; ++o) {
                            const unsigned long long y = s_total[o];
                            r += y > key[j] || (y == key[j] && s_which[o] < which[j]);
                        }
                        rank[j] = r;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (rank[j] < a.n) { s_total[rank[j]] = key[j]; s_which[rank[j]] = which[j]; }
                if (threadIdx.x == 0) s_count = min(have, a.n);
                __syncthreads();
            }
            if (!go_on) break;
        }
    }
    const int have = s_count;
    for (int i = threadIdx.x; i < a.n; i += 256) {
        const long long at = (long long)b * a.n + i;
        const bool there = i < have;
        float score = -INFINITY;
        int parent = -1;
        long long token = -1;
        bool ended = false;
        if (there) {
            const unsigned long long u = s_total[i];
            score = (float)__longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
            parent = (int)(s_which[i] >> 32);
            token = (long long)(s_which[i] & 0xffffffffu);
            ended = s_kind[parent] == 2 || token == a.end;
        }
        a.out_scores[at] = score;
        a.parents[at] = parent;
        a.tokens[at] = token;
        if (a.out_done) a.out_done[at] = ended;
    }
}

bool select_sizes_ok(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
    return batch >= 1 && batch <= P8_BATCH_MAX && beams >= 1 && beams <= P8_BEAMS_MAX && vocab >= 1 && vocab <= INT32_MAX - 65536 && n >= 1 && n <= P8_CANDIDATES_MAX;
}
int64_t splits_of(int64_t batch, int64_t beams, int64_t vocab) { return select_splits(batch * beams, beams, vocab, sm_count(), 4096); }
size_t select_workspace(int64_t batch, int64_t beams, int64_t vocab, int64_t n) { return (size_t)(batch * beams * splits_of(batch, beams, vocab) * (n + 1) * 8); }

p8_status launch_beam_select(const p8_beam_select_args *x, void *workspace, cudaStream_t st) {
    SelectArgs a;
    a.logits = x->logits; a.ls[0] = x->stride[0]; a.ls[1] = x->stride[1];
    a.scores = x->scores; a.done = x->done; a.out_scores = x->out_scores; a.parents = x->parents; a.tokens = (long long *)x->tokens; a.out_done = x->out_done;
    a.end = x->end; a.batch = (int)x->batch; a.beams = (int)x->beams; a.vocab = (int)x->vocab; a.n = (int)x->candidates;
    a.splits = (int)splits_of(x->batch, x->beams, x->vocab);
    a.chunk = (int)(((x->vocab + a.splits - 1) / a.splits + 15) / 16 * 16);
    const int64_t pieces = x->batch * x->beams * a.splits;
    a.best = (unsigned long long *)workspace;
    a.sums = (float2 *)(a.best + pieces * a.n);
    const int es = elem_size(x->type);
    const auto whole = [&](int64_t stride, int64_t rows) { return rows <= 1 || stride * es % 16 == 0; };
    const bool vec = al16(x->logits) && whole(x->stride[0], x->batch) && whole(x->stride[1], x->beams);
    const auto scan = x->type == P8_KV_F32 ? (vec ? k_beam_scan<float, true> : k_beam_scan<float, false>)
                      : x->type == P8_KV_F16 ? (vec ? k_beam_scan<__half, true> : k_beam_scan<__half, false>)
                                             : (vec ? k_beam_scan<__nv_bfloat16, true> : k_beam_scan<__nv_bfloat16, false>);
    if (launch_after(scan, dim3((unsigned int)pieces), dim3(256), 0, st, a) != cudaSuccess) return P8_ERR_CUDA;
    return done(launch_after(k_beam_join, dim3((unsigned int)x->batch), dim3(256), 0, st, a));
}

// ----------------------------------------------------------------------------------------------------------------
// reordering. Which begun page goes where follows from a group's parents alone (ballots, in every warp). The first launch copies the
// begun pages of further children; it reads of the tables only the begun pages' column. The second one, whose blocks start as soon as
// all of the first have passed their own wait, writes the full pages' columns meanwhile, and the begun pages' once the copies are done.
struct ReorderArgs {
    char *kv[2];
    long long st[2][4];  // bytes: layer, page, head, slot
    int *tables;
    const int *parents, *lens;
    long long ts, slots, columns;
    PageDiv div;
    int batch, beams, heads, pages, row_bytes, chunks, alone;  // chunks: blocks of a page; alone: there is no first launch
};
struct BeamPlan {
    bool ok;
    int len, p[2];                          // parents of beams lane and lane + 32
    unsigned long long further, childless;  // beams whose parent has a lower child; beams without one
    __device__ __forceinline__ int parent(int i) const { return __shfl_sync(0xffffffffu, i < 32 ? p[0] : p[1], i & 31); }
};
__device__ __forceinline__ BeamPlan beam_plan(const ReorderArgs &a, int b, int lane) {
    BeamPlan r;
    bool fine = true;
    const long long row = (long long)b * a.beams;
    r.len = a.lens[row];
    if (r.len < 0 || r.len > a.slots) fine = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        r.p[k] = i;
        if (i < a.beams) {
            const int p = a.parents[row + i];
            if (p < -1 || p >= a.beams || a.lens[row + i] != r.len) fine = false;
            else if (p >= 0) r.p[k] = p;
        }
    }
    r.ok = __all_sync(0xffffffffu, fine);
    unsigned long long seen = 0;
    r.further = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        const unsigned int same = __match_any_sync(0xffffffffu, i < a.beams ? r.p[k] : 64 + lane);
        const bool again = i < a.beams && ((same & ((1u << lane) - 1)) || (seen >> (r.p[k] & 63) & 1));
        r.further |= (unsigned long long)__ballot_sync(0xffffffffu, again) << (32 * k);
        const bool low = i < a.beams && r.p[k] < 32, high = i < a.beams && r.p[k] >= 32;
        seen |= __reduce_or_sync(0xffffffffu, low ? 1u << r.p[k] : 0u) | (unsigned long long)__reduce_or_sync(0xffffffffu, high ? 1u << (r.p[k] - 32) : 0u) << 32;
    }
    r.childless = ~seen & (a.beams == 64 ? ~0ull : (1ull << a.beams) - 1);
    return r;
}
// whose begun page beam i goes on with
__device__ __forceinline__ int page_from(const BeamPlan &r, int i) {
    if (!(r.further >> i & 1)) return r.parent(i);
    return nth_bit(r.childless, __popcll(r.further & ((1ull << i) - 1)));
}

constexpr int kMoveUnits = 8;  // 16 bytes each, of a thread

__global__ void __launch_bounds__(256) k_beam_move(const __grid_constant__ ReorderArgs a) {
    after_prior();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, b = row / a.beams, i = row - b * a.beams, lane = threadIdx.x % 32;
    const int layer = blockIdx.y / 2, z = blockIdx.y % 2;
    const BeamPlan r = beam_plan(a, b, lane);
    if (!r.ok || !(r.further >> i & 1)) return;
    const int full = (int)page_of(a.div, (unsigned int)r.len), rest = r.len - full * (int)a.div.size, per = a.row_bytes / 16;
    const int items = rest * a.heads * per, first = chunk * 256 * kMoveUnits;
    if (first >= items) return;
    const int src = a.tables[((long long)b * a.beams + r.parent(i)) * a.ts + full], dst = a.tables[((long long)b * a.beams + page_from(r, i)) * a.ts + full];
    if ((unsigned int)src >= (unsigned int)a.pages || (unsigned int)dst >= (unsigned int)a.pages) {
        if (threadIdx.x == 0) out_of_range();
        return;
    }
    const char *from = a.kv[z] + layer * a.st[z][0] + src * a.st[z][1];
    char *to = a.kv[z] + layer * a.st[z][0] + dst * a.st[z][1];
    uint4 v[kMoveUnits];
    long long at[kMoveUnits];
#pragma unroll
    for (int j = 0; j < kMoveUnits; ++j) {
        const int k = first + 256 * j + threadIdx.x;
        if (k < items) {
            const int unit = k % per, hs = k / per, h = hs / rest, s = hs - h * rest;
            at[j] = h * a.st[z][2] + s * a.st[z][3] + 16 * unit;
            v[j] = *reinterpret_cast<const uint4 *>(from + at[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < kMoveUnits; ++j)
        if (first + 256 * j + (int)threadIdx.x < items) *reinterpret_cast<uint4 *>(to + at[j]) = v[j];
}

constexpr int kColumns = 64;

__global__ void __launch_bounds__(256) k_beam_tables(const __grid_constant__ ReorderArgs a) {
    __shared__ int s_old[P8_BEAMS_MAX][kColumns], s_begun[P8_BEAMS_MAX], s_parent[P8_BEAMS_MAX];
    if (a.alone) after_prior();
    const int b = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const BeamPlan r = beam_plan(a, b, lane);
    if (!r.ok) {
        if (blockIdx.x == 0 && threadIdx.x == 0) out_of_range();
        if (!a.alone) after_prior();
        return;
    }
    int *table = a.tables + (long long)b * a.beams * a.ts;
    const int full = (int)page_of(a.div, (unsigned int)r.len), rest = r.len - full * (int)a.div.size;
    if (warp == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (lane + 32 * k < a.beams) {
                s_parent[lane + 32 * k] = r.p[k];
                if (rest) s_begun[lane + 32 * k] = table[(lane + 32 * k) * a.ts + full];
            }
    }
    for (int c0 = blockIdx.x * kColumns; c0 < full; c0 += gridDim.x * kColumns) {
        __syncthreads();
        for (int k = threadIdx.x; k < a.beams * kColumns; k += 256) {
            const int i = k / kColumns, c = k % kColumns;
            if (c0 + c < full) s_old[i][c] = table[i * a.ts + c0 + c];
        }
        __syncthreads();
        for (int k = threadIdx.x; k < a.beams * kColumns; k += 256) {
            const int i = k / kColumns, c = k % kColumns, p = s_parent[i];
            if (c0 + c < full && p != i) table[i * a.ts + c0 + c] = s_old[p][c];
        }
    }
    if (!a.alone) after_prior();  // the copies have looked their pages up
    if (blockIdx.x == 0 && warp == 0 && rest) {
        __syncwarp();
        for (int i = 0; i < a.beams; ++i) {
            const int from = page_from(r, i);
            if (lane == 0 && from != i) table[i * a.ts + full] = s_begun[from];
        }
    }
}

p8_status launch_beam_reorder(const p8_paged *c, const int32_t *parents, const int32_t *lens, int64_t batch, int64_t beams, cudaStream_t st) {
    ReorderArgs a;
    const int es = elem_size(c->type);
    a.kv[0] = (char *)c->k; a.kv[1] = (char *)c->v;
    for (int i = 0; i < 4; ++i) { a.st[0][i] = c->k_stride[i] * es; a.st[1][i] = c->v_stride[i] * es; }
    a.tables = c->tables; a.parents = parents; a.lens = lens; a.ts = c->table_stride; a.slots = c->columns * c->page; a.columns = c->columns;
    a.div = page_div((uint32_t)c->page);
    a.batch = (int)batch; a.beams = (int)beams; a.heads = (int)c->heads; a.pages = (int)c->pages; a.row_bytes = (int)c->width * es;
    const int64_t units = (c->page - 1) * c->heads * (a.row_bytes / 16), chunks = (units + 256 * kMoveUnits - 1) / (256 * kMoveUnits);
    if (units > INT32_MAX || chunks * c->rows > INT32_MAX) return P8_ERR_UNSUPPORTED;
    a.chunks = (int)chunks;
    a.alone = chunks == 0 || beams == 1;
    if (!a.alone && launch_after(k_beam_move, dim3((unsigned int)(chunks * c->rows), (unsigned int)(2 * c->layers)), dim3(256), 0, st, a) != cudaSuccess) return P8_ERR_CUDA;
    const int64_t across = std::max<int64_t>(1, std::min<int64_t>((c->columns + kColumns - 1) / kColumns, (2 * sm_count() + batch - 1) / batch));
    return done(launch_after(k_beam_tables, dim3((unsigned int)across, (unsigned int)batch), dim3(256), 0, st, a));
}
