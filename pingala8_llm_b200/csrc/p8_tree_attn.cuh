// p8_tree_attn.cuh -- attention of a tree of drafted tokens over a cache, and the attention mass per slot (included by
// p8_cache.cu).
//
// Times here are a call's in a CUDA graph at full clocks (1,965 MHz). Calls that follow one another for seconds draw the
// 1,000 W that the GPU may, at 1.6 GHz in the attention: 24 sequences x 7 tokens then take 91 us, not 79, 64 tokens over
// 131,000 slots 182, not 154. A form that was not kept is given with the kept one's time of the same day.
#pragma once

constexpr unsigned int kWaitNs = 2000000000u;  // what waits are bounded by, unless the host says otherwise

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
    int g0, gc, more;  // mass: the query heads g0 .. g0 + gc - 1 of each group; more: added to what `out` has
    float scale;
    unsigned int wait_ns;  // bound of one wait
};

// A unit is (sequence, cache head, block of query rows); its slots are cut into tiles. All tiles of all units
// form one list, sequence by sequence, with a few places more for the beginning of each unit, and every CTA takes an
// equal contiguous share of it, so that the SMs finish together whatever the lengths are, and one long sequence still
// fills them. A unit that lies in one share is finished there; the parts of the others go to the workspace as (sum of p v,
// maximum, sum of p) and k_attn_join adds them up.
constexpr int kTile = 128;  // of a 16-bit cache; 64 of a 32-bit one (as many bytes)
// What a 16-bit attention segment costs beside its tiles, in tiles: filling and draining its pipeline and, for 256 rows,
// writing 128 KB of sums takes about 9 us where a tile takes 2.3 (24 sequences of 501 to 8,192 slots: 105 us without, 79
// with the queries brought ahead as well; 131,000 slots x 256 rows: 161 us with 1, 155 with 4).
__host__ __device__ constexpr int start_of(int rblock) { return rblock > 128 ? 4 : 1; }
struct Cut {                // how a kernel cuts its work
    int rblock, tile;       // query rows of a unit, slots of a tile
    int least;              // tiles of a share, at least
    int start;              // what it costs to begin a segment, in tiles
};

struct Share {
    int pos, end;           // the CTA's tiles
    int b, off, len, n;     // the sequence that pos lies in, and where in it
};

struct Walk {               // a CTA's way through its share, one segment (the tiles of one unit) at a time
    const AttnArgs &a;
    const Cut cut;
    int pos, end, off, b, len, n, nt, units, u, ta, tb, step;
    bool opens;             // the segment is the share's first
    __device__ Walk(const AttnArgs &a_, Cut c, const Share &s)
        : a(a_), cut(c), pos(s.pos), end(s.end), off(s.off), b(s.b), len(s.len), n(s.n), opens(true) {
        count();
    }
    __device__ void count() {
        nt = n ? (len + n + cut.tile - 1) / cut.tile : 0;
        units = n ? a.kvh * ((n * a.group + cut.rblock - 1) / cut.rblock) : 0;
    }
    __device__ bool next() {
        while (pos < end) {
            const int cost = nt + cut.start;
            if (off >= units * cost) {
                off -= units * cost;
                ++b;
                if (!seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n)) n = 0;
                count();
                continue;
            }
            u = off / cost;
            const int in = off - u * cost;  // the unit's first `start` places stand for its beginning
            ta = max(0, in - cut.start);
            step = min(cost - in, end - pos);
            tb = in + step - cut.start;
            if (tb > ta) return true;
            pos += step;
            off += step;
        }
        return false;
    }
    __device__ void advance() {
        pos += step;
        off += step;
        opens = false;
    }
    __device__ int blocks() const { return units / a.kvh; }
    __device__ int head() const { return u / blocks(); }
    __device__ int row0() const { return u % blocks() * cut.rblock; }
    __device__ bool whole() const { return ta == 0 && tb == nt; }
};

// (the host refuses what would not fit 31 bits)
__device__ __forceinline__ int seq_tiles(const AttnArgs &a, Cut cut, int b, int &len, int &n, bool *bad) {
    if (!seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n)) {
        *bad = true;
        n = 0;
    }
    return n ? a.kvh * ((n * a.group + cut.rblock - 1) / cut.rblock) * ((len + n + cut.tile - 1) / cut.tile + cut.start) : 0;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// tiles of a share, of a list of that many
__device__ __forceinline__ int share_of(int total, Cut cut, int ctas) { return max(cut.least, (int)(((unsigned)total + ctas - 1) / (unsigned)ctas)); }
// the share of one CTA (whole warp)
__device__ __forceinline__ Share find_share(const AttnArgs &a, Cut cut, int lane, int cta, int ctas) {
    bool bad = false;
    int len = 0, n = 0, mine = 0, total = 0;
    for (int b = lane; b < a.batch; b += 32) total += mine = seq_tiles(a, cut, b, len, n, &bad);
    total = __reduce_add_sync(0xffffffffu, total);
    if (bad && cta == 0) atomicOr(&g_cache_error, kErrRange);
    const int each = share_of(total, cut, ctas);
    Share s = {};
    s.pos = (int)min((long long)total, (long long)cta * each);
    s.end = (int)min((long long)total, (long long)s.pos + each);
    int run = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        if (a.batch > 32) mine = b0 + lane < a.batch ? seq_tiles(a, cut, b0 + lane, len, n, &bad) : 0;
        const int incl = run + warp_scan(mine, lane);
        const unsigned int hit = __ballot_sync(0xffffffffu, incl > s.pos);
        if (hit) {
            const int l = __ffs(hit) - 1;
            s.b = b0 + l;
            s.off = s.pos - __shfl_sync(0xffffffffu, incl - mine, l);
            s.len = __shfl_sync(0xffffffffu, len, l);
            s.n = __shfl_sync(0xffffffffu, n, l);
            break;
        }
        run = __shfl_sync(0xffffffffu, incl, 31);
    }
    return s;
}

// Waits give up after `ns` (the kernel's results are then invalid and bit 128 is set); from then on every wait of the CTA that
// is not over within one look returns false. What follows from that goes by the role. A thread that starts something
// asynchronous (TMA loads, cp.async, MMAs) starts nothing more: a stage that was not handed over may still be written or read,
// and its barrier may be inside a phase. Before it goes to the CTA's end it waits for all that it did start (settle, which does
// not ask whether something gave up). The others run through to the end and meet there. Each thread goes by its own waits, also in a
// warp of which one issues: votes between them cost 2 % of the attention.
struct Waits {
    volatile int *gave_up;
    unsigned int ns;
    // whether the barrier's phase is over
    __device__ bool operator()(uint64_t *bar, uint32_t parity) const {
        if (mbar_test_wait(bar, parity)) return true;
        if (ns && mbar_try_wait(bar, parity)) return true;  // stays for up to about 4 us
        if (*gave_up) return false;
        if (ns && poll(bar, parity, ns, gave_up)) return true;
        *gave_up = 1;
        atomicOr(&g_cache_error, kErrWait);
        return false;
    }
    // the same, where the phase is ended by roles that go on arriving after something gave up
    __device__ bool arrivals(uint64_t *bar, uint32_t parity) const { return (*this)(bar, parity) && !*gave_up; }
    // for what this role has started and what ends by itself
    __device__ void settle(uint64_t *bar, uint32_t parity) const {
        if (mbar_try_wait(bar, parity) || poll(bar, parity, kWaitNs, nullptr)) return;
        *gave_up = 1;
        atomicOr(&g_cache_error, kErrWait);
    }
    // A look stays for about 4 us. Beside the time there is a least number of looks, a quarter of it: the clock goes on while the
    // GPU runs something else in this kernel's place, and what the wait is for does not.
    static __device__ bool poll(uint64_t *bar, uint32_t parity, unsigned int ns, volatile int *stop) {
        unsigned long long t0, t;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
        for (unsigned int i = 0;; ++i) {
            if (mbar_try_wait(bar, parity)) return true;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
            if ((stop && *stop) || (i >= ns >> 14 && t - t0 > ns)) return false;
        }
    }
};

__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void map_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// Shared-memory operand of 128-byte rows in the 128-byte swizzle (what the tensor map's loads leave; a stage is `rows`
// rows per 64 columns). Rows as the outer extent (Q, K): groups of 8 rows 1024 bytes apart. Rows as the summed one (V):
// the same bytes read the other way, the next 64 columns a whole stage part (16 KB) on.
__device__ __forceinline__ uint64_t desc_rows(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_cols(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <typename T> struct Half16;  // what differs between the two 16-bit types
template <> struct Half16<__nv_bfloat16> {
    static constexpr bool bf16 = true;
    // The weights p = 2^(s - m + kLift) are rounded to the type. The running maximum m is only raised when the new one
    // is kSlack above it, which saves most passes over the accumulator; p then stays below 2^(kLift + kSlack).
    static constexpr float kLift = 0.f, kSlack = 8.f;
    static constexpr uint32_t kExp = 0x7F80u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};
template <> struct Half16<__half> {
    static constexpr bool bf16 = false;
    // fp16 ends at 2^-24: lifted by 2^10, weights keep their 11 bits down to 2^-24 of the largest (and stay below 2^15)
    static constexpr float kLift = 10.f, kSlack = 5.f;
    static constexpr uint32_t kExp = 0x7C00u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};

template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int n, bool b_cols) {  // f32 accumulator, M = 128
    const uint32_t f = Half16<T>::bf16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_cols ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// One thread of the warp, chosen so that the compiler knows the branch to be the warp's: the MMAs' operands then stay in
// uniform registers (under `lane == 0`, with a descriptor put together for each, an MMA took 91 cycles to issue, where a
// 128 x 128 x 16 one runs for 64).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred P;\n elect.sync _|P, 0xffffffff;\n selp.b32 %0, 1, 0, P;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(da), "l"(db),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(ta), "l"(db),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
#define P8_R32(v) "=r"((v)[0]), "=r"((v)[1]), "=r"((v)[2]), "=r"((v)[3]), "=r"((v)[4]), "=r"((v)[5]), "=r"((v)[6]), "=r"((v)[7]), "=r"((v)[8]), \
    "=r"((v)[9]), "=r"((v)[10]), "=r"((v)[11]), "=r"((v)[12]), "=r"((v)[13]), "=r"((v)[14]), "=r"((v)[15]), "=r"((v)[16]), "=r"((v)[17]), \
    "=r"((v)[18]), "=r"((v)[19]), "=r"((v)[20]), "=r"((v)[21]), "=r"((v)[22]), "=r"((v)[23]), "=r"((v)[24]), "=r"((v)[25]), "=r"((v)[26]), \
    "=r"((v)[27]), "=r"((v)[28]), "=r"((v)[29]), "=r"((v)[30]), "=r"((v)[31])
// 32 lanes x 32 columns of 32 bits; the values are there after tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : P8_R32(v)
        : "r"(at)
        : "memory");
}
#undef P8_R32
#define P8_RW8(v, o) "+r"((v)[o]), "+r"((v)[o + 1]), "+r"((v)[o + 2]), "+r"((v)[o + 3]), "+r"((v)[o + 4]), "+r"((v)[o + 5]), "+r"((v)[o + 6]), "+r"((v)[o + 7])
// the wait names the registers, so that nothing that reads them moves ahead of it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : P8_RW8(v, 0), P8_RW8(v, 8), P8_RW8(v, 16), P8_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_waited(uint32_t (&v)[32]) { asm volatile("" : P8_RW8(v, 0), P8_RW8(v, 8), P8_RW8(v, 16), P8_RW8(v, 24)::"memory"); }
#undef P8_RW8
#define P8_R16(v, o) "r"((v)[o]), "r"((v)[o + 1]), "r"((v)[o + 2]), "r"((v)[o + 3]), "r"((v)[o + 4]), "r"((v)[o + 5]), "r"((v)[o + 6]), "r"((v)[o + 7]), \
    "r"((v)[o + 8]), "r"((v)[o + 9]), "r"((v)[o + 10]), "r"((v)[o + 11]), "r"((v)[o + 12]), "r"((v)[o + 13]), "r"((v)[o + 14]), "r"((v)[o + 15])
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
        P8_R16(v, 0), P8_R16(v, 16)
        : "memory");
}
#undef P8_R16
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows [row0, row0 + 128 tiles) of a unit's queries into swizzled shared memory, by one warp. Places behind the last row
// keep what they had: a row of the products depends on no other. flip: the sign bits (a negative scale is taken as its
// magnitude and -q).
template <typename T, int D>
__device__ __forceinline__ void load_q(char *sq, const AttnArgs &a, int b, int h, int row0, int rows, int tiles, uint32_t flip, int lane) {
    constexpr int C = D / 8, STEP = 32 / C;
    const int c = lane % C, n = min(tiles * 128, rows - row0);
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + c * 8;
    int t = (row0 + lane / C) / a.group, g = row0 + lane / C - t * a.group;
    auto place = [&](int r) { return sq + (r / 128) * (128 * D * 2) + (c / 8) * 16384 + (r % 128) * 128 + (((c % 8) ^ (r % 8)) * 16); };
    for (int r = lane / C; r < n; r += STEP) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(place(r))), "l"(q + t * a.qs[1] + (long long)(h * a.group + g) * a.qs[2]) : "memory");
        for (g += STEP; g >= a.group; g -= a.group) ++t;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (flip)
        for (int r = lane / C; r < n; r += STEP) {
            uint4 *v = reinterpret_cast<uint4 *>(place(r));
            *v = make_uint4(v->x ^ flip, v->y ^ flip, v->z ^ flip, v->w ^ flip);
        }
}

// Which of 32 columns a row sees, where `off` of them are the sequence's and the drafted tokens follow.
__device__ __forceinline__ uint32_t seen32(bool live, unsigned long long sees, int off) {
    uint32_t see = off >= 32 ? ~0u : off > 0 ? (1u << off) - 1 : 0u;
    if (off < 32 && off > -64) see |= off >= 0 ? (uint32_t)sees << off : (uint32_t)(sees >> -off);
    return live ? see : 0u;
}
__device__ __forceinline__ void hide(uint32_t (&x)[32], uint32_t see) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
        if (!(see >> k & 1)) x[k] = 0xFF800000u;  // -infinity
}

// Groups of 16 slots that a step multiplies: those that hold something, and at least one.
__device__ __forceinline__ int live_groups(const Walk &w, int tile, int half) {
    const int real = w.len + w.n - tile * kTile - 64 * half;
    return max(1, min(4, (real + 15) / 16));
}

// A drafted token's infinities and NaN (those of the tokens in `bad`) onto the values that a row has written: x plus
// each of them, in columns [x0, x1).
template <typename T, typename O>
__device__ __noinline__ void add_bad(O *out, const T *v, long long stride, unsigned long long bad, int x0, int x1) {
    for (; bad; bad &= bad - 1) {
        const T *y = v + (__ffsll(bad) - 1) * stride;
        for (int k = x0; k < x1; ++k) {
            const float z = to_f(y[k]);
            if (!isfinite(z)) out[k] = from_f<O>(to_f(out[k]) + z);
        }
    }
}

// The tree attention kernel. Twelve warps: two groups of four for the softmax (thread = query row = TMEM lane), one that
// brings tiles of K and V into a ring by TMA, one that brings queries, and one for each of two streams that issues its
// MMAs. A stream is a softmax group with its scores and its accumulator in TMEM; a step is 64 slots:
//   TWO = false (at most 128 query rows): both streams have the same rows, stream s takes the slots 64 s .. of every
//                tile; the accumulators are joined at the segment's end.
//   TWO = true: stream s has rows 128 s .. of a block of 256 and takes every tile's halves one after the other (K and V
//               come once for 256 rows).
// Step k of a stream: S = Q K^T (128 x 64, into one of the stream's two score buffers) -> softmax group: mask, running
// maximum and sum in base 2, P rounded to the type over S's columns -> O += P V (P from TMEM). With two buffers the next
// scores are computed while this step's are exponentiated.
// TWO = false is bound by K and V from HBM: 64 KB a tile of 128 columns at 1/148 of the bandwidth takes 2.8 k cycles, a
// stream's step 2 k (24 sequences x 7 tokens x 32 heads, fp16: 79 us, 5.4 TB/s). TWO = true is bound by the tensor cores
// and the shared memory that feeds them: a 128 x 64 x 16 product takes 60 cycles there, not 32, for its 4 KB of Q, so a
// tile takes 2.9 k at best and 3.9 k in fact (131,000 slots x 8 heads x 256 rows, bf16: 154 us, 0.9 PFLOP/s). Measured
// there (153 us then) and not kept: 128-slot steps with one buffer a stream (twice the columns a product, but scores, softmax and
// products one after the other) 184 us; weights by the old maximum while the new one is found 159 us; with no
// exponentials at all it would still be 147 us.
template <int D, bool TWO>
struct TcShape {
    static constexpr int kStage = kTile * D * 2;
    static constexpr int kQBufs = TWO ? 1 : 2;
    static constexpr int kQ = 2 * 128 * D * 2;  // of 256 rows, or of 128 for this segment and the next
    static constexpr int kStages = D == 64 ? 10 : 5;
    static constexpr int kRows = TWO ? 256 : 128;
    static constexpr int kLeast = (TWO ? 1 : 2) + start_of(kRows);  // one tile at least, or one for each stream at once
    static constexpr int kThreads = 384;
    static constexpr int kSmem = kQ + kStages * kStage;
};

template <typename T, int D, bool TWO>
__global__ void __launch_bounds__(TcShape<D, TWO>::kThreads, 1) k_tree_attn_tc(const AttnArgs a, const __grid_constant__ CUtensorMap mk,
                                                                              const __grid_constant__ CUtensorMap mv, float *part_o, float2 *part_ml) {
    using S_ = TcShape<D, TWO>;
    using H = Half16<T>;
    constexpr int NST = S_::kStages, NQ = S_::kQBufs, kBoxes = D / 64, kStep = 64, PER = TWO ? 2 : 1;  // PER: a stream's steps of a tile
    constexpr Cut cut{S_::kRows, kTile, S_::kLeast, start_of(S_::kRows)};
    extern __shared__ __align__(1024) char dyn[];  // the swizzle goes by address bits
    char *sq = dyn, *ring = sq + S_::kQ;
    __shared__ uint64_t b_full[NST], b_empty[NST], b_q[2], b_qfree[2], b_s[2][2], b_p[2][2], b_pv[2][2], b_end[2], b_seg, b_read, b_tail;  // [stream][score buffer]
    __shared__ float2 s_ml[2][TWO ? 1 : 128];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ Share s_share;
    __shared__ unsigned long long s_bad[3];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const Waits wait{&s_gave_up, a.wait_ns};
    if (warp == 0) {
        after_prior();
        const Share s = find_share(a, cut, lane, blockIdx.x, gridDim.x);
        if (lane == 0) s_share = s;
    } else if (warp == 9) {
        tmem_alloc(&s_tmem, 512);
    } else if (tid == 256) {
        map_prefetch(&mk);
        map_prefetch(&mv);
        for (int i = 0; i < NST; ++i) {
            mbar_init(b_full + i, 1);
            mbar_init(b_empty + i, 2);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&b_s[0][0] + i, 1);
            mbar_init(&b_p[0][0] + i, 128);
            mbar_init(&b_pv[0][0] + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_q + i, 32);
            mbar_init(b_qfree + i, 2);
            mbar_init(b_end + i, 1);
        }
        mbar_init(&b_seg, 256);
        mbar_init(&b_read, 256);
        mbar_init(&b_tail, 256);
        s_bad[0] = s_bad[1] = s_bad[2] = 0;
        s_gave_up = 0;
        fence_mbar_init();
    }
    after_prior();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = s_tmem;
    Walk w(a, cut, s_share);

    if (warp == 8) {  // ---------------------------------------------------------------- loads
        uint32_t n = 0;
        bool on = true;
        while (on && w.next()) {
            for (int t = w.ta; on && t < w.tb; ++t)
                for (int z = 0; z < 2; ++z, ++n) {
                    const int st = n % NST;
                    if (!(on = wait(b_empty + st, (n / NST & 1) ^ 1))) break;
                    if (lane == 0) {
                        mbar_expect_tx(b_full + st, S_::kStage);
#pragma unroll
                        for (int x = 0; x < kBoxes; ++x)
                            tma_load(ring + st * S_::kStage + x * 16384, z ? &mv : &mk, 64 * x, t * kTile, w.head(), w.b, b_full + st);
                    }
                }
            w.advance();
        }
        // nothing may be in flight into this CTA's shared memory when it ends
        for (uint32_t i = n > NST ? n - NST : 0; lane == 0 && i < n; ++i) wait.settle(b_full + i % NST, i / NST & 1);
    } else if (warp == 11) {  // ---------------------------------------------------------- queries, a segment ahead where there is room
        uint32_t seg = 0;
        while (w.next()) {
            const int qb = seg % NQ;
            if (!__all_sync(0xffffffffu, wait(b_qfree + qb, (seg / NQ & 1) ^ 1))) break;
            load_q<T, D>(sq + qb * (128 * D * 2), a, w.b, w.head(), w.row0(), w.n * a.group, TWO ? 2 : 1, a.scale < 0.f ? 0x80008000u : 0u, lane);
            fence_proxy_async();
            mbar_arrive(b_q + qb);
            ++seg;
            w.advance();
        }
    } else if (warp > 8) {  // ----------------------------------------------------------- MMAs of stream s
        const int s = __shfl_sync(0xffffffffu, warp, 0) - 9;
        constexpr uint32_t id_s = idesc_of<T>(kStep, false), id_o = idesc_of<T>(D, true);
        uint32_t base = 0, seg = 0, step = 0;  // ring position and the stream's step count at the segment's start
        bool on = true;  // (what the thread waited for has come)
        while (w.next()) {
            const int ns = (w.tb - w.ta) * PER, qb = seg % NQ;
            const uint64_t dq = desc_rows(smem_u32(sq) + (TWO ? s : qb) * (128 * D * 2));
            on = wait(b_q + qb, seg / NQ & 1) && on;
            auto scores = [&](int k) {
                const uint32_t at = base + 2 * (k / PER), st = at % NST, g = step + k, buf = g & 1;
                bool ok = g < 2 || wait(&b_pv[s][buf], ((g - 2) / 2) & 1);  // the P that the buffer held is read
                ok = wait(b_full + st, at / NST & 1) && ok;
                on = on && ok;
                tc_fence_after();
                const uint64_t dk = desc_rows(smem_u32(ring + st * S_::kStage) + (TWO ? k & 1 : s) * (kStep * 128));
                const uint32_t to = tmem + 128 * s + 64 * buf;
                if (elect_one() && on) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        constexpr uint32_t kUnit = 16;  // of a descriptor's address
                        const uint32_t o = ((kk / 4) * 16384 + (kk % 4) * 32) / kUnit;
                        mma_ss(to, dq + o, dk + o, id_s, kk != 0);
                    }
                    if (k % PER == PER - 1) umma_commit(b_empty + st);
                    if (k == ns - 1) umma_commit(b_qfree + qb);
                    umma_commit(&b_s[s][buf]);
                }
                __syncwarp();
            };
            scores(0);
            if (ns > 1) scores(1);
            for (int k = 0; k < ns; ++k) {
                const uint32_t at = base + 2 * (k / PER) + 1, st = at % NST, buf = (step + k) & 1, use = (step + k) / 2 & 1;
                on = wait(&b_p[s][buf], use) && on;
                on = wait(b_full + st, at / NST & 1) && on;
                tc_fence_after();
                const int half = TWO ? k & 1 : s;
                const uint64_t dv = desc_cols(smem_u32(ring + st * S_::kStage) + half * (kStep * 128));
                const uint32_t to = tmem + 256 + 128 * s, from = tmem + 128 * s + 64 * buf;
                // slots behind the drafted tokens are not multiplied, but for the rest of a group of 16
                const int groups = live_groups(w, w.ta + k / PER, half);
                if (elect_one() && on) {
                    if (groups == kStep / 16) {
#pragma unroll
                        for (int kk = 0; kk < kStep / 16; ++kk) mma_ts(to, from + 8 * kk, dv + kk * 128, id_o, (k | kk) != 0);
                    } else {
                        for (int kk = 0; kk < groups; ++kk) mma_ts(to, from + 8 * kk, dv + kk * 128, id_o, (k | kk) != 0);
                    }
                    if (k % PER == PER - 1) umma_commit(b_empty + st);
                    umma_commit(&b_pv[s][buf]);
                }
                __syncwarp();
                if (k + 2 < ns) scores(k + 2);
            }
            base += 2 * (w.tb - w.ta);
            step += ns;
            ++seg;
            w.advance();
        }
        // nor may a product be on its way when TMEM is given back
        if (elect_one()) umma_commit(b_end + s);
        __syncwarp();
        wait.settle(b_end + s, 0);
    } else {  // -------------------------------------------------------------------------- softmax
        const int s = warp / 4, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, tO = tmem + 256 + 128 * s + lanes;
        const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);  // scores in base 2; 0 as a number that vanishes beside them
        uint32_t base = 0, seg = 0, step = 0, tails = 0;
        while (w.next()) {
            const int ns = (w.tb - w.ta) * PER, h = w.head(), row0 = w.row0(), rows = w.n * a.group;
            const int row = row0 + (TWO ? 128 * s : 0) + r;
            const bool live = row < rows;
            const bool warp_live = row0 + (TWO ? 128 * s : 0) + (warp & 3) * 32 < rows;
            if (tid == 0) s_bad[(seg + 1) % 3] = 0;  // last read two segments ago, next written after this one's b_seg
            unsigned long long sees = 0;
            if (live) {
                const int t = row / a.group;
                sees = a.mask ? a.mask[w.b * a.mask_stride + t] : ~0ull >> (63 - t);
                if (w.n < 64) sees &= (1ull << w.n) - 1;
            }
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int k = 0; k < ns; ++k) {
                const int half = TWO ? k & 1 : s, key0 = (w.ta + k / PER) * kTile + half * kStep;
                const bool tail = key0 + kStep > w.len;
                const uint32_t buf = (step + k) & 1, use = (step + k) / 2 & 1, tS = tmem + 128 * s + 64 * buf + lanes;
                wait(&b_s[s][buf], use);
                tc_fence_after();
                if (warp_live) {
                    uint32_t x[2][32], p[32];
                    tmem_ld32(tS, x[0]);
                    tmem_ld32(tS + 32, x[1]);
                    tmem_wait_ld(x[0]);
                    tmem_waited(x[1]);
                    if (tail) {
                        const int off = w.len - key0;  // the step's columns before it are the sequence's
                        hide(x[0], seen32(live, sees, off));
                        hide(x[1], seen32(live, sees, off - 32));
                    }
                    float t4[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) t4[j] = fmaxf(__uint_as_float(x[0][j]), __uint_as_float(x[1][j]));
#pragma unroll
                    for (int j = 4; j < 32; ++j) t4[j & 3] = fmaxf(t4[j & 3], fmaxf(__uint_as_float(x[0][j]), __uint_as_float(x[1][j])));
                    float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                    top = top == -INFINITY ? m : fmaxf(m, top * c);
                    if (m == -INFINITY) m = top;  // nothing summed so far
                    const bool raise = top > m + H::kSlack;
                    if (__any_sync(0xffffffffu, raise)) {
                        wait(&b_pv[s][buf ^ 1], (step + k - 1) / 2 & 1);  // the step before has added its products (a first step never raises)
                        tc_fence_after();
                        const float f = raise ? ex2(m - top) : 1.f;
                        if (raise) m = top;
                        l *= f;
#pragma unroll 1
                        for (int j = 0; j < D / 32; ++j) {
                            tmem_ld32(tO + 32 * j, p);
                            tmem_wait_ld(p);
#pragma unroll
                            for (int i = 0; i < 32; ++i) p[i] = __float_as_uint(__uint_as_float(p[i]) * f);
                            tmem_st32(tO + 32 * j, p);
                        }
                    }
                    const float sub = m == -INFINITY ? 0.f : H::kLift - m;
                    float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float p0 = ex2(fmaf(__uint_as_float(x[j / 16][2 * (j % 16)]), c, sub));
                        const float p1 = ex2(fmaf(__uint_as_float(x[j / 16][2 * (j % 16) + 1]), c, sub));
                        l4[j & 1] += p0;
                        l4[2 + (j & 1)] += p1;
                        p[j] = H::pack(p0, p1);
                    }
                    tmem_st32(tS, p);  // over the scores
                    l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                    tmem_wait_st();
                }
                if (tail) {
                    // Weights are 0 where a row does not see a slot, but 0 times an infinity is not: rows of V behind the
                    // drafted tokens (up to the next 16) become zero, and so do a drafted token's infinities and NaN, which
                    // reach the rows that do see it at the segment's end. TWO: both groups use these rows, and clean every
                    // other one.
                    const uint32_t at = base + 2 * (k / PER) + 1, st = at % NST;
                    wait(b_full + st, at / NST & 1);
                    const int first = max(0, w.len - key0), real = w.len + w.n - key0, last = 16 * live_groups(w, w.ta + k / PER, half);
                    for (int i = TWO ? 2 * r + s : r; i < (last - first) * (D / 8); i += TWO ? 256 : 128) {
                        const int y = first + i / (D / 8), ch = i % (D / 8);
                        uint4 *v = reinterpret_cast<uint4 *>(ring + st * S_::kStage + (ch / 8) * 16384 + (half * kStep + y) * 128 + ((ch % 8) ^ (y % 8)) * 16);
                        if (y >= real) {
                            *v = make_uint4(0, 0, 0, 0);
                        } else {
                            uint32_t q[4] = {v->x, v->y, v->z, v->w};
                            bool bad = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((q[e] & H::kExp) == H::kExp) { q[e] &= 0xFFFF0000u; bad = true; }
                                if ((q[e] >> 16 & H::kExp) == H::kExp) { q[e] &= 0x0000FFFFu; bad = true; }
                            }
                            if (bad) {
                                *v = make_uint4(q[0], q[1], q[2], q[3]);
                                atomicOr(&s_bad[seg % 3], 1ull << (key0 + y - w.len));
                            }
                        }
                    }
                    fence_proxy_async();
                    if (TWO) {
                        mbar_arrive(&b_tail);
                        wait(&b_tail, tails++ & 1);
                    }
                }
                tc_fence_before();
                if (!TWO && k == 0 && seg > 0) wait(&b_read, (seg - 1) & 1);  // both groups have read both accumulators
                mbar_arrive(&b_p[s][buf]);
            }
            const uint32_t last = step + ns - 1;
            wait(&b_pv[s][last & 1], last / 2 & 1);
            tc_fence_after();
            if (!TWO) s_ml[s][r] = make_float2(m, l);
            mbar_arrive(&b_seg);
            wait(&b_seg, seg & 1);
            tc_fence_after();
            const unsigned long long bad = s_bad[seg % 3] & sees;
            // out = sum over this thread's streams of f O, in columns [x0, x0 + width)
            float f0 = 1.f, f1 = 0.f;
            constexpr int width = TWO ? D : D / 2;
            const int x0 = TWO ? 0 : s * width;
            if (!TWO) {
                const float2 o = s_ml[s ^ 1][r];
                const float m0 = s ? o.x : m, m1 = s ? m : o.x, l0 = s ? o.y : l, l1 = s ? l : o.y;
                m = fmaxf(m0, m1);
                f0 = m0 == m ? 1.f : ex2(m0 - m);
                f1 = m1 == m ? 1.f : ex2(m1 - m);
                l = l0 * f0 + l1 * f1;
            }
            if (warp_live) {
                const bool whole = w.whole();
                const int t = row / a.group, head = h * a.group + row % a.group;
                const long long pr = ((long long)blockIdx.x * 2 + (w.opens ? 0 : 1)) * S_::kRows + (TWO ? 128 * s : 0) + r;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                T *out = static_cast<T *>(a.out) + w.b * a.os[0] + t * a.os[1] + (long long)head * a.os[2];
                float *po = part_o + pr * D;
                const uint32_t t0 = tmem + 256 + lanes + (TWO ? 128 * s : 0) + x0;
#pragma unroll 1
                for (int j = 0; j < width; j += 32) {
                    uint32_t o[32];
                    tmem_ld32(t0 + j, o);
                    tmem_wait_ld(o);
                    if (!TWO) {
                        uint32_t o1[32];
                        tmem_ld32(t0 + 128 + j, o1);
                        tmem_wait_ld(o1);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(o1[i]), f1, __uint_as_float(o[i]) * f0));
                    }
                    if (live && whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t q[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) q[e] = H::pack(__uint_as_float(o[i + 2 * e]) * inv, __uint_as_float(o[i + 2 * e + 1]) * inv);
                            *reinterpret_cast<uint4 *>(out + x0 + j + i) = make_uint4(q[0], q[1], q[2], q[3]);
                        }
                    } else if (live) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8)  // a whole sector a thread: half as many requests to L2 as with 16 bytes
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(po + x0 + j + i), "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]),
                                         "r"(o[i + 3]), "r"(o[i + 4]), "r"(o[i + 5]), "r"(o[i + 6]), "r"(o[i + 7])
                                         : "memory");
                    }
                }
                if (live && bad) {
                    const T *v = static_cast<const T *>(a.v) + w.b * a.vs[0] + h * a.vs[1] + (long long)w.len * a.vs[2];
                    if (whole) add_bad(out, v, a.vs[2], bad, x0, x0 + width);
                    else add_bad(po, v, a.vs[2], bad, x0, x0 + width);
                }
                if (live && x0 == 0) {
                    if (!whole) part_ml[pr] = make_float2(m, l);
                    else if (a.lse) a.lse[((long long)w.b * a.tokens + t) * a.heads + head] = l == 0.f ? -INFINITY : (m - H::kLift + log2f(l)) * 0.6931471805599453f;
                }
            }
            tc_fence_before();
            if (!TWO) mbar_arrive(&b_read);
            base += 2 * (w.tb - w.ta);
            step += ns;
            ++seg;
            w.advance();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

// Adds up a unit's parts in their order, one warp per query row, AHEAD parts a round of loads. Bound by its rounds where
// rows are few, by how many blocks fit an SM where they are many (fewer loads ahead, fewer registers).
template <typename T, int D, int AHEAD>
__global__ void __launch_bounds__(256) k_attn_join(const AttnArgs a, Cut cut, int ctas, float lift, const float *part_o, const float2 *part_ml) {
    // Everything up to the wait comes from the call's inputs; the parts are the attention kernel's outputs. The blocks start
    // early where an SM has room: on one without an attention CTA, or whose CTA has ended. Beside a CTA their registers fit only with
    // 32-bit caches and one row tile (a 16-bit one leaves 7 K of 65,536, a block wants 12 K to 27 K). Every warp waits, with or without
    // something to add: what follows in the stream waits for this launch alone.
    constexpr int W = D / 32;
    const int lane = threadIdx.x % 32;
    const long long id = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    const bool is = id < (long long)a.batch * a.tokens * a.heads;
    const int head = is ? (int)(id % a.heads) : 0, t = is ? (int)(id / a.heads % a.tokens) : 0, b = is ? (int)(id / a.heads / a.tokens) : 0;
    int len, n, u0 = 0, each = 1, c0 = 0, c1 = 0;
    const bool ok = seq_range(a.lens, a.counts, b, a.tokens, a.slots, len, n) && t < n && is;
    const int h = head / a.group, row = t * a.group + head % a.group;
    if (ok) {
        bool bad = false;
        int total = 0, before = 0, l_, n_;
        for (int x = lane; x < a.batch; x += 32) {
            const int k = seq_tiles(a, cut, x, l_, n_, &bad);
            total += k;
            before += x < b ? k : 0;
        }
        total = __reduce_add_sync(0xffffffffu, total);
        before = __reduce_add_sync(0xffffffffu, before);
        each = share_of(total, cut, ctas);
        const int blocks = (n * a.group + cut.rblock - 1) / cut.rblock, nt = (len + n + cut.tile - 1) / cut.tile;
        u0 = before + (h * blocks + row / cut.rblock) * (nt + cut.start);
        c0 = (u0 + cut.start) / each;
        c1 = (u0 + cut.start + nt - 1) / each;
    }
    after_prior();
    if (c0 == c1) return;  // finished by that CTA, or not there
    auto at = [&](int c) { return ((long long)c * 2 + (c == c0 && c0 * each < u0 ? 1 : 0)) * cut.rblock + row % cut.rblock; };
    float m = -INFINITY, l = 0.f, acc[W] = {};
    for (int c = c0; c <= c1; c += AHEAD) {  // all loads of AHEAD parts at once; lane i has the statistics of part c + i
        const int cnt = min(AHEAD, c1 - c + 1);
        const float2 ml = lane < cnt ? part_ml[at(c + lane)] : make_float2(-INFINITY, 0.f);
        float v[AHEAD][W];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (i < cnt) {
                const float *p = part_o + at(c + i) * D + lane * W;
                if (W == 4) *reinterpret_cast<float4 *>(v[i]) = *reinterpret_cast<const float4 *>(p);
                else *reinterpret_cast<float2 *>(v[i]) = *reinterpret_cast<const float2 *>(p);
            }
        float top = ml.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, m);
        const float f = ml.x == top ? 1.f : ex2(ml.x - top), old = m == top ? 1.f : ex2(m - top);
        m = top;
        float sum = ml.y * f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, old, sum);
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] *= old;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float fi = __shfl_sync(0xffffffffu, f, i);
            if (i < cnt)
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k] = fmaf(v[i][k], fi, acc[k]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *out = static_cast<T *>(a.out) + b * a.os[0] + t * a.os[1] + (long long)head * a.os[2] + lane * W;
#pragma unroll
    for (int k = 0; k < W; ++k) out[k] = from_f<T>(acc[k] * inv);
    if (a.lse && lane == 0) a.lse[((long long)b * a.tokens + t) * a.heads + head] = l == 0.f ? -INFINITY : (m - lift + log2f(l)) * 0.6931471805599453f;
}

// The mass kernel: S^T = K Q^T, a tile's 128 slots as the TMEM lanes and the query rows as its columns, so that a thread
// holds one slot and sums it over rows. Four score buffers of 128 columns, each with four warps of its own: with more than
// 32 rows two of them take the halves of a tile's rows, so that two tiles are under way, with fewer rows four tiles are. A
// buffer is given back once its last columns are in registers, before their exponentials. Keys come through a TMA ring,
// the unit's query rows and their -lse stay in shared memory. Bound by K from HBM up to about 170 rows (32 KB a tile: 1.4 k
// cycles at 1/148 of the bandwidth; 7 tokens x 32 heads over 24 x 8 k slots: 69 us, 6.0 TB/s), by the exponentials (8 cycles
// a row and tile) beyond: 64 tokens x 32 heads over 2 x 32 k slots 54 us (50 of keys that are partly in
// L2), of which the exponentials are 29. That case, of such keys, took 84 us with one group a buffer, 66 with two that shared one
// and with the query rows loaded one piece after the other, 55 without what mass_cut counts. With few rows it costs up to 4 us in 28 to have more than four stages.
template <int D, int ROWS>
struct MassShape {
    static constexpr int kStage = kTile * D * 2;
    static constexpr int kQ = ROWS * D * 2;
    static constexpr int kStages = D == 64 ? 6 : ROWS == 512 ? 2 : 4;
    static constexpr int kSmem = kQ + kStages * kStage;
};

// With many rows it takes as long as four tiles to load them behind the first tiles of K and to fill and drain the buffers.
__host__ __device__ constexpr Cut mass_cut(int rows) { return {1 << 30, kTile, 1, rows > 128 ? 4 : 0}; }

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(576, 1) k_attn_mass_tc(const AttnArgs a, const __grid_constant__ CUtensorMap mk) {
    using S_ = MassShape<D, ROWS>;
    constexpr int NST = S_::kStages, kBoxes = D / 64, C = D / 8, kAtom = ROWS * 128;
    constexpr bool SPLIT = ROWS > 32;          // halves of the rows, or every group has tiles of its own
    constexpr int kTurns = SPLIT ? 2 : 4;
    extern __shared__ __align__(1024) char dyn[];
    char *sq = dyn, *ring = sq + S_::kQ;
    __shared__ uint64_t b_full[NST], b_empty[NST], b_s[4], b_free[4], b_q, b_seg, b_end;
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ Share s_share;
    __shared__ alignas(16) float s_nl[ROWS];
    __shared__ float s_sum[2][2][128];
    __shared__ int s_skips;  // 1 + the last segment with a row that counts for nothing
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const Waits wait{&s_gave_up, a.wait_ns};
    const Cut cut = mass_cut(a.tokens * a.gc);
    if (warp == 0) {
        after_prior();
        const Share s = find_share(a, cut, lane, blockIdx.x, gridDim.x);
        if (lane == 0) s_share = s;
    } else if (warp == 17) {
        tmem_alloc(&s_tmem, 512);
    } else if (tid == 512) {
        map_prefetch(&mk);
        for (int i = 0; i < NST; ++i) {
            mbar_init(b_full + i, 1);
            mbar_init(b_empty + i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(b_s + i, 1);
            mbar_init(b_free + i, 128);
        }
        mbar_init(&b_q, 512);
        mbar_init(&b_seg, 512);
        mbar_init(&b_end, 1);
        s_gave_up = 0;
        s_skips = 0;
        fence_mbar_init();
    }
    after_prior();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    Walk w(a, cut, s_share);

    if (warp == 16) {  // ---------------------------------------------------------------- loads
        uint32_t n = 0;
        bool on = true;
        while (on && w.next()) {
            for (int t = w.ta; t < w.tb; ++t, ++n) {
                const int st = n % NST;
                if (n == 2 && w.opens && w.n * a.gc > 64) on = wait(&b_q, 0);  // the first query rows before the rest of the ring: 0.7 us
                if (!(on = on && wait(b_empty + st, (n / NST & 1) ^ 1))) break;
                if (lane == 0) {
                    mbar_expect_tx(b_full + st, S_::kStage);
#pragma unroll
                    for (int x = 0; x < kBoxes; ++x) tma_load(ring + st * S_::kStage + x * 16384, &mk, 64 * x, t * kTile, w.u, w.b, b_full + st);
                }
            }
            w.advance();
        }
        for (uint32_t i = n > NST ? n - NST : 0; lane == 0 && i < n; ++i) wait.settle(b_full + i % NST, i / NST & 1);
    } else if (warp == 17) {  // ----------------------------------------------------------- MMAs
        uint32_t n = 0, seg = 0, held = 0;  // (bit: the phase of b_free)
        bool on = true;
        while (w.next()) {
            const int rows = w.n * a.gc;
            on = wait(&b_q, seg & 1) && on;
            tc_fence_after();
            for (int t = w.ta; t < w.tb; ++t, ++n) {
                const int st = n % NST, s = (t - w.ta) % kTurns;
                on = wait(b_full + st, n / NST & 1) && on;
                for (int r0 = 0; r0 < rows; r0 += 256) {
                    const int all = min(rows - r0, 256), mid = min((all + 63) / 64 * 32, all);
                    for (int half = 0; half < 2; ++half) {
                        const int from = half ? mid : 0, cols = ((half ? all : mid) - from + 15) / 16 * 16, g = SPLIT ? 2 * s + half : s;
                        if (!cols) break;
                        on = wait(b_free + g, (held >> g & 1) ^ 1) && on;
                        held ^= 1u << g;
                        tc_fence_after();
                        const uint64_t dk = desc_rows(smem_u32(ring + st * S_::kStage)), dq = desc_rows(smem_u32(sq) + (r0 + from) * 128);
                        const uint32_t id = idesc_of<T>(cols, false), to = tmem + 128 * g;
                        if (elect_one() && on) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk)
                                mma_ss(to, dk + ((kk / 4) * 16384 + (kk % 4) * 32) / 16, dq + ((kk / 4) * kAtom + (kk % 4) * 32) / 16, id, kk != 0);
                            if (r0 + 256 >= rows && (half || mid == all)) umma_commit(b_empty + st);
                            umma_commit(b_s + g);
                        }
                        __syncwarp();
                    }
                }
            }
            ++seg;
            w.advance();
        }
        if (elect_one()) umma_commit(&b_end);  // nothing may be on its way when TMEM is given back
        __syncwarp();
        wait.settle(&b_end, 0);
    } else {  // -------------------------------------------------------------------------- sums
        const int s = warp / 4 % kTurns, half = SPLIT ? warp / 8 : 0, g = SPLIT ? 2 * s + half : s, r = tid & 127;
        const uint32_t tS = tmem + 128 * g + ((uint32_t)(warp & 3) << 21);
        const float c = a.scale * 1.4426950408889634f;
        uint32_t seg = 0, c_s = 0, it = 0;
        while (w.next()) {
            const int rows = w.n * a.gc, h = w.u;
            // Query rows warp, warp + 16, ..: lane i finds where the i-th lies and its lse, then 16 bytes a lane, eight loads
            // under way. (Rows that count for nothing are kept out of the sums; what their queries are does not matter.)
            long long at = -1;
            if (const int row = warp + 16 * lane; row < rows) {
                const int k = row / a.gc, head = h * a.group + a.g0 + row - k * a.gc;
                const int src = a.rows ? a.rows[(long long)w.b * a.tokens + k] : k;
                float nl = -INFINITY;
                if (src < 0 || src >= a.tokens) {
                    atomicOr(&g_cache_error, kErrRange);
                } else {
                    at = w.b * a.qs[0] + src * a.qs[1] + (long long)head * a.qs[2];
                    const float lse = a.lse_in[((long long)w.b * a.tokens + src) * a.heads + head];
                    if (lse != -INFINITY) nl = lse * -1.4426950408889634f;
                }
                s_nl[row] = nl;
                if (nl == -INFINITY) s_skips = seg + 1;
            }
            constexpr int kPer = 32 / C, kAhead = SPLIT ? 8 : 1;  // rows of a load, loads (32 rows: one)
            const int ch = lane % C;
            for (int i0 = 0; warp + 16 * i0 < rows; i0 += kPer * kAhead) {
                uint4 v[kAhead];
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
                    const int i = i0 + kPer * x + lane / C;
                    const long long from = __shfl_sync(0xffffffffu, at, i & 31);
                    v[x] = make_uint4(0, 0, 0, 0);
                    if (warp + 16 * i < rows && from >= 0) v[x] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + from + ch * 8);
                }
#pragma unroll
                for (int x = 0; x < kAhead; ++x)
                    if (const int row = warp + 16 * (i0 + kPer * x + lane / C); row < rows)
                        *reinterpret_cast<uint4 *>(sq + (ch / 8) * kAtom + row * 128 + ((ch ^ row) & 7) * 16) = v[x];
            }
            fence_proxy_async();
            mbar_arrive(&b_q);
            wait(&b_q, seg & 1);  // s_nl is there
            const bool skips = s_skips == seg + 1;  // (then the sums leave them out)
            const float *min_ = a.mass + w.b * a.ms[0] + h * a.ms[1];
            float *mout = a.mass_out + w.b * a.mos[0] + h * a.mos[1];
            for (int t = w.ta + s; t < w.tb; t += kTurns) {
                const int key = t * kTile + r, late = key - w.len;
                const bool tail = t * kTile + kTile > w.len;
                float before = 0.f;
                if (half == 0) {
                    if (late < 0) before = min_[key];
                    else if (a.more && late < w.n) before = mout[key];
                }
                const int from = late > 0 ? (late < w.n ? late * a.gc : rows) : 0;  // the first row that sees the slot
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                for (int r0 = 0; r0 < rows; r0 += 256) {
                    const int all = min(rows - r0, 256), mid = min((all + 63) / 64 * 32, all), cnt = half ? all : mid;
                    if (half && mid == all) break;
                    wait(b_s + g, c_s++ & 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int j = half ? mid : 0; j < cnt; j += 32) {
                        uint32_t x[32];
                        tmem_ld32(half ? tS + j - mid : tS + j, x);
                        tmem_wait_ld(x);
                        if (j + 32 >= cnt) {  // all read: the next scores may come
                            tc_fence_before();
                            mbar_arrive(b_free + g);
                        }
                        const float4 *nl = reinterpret_cast<const float4 *>(s_nl + r0 + j);
                        if (tail || skips || j + 32 > cnt) {
                            const int lo = from - r0 - j, hi = cnt - j;
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                const float n1 = k < hi ? s_nl[r0 + j + k] : -INFINITY, p = ex2(fmaf(__uint_as_float(x[k]), c, n1));
                                sum[k & 3] += k >= lo && n1 != -INFINITY ? p : 0.f;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float4 n4 = nl[k];
                                sum[0] += ex2(fmaf(__uint_as_float(x[4 * k]), c, n4.x));
                                sum[1] += ex2(fmaf(__uint_as_float(x[4 * k + 1]), c, n4.y));
                                sum[2] += ex2(fmaf(__uint_as_float(x[4 * k + 2]), c, n4.z));
                                sum[3] += ex2(fmaf(__uint_as_float(x[4 * k + 3]), c, n4.w));
                            }
                        }
                    }
                }
                float sums = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (SPLIT && rows > 32) {  // the other half's; two places by turns, so that one barrier a tile is enough
                    float *other = &s_sum[s][it++ & 1][r];
                    if (half) *other = sums;
                    asm volatile("bar.sync %0, 256;" ::"r"(1 + s) : "memory");
                    if (!half) sums += *other;
                }
                if (!half && late < w.n) mout[key] = before + sums;
            }
            mbar_arrive(&b_seg);  // all groups have seen all of the segment's scores: its query rows are done with
            wait(&b_seg, seg & 1);
            ++seg;
            w.advance();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 17) tmem_dealloc(tmem, 512);
}

// ================================================================================================================
// 32-bit caches: products of 32-bit values on the tensor cores
// ================================================================================================================
// x = hi + lo, both TF32 (8 + 11 bits; hi rounded, so that lo has either sign): x y = hi hi' + hi lo' + lo hi' up to
// 2^-21 |x y|, three mma.sync products with fp32 sums. The tensor cores cut what they add off, they do not round it: so
// products with a small piece have sums of their own, a tile's products of weights and values are added to the
// accumulator by fp32 additions, and scores have two sums (all in one, and hi cut off: 2.8e-6 off 64 bits instead of
// 0.6e-6, where a plain fp32 product is 1.2e-6 off; at 12 tokens x 32 heads over 2,047 slots it
// cost 2.5 us of 27). (tcgen05 takes its operands from shared memory, where the split of K and V would have to be written back: more
// shared-memory traffic than the products take. From registers a split costs three integer or fp32 operations.)
// A product waits for the one before it on the same sum (four of them take that long to issue), so the order is by piece,
// through as many sums as there are.
struct Split {
    uint32_t hi, lo;  // the tensor cores leave out the last 13 bits
};
// kAny: x may be anything. Rounding carries the last 2^12 numbers below infinity over to it, so hi comes from a magnitude
// below them (lo then has up to 13 bits); an infinity stays one, in lo. It is the fourth operation of a split: 12 tokens x 32
// heads over 2,047 slots take 28.7 us, not 27.8, 64 tokens over 8,192 slots 217, not 207, masses of 12 tokens over 32,768 slots
// 81, not 78. Weights are never that large, and queries are kept below it when they are staged.
constexpr uint32_t kRounds = 0x7F7FEFFFu;  // the largest number that is rounded to a finite one
template <bool kAny>
__device__ __forceinline__ Split split(float x) {
    float y = x;
    if (kAny) asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(__uint_as_float(kRounds)));
    Split s;
    s.hi = (__float_as_uint(y) + 0x1000u) & 0xFFFFE000u;
    s.lo = __float_as_uint(x - __uint_as_float(s.hi));
    return s;
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
struct Frag {  // a 16 x 8 left operand: queries or weights
    Split x[4];
    __device__ __forceinline__ Frag(float x0, float x1, float x2, float x3) {
        x[0] = split<false>(x0);
        x[1] = split<false>(x1);
        x[2] = split<false>(x2);
        x[3] = split<false>(x3);
    }
};
// a query's value times the scale, finite ones below what split<false> can take
__device__ __forceinline__ float staged(float x, float c) {
    const float y = x * c;
    return isfinite(y) ? copysignf(fminf(fabsf(y), __uint_as_float(kRounds)), y) : y;
}
__device__ __forceinline__ void mma_part(float (&c)[4], const Frag &a, int part, const Split &u, const Split &v) {  // the small pieces first
    if (part == 0) mma8(c, a.x[0].hi, a.x[1].hi, a.x[2].hi, a.x[3].hi, u.lo, v.lo);
    else if (part == 1) mma8(c, a.x[0].lo, a.x[1].lo, a.x[2].lo, a.x[3].lo, u.hi, v.hi);
    else mma8(c, a.x[0].hi, a.x[1].hi, a.x[2].hi, a.x[3].hi, u.hi, v.hi);
}
// c[i] += a (b0[i], b1[i]) for four sums of the large pieces' products, x[i] for those with a small one
__device__ __forceinline__ void mma_four(float (&c)[4][4], float (&x)[4][4], const Frag &a, const float4 &b0, const float4 &b1) {
    const Split u[4] = {split<true>(b0.x), split<true>(b0.y), split<true>(b0.z), split<true>(b0.w)};
    const Split v[4] = {split<true>(b1.x), split<true>(b1.y), split<true>(b1.z), split<true>(b1.w)};
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_part(part < 2 ? x[i] : c[i], a, part, u[i], v[i]);
}
// 16 columns of scores: c[0] and c[1] each take half of the columns' large pieces, c[2] the products with a small one, for N
// groups of slots (k[j]: a lane's four columns)
template <int N>
__device__ __forceinline__ void mma_scores(float (&c)[3][N][4], const float4 &q0, const float4 &q1, const float4 (&k)[N]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const Frag a = half ? Frag(q0.z, q1.z, q0.w, q1.w) : Frag(q0.x, q1.x, q0.y, q1.y);
        Split s[N][2];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            s[j][0] = split<true>(half ? k[j].z : k[j].x);
            s[j][1] = split<true>(half ? k[j].w : k[j].y);
        }
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int j = 0; j < N; ++j) mma_part(c[part < 2 ? 2 : half][j], a, part, s[j][0], s[j][1]);
    }
}
constexpr int kTile32 = 64;
// A stage holds 64 slots in parts of 32 columns as the tensor map's loads leave them: 128-byte rows, the 16-byte pieces
// exchanged by the row's last three bits.
__device__ __forceinline__ float4 stage32(const char *st, int slot, int col4) {  // columns 4 col4 ..
    return *reinterpret_cast<const float4 *>(st + (col4 / 8) * 8192 + slot * 128 + ((col4 % 8) ^ (slot % 8)) * 16);
}
// Query rows: 16-byte pieces exchanged between the halves of 128 bytes in every other row (two rows are read at a time).
template <int D>
__device__ __forceinline__ float4 *query32(char *sq, int row, int col4) {
    return reinterpret_cast<float4 *>(sq + row * (D * 4) + (col4 ^ ((row & 1) << 2)) * 16);
}

// A group of four warps has 16 query rows. In a tile of 64 slots warp w of it computes the scores of slots 16 w .., the
// group agrees on the running maximum, the weights go through shared memory, and warp w adds up the columns 32 w .. (of 64
// columns: of half of the slots) of all weights and values. So every group keeps all four schedulers busy whatever the
// number of row tiles, and a warp holds 16 accumulators a thread, not 64 (eight warps with all columns of their own slots
// took 28.1 us where this took 24.7, 12 tokens x 32 heads over 2,047 slots). RT row tiles share every tile of K and V;
// with fewer than four, two such sets of groups take the tiles in turn (NS) and are joined at the segment's end.
// Within the products the columns of K (and the slots in S and P) are taken in the order in which a lane finds them in 16
// consecutive bytes: the sums do not depend on it.
// Bound by K and V from HBM for up to 16 rows, by the products beyond.
template <int D, int RT>
struct F32Shape {
    static constexpr int NS = RT == 4 ? 1 : 2, kGroups = RT * NS, kWarps = 4 * kGroups, kThreads = kWarps * 32 + 32;
    static constexpr int kSlices = D / 32, kParts = 4 / kSlices;  // of the columns; of the slots for each
    static constexpr int kStage = kTile32 * D * 4;
    static constexpr int kStages = D == 64 ? 8 : 5;
    static constexpr int kP = 68;  // a row of weights, so that rows start four banks apart
    static constexpr int kQ = RT * 16 * D * 4, kWeights = kGroups * 16 * kP * 4, kJoin = (NS * kParts - 1) * RT * 16 * D * 4;
    static constexpr int kSmem = kStages * kStage + kQ + kWeights + kJoin;
};

template <int D, int RT>
__global__ void __launch_bounds__(F32Shape<D, RT>::kThreads, 1) k_tree_attn_f32(const AttnArgs a, const __grid_constant__ CUtensorMap mk,
                                                                               const __grid_constant__ CUtensorMap mv, float *part_o, float2 *part_ml) {
    using S_ = F32Shape<D, RT>;
    constexpr int NST = S_::kStages, NS = S_::NS, PARTS = S_::kParts, R = RT * 16, P = S_::kP, ALL = S_::kWarps * 32;
    constexpr Cut cut{R, kTile32, 1, 0};
    extern __shared__ __align__(1024) char dyn[];
    char *ring = dyn, *sq = ring + NST * S_::kStage;
    float *weights = reinterpret_cast<float *>(sq + S_::kQ), *join = weights + S_::kWeights / 4;
    __shared__ uint64_t b_full[NST], b_empty[NST];
    __shared__ int s_gave_up;
    __shared__ Share s_share;
    __shared__ float s_max[S_::kGroups][4][16], s_sum[S_::kGroups][4][16], s_m[S_::kGroups][16];
    __shared__ unsigned long long s_bad;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const Waits wait{&s_gave_up, a.wait_ns};
    if (warp == 0) {
        after_prior();
        const Share s = find_share(a, cut, lane, blockIdx.x, gridDim.x);
        if (lane == 0) s_share = s;
    } else if (tid == ALL) {
        map_prefetch(&mk);
        map_prefetch(&mv);
        for (int i = 0; i < NST; ++i) {
            mbar_init(b_full + i, 1);
            mbar_init(b_empty + i, 4 * RT);
        }
        s_gave_up = 0;
        s_bad = 0;
        fence_mbar_init();
    }
    after_prior();
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Walk w(a, cut, s_share);
    if (tid >= ALL) {  // loads
        uint32_t n = 0;
        bool on = true;
        while (on && w.next()) {
            for (int t = w.ta; on && t < w.tb; ++t)
                for (int z = 0; z < 2; ++z, ++n) {
                    const int st = n % NST;
                    if (!(on = wait.arrivals(b_empty + st, (n / NST & 1) ^ 1))) break;
                    if (lane == 0) {
                        mbar_expect_tx(b_full + st, S_::kStage);
#pragma unroll
                        for (int x = 0; x < D / 32; ++x)
                            tma_load(ring + st * S_::kStage + x * 8192, z ? &mv : &mk, 32 * x, t * kTile32, w.head(), w.b, b_full + st);
                    }
                }
            w.advance();
        }
        for (uint32_t i = n > NST ? n - NST : 0; lane == 0 && i < n; ++i) wait.settle(b_full + i % NST, i / NST & 1);
        return;
    }
    const int group = warp / 4, rt = group % RT, ns = group / RT, wq = warp % 4, g = lane / 4, t = lane % 4;
    const int slice = wq % S_::kSlices, part = wq / S_::kSlices, contrib = ns * PARTS + part;
    auto sync_group = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
    auto sync_all = [&] { asm volatile("bar.sync 8, %0;" ::"n"(ALL) : "memory"); };
    float *pw = weights + group * 16 * P;
    const float c = a.scale * 1.4426950408889634f;
    uint32_t base = 0;
    while (w.next()) {
        const int h = w.head(), row0 = w.row0(), rows = w.n * a.group;
        const float *q = static_cast<const float *>(a.q) + w.b * a.qs[0];
        constexpr int C = D / 4, QN = (R * C + ALL - 1) / ALL;  // a thread's pieces of the query rows, all in flight at once
        float4 qv[QN];
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = tid / C + i * (ALL / C), row = row0 + r, tok = row / a.group;
            qv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < R && row < rows) qv[i] = *reinterpret_cast<const float4 *>(q + tok * a.qs[1] + (long long)(h * a.group + row - tok * a.group) * a.qs[2] + 4 * (tid % C));
        }
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const float4 v = qv[i];
            const int r = tid / C + i * (ALL / C);
            if (r < R) *query32<D>(sq, r, tid % C) = make_float4(staged(v.x, c), staged(v.y, c), staged(v.z, c), staged(v.w, c));  // scores in base 2
        }
        sync_all();
        const bool live = row0 + 16 * rt < rows;  // the group has rows
        unsigned long long sees[2] = {0, 0};
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[4][4] = {};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int row = row0 + 16 * rt + g + 8 * y;
            if (row < rows) {
                const int tok = row / a.group;
                sees[y] = a.mask ? a.mask[w.b * a.mask_stride + tok] : ~0ull >> (63 - tok);
                if (w.n < 64) sees[y] &= (1ull << w.n) - 1;
            }
        }
#pragma unroll 1
        for (int tile = w.ta + ns; tile < w.tb; tile += NS) {
            const uint32_t nk = base + 2 * (tile - w.ta), nv = nk + 1;
            const int stk = nk % NST, stv = nv % NST;
            const int key0 = tile * kTile32, off = key0 + 16 * wq;  // off: the first slot of the warp's scores
            const bool tail = key0 + kTile32 > w.len;
            float s[2][4];
            wait(b_full + stk, nk / NST & 1);
            if (live) {
                const char *st = ring + stk * S_::kStage;
                const int slot = 16 * wq + (g >> 1) + ((g & 1) << 2);
                float s2[3][2][4] = {};
#pragma unroll 1
                for (int d = 0; d < D / 16; ++d) {
                    const float4 k[2] = {stage32(st, slot, 4 * d + t), stage32(st, slot + 8, 4 * d + t)};
                    mma_scores(s2, *query32<D>(sq, 16 * rt + g, 4 * d + t), *query32<D>(sq, 16 * rt + g + 8, 4 * d + t), k);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = (s2[0][j][e] + s2[1][j][e]) + s2[2][j][e];  // row g + 8 (e / 2), slot off + 8 j + t + 4 (e % 2)
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(b_empty + stk);
            if (live) {
                if (tail) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int at = off + 8 * j + t + 4 * (e & 1) - w.len, row = row0 + 16 * rt + g + 8 * (e >> 1);
                            if (row >= rows || (at >= 0 && (at >= w.n || !(sees[e >> 1] >> at & 1)))) s[j][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float top = fmaxf(fmaxf(s[0][2 * y], s[0][2 * y + 1]), fmaxf(s[1][2 * y], s[1][2 * y + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (t == 0) s_max[group][wq][g + 8 * y] = top;
                }
                sync_group();
                float f[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int r = g + 8 * y;
                    const float top = fmaxf(fmaxf(fmaxf(s_max[group][0][r], s_max[group][1][r]), fmaxf(s_max[group][2][r], s_max[group][3][r])), m[y]);
                    f[y] = top == m[y] ? 1.f : ex2(m[y] - top);
                    m[y] = top;
                    const float sub = top == -INFINITY ? 0.f : top;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float p = ex2(s[j][2 * y + e] - sub);
                            sum += p;
                            pw[r * P + 16 * wq + 8 * j + t + 4 * e] = p;
                        }
                    l[y] = l[y] * f[y] + sum;
                }
                if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[i][0] *= f[0];
                        o[i][1] *= f[0];
                        o[i][2] *= f[1];
                        o[i][3] *= f[1];
                    }
                }
            }
            wait(b_full + stv, nv / NST & 1);
            if (live) {
                char *st = ring + stv * S_::kStage;
                const int eights = (w.len + w.n - key0 + 7) / 8;  // of the tile's slots that hold something; the others are not multiplied
                if (tail) {
                    // A weight of 0 times an infinity is not 0: slots that no row sees become zero (as far as they are multiplied),
                    // and so do a drafted token's infinities and NaN (they reach the rows that see it at the segment's end).
                    // Groups with other rows of the same slots write the same zeros.
#pragma unroll 1
                    for (int i = max(0, w.len - key0) * (D / 4) + wq * 32 + lane; i < min(8, eights) * 8 * (D / 4); i += 128) {
                        const int slot = i / (D / 4), col4 = i % (D / 4), at = key0 + slot - w.len;
                        float4 *v = reinterpret_cast<float4 *>(st + (col4 / 8) * 8192 + slot * 128 + ((col4 % 8) ^ (slot % 8)) * 16);
                        const float4 x = *v;
                        if (at < w.n && isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w)) continue;
                        if (at < w.n) atomicOr(&s_bad, 1ull << at);
                        const bool real = at < w.n;
                        *v = make_float4(real && isfinite(x.x) ? x.x : 0.f, real && isfinite(x.y) ? x.y : 0.f, real && isfinite(x.z) ? x.z : 0.f,
                                         real && isfinite(x.w) ? x.w : 0.f);
                    }
                    fence_proxy_async();  // the stage is the TMA's again after this tile
                }
                sync_group();  // the weights are there
                const int j1 = min((part + 1) * (8 / PARTS), eights), col4 = 8 * slice + (g >> 1) + ((g & 1) << 2);
                float large[4][4] = {}, small[4][4] = {};
#pragma unroll 1
                for (int j = part * (8 / PARTS); j < j1; ++j) {
                    const float *x = pw + g * P + 8 * j + t;
                    mma_four(large, small, Frag(x[0], x[8 * P], x[4], x[8 * P + 4]), stage32(st, 8 * j + t, col4), stage32(st, 8 * j + t + 4, col4));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] += large[i][e] + small[i][e];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(b_empty + stv);
        }
        // o[i][2 y + e]: row g + 8 y, column 32 slice + 16 e + 4 t + i
        if (live) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
                l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
                if (t == 0) {
                    s_sum[group][wq][g + 8 * y] = l[y];
                    if (wq == 0) s_m[group][g + 8 * y] = m[y];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (contrib > 0)
                        *reinterpret_cast<float4 *>(join + (((contrib - 1) * RT + rt) * 16 + g + 8 * y) * D + 32 * slice + 16 * e + 4 * t) =
                            make_float4(o[0][2 * y + e], o[1][2 * y + e], o[2][2 * y + e], o[3][2 * y + e]);
            }
        }
        sync_all();
        if (contrib == 0 && live) {
            const bool whole = w.whole();
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int r = g + 8 * y, row = row0 + 16 * rt + r;
                float top = m[y], f[NS], sum = 0.f;
#pragma unroll
                for (int x = 0; x < NS; ++x) top = fmaxf(top, s_m[x * RT + rt][r]);
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const float mx = s_m[x * RT + rt][r];
                    f[x] = mx == top ? 1.f : ex2(mx - top);
                    sum += f[x] * ((s_sum[x * RT + rt][0][r] + s_sum[x * RT + rt][1][r]) + (s_sum[x * RT + rt][2][r] + s_sum[x * RT + rt][3][r]));
                }
                if (row >= rows) continue;
                const int tok = row / a.group, head = h * a.group + row - tok * a.group;
                const long long pr = ((long long)blockIdx.x * 2 + (w.opens ? 0 : 1)) * R + 16 * rt + r;
                const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                float *out = whole ? static_cast<float *>(a.out) + w.b * a.os[0] + tok * a.os[1] + (long long)head * a.os[2] : part_o + pr * D;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = 32 * slice + 16 * e + 4 * t;
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = o[i][2 * y + e] * f[0];
#pragma unroll
                    for (int x = 1; x < NS * PARTS; ++x) {
                        const float4 z = *reinterpret_cast<const float4 *>(join + (((x - 1) * RT + rt) * 16 + r) * D + col);
                        const float fx = f[x / PARTS];
                        v[0] = fmaf(z.x, fx, v[0]);
                        v[1] = fmaf(z.y, fx, v[1]);
                        v[2] = fmaf(z.z, fx, v[2]);
                        v[3] = fmaf(z.w, fx, v[3]);
                    }
                    *reinterpret_cast<float4 *>(out + col) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                }
                const unsigned long long bad = s_bad & sees[y];
                if (bad) {  // the thread's own columns
                    const float *v = static_cast<const float *>(a.v) + w.b * a.vs[0] + h * a.vs[1] + (long long)w.len * a.vs[2];
                    for (int e = 0; e < 2; ++e) add_bad(out, v, a.vs[2], bad, 32 * slice + 16 * e + 4 * t, 32 * slice + 16 * e + 4 * t + 4);
                }
                if (t == 0 && wq == 0) {
                    if (!whole) part_ml[pr] = make_float2(top, sum);
                    else if (a.lse) a.lse[((long long)w.b * a.tokens + tok) * a.heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
                }
            }
        }
        sync_all();
        if (tid == 0) s_bad = 0;  // the next segment's first barrier comes before its first use
        base += 2 * (w.tb - w.ta);
        w.advance();
    }
}

// The masses of a 32-bit cache. Four groups of four warps take the tiles in turn; a warp has 16 of the 64 slots and goes
// through the query rows 16 at a time. A lane's four slots are summed over its rows, and over the eight lanes that share
// them at the end. 12 tokens x 32 heads over 65,536 slots take 147 us, one token 59 us, 4.6 TB/s (eight warps with eight
// slots of every tile each took 200 and 110 us where this took 141 and 57). Bound by K from HBM for up to 16 rows, by the products beyond.
template <int D>
struct F32Mass {
    static constexpr int kRows = 128, kGroups = 4, kThreads = 4 * kGroups * 32 + 32;
    static constexpr int kStage = kTile32 * D * 4;
    static constexpr int kStages = D == 64 ? 8 : 5;
    static constexpr int kSmem = kStages * kStage + kRows * D * 4;
};
template <int D>
__global__ void __launch_bounds__(F32Mass<D>::kThreads, 1) k_attn_mass_f32(const AttnArgs a, const __grid_constant__ CUtensorMap mk) {
    using S_ = F32Mass<D>;
    constexpr int NST = S_::kStages, NG = S_::kGroups, ALL = NG * 128;
    constexpr Cut cut{1 << 30, kTile32, 1, 0};
    extern __shared__ __align__(1024) char dyn[];
    char *ring = dyn, *sq = ring + NST * S_::kStage;
    __shared__ uint64_t b_full[NST], b_empty[NST];
    __shared__ int s_gave_up;
    __shared__ Share s_share;
    __shared__ float s_nl[S_::kRows];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const Waits wait{&s_gave_up, a.wait_ns};
    if (warp == 0) {
        after_prior();
        const Share s = find_share(a, cut, lane, blockIdx.x, gridDim.x);
        if (lane == 0) s_share = s;
    } else if (tid == ALL) {
        map_prefetch(&mk);
        for (int i = 0; i < NST; ++i) {
            mbar_init(b_full + i, 1);
            mbar_init(b_empty + i, 4);
        }
        s_gave_up = 0;
        fence_mbar_init();
    }
    after_prior();
    __syncthreads();
    Walk w(a, cut, s_share);
    if (tid >= ALL) {
        uint32_t n = 0;
        bool on = true;
        while (on && w.next()) {
            for (int t = w.ta; t < w.tb; ++t, ++n) {
                const int st = n % NST;
                if (!(on = wait.arrivals(b_empty + st, (n / NST & 1) ^ 1))) break;
                if (lane == 0) {
                    mbar_expect_tx(b_full + st, S_::kStage);
#pragma unroll
                    for (int x = 0; x < D / 32; ++x) tma_load(ring + st * S_::kStage + x * 8192, &mk, 32 * x, t * kTile32, w.u, w.b, b_full + st);
                }
            }
            w.advance();
        }
        for (uint32_t i = n > NST ? n - NST : 0; lane == 0 && i < n; ++i) wait.settle(b_full + i % NST, i / NST & 1);
        return;
    }
    auto sync_all = [&] { asm volatile("bar.sync 1, %0;" ::"n"(ALL) : "memory"); };
    const int group = warp / 4, wq = warp % 4, g = lane / 4, t = lane % 4;
    const float c = a.scale * 1.4426950408889634f;
    uint32_t base = 0;
    while (w.next()) {
        const int rows = w.n * a.gc, h = w.u, padded = (rows + 15) / 16 * 16;
        for (int i = tid; i < padded * (D / 4); i += ALL) {
            const int col4 = i % (D / 4), row = i / (D / 4);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float nl = -INFINITY;
            if (row < rows) {
                const int k = row / a.gc, head = h * a.group + a.g0 + row - k * a.gc;
                const int src = a.rows ? a.rows[(long long)w.b * a.tokens + k] : k;
                if (src < 0 || src >= a.tokens) {
                    if (col4 == 0) atomicOr(&g_cache_error, kErrRange);
                } else {
                    const float lse = a.lse_in[((long long)w.b * a.tokens + src) * a.heads + head];
                    if (lse != -INFINITY) {
                        nl = lse * -1.4426950408889634f;
                        v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + w.b * a.qs[0] + src * a.qs[1] + (long long)head * a.qs[2] + 4 * col4);
                        v = make_float4(staged(v.x, c), staged(v.y, c), staged(v.z, c), staged(v.w, c));
                    }
                }
            }
            *query32<D>(sq, row, col4) = v;
            if (col4 == 0) s_nl[row] = nl;
        }
        sync_all();
        const float *min_ = a.mass + w.b * a.ms[0] + h * a.ms[1];
        float *mout = a.mass_out + w.b * a.mos[0] + h * a.mos[1];
#pragma unroll 1
        for (int tile = w.ta + group; tile < w.tb; tile += NG) {
            const uint32_t n = base + tile - w.ta;
            const char *st = ring + n % NST * S_::kStage;
            const int key0 = tile * kTile32 + 16 * wq, end = w.len + w.n, slot = 16 * wq + (g >> 1) + ((g & 1) << 2);
            float before = 0.f;  // of slot key0 + lane
            if (lane < 16 && key0 + lane < end) before = key0 + lane < w.len ? min_[key0 + lane] : a.more ? mout[key0 + lane] : 0.f;
            wait(b_full + n % NST, n / NST & 1);
            float sum[2][2] = {};
            if (key0 < end) {
                int from[2][2];  // the first row that sees the slot
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int late = key0 + 8 * j + t + 4 * e - w.len;
                        from[j][e] = late <= 0 ? 0 : late < w.n ? late * a.gc : rows;
                    }
#pragma unroll 1
                for (int r0 = 0; r0 < padded; r0 += 16) {
                    float s2[3][2][4] = {};
#pragma unroll 2
                    for (int d = 0; d < D / 16; ++d) {
                        const float4 k[2] = {stage32(st, slot, 4 * d + t), stage32(st, slot + 8, 4 * d + t)};
                        mma_scores(s2, *query32<D>(sq, r0 + g, 4 * d + t), *query32<D>(sq, r0 + g + 8, 4 * d + t), k);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = r0 + g + 8 * (e >> 1);
                        const float nl = s_nl[row];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float p = ex2((s2[0][j][e] + s2[1][j][e]) + (s2[2][j][e] + nl));
                            if (row >= from[j][e & 1] && nl != -INFINITY) sum[j][e & 1] += p;  // (nor of rows behind the last)
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(b_empty + n % NST);
            // lane i < 16 writes slot key0 + i: the sum that lanes t = i % 4 hold as (j, e) = (i / 8, i / 4 % 2)
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) sum[j][e] += __shfl_xor_sync(0xffffffffu, sum[j][e], x);
                    if (lane / 4 == 2 * j + e) mine = sum[j][e];
                }
            if (lane < 16 && key0 + lane < end) mout[key0 + lane] = before + mine;
        }
        sync_all();  // the query rows are done with
        base += w.tb - w.ta;
        w.advance();
    }
}

// ----------------------------------------------------------------------------------------------------------------
// host side
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {  // from the driver, so that the library does not link against it
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}
// 128 bytes of columns x a tile of slots of one head, in the 128-byte swizzle; slots behind the last read as zero
bool cache_map(CUtensorMap *m, const p8_kv *c, const void *base, const int64_t *st) {
    const EncodeTiled f = encode_tiled();
    const cuuint64_t dims[4] = {(cuuint64_t)c->width, (cuuint64_t)c->slots, (cuuint64_t)c->heads, (cuuint64_t)c->batch};
    // the stride of a dimension of one is never used, but has to be a valid one
    const bool wide = c->type == P8_KV_F32;
    const cuuint64_t es = wide ? 4 : 2, row = (cuuint64_t)c->width * es;
    const cuuint64_t strides[3] = {c->slots > 1 ? (cuuint64_t)st[3] * es : row, c->heads > 1 ? (cuuint64_t)st[2] * es : row, c->batch > 1 ? (cuuint64_t)st[1] * es : row};
    const cuuint32_t box[4] = {wide ? 32u : 64u, (cuuint32_t)(wide ? kTile32 : kTile), 1, 1}, one[4] = {1, 1, 1, 1};
    return f(m, wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : c->type == P8_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool TWO>
void allow_attn() {
    cudaFuncSetAttribute(k_tree_attn_tc<T, D, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<D, TWO>::kSmem);
}
template <typename T, int D>
void allow() {
    allow_attn<T, D, false>();
    allow_attn<T, D, true>();
    cudaFuncSetAttribute(k_attn_mass_tc<T, D, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, MassShape<D, 32>::kSmem);
    cudaFuncSetAttribute(k_attn_mass_tc<T, D, 256>, cudaFuncAttributeMaxDynamicSharedMemorySize, MassShape<D, 256>::kSmem);
    cudaFuncSetAttribute(k_attn_mass_tc<T, D, 512>, cudaFuncAttributeMaxDynamicSharedMemorySize, MassShape<D, 512>::kSmem);
}
template <int D>
void allow32() {
    cudaFuncSetAttribute(k_tree_attn_f32<D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, F32Shape<D, 1>::kSmem);
    cudaFuncSetAttribute(k_tree_attn_f32<D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, F32Shape<D, 2>::kSmem);
    cudaFuncSetAttribute(k_tree_attn_f32<D, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, F32Shape<D, 4>::kSmem);
    cudaFuncSetAttribute(k_attn_mass_f32<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, F32Mass<D>::kSmem);
}
// SM count of the current device; the first call on a device raises the kernels' shared-memory limits there
int sm_count() {
    static std::atomic<int> n[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int v = n[dev].load(std::memory_order_acquire);
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
        allow<__half, 64>();
        allow<__half, 128>();
        allow<__nv_bfloat16, 64>();
        allow<__nv_bfloat16, 128>();
        allow32<64>();
        allow32<128>();
        n[dev].store(v, std::memory_order_release);
    }
    return v;
}

// Query rows of a unit. 16-bit: one block for up to 256, so that K and V are read once. 32-bit: up to 64, since the
// products bound more rows anyway; further blocks read K and V from L2 again, at less than half of its rate.
Cut attn_cut(const p8_kv *c, int64_t rows) {
    if (c->type != P8_KV_F32) return rows > 128 ? Cut{256, kTile, TcShape<64, true>::kLeast, start_of(256)} : Cut{128, kTile, TcShape<64, false>::kLeast, start_of(128)};
    return {rows <= 16 ? 16 : rows <= 32 ? 32 : 64, kTile32, 1, 0};
}
int64_t attn_tiles(const p8_kv *c, int64_t rows, Cut cut) {
    return c->batch * c->heads * ((rows + cut.rblock - 1) / cut.rblock) * ((c->slots + cut.tile - 1) / cut.tile + cut.start);
}
// CTAs of a call: no more than there can be tiles
int attn_ctas(const p8_kv *c, int64_t rows, Cut cut) { return (int)std::min<int64_t>(sm_count(), attn_tiles(c, rows, cut)); }

size_t tree_attn_workspace(const p8_kv *c, int64_t tokens, int64_t heads) {  // two parts a CTA, each with the rows' two statistics
    const int64_t rows = tokens * (heads / c->heads);
    const Cut cut = attn_cut(c, rows);
    return (size_t)2 * attn_ctas(c, rows, cut) * cut.rblock * ((size_t)c->width * 4 + 8);
}

// k_attn_join with 16 parts a round has 107 (64 columns: 72) registers a thread, so 2 (3) blocks of eight rows fit an SM; with
// 8 parts, 64 (48). Sixteen are used as long as all blocks run at once, 2,368 (3,552) rows of 148 SMs; beyond, the blocks behind the
// first wave cost more than the loads save. Times of a call, 16 against 8 parts, 16 bit, 128 columns: 256 rows of 65,000 slots
// 55.3 : 57.9 us, 2,304 rows of them 117.4 : 119.6; 2,560 rows of 3,000 slots 32.9 : 29.9, 16,384 rows of 2,000 slots 76.1 :
// 66.3. 64 columns: 2,560 rows of 3,000 slots 24.1 : 25.0, 3,584 rows of 4,000 slots 44.4 : 43.0.
template <int D>
constexpr int kJoinBlocks = D == 128 ? 2 : 3;
template <typename T, int D, typename K>
p8_status run_attn(K kernel, int threads, int smem, float lift, const p8_kv *c, const AttnArgs &a, void *ws, cudaStream_t st) {
    CUtensorMap mk, mv;
    if (!encode_tiled()) return P8_ERR_CUDA;
    if (!cache_map(&mk, c, c->k, c->k_stride) || !cache_map(&mv, c, c->v, c->v_stride)) return P8_ERR_UNSUPPORTED;
    const Cut cut = attn_cut(c, (int64_t)a.tokens * a.group);
    const int ctas = attn_ctas(c, (int64_t)a.tokens * a.group, cut);
    float *po = static_cast<float *>(ws);
    float2 *ml = reinterpret_cast<float2 *>(po + (size_t)2 * ctas * cut.rblock * D);
    if (launch_after(kernel, dim3(ctas), dim3(threads), (size_t)smem, st, a, mk, mv, po, ml) != cudaSuccess) return P8_ERR_CUDA;
    const long long rows = (long long)a.batch * a.tokens * a.heads;
    const dim3 grid((unsigned int)((rows + 7) / 8));
    const auto join = rows <= 8ll * kJoinBlocks<D> * sm_count() ? k_attn_join<T, D, 16> : k_attn_join<T, D, 8>;
    return launch_after(join, grid, dim3(256), 0, st, a, cut, ctas, lift, (const float *)po, (const float2 *)ml) == cudaSuccess ? P8_OK : P8_ERR_CUDA;
}
template <typename T, int D>
p8_status run_tc(const p8_kv *c, const AttnArgs &a, void *ws, cudaStream_t st) {
    constexpr float lift = Half16<T>::kLift;
    if (a.tokens * a.group > 128) return run_attn<T, D>(k_tree_attn_tc<T, D, true>, TcShape<D, true>::kThreads, TcShape<D, true>::kSmem, lift, c, a, ws, st);
    return run_attn<T, D>(k_tree_attn_tc<T, D, false>, TcShape<D, false>::kThreads, TcShape<D, false>::kSmem, lift, c, a, ws, st);
}
template <int D>
p8_status run_f32(const p8_kv *c, const AttnArgs &a, void *ws, cudaStream_t st) {
    switch (attn_cut(c, (int64_t)a.tokens * a.group).rblock) {
        case 16: return run_attn<float, D>(k_tree_attn_f32<D, 1>, F32Shape<D, 1>::kThreads, F32Shape<D, 1>::kSmem, 0.f, c, a, ws, st);
        case 32: return run_attn<float, D>(k_tree_attn_f32<D, 2>, F32Shape<D, 2>::kThreads, F32Shape<D, 2>::kSmem, 0.f, c, a, ws, st);
        default: return run_attn<float, D>(k_tree_attn_f32<D, 4>, F32Shape<D, 4>::kThreads, F32Shape<D, 4>::kSmem, 0.f, c, a, ws, st);
    }
}
// At most `most` rows a launch (what its shared memory holds); the later launches add to the first one's sums.
template <typename F>
p8_status mass_launches(AttnArgs a, int most, F launch) {
    for (a.g0 = 0; a.g0 < a.group; a.g0 += a.gc) {
        a.gc = std::min(most / a.tokens, a.group - a.g0);
        a.more = a.g0 > 0;
        if (a.more) {
            a.mass = a.mass_out;
            for (int i = 0; i < 2; ++i) a.ms[i] = a.mos[i];
        }
        if (launch(a) != cudaSuccess) return P8_ERR_CUDA;
    }
    return P8_OK;
}
template <typename T, int D>
p8_status run_mass_tc(const p8_kv *c, const AttnArgs &a, cudaStream_t st) {
    CUtensorMap mk;
    if (!encode_tiled()) return P8_ERR_CUDA;
    if (!cache_map(&mk, c, c->k, c->k_stride)) return P8_ERR_UNSUPPORTED;
    const int ctas = attn_ctas(c, 1, mass_cut(std::min(512 / a.tokens, a.group) * a.tokens));
    return mass_launches(a, 512, [&](const AttnArgs &x) {
        const int rows = x.tokens * x.gc;
        if (rows <= 32) return launch_after(k_attn_mass_tc<T, D, 32>, dim3(ctas), dim3(576), (size_t)MassShape<D, 32>::kSmem, st, x, mk);
        return launch_after(rows <= 256 ? k_attn_mass_tc<T, D, 256> : k_attn_mass_tc<T, D, 512>, dim3(ctas), dim3(576),
                            (size_t)(rows <= 256 ? MassShape<D, 256>::kSmem : MassShape<D, 512>::kSmem), st, x, mk);
    });
}
template <int D>
p8_status run_mass_f32(const p8_kv *c, const AttnArgs &a, cudaStream_t st) {
    CUtensorMap mk;
    if (!encode_tiled()) return P8_ERR_CUDA;
    if (!cache_map(&mk, c, c->k, c->k_stride)) return P8_ERR_UNSUPPORTED;
    const int ctas = attn_ctas(c, 1, Cut{1, kTile32, 1, 0});
    return mass_launches(a, F32Mass<D>::kRows, [&](const AttnArgs &x) { return launch_after(k_attn_mass_f32<D>, dim3(ctas), dim3(F32Mass<D>::kThreads), (size_t)F32Mass<D>::kSmem, st, x, mk); });
}
template <int D>
p8_status run_width(const p8_kv *c, const AttnArgs &a, bool mass, void *ws, cudaStream_t st) {
    if (c->type == P8_KV_F32) return mass ? run_mass_f32<D>(c, a, st) : run_f32<D>(c, a, ws, st);
    if (c->type == P8_KV_F16) return mass ? run_mass_tc<__half, D>(c, a, st) : run_tc<__half, D>(c, a, ws, st);
    return mass ? run_mass_tc<__nv_bfloat16, D>(c, a, st) : run_tc<__nv_bfloat16, D>(c, a, ws, st);
}

std::atomic<unsigned int> g_wait_ns{kWaitNs};
void base_args(AttnArgs &x, const p8_kv *c, const void *q, const int64_t *qs, int64_t tokens, int64_t heads) {
    memset(&x, 0, sizeof(x));
    x.q = q; x.k = c->k; x.v = c->v;
    for (int i = 0; i < 3; ++i) { x.qs[i] = qs[i]; x.ks[i] = c->k_stride[1 + i]; x.vs[i] = c->v_stride[1 + i]; }
    x.slots = c->slots; x.batch = (int)c->batch; x.tokens = (int)tokens; x.heads = (int)heads; x.kvh = (int)c->heads;
    x.group = (int)(heads / c->heads);
    x.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
}

p8_status launch_attn(const p8_kv *c, const AttnArgs &x, bool mass, void *ws, cudaStream_t st) {
    const int64_t rows = mass ? 1 : (int64_t)x.tokens * x.group;
    if (attn_tiles(c, rows, mass && c->type != P8_KV_F32 ? mass_cut(512) : attn_cut(c, rows)) > INT32_MAX / 2 || c->batch * x.tokens * x.heads > INT32_MAX) return P8_ERR_UNSUPPORTED;
    return c->width == 128 ? run_width<128>(c, x, mass, ws, st) : run_width<64>(c, x, mass, ws, st);
}

p8_status launch_tree_attn(const p8_kv *c, const p8_tree_attn_args *a, void *ws, cudaStream_t st) {
    AttnArgs x;
    base_args(x, c, a->q, a->q_stride, a->tokens, a->heads);
    x.lens = a->lens; x.counts = a->counts; x.mask = (const unsigned long long *)a->mask; x.mask_stride = a->mask_stride;
    x.scale = (float)a->scale; x.out = a->out; x.lse = a->lse;
    for (int i = 0; i < 3; ++i) x.os[i] = a->out_stride[i];
    return launch_attn(c, x, false, ws, st);
}

p8_status launch_attn_mass(const p8_kv *c, const p8_attn_mass_args *a, cudaStream_t st) {
    AttnArgs x;
    base_args(x, c, a->q, a->q_stride, a->tokens, a->heads);
    x.lens = a->lens; x.counts = a->counts; x.rows = a->rows; x.lse_in = a->lse; x.scale = (float)a->scale;
    x.mass = a->mass; x.mass_out = a->out;
    for (int i = 0; i < 2; ++i) { x.ms[i] = a->mass_stride[i]; x.mos[i] = a->out_stride[i]; }
    return launch_attn(c, x, true, nullptr, st);
}
