// What a row of logits says about given tokens: the log probability and rank of one token, the entropy of the distribution and
// its best alternatives, in one pass over the logits. The reference answers with the argmax alone (k_argmax,
// engine/faie2fn.cu:1910-1935).
//
//   m = max x, Z = sum e^(x - m), logprob = x_t - m - ln Z, entropy = ln Z - sum e^(x - m) (x - m) / Z,
//   rank = the entries before t by (value, lower index), alternatives = the first k of that order
//
// Every thread keeps the running maximum, sum and weighted sum of its own 16-byte words of the row (rescaled when its maximum
// moves); a CTA, or a cluster of CTAs where the rows are few, joins them through (distributed) shared memory. No workspace, no
// atomics on memory: the same bits every time.
//
// The alternatives cost no second pass: the threads' maxima are there already, and their k-th largest is a bound that no
// alternative of the CTA's part falls below, so only what can reach it is read again: the segments (of a thread's words) whose own
// maximum does, about k of 4096, spread over all threads, which list what reaches it. (If equal entries are too many to be listed, every
// warp keeps its best 32 sorted over its lanes.)
//
// What bounds it: with many rows in bf16 instruction issue (11.5 an entry in all; 2048 x 151936: 135 us with 20 alternatives and tokens, 109 with
// neither, where the bytes take 95 at the copy rate), in fp32 the loads (1024 rows: 117, the bytes 95); with few rows the chain of steps behind the
// pass (32 rows of fp32: 11.5 us, without alternatives 8.0, where the bytes take 3).
#include <cuda_bf16.h>

#include <utility>

#include "fn_argmax.cuh"
#include "fn_engine.h"
#include "fn_kv4.h"

namespace fn {

constexpr int LP_MAX_TOP = 32, LP_MAX_CLUSTER = 8;
constexpr float LP_LOWEST = -3.402823466e38f, LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;
constexpr float LP_FAR = -1000.0f;  // exponents below it stand for nothing: 2^-1000 is 0, and 0 * -1000 too (0 * -inf is not)

struct LpArgs {
    const void *logits;
    int64_t stride;  // elements from row to row
    int rows, vocab, top;
    const int *tokens;
    float *logprob;
    int *rank;
    float *entropy;
    int *top_ids;
    float *top_logprobs;
    uint32_t *err;
};

// m: the largest entry (-inf: none above it); b = max(m, lowest) is what exponents count from; s = sum 2^y, t = sum 2^y y with
// y = (x - b) log2 e
struct LpSum {
    float m, b, s, t;
};

__device__ __forceinline__ float lp_ex2(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {
    float e;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(a), "f"(b));
    return e;
}
__device__ __forceinline__ void lp_raise(LpSum &a, float m) {
    const float b = fmaxf(m, LP_LOWEST), y = fmaxf((a.b - b) * LP_LOG2E, LP_FAR), f = lp_ex2(y);
    a.t = f * (a.t + y * a.s);
    a.s *= f;
    a.m = m;
    a.b = b;
}
__device__ __forceinline__ void lp_join(LpSum &a, LpSum c) {
    const float m = fmaxf(a.m, c.m);
    lp_raise(a, m);
    lp_raise(c, m);
    a.s += c.s;
    a.t += c.t;
}

// two fp32 values in one register pair: half the instructions of the sums
__device__ __forceinline__ uint64_t lp_two(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void lp_untwo(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t lp_mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

__device__ __forceinline__ uint32_t lp_max2(uint32_t a, uint32_t b) {
    uint32_t v;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
    return v;
}
__device__ __forceinline__ uint32_t lp_max2_nan(uint32_t a, uint32_t b) {
    uint32_t v;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
    return v;
}
__device__ __forceinline__ float lp_low(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float lp_high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// the smallest number above v (of +0 as of -0: the smallest positive); NaN above +inf
__device__ __forceinline__ float lp_above(float v) {
    if (v == 0.0f) return __uint_as_float(1u);
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float(v > 0.0f ? u + 1 : u - 1);
}

// A thread's sums on their way, s and t in two halves each, and what depends on the type: words of 16 bytes, and how their entries are
// added and counted.
template <typename T> struct LpAcc;
template <> struct LpAcc<float> {
    static constexpr int N = 4;  // entries of a word
    static constexpr uint32_t NOTHING = 0xff800000u;  // what an empty word is made of: -inf
    float m = -INFINITY, b = LP_LOWEST;
    uint64_t minus_b = lp_two(-LP_LOWEST, -LP_LOWEST), s = 0, t = 0;
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    __device__ __forceinline__ void raise(float to) {
        const float c = fmaxf(to, LP_LOWEST), y = fmaxf((b - c) * LP_LOG2E, LP_FAR), f = lp_ex2(y);
        t = lp_mul2(lp_two(f, f), lp_fma2(lp_two(y, y), s, t));
        s = lp_mul2(lp_two(f, f), s);
        m = to;
        b = c;
        minus_b = lp_two(-c, -c);
    }
    __device__ __forceinline__ void pair(float x0, float x1) {
        float y0, y1;
        lp_untwo(lp_mul2(lp_add2(lp_two(x0, x1), minus_b), lp_two(LP_LOG2E, LP_LOG2E)), y0, y1);
        y0 = lp_max_nan(y0, LP_FAR), y1 = lp_max_nan(y1, LP_FAR);
        const uint64_t e = lp_two(lp_ex2(y0), lp_ex2(y1));
        s = lp_add2(s, e);
        t = lp_fma2(e, lp_two(y0, y1), t);
    }
    typedef float Most;  // the largest entry of some
    static __device__ __forceinline__ float none() { return -INFINITY; }
    static __device__ __forceinline__ float larger(float a, float c) { return fmaxf(a, c); }
    static __device__ __forceinline__ float value(float a) { return a; }
    template <int U> __device__ __forceinline__ float words(const uint4 (&w)[U]) {  // adds them and returns their largest entry
        float x[U][4], most = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unpack(w[u], x[u]);
            most = fmaxf(most, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
        }
        if (most > m) raise(most);
#pragma unroll
        for (int u = 0; u < U; ++u) pair(x[u][0], x[u][1]), pair(x[u][2], x[u][3]);
        return most;
    }
    __device__ __forceinline__ void one(float x) {
        if (x > m) raise(x);
        pair(x, -INFINITY);
    }
    __device__ __forceinline__ void clear() { s = t = 0; }
    __device__ __forceinline__ LpSum sum() const {
        float s0, s1, t0, t1;
        lp_untwo(s, s0, s1);
        lp_untwo(t, t0, t1);
        return LpSum{m, b, s0 + s1, t0 + t1};
    }
    // how many entries are at least `bar`: whole numbers in fp32, two at a time
    struct Counter {
        uint64_t n = 0;
        __device__ __forceinline__ void add(uint4 w, float bar) {
            const float b[4] = {at_least(w.x, bar), at_least(w.y, bar), at_least(w.z, bar), at_least(w.w, bar)};
            n = lp_add2(n, lp_add2(lp_two(b[0], b[1]), lp_two(b[2], b[3])));
        }
        __device__ __forceinline__ void flush(int &) {}  // (2^24 of a thread's would be too many)
        __device__ __forceinline__ void end(int &before) {
            float x, y;
            lp_untwo(n, x, y);
            before += (int)x + (int)y;
        }
        static __device__ __forceinline__ float at_least(uint32_t x, float bar) {
            float v;
            asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(v) : "f"(__uint_as_float(x)), "f"(bar));
            return v;
        }
    };
    static __device__ __forceinline__ float above(float v) { return lp_above(v); }
};
// bf16 has half the bytes an entry, so it is instructions that bound it. Exponents count from a whole number c near b log2 e, so that
// one fused multiply-add makes them (rounded once; and c's steps are exact powers of two); that log2 e itself is rounded makes every
// difference of two entries 1.3e-8 of itself larger. Entries far below b, -inf among them, are raised to a number that still stands for
// nothing, two at a time. From |b| = 2^17 on the next bf16 number below b is 512 away and more: there only entries equal to b count.
template <> struct LpAcc<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t NOTHING = 0xff80ff80u;
    float m = -INFINITY, b = LP_LOWEST, c = 0.0f;
    uint32_t m2 = 0xff80ff80u, floor = 0;  // m twice; what entries are raised to, twice
    bool far = true;
    float s0 = 0.0f, s1 = 0.0f, t0 = 0.0f, t1 = 0.0f;
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = lp_low(v[i]), x[2 * i + 1] = lp_high(v[i]);
    }
    __device__ __forceinline__ void raise(float to) {
        const bool was_far = far;
        const float was = c;
        m = to;
        b = fmaxf(to, LP_LOWEST);
        const uint32_t h = __float_as_uint(to) >> 16;
        m2 = h << 16 | h;
        far = fabsf(b) >= 131072.0f;
        c = far ? 0.0f : rintf(b * LP_LOG2E);
        const float y = was_far || far ? LP_FAR : fmaxf(was - c, LP_FAR), f = lp_ex2(y);
        t0 = f * fmaf(y, s0, t0), t1 = f * fmaf(y, s1, t1);
        s0 *= f, s1 *= f;
        const float low = b - fmaxf(700.0f, fabsf(b) * 0.015625f);
        const __nv_bfloat162 p = __floats2bfloat162_rn(low, low);
        memcpy(&floor, &p, 4);
    }
    __device__ __forceinline__ void equal(float x) {  // far: entries equal to b, and NaN
        s0 += x == b ? (b == INFINITY ? NAN : 1.0f) : x == x ? 0.0f : x;
    }
    __device__ __forceinline__ void pair(uint32_t v) {
        const uint32_t q = lp_max2_nan(v, floor);
        const float y0 = fmaf(lp_low(q), LP_LOG2E, -c), y1 = fmaf(lp_high(q), LP_LOG2E, -c), e0 = lp_ex2(y0), e1 = lp_ex2(y1);
        s0 += e0, s1 += e1;
        t0 = fmaf(e0, y0, t0), t1 = fmaf(e1, y1, t1);
    }
    typedef uint32_t Most;  // the largest entry of some: the larger of two
    static __device__ __forceinline__ uint32_t none() { return 0xff80ff80u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t c) { return lp_max2(a, c); }
    static __device__ __forceinline__ float value(uint32_t a) { return fmaxf(lp_low(a), lp_high(a)); }
    template <int U> __device__ __forceinline__ uint32_t words(const uint4 (&w)[U]) {  // adds them and returns their largest entry
        uint32_t p = none();
#pragma unroll
        for (int u = 0; u < U; ++u) p = lp_max2(p, lp_max2(lp_max2(w[u].x, w[u].y), lp_max2(w[u].z, w[u].w)));
        if (lp_max2(p, m2) != m2) {
            const float most = value(p);
            if (most > m) raise(most);
        }
        if (far) {
#pragma unroll 1
            for (int u = 0; u < U; ++u) {
                uint4 now = w[0];
#pragma unroll
                for (int i = 1; i < U; ++i)
                    if (u == i) now = w[i];
                const uint32_t v[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) equal(lp_low(v[i])), equal(lp_high(v[i]));
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) pair(w[u].x), pair(w[u].y), pair(w[u].z), pair(w[u].w);
        }
        return p;
    }
    __device__ __forceinline__ void one(float x) {
        if (x > m) raise(x);
        if (far) equal(x);
        else pair(__float_as_uint(x) >> 16 | 0xff800000u);  // (beside -inf)
    }
    __device__ __forceinline__ void clear() { s0 = s1 = t0 = t1 = 0.0f; }
    __device__ __forceinline__ LpSum sum() const {  // counted from b
        const float y = far ? 0.0f : fmaf(b, LP_LOG2E, -c), f = lp_ex2(-y), z = s0 + s1;
        return LpSum{m, b, f * z, f * (t0 + t1 - y * z)};
    }
    // How many entries are at least `bar`, two at a time: a mask of ones for each that is, added up as 32-bit numbers. `low` masks in the
    // low halves and `high` ones make 0xffff (low + 65536 high) = 65536 (low - high) - low, from which both are read back.
    struct Counter {
        uint32_t n = 0;
        __device__ __forceinline__ void add(uint4 w, float bar) {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
            const __nv_bfloat162 b = __floats2bfloat162_rn(bar, bar);  // (exact)
            uint32_t k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __nv_bfloat162 x;
                memcpy(&x, &v[i], 4);
                k[i] = __hge2_mask(x, b);
            }
            n += k[0] + k[1];
            n += k[2] + k[3];
        }
        __device__ __forceinline__ void flush(int &before) {  // before 65536 of a half
            const uint32_t low = (0u - n) & 0xffff, high = (low - ((n + low) >> 16)) & 0xffff;
            before += low + high;
            n = 0;
        }
        __device__ __forceinline__ void end(int &before) { flush(before); }
    };
    static __device__ __forceinline__ float above(float v) {  // the next bf16 number up
        if (v == 0.0f) return __uint_as_float(0x10000u);
        const uint32_t u = __float_as_uint(v);
        return __uint_as_float(v > 0.0f ? u + 0x10000u : u - 0x10000u);
    }
};

__device__ __forceinline__ bool lp_stands_before(float x, int i, int token, float given, float above) { return x >= (i < token ? given : above); }

__device__ __forceinline__ uint32_t lp_order(float v) { return (uint32_t)(amax_key(v, 0) >> 32); }  // 0: no candidate

// `list`: a warp's best entries, descending over the lanes (0: none); takes every lane's key and returns the new list
__device__ __noinline__ unsigned long long lp_insert(unsigned long long list, unsigned long long key, int lane, int top) {
    for (;;) {
        const unsigned long long last = __shfl_sync(0xffffffffu, list, top - 1);
        const uint32_t want = __ballot_sync(0xffffffffu, key > last);
        if (!want) return list;
        const int from = __ffs(want) - 1;
        const unsigned long long k = __shfl_sync(0xffffffffu, key, from), up = __shfl_up_sync(0xffffffffu, list, 1);
        const int at = __popc(__ballot_sync(0xffffffffu, list > k));
        list = lane < at ? list : lane == at ? k : up;
        if (lane == from) key = 0;
    }
}

__device__ __forceinline__ uint32_t lp_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// p of CTA `rank` of the cluster = v
template <typename P> __device__ __forceinline__ void lp_store(P *p, uint32_t rank, P v) {
    static_assert(sizeof(P) == 4 || sizeof(P) == 8, "");
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    if constexpr (sizeof(P) == 4) {
        uint32_t u;
        memcpy(&u, &v, 4);
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(u) : "memory");
    } else {
        unsigned long long u;
        memcpy(&u, &v, 8);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(u) : "memory");
    }
}

// Rounds of words that a thread's sums take in fp32 (up to 512 terms each, whose additions are off by 2^-15 of it at the very worst) before
// they join sums in 64 bits: in fp32 alone rows of 2^26 entries lost up to 5e-4.
constexpr int LP_FOLD = 32;
template <int THREADS> struct LpFold {  // every thread's own: sums counted from b
    double s[THREADS], t[THREADS];
    float b[THREADS];
    __device__ __forceinline__ void add(const LpSum &c, bool first) {
        double s0 = 0.0, t0 = 0.0;
        if (!first) {
            const float y = fmaxf((b[threadIdx.x] - c.b) * LP_LOG2E, LP_FAR), f = lp_ex2(y);
            s0 = f * s[threadIdx.x], t0 = f * (t[threadIdx.x] + y * s[threadIdx.x]);
        }
        s[threadIdx.x] = s0 + c.s, t[threadIdx.x] = t0 + c.t;
        b[threadIdx.x] = c.b;
    }
};

template <int THREADS> struct LpShared {
    static constexpr int W = THREADS / 32, SEGMENTS = 4096 / THREADS;
    LpSum sums[W];
    int before[W];
    uint32_t ends[2][W];
    union {
        LpFold<THREADS> fold;  // while the words are read; then
        struct {
            unsigned long long keys[W * LP_MAX_TOP];  // (as many as a cluster's at least)
            int columns[THREADS];                     // segments that are read again
        };
    };
    unsigned long long best[LP_MAX_TOP];  // this CTA's alternatives, in order
    LpSum sum;                            // the row's
    LpSum part[LP_MAX_CLUSTER];           // what the cluster's CTAs found
    int before_of[LP_MAX_CLUSTER];
    unsigned long long keys_of[LP_MAX_CLUSTER][LP_MAX_TOP];
    int count, n_keys, n_columns;
    uint32_t most[SEGMENTS][THREADS];  // the largest entry (in order) of every segment
};

// What a CTA does once a row is out of line and rolled where it is called more than once: of a short call's time a good part is fetching
// code that has not run yet.
//
// n keys (distinct, or 0) put in order: the first `top` into best, which holds zeros. THREADS / 256 neighbours count a key against the others.
template <int THREADS> __device__ __noinline__ void lp_rank_keys(const unsigned long long *keys, int n, int top, unsigned long long *best) {
    constexpr int Q = THREADS / 256;
    for (int i0 = (threadIdx.x & ~31) / Q; i0 < n; i0 += 256) {  // (a warp without a key is done)
        const int i = i0 + (threadIdx.x & 31) / Q;
        const unsigned long long k = i < n ? keys[i] : 0;
        int at = 0;
#pragma unroll 4
        for (int j = threadIdx.x % Q; j < n; j += Q) at += keys[j] > k;
#pragma unroll
        for (int o = 1; o < Q; o <<= 1) at += __shfl_xor_sync(0xffffffffu, at, o);
        if (threadIdx.x % Q == 0 && k && at < top) best[at] = k;
    }
}
// the lanes' sums joined, in every lane
__device__ __forceinline__ LpSum lp_warp_join(LpSum a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpSum c;
        c.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        c.b = __shfl_xor_sync(0xffffffffu, a.b, o);
        c.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        c.t = __shfl_xor_sync(0xffffffffu, a.t, o);
        lp_join(a, c);
    }
    return a;
}

constexpr int LP_MAX_VOCAB = 1 << 28;  // so a segment has up to 2048 rounds, each with up to 16 entries of a half of the counter
// CTAs of 256 threads on an SM: five where instructions bound it (bf16, 2048 rows of 151936: 135 us, by four 145; 200 rows, where
// latency counts, 27.2 and 26.9), four where loads do (fp32, 1024 rows: 117 us, by five 126)
constexpr int lp_ctas(int size) { return size == 2 ? 5 : 4; }

// grid: rows x C CTAs in clusters of C (a power of two up to 8) for a row
template <typename T, int LP_T> __global__ void __launch_bounds__(LP_T, LP_T == 1024 ? 1 : lp_ctas(sizeof(T))) k_logprobs(const LpArgs a, int C) {
    constexpr int N = LpAcc<T>::N, U = 4, LP_W = LP_T / 32, SEGMENTS = LpShared<LP_T>::SEGMENTS;  // entries of a word; words in flight per thread
    static_assert(LP_W >= LP_MAX_CLUSTER, "");
    __shared__ LpShared<LP_T> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / C;
    const uint32_t part = C > 1 ? lp_cluster_rank() : 0;
    if (C > 1) lp_cluster_arrive();  // that this CTA's shared memory is there
    if (tid == 0) sh.n_keys = sh.n_columns = 0;
    if (tid < LP_MAX_TOP) sh.best[tid] = 0;
    pdl_wait();
    pdl_trigger();
    const T *x = (const T *)after_wait(a.logits) + row * a.stride;
    const int token = a.tokens ? after_wait(a.tokens)[row] : -1;
    const bool known = token >= 0 && token < a.vocab;
    // whole 16-byte words, and the entries before and behind them
    const int head = min(a.vocab, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T))), words = (a.vocab - head) / N;
    const int tail0 = head + words * N, tail = a.vocab - tail0;
    const int w0 = (int)((int64_t)words * part / C), w1 = (int)((int64_t)words * (part + 1) / C);
    const uint4 *v = (const uint4 *)(x + head);
    const float given = known ? (float)x[token] + 0.0f : NAN, above = LpAcc<T>::above(given);
    const int own_word = token >= head ? (token - head) / N : -1;  // the word that holds the token: counted as those behind it, then put right
    LpAcc<T> acc;
    int before = 0;
    typename LpAcc<T>::Counter counter;
    // what a thread meets in a segment of the row: its largest entry
    const int rounds = (w1 - w0 + U * LP_T - 1) / (U * LP_T), per = max(1, (rounds + SEGMENTS - 1) / SEGMENTS);
    for (int i = 0, seg = 0; i < rounds; ++seg) {
        typename LpAcc<T>::Most most = LpAcc<T>::none();
#pragma unroll 1
        for (const int end = min(rounds, i + per); i < end; ++i) {
            if (i && i % LP_FOLD == 0) sh.fold.add(acc.sum(), i == LP_FOLD), acc.clear();
            const int w = w0 + i * U * LP_T + tid;
            const uint4 *p = v + w;
            uint4 r[U];
            if (LP_T < 1024 && w0 + (i + 1) * U * LP_T <= w1) {  // all words of all threads (of long loops; else it is more code to fetch)
#pragma unroll
                for (int u = 0; u < U; ++u) r[u] = p[u * LP_T];
                most = LpAcc<T>::larger(most, acc.words(r));
                if (known) {
                    const int ahead = own_word - (w0 + i * U * LP_T);  // words of this round before the token's
                    if (ahead <= 0 || ahead >= U * LP_T) {
                        const float bar = ahead <= 0 ? above : given;
#pragma unroll
                        for (int u = 0; u < U; ++u) counter.add(r[u], bar);
                    } else {
#pragma unroll
                        for (int u = 0; u < U; ++u) counter.add(r[u], w + u * LP_T < own_word ? given : above);
                    }
                }
            } else {
                constexpr uint32_t x = LpAcc<T>::NOTHING;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    r[u] = make_uint4(x, x, x, x);
                    if (w + u * LP_T < w1) r[u] = p[u * LP_T];
                }
                most = LpAcc<T>::larger(most, acc.words(r));
                if (known) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (w + u * LP_T < w1) counter.add(r[u], w + u * LP_T < own_word ? given : above);
                }
            }
        }
        if (known) counter.flush(before);
        if (a.top) sh.most[seg][tid] = lp_order(LpAcc<T>::value(most));
    }
    if (known) counter.end(before);
    if (known && own_word >= w0 && own_word < w1 && (own_word - w0) % LP_T == tid) {
        const int i0 = head + own_word * N;
        for (int i = i0; i < token; ++i) before += (float)x[i] == given;
    }
    // the entries outside whole words: one a thread, of the first CTA
    const int odd = part == 0 && tid < head + tail ? (tid < head ? tid : tail0 + tid - head) : -1;
    if (odd >= 0) {
        const float e = (float)x[odd];
        acc.one(e);
        if (known) before += lp_stands_before(e, odd, token, given, above);
    }
    LpSum sum = acc.sum();
    if (rounds > LP_FOLD) {
        sh.fold.add(sum, false);
        sum.s = (float)sh.fold.s[tid], sum.t = (float)sh.fold.t[tid];
    }
    const uint32_t mine = lp_order(sum.m);
    const LpSum all = lp_warp_join(sum);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) sh.sums[warp] = all, sh.before[warp] = before;
    if (a.top) {
        // a bound that at least `top` threads' maxima reach (0: all), by halving the interval between the bound that all reach
        // and the one that none does, until at most half as many again do
        uint32_t lo = 0, hi = 0xffffffffu;
        {
            const uint32_t wmin = __reduce_min_sync(0xffffffffu, mine), wmax = __reduce_max_sync(0xffffffffu, mine);
            if (lane == 0) sh.ends[0][warp] = wmin, sh.ends[1][warp] = wmax;
            __syncthreads();
            lo = __reduce_min_sync(0xffffffffu, sh.ends[0][lane % LP_W]);
            hi = __reduce_max_sync(0xffffffffu, sh.ends[1][lane % LP_W]);
        }
        if (a.top == 1) lo = hi;  // (the largest itself)
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = __syncthreads_count(mine >= mid);
            if (n >= a.top) {
                lo = mid;
                if (n <= a.top + a.top / 2) break;
            } else hi = mid;
        }
        const uint32_t bound = lo;
        if (mine && mine >= bound)
            for (int i = 0; i * per < rounds; ++i)
                if (const uint32_t o = sh.most[i][tid]; o && o >= bound) {
                    const int at = atomicAdd(&sh.n_columns, 1);
                    if (at < LP_T) sh.columns[at] = i * LP_T + tid;
                }
        __syncthreads();
        const int n = sh.n_columns;
        // segments that reach the bound, or all of them if they are too many to be listed
        const bool listed = n <= LP_T;
        const int each = per * U, count = (listed ? n : LP_T * ((rounds + per - 1) / per)) * each;  // words of a segment; words to read
        auto word = [&](int i) {  // word i of those to read, w1 if there is none
            const int c = i / each, column = listed ? sh.columns[min(c, LP_T - 1)] : c;
            return i < count ? w0 + (column / LP_T * each + i - c * each) * LP_T + column % LP_T : w1;
        };
        constexpr int KEYS = LP_W * LP_MAX_TOP;  // that sh.keys holds
#pragma unroll 1
        for (int i = tid; i < count; i += LP_T) {
            const int w = word(i);
            if (w >= w1) continue;
            float e[N];
            LpAcc<T>::unpack(v[w], e);
            float m = e[0];
#pragma unroll
            for (int j = 1; j < N; ++j) m = fmaxf(m, e[j]);
            if (lp_order(m) < bound || !(m > -INFINITY)) continue;
            uint32_t reach = 0;  // the entries that reach the bound
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (const uint32_t o = lp_order(e[j]); o && o >= bound) reach |= 1u << j;
#pragma unroll 1
            for (; reach; reach &= reach - 1) {
                const int j = __ffs(reach) - 1, at = atomicAdd(&sh.n_keys, 1);
                if (at < KEYS) sh.keys[at] = amax_key((float)x[head + w * N + j], head + w * N + j);
            }
        }
        if (odd >= 0) {
            const unsigned long long key = amax_key((float)x[odd], odd);
            if (key && (uint32_t)(key >> 32) >= bound) {
                const int at = atomicAdd(&sh.n_keys, 1);
                if (at < KEYS) sh.keys[at] = key;
            }
        }
        __syncthreads();
        if (sh.n_keys > KEYS) {  // many equal entries: every warp keeps its best
            __syncthreads();
            if (tid == 0) sh.n_keys = 0;
            unsigned long long list = 0;
#pragma unroll 1
            for (int i = tid; i - lane < count; i += LP_T) {
                const int w = word(i);
#pragma unroll 1
                for (int j = 0; j < N; ++j) list = lp_insert(list, w < w1 ? amax_key((float)x[head + w * N + j], head + w * N + j) : 0ull, lane, a.top);
            }
            if (part == 0 && warp == 0) list = lp_insert(list, odd >= 0 ? amax_key((float)x[odd], odd) : 0ull, lane, a.top);
            __syncthreads();
            if (list && lane < a.top) sh.keys[atomicAdd(&sh.n_keys, 1)] = list;
            __syncthreads();
        }
        lp_rank_keys<LP_T>(sh.keys, sh.n_keys, a.top, sh.best);
    }
    __syncthreads();
    const LpSum nothing{-INFINITY, LP_LOWEST, 0.0f, 0.0f};
    if (warp == 0) {
        const LpSum z = lp_warp_join(lane < LP_W ? sh.sums[lane] : nothing);
        const int n = __reduce_add_sync(0xffffffffu, lane < LP_W ? sh.before[lane] : 0);
        if (C == 1) {
            if (lane == 0) sh.sum = z, sh.count = n;
        } else {  // to the first CTA
            lp_cluster_wait();
            if (lane < a.top) lp_store(&sh.keys_of[part][lane], 0, sh.best[lane]);
            if (lane == 0) {
                lp_store(&sh.part[part].m, 0, z.m);
                lp_store(&sh.part[part].b, 0, z.b);
                lp_store(&sh.part[part].s, 0, z.s);
                lp_store(&sh.part[part].t, 0, z.t);
                lp_store(&sh.before_of[part], 0, n);
            }
        }
    } else if (C > 1) lp_cluster_wait();
    if (C > 1) {
        __syncthreads();
        lp_cluster_arrive();
        lp_cluster_wait();
        if (part) return;
        if (warp == 0) {
            const LpSum z = lp_warp_join(lane < C ? sh.part[lane] : nothing);
            const int n = __reduce_add_sync(0xffffffffu, lane < C ? sh.before_of[lane] : 0);
            if (lane == 0) sh.sum = z, sh.count = n;
        }
        if (a.top) {
            if (tid < LP_MAX_TOP) sh.best[tid] = 0;
            if (tid < C * a.top) sh.keys[tid] = sh.keys_of[tid / a.top][tid % a.top];
            __syncthreads();
            lp_rank_keys<LP_T>(sh.keys, C * a.top, a.top, sh.best);
        }
    }
    __syncthreads();
    const LpSum z = sh.sum;
    const bool none = z.s == 0.0f;  // nothing above -inf
    const float ln = logf(z.s);
    if (tid < a.top) {
        const unsigned long long k = sh.best[tid];
        const uint32_t o = (uint32_t)(k >> 32);
        const float value = __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
        a.top_ids[row * a.top + tid] = k ? amax_index(k) : -1;
        a.top_logprobs[row * a.top + tid] = k ? value - z.b - ln : -INFINITY;
    }
    if (tid == 0) {
        if (token >= a.vocab) dev_fail(a.err, DEV_BAD_ARG);
        if (a.logprob) a.logprob[row] = token < 0 ? 0.0f : !known ? NAN : none ? -INFINITY : given - z.b - ln;
        if (a.rank) a.rank[row] = known && given == given ? sh.count : -1;
        if (a.entropy) a.entropy[row] = none ? 0.0f : ln - LP_LN2 * z.t / z.s;
    }
}

}  // namespace fn

using namespace fn;

FN_API int fn_logprobs(uint32_t type, const void *logits, int64_t stride, int rows, int vocab, const int *tokens, float *logprob,
                       int *rank, float *entropy, int top, int *top_ids, float *top_logprobs, void *stream) {
    return kv4_entry("logprobs", [&]() -> int {
        if (type != T_F32 && type != T_BF16) return fail("logprobs: logits must be F32 or BF16");
        if (rows < 0 || vocab < 1 || vocab > LP_MAX_VOCAB) return fail("logprobs: bad row / vocabulary counts");
        if (top < 0 || top > LP_MAX_TOP) return fail("logprobs: top out of range (0..32)");
        if (rows == 0) return 0;
        if (!logits || (top && (!top_ids || !top_logprobs))) return fail("logprobs: null pointer");
        if (!tokens && (logprob || rank)) return fail("logprobs: log probabilities and ranks want tokens");
        const int64_t size = type == T_F32 ? 4 : 2, one = (int64_t)rows * 4;
        if ((uintptr_t)logits % size) return fail("logprobs: logits must be aligned to their type");
        for (const auto &[out, n] : {std::pair<const void *, int64_t>(logprob, one), {rank, one}, {entropy, one}, {top_ids, one * top}, {top_logprobs, one * top}})
            if (rows_meet_bytes(logits, stride * size, rows, vocab * size, out, n) || ((out != tokens || n != one) && rows_meet_bytes(tokens, 0, 1, one, out, n)))
                return fail("logprobs: results lie over logits or tokens");
        // rows that the SMs can take at once get CTAs of 1024 threads, and up to 8 of them (of 4096 entries and more) where they are fewer;
        // else CTAs of 256 share an SM
        const bool large = rows <= num_sms();
        int C = 1;
        while (large && C < LP_MAX_CLUSTER && (int64_t)rows * C * 2 <= num_sms() && vocab / (2 * C) >= 4096) C *= 2;
        const LpArgs a{logits, stride, rows, vocab, top, tokens, logprob, rank, entropy, top_ids, top_logprobs, dev_error_ptr()};
        const dim3 grid((unsigned)(rows * C)), block(large ? 1024 : 256);
        auto *k = type == T_F32 ? (large ? k_logprobs<float, 1024> : k_logprobs<float, 256>)
                                : (large ? k_logprobs<__nv_bfloat16, 1024> : k_logprobs<__nv_bfloat16, 256>);
        const cudaError_t e = C > 1 ? launch_kc(k, grid, block, (unsigned)C, 0, (cudaStream_t)stream, a, C)
                                    : launch_k(k, grid, block, 0, (cudaStream_t)stream, a, C);
        if (e != cudaSuccess) return fail(std::string("logprobs launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
