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
// alternative of the CTA's part falls below, so only the words of threads whose maximum reaches it are read again (about k
// threads of the CTA, from L2), each by a warp that keeps its best 32 entries sorted over its lanes.
#include <cuda_bf16.h>

#include "fn_argmax.cuh"
#include "fn_engine.h"
#include "fn_kv4.h"

namespace fn {

constexpr int LP_T = 256, LP_W = LP_T / 32, LP_MAX_TOP = 32, LP_MAX_CLUSTER = 8;
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

template <typename T> struct LpWord;  // 16 bytes of logits
template <> struct LpWord<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
};
template <> struct LpWord<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
};

// the smallest number above v (of +0 as of -0: the smallest positive); NaN above +inf
__device__ __forceinline__ float lp_above(float v) {
    if (v == 0.0f) return __uint_as_float(1u);
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float(v > 0.0f ? u + 1 : u - 1);
}

// entries x[0..N) from index i0: an entry stands before the token if it is at least `given` (lower index) or above it
template <int N> __device__ __forceinline__ void lp_add(const float (&x)[N], LpSum &a) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > a.m) lp_raise(a, m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = lp_max_nan((x[i] - a.b) * LP_LOG2E, LP_FAR), e = lp_ex2(y);
        a.s += e;
        a.t = fmaf(e, y, a.t);
    }
}
template <int N> __device__ __forceinline__ void lp_count(const float (&x)[N], int i0, int token, float given, float above, int &before) {
    if (i0 + N <= token || i0 > token) {
        const float bar = i0 > token ? above : given;
#pragma unroll
        for (int i = 0; i < N; ++i) before += x[i] >= bar;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) before += x[i] >= (i0 + i < token ? given : above);
    }
}

__device__ __forceinline__ uint32_t lp_order(float v) { return (uint32_t)(amax_key(v, 0) >> 32); }  // 0: no candidate

// `list`: a warp's best entries, descending over the lanes (0: none); takes every lane's key
__device__ __forceinline__ void lp_insert(unsigned long long &list, unsigned long long key, int lane, int top) {
    for (;;) {
        const unsigned long long last = __shfl_sync(0xffffffffu, list, top - 1);
        const uint32_t want = __ballot_sync(0xffffffffu, key > last);
        if (!want) return;
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
__device__ __forceinline__ void lp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// p of CTA `rank` of the cluster
template <typename P> __device__ __forceinline__ P lp_load(const P *p, uint32_t rank) {
    static_assert(sizeof(P) == 4 || sizeof(P) == 8, "");
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    P v;
    if constexpr (sizeof(P) == 4) {
        uint32_t u;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(u) : "r"(a) : "memory");
        memcpy(&v, &u, 4);
    } else {
        unsigned long long u;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(u) : "r"(a) : "memory");
        memcpy(&v, &u, 8);
    }
    return v;
}

struct LpShared {
    LpSum sums[LP_W];
    int before[LP_W];
    unsigned long long keys[LP_MAX_CLUSTER > LP_W ? LP_MAX_CLUSTER * LP_MAX_TOP : LP_W * LP_MAX_TOP];
    unsigned long long best[LP_MAX_TOP];  // this CTA's alternatives, in order
    LpSum sum;                            // this CTA's part
    int count, n_keys, n_columns;
    short columns[LP_T];                  // threads whose words are read again
};

// the n keys in sh.keys put in order: the first `top` into sh.best
__device__ __forceinline__ void lp_rank_keys(LpShared &sh, int n, int top) {
    for (int i = threadIdx.x; i < n; i += LP_T) {
        const unsigned long long k = sh.keys[i];
        int at = 0;
        for (int j = 0; j < n; ++j) at += sh.keys[j] > k;
        if (k && at < top) sh.best[at] = k;
    }
}

// grid: rows x C CTAs in clusters of C (a power of two up to 8) for a row
template <typename T> __global__ void __launch_bounds__(LP_T, 4) k_logprobs(const LpArgs a, int C) {
    constexpr int N = LpWord<T>::N, U = 4;  // entries of a word; words in flight per thread
    __shared__ LpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / C;
    const uint32_t part = C > 1 ? lp_cluster_rank() : 0;
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
    const float given = known ? (float)x[token] + 0.0f : NAN, above = lp_above(given);
    LpSum sum{-INFINITY, LP_LOWEST, 0.0f, 0.0f};
    int before = 0;
    for (int w = w0 + tid; w < w1; w += U * LP_T) {
        uint4 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (w + u * LP_T < w1) r[u] = v[w + u * LP_T];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (w + u * LP_T >= w1) break;
            float e[N];
            LpWord<T>::unpack(r[u], e);
            lp_add<N>(e, sum);
            if (known) lp_count<N>(e, head + (w + u * LP_T) * N, token, given, above, before);
        }
    }
    // the entries outside whole words: one a thread, of the first CTA
    const int odd = part == 0 && tid < head + tail ? (tid < head ? tid : tail0 + tid - head) : -1;
    if (odd >= 0) {
        const float e[1] = {(float)x[odd]};
        lp_add<1>(e, sum);
        if (known) lp_count<1>(e, odd, token, given, above, before);
    }
    const uint32_t mine = lp_order(sum.m);
    LpSum all = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpSum c;
        c.m = __shfl_xor_sync(0xffffffffu, all.m, o);
        c.b = __shfl_xor_sync(0xffffffffu, all.b, o);
        c.s = __shfl_xor_sync(0xffffffffu, all.s, o);
        c.t = __shfl_xor_sync(0xffffffffu, all.t, o);
        lp_join(all, c);
    }
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) sh.sums[warp] = all, sh.before[warp] = before;
    if (a.top) {
        // a bound that at least `top` threads' maxima reach (0: all), by halving the interval between the bound that all reach
        // and the one that none does, until at most half as many again do
        uint32_t lo = 0, hi = 0xffffffffu;
        {
            const uint32_t wmin = __reduce_min_sync(0xffffffffu, mine), wmax = __reduce_max_sync(0xffffffffu, mine);
            __shared__ uint32_t ends[2][LP_W];
            if (lane == 0) ends[0][warp] = wmin, ends[1][warp] = wmax;
            __syncthreads();
            uint32_t l = ends[0][0], h = ends[1][0];
#pragma unroll
            for (int i = 1; i < LP_W; ++i) l = min(l, ends[0][i]), h = max(h, ends[1][i]);
            lo = l, hi = h;
        }
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = __syncthreads_count(mine >= mid);
            if (n >= a.top) {
                lo = mid;
                if (n <= a.top + a.top / 2) break;
            } else hi = mid;
        }
        const uint32_t bound = lo;
        if (mine && mine >= bound) sh.columns[atomicAdd(&sh.n_columns, 1)] = (short)tid;
        __syncthreads();
        const int n = sh.n_columns;
        unsigned long long list = 0;
        auto take = [&](unsigned long long key) {
            if ((uint32_t)(key >> 32) < bound) key = 0;
            lp_insert(list, key, lane, a.top);
        };
        for (int c = warp; c < n; c += LP_W) {
            const int first = w0 + sh.columns[c];
            for (int w = first; w < w1; w += 32 * LP_T) {
                const int at = w + lane * LP_T;
                float e[N];
#pragma unroll
                for (int i = 0; i < N; ++i) e[i] = NAN;
                if (at < w1) LpWord<T>::unpack(v[at], e);
                float m = e[0];
#pragma unroll
                for (int i = 1; i < N; ++i) m = fmaxf(m, e[i]);
                const uint32_t o = lp_order(m);
                if (!__any_sync(0xffffffffu, o && o >= bound)) continue;
#pragma unroll
                for (int i = 0; i < N; ++i) take(amax_key(e[i], head + at * N + i));
            }
        }
        if (part == 0 && warp == 0) take(lane < head + tail ? amax_key((float)x[odd], odd) : 0ull);
        if (list && lane < a.top) sh.keys[atomicAdd(&sh.n_keys, 1)] = list;
        __syncthreads();
        lp_rank_keys(sh, sh.n_keys, a.top);
    }
    __syncthreads();
    if (tid == 0) {
        LpSum z = sh.sums[0];
        int n = sh.before[0];
        for (int i = 1; i < LP_W; ++i) lp_join(z, sh.sums[i]), n += sh.before[i];
        sh.sum = z;
        sh.count = n;
    }
    if (C > 1) {
        __syncthreads();
        lp_cluster_sync();
        if (part == 0) {
            if (tid < C * a.top) sh.keys[tid] = lp_load(&sh.best[tid % a.top], tid / a.top);
            if (tid == 0) {
                LpSum z = sh.sum;
                int n = sh.count;
                for (int i = 1; i < C; ++i) {
                    lp_join(z, LpSum{lp_load(&sh.sum.m, i), lp_load(&sh.sum.b, i), lp_load(&sh.sum.s, i), lp_load(&sh.sum.t, i)});
                    n += lp_load(&sh.count, i);
                }
                sh.sum = z;
                sh.count = n;
            }
        }
        __syncthreads();
        lp_cluster_sync();  // the others' shared memory has been read
        if (part) return;
        if (a.top) {
            if (tid < LP_MAX_TOP) sh.best[tid] = 0;
            __syncthreads();
            lp_rank_keys(sh, C * a.top, a.top);
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
        if (rows < 0 || vocab < 1 || vocab > 1 << 30) return fail("logprobs: bad row / vocabulary counts");
        if (top < 0 || top > LP_MAX_TOP) return fail("logprobs: top out of range (0..32)");
        if (rows == 0) return 0;
        if (!logits || (top && (!top_ids || !top_logprobs))) return fail("logprobs: null pointer");
        if (!tokens && (logprob || rank)) return fail("logprobs: log probabilities and ranks want tokens");
        if ((uintptr_t)logits % (type == T_F32 ? 4 : 2)) return fail("logprobs: logits must be aligned to their type");
        // rows too few for the SMs (4 CTAs of 256 threads each) share theirs between up to 8 CTAs of 4096 entries and more
        int C = 1;
        while (C < LP_MAX_CLUSTER && (int64_t)rows * C * 2 <= 4 * num_sms() && vocab / (2 * C) >= 4096) C *= 2;
        if ((int64_t)rows * C > INT32_MAX) return fail("logprobs: too many rows");
        const LpArgs a{logits, stride, rows, vocab, top, tokens, logprob, rank, entropy, top_ids, top_logprobs, dev_error_ptr()};
        const dim3 grid((unsigned)(rows * C));
        auto *k = type == T_F32 ? k_logprobs<float> : k_logprobs<__nv_bfloat16>;
        const cudaError_t e = C > 1 ? launch_kc(k, grid, dim3(LP_T), (unsigned)C, 0, (cudaStream_t)stream, a, C)
                                    : launch_k(k, grid, dim3(LP_T), 0, (cudaStream_t)stream, a, C);
        if (e != cudaSuccess) return fail(std::string("logprobs launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
