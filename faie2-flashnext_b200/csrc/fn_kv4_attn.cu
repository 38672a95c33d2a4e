// Attention over the paged 4-bit KV cache (fn_kv4.h): softmax(scale q k^T) v per query row, causal, grouped heads.
// The reference's attention reads dense fp32 caches at one position for all (k_attn_split + k_attn_combine,
// engine/faie2fn.cu:1598-1690).
//
// Mathematics. With codes c (0..15) and one scale d per 64 dims G of a token, s = q . k = sum_G dk[G] (sum_{i in G} q_i c_i
// - 8 sum_{i in G} q_i), and out_i = sum_t p_t dv[t][G] c_ti - 8 sum_t p_t dv[t][G]. The inner sums are matrix products
// with the codes themselves, so nothing is dequantised: a nibble in the low bits of a half is the fp16 number c 2^-24 (or
// c 2^-20 four bits higher), exact, and the tensor cores take it as it is. One mask per two codes replaces the
// conversion; the offset's term enters as the product's initial accumulator (K) or is subtracted at the end (V).
//
// Orientation. Codes are the A operand (16 tokens x 16 dims for K, 16 dims x 16 tokens for V) and the query rows the B
// operand's 8 columns: a group of 8 heads fills the instruction. The weights p dv come out of the score product with tokens
// down and rows across and are turned by movmatrix, 8 x 8 at a time, into the second product's B operand.
//
// Precision. bf16 rows: q is exact in fp16 after scaling, p dv is rounded once to 11 bits (the output has 8). fp32 rows: q
// and p dv are split into two fp16 numbers, 22 bits together, which costs a second instruction each. A tensor core drops
// what lies some 24 bits below the nominal size of its largest term, and a code as a subnormal fp16 number lies up to 10
// bits below its nominal size; so both first halves are whole numbers up to 2^11 (q scaled per row by a power of two, p dv by
// the softmax's reference): all their products and sums are multiples of one unit, and exact. Floating halves lost 2.5e-6
// of the output where this form loses 3e-7. Sums over more than 32 tokens are added in fp32 outside the tensor core, whose
// own accumulation cuts instead of rounding. The softmax runs in base 2 with one reference per row, the running maximum
// plus the running exponent of the largest |dv|, so that p dv uses fp16's range whatever the size of V.
//
// Work. A unit is 64 tokens of one kv head for one row tile (8 or 16 rows: the heads of a group, token after token). All
// units of the call in a row are cut into equal runs, one per CTA, whatever request they belong to: each CTA finds its run
// from the lengths by a prefix sum, so nothing about the lengths is known on the host and a captured call serves any.
// A row tile whose units lie in several CTAs is joined by the last of them to finish (groups of 16 first, then the
// groups), in the order of the CTAs, so the result does not depend on timing.
//
// A CTA: one warp copies pages into a ring (one bulk copy per page and head: codes and scales of K and V), four warps
// compute, two on each 64-token stage, 32 tokens each, with their own running softmax; they merge at the end of a run.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "fn_kv4.h"

namespace fn {

constexpr int KA_TOK = 64;                    // tokens of a stage
constexpr int KA_CONS = 4;                    // computing warps
constexpr int KA_THREADS = 256;               // the computing warpgroup, and one of which a warp copies
// registers: 256 threads x 128 at launch; the copying warpgroup gives up what the computing one takes (40 + 216 = 2 x 128),
// which holds 8 or 16 rows of 256 sums
constexpr int KA_REG_COPY = 40, KA_REG_COMP = 216;
constexpr int KA_CTAS = 2;                    // per SM
constexpr int KA_FAN = 16;                    // partial results joined at once
constexpr int KA_JOIN = 32;                   // .. and at most in the second round
constexpr int KA_MAX_GRID = KA_FAN * KA_JOIN; // CTAs at most

struct Kv4AttnArgs {
    Kv4Lay l;
    int n, rows, nh, group, max_pages, vec;
    const void *q, *gate;
    int64_t qt, qh, gt, gh, ot;
    void *out;
    const int *cu, *kv_len, *table;
    float scale;
    float *part;     // [CTA][2]: a row tile's sums [rows][hd], references [rows], sums of weights [rows]
    uint32_t *cnt;   // [3][KA_MAX_GRID] arrivals, zero between calls
    uint32_t *err;
};

// a request's share of the work
struct KaReq {
    int first, fresh, len, tiles, rt;  // first row, rows, tokens, 64-token tiles, row tiles
};
template <int ROWS> __device__ __forceinline__ KaReq ka_req(const Kv4AttnArgs &a, int r) {
    KaReq q;
    const int c0 = after_wait(a.cu)[r], c1 = after_wait(a.cu)[r + 1];
    q.first = min(max(c0, 0), a.rows);
    q.fresh = min(max(c1, q.first), a.rows) - q.first;
    const long long cap = (long long)a.max_pages * a.l.bs;
    q.len = (int)min((long long)max(after_wait(a.kv_len)[r], 0), cap);
    q.tiles = max((q.len + KA_TOK - 1) / KA_TOK, 1);  // an empty request's rows are written too
    q.rt = (int)(((long long)q.fresh * a.group + ROWS - 1) / ROWS);
    return q;
}

__device__ __forceinline__ void ka_mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t ka_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ float2 ka_unpack(uint32_t w) { return __half22float2(*(const __half2 *)&w); }
// an 8 x 8 matrix of halves, row g columns 2t, 2t + 1 in lane 4 g + t, turned
__device__ __forceinline__ uint32_t ka_turn(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ float ka_half(const uint8_t *p) { return __half2float(*(const __half *)p); }
// the weight of a part whose reference is `ref` beside the common one; a part without a key has none, and a row that has
// nothing but NaN scores keeps them through the reference 0
__device__ __forceinline__ float ka_weight(float ref, float common) {
    return ka_exp2(ref == -INFINITY ? (common == -INFINITY ? 0.0f : -INFINITY) : ref - common);
}
__device__ __forceinline__ void ka_bar() { asm volatile("bar.sync 1, %0;" ::"n"(32 * KA_CONS) : "memory"); }
// the same, and whether any thread brought `p`
__device__ __forceinline__ bool ka_bar_or(bool p) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"((uint32_t)p), "n"(32 * KA_CONS)
        : "memory");
    return any != 0;
}
__device__ __forceinline__ void ka_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
template <typename T> __device__ __forceinline__ float ka_f(T x);
template <> __device__ __forceinline__ float ka_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float ka_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <int HD, bool HL, int NT> struct KaCfg {
    using T = std::conditional_t<HL, float, __nv_bfloat16>;
    static constexpr int NG = HD / KV4_GROUP, ROWS = 8 * NT;
    static constexpr int OS = HD + 1;                         // floats between rows of the merged sums (banks)
    static constexpr uint32_t STAGE = KA_TOK * HD / 16 * 17;  // bytes of 64 tokens of one head
    static constexpr uint32_t QF = NT * NG * 4 * 32 * (HL ? 16 : 8);  // q as B operands: [n-tile][group][step][lane]
    static constexpr uint32_t OB = (ROWS * OS * 4 + 127) / 128 * 128;
    // the merged sums share their place with q, which is rebuilt for the next row tile
    static constexpr uint32_t Q_OFF = 1024, ST_OFF = Q_OFF + (QF > OB ? QF : OB);
    static constexpr uint32_t SMEM_MAX = 112 * 1024;          // of two CTAs on an SM (114 KB each, less static memory)
    // stages, an even number: a slot then always belongs to the same pair of warps, whose waits see each of its phases
    static constexpr int S = (SMEM_MAX - ST_OFF) / STAGE > 16 ? 16 : (SMEM_MAX - ST_OFF) / STAGE / 2 * 2;
    static constexpr uint32_t SMEM = ST_OFF + S * STAGE;
};
constexpr int KA_PART_MAX = 16 * 256 + 32;

template <int HD, bool HL, int NT> __global__ void __launch_bounds__(KA_THREADS, KA_CTAS) k_kv4_attn(const __grid_constant__ Kv4AttnArgs a) {
    using C = KaCfg<HD, HL, NT>;
    using T = typename C::T;
    constexpr int NG = C::NG, ROWS = C::ROWS, S = C::S, OS = C::OS;
    using QF = std::conditional_t<HL, uint4, uint2>;
    extern __shared__ __align__(128) uint8_t sm_ka[];
    __shared__ long long red[KA_THREADS / 32], s_off;
    __shared__ int s_req;
    __shared__ volatile int s_fail;
    __shared__ float s_rs[ROWS], s_qs[2][ROWS][NG], s_ref[KA_CONS][ROWS], s_l[KA_CONS][ROWS], s_mref[ROWS], s_ml[ROWS];
    __shared__ float s_join[KA_JOIN][ROWS];
    __shared__ int s_last;
    __shared__ uint32_t s_valid[S];
    uint64_t *full = (uint64_t *)sm_ka, *empty = full + S;
    QF *qf = (QF *)(sm_ka + C::Q_OFF);
    float *ob = (float *)(sm_ka + C::Q_OFF);
    uint8_t *ring = sm_ka + C::ST_OFF;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 2);
        }
        mbar_fence_init();
        s_fail = 0;
    }
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's run of units: prefix sum over the requests, a contiguous share of them per thread
    const int per_t = (a.n + KA_THREADS - 1) / KA_THREADS, r0 = min(tid * per_t, a.n), r1 = min(r0 + per_t, a.n);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) {
        const KaReq q = ka_req<ROWS>(a, r);
        mine += (long long)q.rt * a.l.nkv * q.tiles;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    long long before = incl - mine, units = 0;
    for (int w = 0; w < KA_THREADS / 32; ++w) {
        if (w < warp) before += red[w];
        units += red[w];
    }
    const long long per = max((units + gridDim.x - 1) / gridDim.x, 2ll);
    const long long u0 = blockIdx.x * per, u1 = min(u0 + per, units);
    if (u0 < u1 && u0 >= before && u0 < before + mine) {
        long long at = before;
        for (int r = r0; r < r1; ++r) {
            const KaReq q = ka_req<ROWS>(a, r);
            const long long w = (long long)q.rt * a.l.nkv * q.tiles;
            if (u0 < at + w) {
                s_req = r;
                s_off = u0 - at;
                break;
            }
            at += w;
        }
    }
    // rows that belong to no request
    {
        const int live = min(max(after_wait(a.cu)[a.n], 0), a.rows);
        const long long left = (long long)(a.rows - live) * a.nh * HD;
        for (long long i = (long long)blockIdx.x * KA_THREADS + tid; i < left; i += (long long)gridDim.x * KA_THREADS) {
            const long long row = i / (a.nh * HD);
            ((T *)a.out)[(live + row) * a.ot + (i - row * a.nh * HD)] = (T)0.0f;
        }
    }
    __syncthreads();
    if (u0 >= u1) return;

    int r = s_req;
    KaReq rq = ka_req<ROWS>(a, r);
    int item = (int)(s_off / rq.tiles), k = (int)(s_off - (long long)item * rq.tiles);
    // to the next row tile of the run
    auto next = [&]() {
        k = 0;
        if (++item < rq.rt * a.l.nkv) return;
        item = 0;
        do rq = ka_req<ROWS>(a, ++r);
        while (rq.rt == 0);
    };
    auto wt = [&](uint64_t *bar, uint32_t par) {
        if (s_fail) return false;
        if (mbar_park(bar, par)) return true;
        s_fail = 1;
        dev_fail(a.err, DEV_WAIT_TIMEOUT);
        return false;
    };
    const int ppt = KA_TOK / a.l.bs;  // pages of a stage

    if (warp >= KA_CONS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KA_REG_COPY));
        if (warp > KA_CONS) return;
        // ---- copies: lane p fetches page p of a stage; a lane holds one entry of the next 32 pages' ids
        int it = 0;
        for (long long u = u0; u < u1;) {
            const int kend = (int)min((long long)rq.tiles, k + (u1 - u)), kv = item / rq.rt;
            const int pages = (rq.len + a.l.bs - 1) / a.l.bs;
            const int *tab = after_wait(a.table) + (size_t)r * a.max_pages;
            const int p0 = k * ppt;
            int cur = p0 + lane < pages ? tab[p0 + lane] : -1, nxt = p0 + 32 + lane < pages ? tab[p0 + 32 + lane] : -1, base = p0;
            for (int j = k; j < kend; ++j, ++it) {
                const int sl = it % S, pg = j * ppt;
                if (pg >= base + 32) {
                    cur = nxt;
                    base += 32;
                    nxt = base + 32 + lane < pages ? tab[base + 32 + lane] : -1;
                }
                const int id = __shfl_sync(0xffffffffu, cur, (pg - base + (lane < ppt ? lane : 0)) & 31);
                const bool want = lane < ppt && pg + lane < pages, ok = want && id >= 0 && id < a.l.n_pages;
                if (want && !ok) dev_fail(a.err, DEV_BAD_ARG);
                const uint32_t m = __ballot_sync(0xffffffffu, ok);
                bool go = true;
                if (lane == 0) {
                    go = it < S || wt(&empty[sl], (uint32_t)(it / S - 1) & 1u);
                    if (go) {
                        s_valid[sl] = m;
                        mbar_arrive_tx(&full[sl], (uint32_t)__popc(m) * a.l.rec);
                    }
                }
                go = __shfl_sync(0xffffffffu, (int)go, 0);
                if (!go) goto drained;
                if (ok)
                    bulk_g2s(ring + (size_t)sl * C::STAGE + lane * a.l.rec,
                             a.l.pages + ((int64_t)id * a.l.nkv + kv) * (int64_t)a.l.rec, a.l.rec, &full[sl]);
            }
            u += kend - k;
            if (u < u1) next();
        }
    drained:
        // a CTA that gave up must not leave with copies into its shared memory in flight
        if (s_fail && lane == 0)
            for (int i = max(it - S, 0); i < it; ++i) mbar_park(&full[i % S], (uint32_t)(i / S) & 1u);
        return;
    }

    // ---- compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KA_REG_COMP));
    const int g = lane >> 2, t = lane & 3, half = warp & 1, pair = warp >> 1;
    // index n of 8 tokens is token n ^ (n >> 2): with it both the K reads (8 bytes of 8 tokens x 4 lanes, 16 lanes at a
    // time) and the V reads (4 bytes of 4 tokens x 8 words) touch 32 different banks
    const int tk = g ^ (g >> 2);
    const int tv0 = (2 * t) ^ (t >> 1), tv1 = (2 * t + 1) ^ (t >> 1);
    int it = 0;
    for (long long u = u0; u < u1;) {
        const int kend = (int)min((long long)rq.tiles, k + (u1 - u)), kv = item / rq.rt, tile = item - kv * rq.rt;
        const int nrow = min(ROWS, rq.fresh * a.group - tile * ROWS);
        // ---- q of the row tile into B operands
        ka_bar();
        {
            constexpr int L = 32 * KA_CONS / ROWS, PG = KV4_GROUP / L;  // lanes of a row; dims of a group each takes
            const int i = tid / L, sub = tid % L, flat = tile * ROWS + i, tok = flat / a.group;
            const T *src = (const T *)after_wait(a.q) + (int64_t)(rq.first + tok) * a.qt +
                           (int64_t)(kv * a.group + flat - tok * a.group) * a.qh + sub * PG;
            float x[NG][PG], mx = 0.0f;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                for (int j = 0; j < PG; ++j) {
                    x[gi][j] = i < nrow ? ka_f<T>(src[gi * KV4_GROUP + j]) : 0.0f;
                    mx = fmaxf(mx, fabsf(x[gi][j]));
                }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const int e = min(max(10 - ((int)(__float_as_uint(mx) >> 23) - 127), -90), 120);
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                float sum = 0.0f, sum_lo = 0.0f;
#pragma unroll
                for (int j = 0; j < PG; ++j) {
                    const int d = sub * PG + j, w = d >> 3, nib = d & 7, step = (w & 1) * 2 + ((nib & 3) >> 1);
                    const float f = x[gi][j] * up, fh = HL ? rintf(f) : f, fl = f - fh;
                    const float sc = nib & 1 ? 0.0625f : 1.0f;  // odd nibbles stand 16 times as high
                    const __half lo = __float2half_rn(fl);
                    sum += fh;
                    sum_lo += __half2float(lo);
                    __half *dst = (__half *)&qf[(((i >> 3) * NG + gi) * 4 + step) * 32 + (i & 7) * 4 + (w >> 1)];
                    dst[(nib & 1) * 2 + (nib >> 2)] = __float2half_rn(fh * sc);
                    if constexpr (HL) dst[(2 + (nib & 1)) * 2 + (nib >> 2)] = __float2half_rn(__half2float(lo) * sc);
                }
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (HL) sum_lo += __shfl_xor_sync(0xffffffffu, sum_lo, o);
                }
                if (sub == 0) {
                    s_qs[0][i][gi] = sum * (-8.0f / 16777216.0f);
                    if (HL) s_qs[1][i][gi] = sum_lo * (-8.0f / 16777216.0f);
                }
            }
            // scores in base 2: undo the scaling and the codes' 2^-24
            if (sub == 0) s_rs[i] = a.scale * 1.44269504f * __uint_as_float((uint32_t)(24 - e + 127) << 23);
        }
        ka_bar();
        // rows see tokens below their limit; rows past the tile's last see what the last sees (their results are dropped)
        auto limit = [&](int i) {
            const int f = tile * ROWS + min(i, nrow - 1);
            return min(max(rq.len - rq.fresh + f / a.group + 1, 0), rq.len);
        };
        const int lo_lim = limit(0), hi_lim = limit(ROWS - 1);
        int lim[NT][2];
        // o[n-tile][group][byte]: rows 2t, 2t + 1 of the tile for dim 8 g + 2 byte, then for the dim after it
        float o[NT][NG][4][4], corr[NT][NG][2], m[NT][2], l[NT][2], ref[NT][2];
        int ev = -40;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                lim[n][c] = limit(8 * n + 2 * t + c);
                m[n][c] = ref[n][c] = -INFINITY;
                l[n][c] = 0.0f;
            }
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                corr[n][gi][0] = corr[n][gi][1] = 0.0f;
#pragma unroll
                for (int by = 0; by < 4; ++by) o[n][gi][by][0] = o[n][gi][by][1] = o[n][gi][by][2] = o[n][gi][by][3] = 0.0f;
            }
        }
        bool alive = true;
        for (int j = k; j < kend; ++j, ++it) {
            if ((it & 1) != pair) continue;
            const int sl = it % S;
            if (!wt(&full[sl], (uint32_t)(it / S) & 1u)) {
                alive = false;
                break;
            }
            const uint8_t *st = ring + (size_t)sl * C::STAGE;
            const int t0 = j * KA_TOK + half * 32;  // this warp's first token
            const uint32_t valid = s_valid[sl];
            const bool masked = t0 + 32 > lo_lim || valid != (1u << ppt) - 1u;
            // record and place of this warp's two runs of 16 tokens
            const uint8_t *rec[2];
            int pl[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int at = half * 32 + b * 16, pg = at / a.l.bs;
                rec[b] = st + pg * a.l.rec;
                pl[b] = at - pg * a.l.bs;
            }
            // ---- scores sc[n-tile][run][tokens tk, tk + 8][rows 2t, 2t + 1]
            float sc[NT][2][2][2] = {};
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                QF B[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) B[n][x] = qf[((n * NG + gi) * 4 + x) * 32 + lane];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int line = gi * a.l.bs + pl[b] + tk;
                    const uint2 w = *(const uint2 *)(rec[b] + line * 32 + t * 8), v = *(const uint2 *)(rec[b] + (line + 8) * 32 + t * 8);
                    const float d0 = ka_half(rec[b] + 2 * a.l.kb + line * 2), d1 = ka_half(rec[b] + 2 * a.l.kb + (line + 8) * 2);
                    const uint4 A0 = make_uint4(w.x & 0x000f000fu, v.x & 0x000f000fu, w.x & 0x00f000f0u, v.x & 0x00f000f0u);
                    const uint4 A1 = make_uint4((w.x >> 8) & 0x000f000fu, (v.x >> 8) & 0x000f000fu, (w.x >> 8) & 0x00f000f0u, (v.x >> 8) & 0x00f000f0u);
                    const uint4 A2 = make_uint4(w.y & 0x000f000fu, v.y & 0x000f000fu, w.y & 0x00f000f0u, v.y & 0x00f000f0u);
                    const uint4 A3 = make_uint4((w.y >> 8) & 0x000f000fu, (v.y >> 8) & 0x000f000fu, (w.y >> 8) & 0x00f000f0u, (v.y >> 8) & 0x00f000f0u);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float i0 = s_qs[0][8 * n + 2 * t][gi], i1 = s_qs[0][8 * n + 2 * t + 1][gi];
                        float acc[4] = {i0, i1, i0, i1};
                        ka_mma(acc, A0, B[n][0].x, B[n][0].y);
                        ka_mma(acc, A1, B[n][1].x, B[n][1].y);
                        ka_mma(acc, A2, B[n][2].x, B[n][2].y);
                        ka_mma(acc, A3, B[n][3].x, B[n][3].y);
                        if constexpr (HL) {
                            const float j0 = s_qs[1][8 * n + 2 * t][gi], j1 = s_qs[1][8 * n + 2 * t + 1][gi];
                            float low[4] = {j0, j1, j0, j1};
                            ka_mma(low, A0, B[n][0].z, B[n][0].w);
                            ka_mma(low, A1, B[n][1].z, B[n][1].w);
                            ka_mma(low, A2, B[n][2].z, B[n][2].w);
                            ka_mma(low, A3, B[n][3].z, B[n][3].w);
#pragma unroll
                            for (int x = 0; x < 4; ++x) acc[x] += low[x];
                        }
                        sc[n][b][0][0] += acc[0] * d0;
                        sc[n][b][0][1] += acc[1] * d0;
                        sc[n][b][1][0] += acc[2] * d1;
                        sc[n][b][1][1] += acc[3] * d1;
                    }
                }
            }
            // ---- V scales of this lane's tokens, and the largest among the warp's
            float dv[2][2][NG], dm = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int tok = t0 + b * 16 + h * 8 + tk;
                    const bool drop = masked && (!(valid >> ((half * 32 + b * 16 + h * 8) / a.l.bs) & 1u) || tok >= hi_lim);
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) {
                        const float d = ka_half(rec[b] + 2 * a.l.kb + a.l.sb + (gi * a.l.bs + pl[b] + h * 8 + tk) * 2);
                        dv[b][h][gi] = drop ? 0.0f : d;  // what nobody sees counts for nothing, whatever is there
                        dm = fmaxf(dm, fabsf(dv[b][h][gi]));
                    }
                }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, x));
            ev = max(ev, (int)(__float_as_uint(dm) >> 23) - 127);
            // ---- running softmax in base 2: p = exp2(s - reference), |p dv| < 2^11
            bool moved = false;
            float z[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float rs = s_rs[8 * n + 2 * t + c];
                    float mx = m[n][c];
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float s = sc[n][b][h][c] * rs;
                            if (masked) {
                                const int tok = t0 + b * 16 + h * 8 + tk;
                                if (!(valid >> ((half * 32 + b * 16 + h * 8) / a.l.bs) & 1u) || tok >= lim[n][c]) s = -INFINITY;
                            }
                            sc[n][b][h][c] = s;
                            mx = fmaxf(mx, s);
                        }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                    m[n][c] = mx;
                    const float nr = mx + (float)(ev - 10);
                    moved |= nr != ref[n][c];
                    z[n][c] = nr == -INFINITY ? 0.0f : nr;
                }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float f0 = ka_exp2(ref[n][0] - z[n][0]), f1 = ka_exp2(ref[n][1] - z[n][1]);
                    l[n][0] *= f0;
                    l[n][1] *= f1;
                    ref[n][0] = m[n][0] + (float)(ev - 10);
                    ref[n][1] = m[n][1] + (float)(ev - 10);
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) {
                        corr[n][gi][0] *= f0;
                        corr[n][gi][1] *= f1;
#pragma unroll
                        for (int by = 0; by < 4; ++by) {
                            o[n][gi][by][0] *= f0;
                            o[n][gi][by][1] *= f1;
                            o[n][gi][by][2] *= f0;
                            o[n][gi][by][3] *= f1;
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            sc[n][b][h][c] = ka_exp2(sc[n][b][h][c] - z[n][c]);
                            l[n][c] += sc[n][b][h][c];
                        }
            // ---- out += c (p dv)
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                uint32_t P[NT][2][2], Q[NT][2][2];  // B operands: tokens 2t, 2t + 1 (+ 8) of row g; second halves
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float p0 = sc[n][b][h][0], p1 = sc[n][b][h][1], d = dv[b][h][gi];
                            // a token that a row does not see weighs nothing whatever its scale is (NaN)
                            const float x0 = masked && p0 == 0.0f ? 0.0f : p0 * d, x1 = masked && p1 == 0.0f ? 0.0f : p1 * d;
                            corr[n][gi][0] += x0;
                            corr[n][gi][1] += x1;
                            if constexpr (HL) {
                                const float big = 12582912.0f;  // 1.5 2^23: adding it rounds to whole numbers
                                const float h0 = __fadd_rn(__fadd_rn(x0, big), -big), h1 = __fadd_rn(__fadd_rn(x1, big), -big);
                                P[n][b][h] = ka_turn(ka_pack(h0, h1));
                                Q[n][b][h] = ka_turn(ka_pack(x0 - h0, x1 - h1));
                            } else {
                                P[n][b][h] = ka_turn(ka_pack(x0, x1));
                            }
                        }
                uint32_t w[2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint8_t *vc = rec[b] + a.l.kb + (gi * a.l.bs + pl[b]) * 32 + g * 4;
                    w[b][0] = *(const uint32_t *)(vc + tv0 * 32);
                    w[b][1] = *(const uint32_t *)(vc + tv1 * 32);
                    w[b][2] = *(const uint32_t *)(vc + (8 + tv0) * 32);
                    w[b][3] = *(const uint32_t *)(vc + (8 + tv1) * 32);
                }
#pragma unroll
                for (int by = 0; by < 4; ++by) {
                    const uint32_t sel = (uint32_t)(by | by << 4 | (4 + by) << 8 | (4 + by) << 12);
                    uint4 A[2];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t x = __byte_perm(w[b][0], w[b][1], sel), y = __byte_perm(w[b][2], w[b][3], sel);
                        A[b] = make_uint4(x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if constexpr (HL) {
                            float acc[4] = {};
                            ka_mma(acc, A[0], P[n][0][0], P[n][0][1]);
                            ka_mma(acc, A[1], P[n][1][0], P[n][1][1]);
                            ka_mma(acc, A[0], Q[n][0][0], Q[n][0][1]);
                            ka_mma(acc, A[1], Q[n][1][0], Q[n][1][1]);
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[n][gi][by][x] += acc[x];
                        } else {
                            ka_mma(o[n][gi][by], A[0], P[n][0][0], P[n][0][1]);
                            ka_mma(o[n][gi][by], A[1], P[n][1][0], P[n][1][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ka_arrive(&empty[sl]);
        }

        // ---- merge the four warps: one reference per row, sums added quarter by quarter in a fixed order
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) corr[n][gi][c] += __shfl_xor_sync(0xffffffffu, corr[n][gi][c], x);
                }
        if (g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    s_ref[warp][8 * n + 2 * t + c] = ref[n][c];
                    s_l[warp][8 * n + 2 * t + c] = l[n][c];
                }
        }
        if (ka_bar_or(!alive)) return;  // a wait gave up: all warps leave here together
        auto top = [&](int i) { return fmaxf(fmaxf(s_ref[0][i], s_ref[1][i]), fmaxf(s_ref[2][i], s_ref[3][i])); };
        float wf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) wf[n][c] = ka_weight(ref[n][c], top(8 * n + 2 * t + c));
        if (tid < ROWS) {
            const float tt = top(tid);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < KA_CONS; ++w) sum += s_l[w][tid] * ka_weight(s_ref[w][tid], tt);
            s_mref[tid] = tt;
            s_ml[tid] = sum;
        }
        for (int round = 0; round < 4; ++round) {
#pragma unroll
            for (int by = 0; by < 4; ++by) {
                if (((warp + round) & 3) != by) continue;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float v = (o[n][gi][by][x] * (x >= 2 ? 1048576.0f : 16777216.0f) - 8.0f * corr[n][gi][x & 1]) * wf[n][x & 1];
                            float *p = ob + (8 * n + 2 * t + (x & 1)) * OS + gi * KV4_GROUP + 8 * g + 2 * by + (x >> 1);
                            *p = round ? *p + v : v;
                        }
            }
            ka_bar();
        }
        // the row tile's output: a warp takes a row at a time
        auto emit = [&]() {
            for (int i = warp; i < nrow; i += KA_CONS) {
                const int f = tile * ROWS + i, tok = f / a.group, h = kv * a.group + f - tok * a.group;
                const int64_t row = rq.first + tok;
                const bool sees = limit(i) > 0;
                const float inv = s_ml[i];
                for (int d = lane; d < HD; d += 32) {
                    float y = sees ? ob[i * OS + d] / inv : 0.0f;
                    if (a.gate && sees) y *= sigm(ka_f<T>(((const T *)after_wait(a.gate))[row * a.gt + h * a.gh + d]));
                    ((T *)a.out)[row * a.ot + (int64_t)h * HD + d] = (T)y;
                }
            }
        };
        if (k == 0 && kend == rq.tiles) {
            emit();
        } else {
            // ---- a part of a row tile: into the workspace; the last CTA of 16 joins them, the last of those the rest
            const long long first = u - k;  // the row tile's first unit
            const int c0 = (int)(first / per), c1 = (int)((first + rq.tiles - 1) / per), c = blockIdx.x;
            const int edge = first != c0 * per;  // a CTA's part lies at its run's start (0) or after it (1)
            auto slot = [&](int cta) { return a.part + ((size_t)cta * 2 + (cta == c0 ? edge : 0)) * KA_PART_MAX; };
            auto put = [&](float *to) {
                for (int e = tid; e < nrow * HD; e += 32 * KA_CONS) __stcg(to + e, ob[e / HD * OS + e % HD]);
                if (tid < ROWS) {
                    __stcg(to + ROWS * HD + tid, s_mref[tid]);
                    __stcg(to + ROWS * HD + ROWS + tid, s_ml[tid]);
                }
            };
            put(slot(c));
            // joins the parts of CTAs b, b + step, .. into ob, s_mref and s_ml
            auto join = [&](int b, int step, int count) {
                for (int x = tid; x < count * ROWS; x += 32 * KA_CONS)
                    s_join[x / ROWS][x % ROWS] = __ldcg(slot(b + x / ROWS * step) + ROWS * HD + x % ROWS);
                ka_bar();
                if (tid < ROWS) {
                    float mx = -INFINITY, sum = 0.0f;
                    for (int x = 0; x < count; ++x) mx = fmaxf(mx, s_join[x][tid]);
#pragma unroll 8
                    for (int x = 0; x < count; ++x) {
                        const float f = ka_weight(s_join[x][tid], mx);
                        s_join[x][tid] = f;
                        sum += f * __ldcg(slot(b + x * step) + ROWS * HD + ROWS + tid);
                    }
                    s_mref[tid] = mx;
                    s_ml[tid] = sum;
                }
                ka_bar();
                constexpr int E = ROWS * HD / (32 * KA_CONS * 4), U = E >= 8 ? 1 : E >= 4 ? 2 : 4;  // loads in flight: 8 at least
                float4 y[E] = {};
                for (int x0 = 0; x0 < count; x0 += U) {
                    float4 v[U][E];
#pragma unroll
                    for (int x = 0; x < U; ++x)
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (x0 + x < count) v[x][e] = __ldcg((const float4 *)(slot(b + (x0 + x) * step)) + tid + e * 32 * KA_CONS);
#pragma unroll
                    for (int x = 0; x < U; ++x)
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (x0 + x < count) {
                                const float f = s_join[x0 + x][(tid + e * 32 * KA_CONS) * 4 / HD];
                                y[e].x += f * v[x][e].x, y[e].y += f * v[x][e].y, y[e].z += f * v[x][e].z, y[e].w += f * v[x][e].w;
                            }
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int at = (tid + e * 32 * KA_CONS) * 4;
                    float *p = ob + at / HD * OS + at % HD;
                    p[0] = y[e].x, p[1] = y[e].y, p[2] = y[e].z, p[3] = y[e].w;
                }
                ka_bar();
            };
            // true for the last of `count` arrivals (all that the others stored before theirs is visible to it)
            auto last_of = [&](uint32_t *counter, int count) {
                __threadfence();
                ka_bar();
                if (tid == 0) {
                    const bool last = atomicAdd(counter, 1u) == (uint32_t)count - 1;
                    if (last) *counter = 0;
                    __threadfence();
                    s_last = last;
                }
                ka_bar();
                return s_last != 0;
            };
            const int parts = c1 - c0 + 1, gr = (c - c0) / KA_FAN, gb = c0 + gr * KA_FAN, gn = min(KA_FAN, c1 - gb + 1);
            bool mineis = last_of(a.cnt + (gr ? KA_MAX_GRID : 0) + gb, gn);
            int jb = gb, step = 1, count = gn;
            while (mineis) {
                join(jb, step, count);
                if (step == KA_FAN || parts <= KA_FAN) break;
                put(slot(gb));
                jb = c0, step = KA_FAN, count = (parts + KA_FAN - 1) / KA_FAN;
                mineis = last_of(a.cnt + 2 * KA_MAX_GRID + c0, count);
            }
            if (mineis) emit();
        }
        u += kend - k;
        if (u < u1) next();
    }
}

}  // namespace fn

using namespace fn;

// counters, then every CTA's two partial results
FN_API uint64_t fn_kv4_attn_workspace(void) {
    return 3 * KA_MAX_GRID * 4 + (uint64_t)std::min(num_sms() * KA_CTAS, KA_MAX_GRID) * 2 * KA_PART_MAX * 4;
}

template <int HD, bool HL, int NT> static cudaError_t attn_launch(const Kv4AttnArgs &a, long long units, cudaStream_t s) {
    const cudaError_t e = allow_max_dynamic_smem(k_kv4_attn<HD, HL, NT>);
    if (e != cudaSuccess) return e;
    const int grid = (int)std::min(std::max(units / 2, 1ll), (long long)std::min(num_sms() * KA_CTAS, KA_MAX_GRID));
    return launch_k(k_kv4_attn<HD, HL, NT>, dim3(grid), dim3(KA_THREADS), KaCfg<HD, HL, NT>::SMEM, s, a);
}
template <int HD> static cudaError_t attn_go(const Kv4AttnArgs &a, bool f32, int max_new, cudaStream_t s) {
    // requests whose rows fill one column tile of 8 take the narrow form
    const long long rows = (long long)std::min(max_new, a.rows) * a.group;
    const int nt = rows <= 8 ? 1 : 2;
    // the most units there can be: no more CTAs than pairs of them
    const long long tiles = ((long long)a.max_pages * a.l.bs + KA_TOK - 1) / KA_TOK;
    const long long units = (long long)a.n * a.l.nkv * std::max((rows + 8 * nt - 1) / (8 * nt), 1ll) * tiles;
    if (nt == 1) return f32 ? attn_launch<HD, true, 1>(a, units, s) : attn_launch<HD, false, 1>(a, units, s);
    return f32 ? attn_launch<HD, true, 2>(a, units, s) : attn_launch<HD, false, 2>(a, units, s);
}

FN_API int fn_kv4_attn(const fn_kv4_t *c, uint32_t type, int n, int rows, int nh, const void *q, int64_t q_token,
                       int64_t q_head, const void *gate, int64_t gate_token, int64_t gate_head, void *out,
                       int64_t out_token, const int *cu, const int *kv_len, const int *table, int max_pages, int max_new,
                       float scale, void *ws, uint64_t ws_bytes, void *stream) {
    return kv4_entry("kv4 attn", [&]() -> int {
        Kv4AttnArgs a{};
        if (kv4_layout(c, a.l, "kv4 attn")) return -1;
        if (type != T_F32 && type != T_BF16) return fail("kv4 attn: rows must be F32 or BF16");
        if (n < 1 || n > KV4_MAX_REQ) return fail("kv4 attn: requests out of range (1..4096)");
        if (nh < 1 || nh % c->nkv || nh / c->nkv > 64) return fail("kv4 attn: bad head counts");
        if (rows < 0 || max_pages < 1 || max_new < 0) return fail("kv4 attn: bad row / page counts");
        if (rows == 0) return 0;
        if (!q || !out || !cu || !kv_len || !table || !ws) return fail("kv4 attn: null pointer");
        if (ws_bytes < fn_kv4_attn_workspace() || (uintptr_t)ws % 256) return fail("kv4 attn: workspace too small or unaligned");
        a.n = n, a.rows = rows, a.nh = nh, a.max_pages = max_pages;
        a.q = q, a.gate = gate, a.out = out;
        a.qt = q_token, a.qh = q_head, a.gt = gate_token, a.gh = gate_head, a.ot = out_token;
        a.cu = cu, a.kv_len = kv_len, a.table = table;
        a.scale = scale;
        a.err = dev_error_ptr();
        a.group = nh / c->nkv;
        a.cnt = (uint32_t *)ws;
        a.part = (float *)((uint8_t *)ws + 3 * KA_MAX_GRID * 4);
        const bool f32 = type == T_F32;
        const cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e = c->hd == 64 ? attn_go<64>(a, f32, max_new, s)
                            : c->hd == 128 ? attn_go<128>(a, f32, max_new, s)
                                           : attn_go<256>(a, f32, max_new, s);
        if (e != cudaSuccess) return fail(std::string("kv4 attn launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
