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
// Precision. fp32 rows: q (scaled per row by a power of two so that its largest value is 2^10..2^11) and p dv are split
// into two fp16 numbers, 22 bits together, in two of the 16 rows of a matrix instruction (rows g and g + 8 of the A
// operand), so the second half costs no instruction: an 8-row tile fills the 16. Their sums are fp32. bf16 rows: q is
// exact in fp16 after scaling, p dv is rounded once to 11 bits (the output has 8), and a tile holds 16 rows. The softmax
// runs in base 2 with one reference per row, the running maximum plus the running exponent of the largest dv, so p dv uses
// fp16's range whatever the size of V; the reference changes scale the sums exactly like a new maximum does.
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
constexpr int KA_MAX_GRID = 2048;             // CTAs the workspace has room for

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

template <int HD, bool HL> struct KaCfg {
    using T = std::conditional_t<HL, float, __nv_bfloat16>;
    static constexpr int NG = HD / KV4_GROUP, ROWS = HL ? 8 : 16;
    static constexpr uint32_t STAGE = KA_TOK * HD / 16 * 17;  // bytes of 64 tokens of one head
    static constexpr uint32_t QF = NG * 4 * 32 * 16;          // q as A operands: [group][step][lane] x 16 bytes
    static constexpr uint32_t OB = ROWS * HD * 4;
    // the merged sums share their place with q, which is rebuilt for the next row tile
    static constexpr uint32_t Q_OFF = 1024, ST_OFF = Q_OFF + (QF > OB ? QF : OB);
    static constexpr uint32_t SMEM_MAX = 111 * 1024;          // of two CTAs on an SM (113 KB each, less static memory)
    // stages, an even number: a slot then always belongs to the same pair of warps, whose waits see each of its phases
    static constexpr int S = (SMEM_MAX - ST_OFF) / STAGE > 16 ? 16 : (SMEM_MAX - ST_OFF) / STAGE / 2 * 2;
    static constexpr uint32_t SMEM = ST_OFF + S * STAGE;
    static constexpr int PART = ROWS * HD + 2 * ROWS;         // floats of a partial result
};
constexpr int KA_PART_MAX = 16 * 256 + 32;

template <int HD, bool HL> __global__ void __launch_bounds__(KA_THREADS, KA_CTAS) k_kv4_attn(const __grid_constant__ Kv4AttnArgs a) {
    using C = KaCfg<HD, HL>;
    using T = typename C::T;
    constexpr int NG = C::NG, ROWS = C::ROWS, S = C::S;
    extern __shared__ __align__(128) uint8_t sm_ka[];
    __shared__ long long red[KA_THREADS / 32], s_off;
    __shared__ int s_req;
    __shared__ volatile int s_fail;
    __shared__ float s_rs[16], s_qs[16][NG], s_ref[KA_CONS][16], s_l[KA_CONS][16], s_mref[16], s_ml[16];
    __shared__ int s_last;
    __shared__ uint32_t s_valid[S];
    uint64_t *full = (uint64_t *)sm_ka, *empty = full + S;
    uint4 *qf = (uint4 *)(sm_ka + C::Q_OFF);
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
    // column n of an 8-token product is token n ^ (n >> 2): with it both the K reads (8 bytes of 4 tokens x 4 lanes) and
    // the V reads (4 bytes of 4 tokens x 8 words) touch 32 different banks
    const int tk = g ^ (g >> 2);
    const int tv0 = (2 * t) ^ (t >> 1), tv1 = (2 * t + 1) ^ (t >> 1);  // columns 2t, 2t + 1: one aligned pair of tokens
    const bool swap = t >= 2;                                          // whose second is column 2t
    const int tp = tv0 & ~1;
    int it = 0;
    for (long long u = u0; u < u1;) {
        const int kend = (int)min((long long)rq.tiles, k + (u1 - u)), kv = item / rq.rt, tile = item - kv * rq.rt;
        const int nrow = min(ROWS, rq.fresh * a.group - tile * ROWS);
        // ---- q of the row tile into A operands
        ka_bar();
        {
            constexpr int L = 32 * KA_CONS / ROWS, PG = KV4_GROUP / L;  // lanes of a row; dims of a group each takes
            const int i = tid / L, sub = tid % L, flat = tile * ROWS + i, tok = flat / a.group;
            const T *src = (const T *)after_wait(a.q) + (int64_t)(rq.first + tok) * a.qt +
                           (int64_t)(kv * a.group + flat - tok * a.group) * a.qh;
            float x[NG][PG], mx = 0.0f;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                for (int j = 0; j < PG; ++j) {
                    x[gi][j] = i < nrow ? ka_f<T>(src[gi * KV4_GROUP + sub * PG + j]) : 0.0f;
                    mx = fmaxf(mx, fabsf(x[gi][j]));
                }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const int e = min(max(10 - ((int)(__float_as_uint(mx) >> 23) - 127), -90), 120);
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < PG; ++j) {
                    const int d = sub * PG + j, w = d >> 3, nib = d & 7, step = (w & 1) * 2 + ((nib & 3) >> 1);
                    const float f = x[gi][j] * up * (nib & 1 ? 0.0625f : 1.0f);
                    const __half hi = __float2half_rn(f), lo = __float2half_rn(f - __half2float(hi));
                    sum += (__half2float(hi) + (HL ? __half2float(lo) : 0.0f)) * (nib & 1 ? 16.0f : 1.0f);
                    __half *dst = (__half *)&qf[(gi * 4 + step) * 32 + (i & 7) * 4 + (w >> 1)];
                    // A registers: 0 = row g, 1 = row g + 8 (k low), 2, 3 the same (k high)
                    const int reg = (nib & 1) * 2;
                    if constexpr (HL) {
                        dst[reg * 2 + (nib >> 2)] = hi;
                        dst[(reg + 1) * 2 + (nib >> 2)] = lo;
                    } else {
                        dst[(reg + (i >> 3)) * 2 + (nib >> 2)] = hi;
                    }
                }
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (sub == 0) s_qs[i][gi] = sum * (-8.0f / 16777216.0f);
            }
            // scores in base 2: undo the scaling and the codes' 2^-24
            if (sub == 0) s_rs[i] = a.scale * 1.44269504f * __uint_as_float((uint32_t)(24 - e + 127) << 23);
        }
        ka_bar();
        // rows see tokens below lim; rows past the tile's last see what the last sees (their results are dropped)
        auto limit = [&](int i) {
            const int f = tile * ROWS + min(i, nrow - 1);
            return min(max(rq.len - rq.fresh + f / a.group + 1, 0), rq.len);
        };
        const int lim0 = limit(g), lim1 = HL ? lim0 : limit(g + 8), lo_lim = limit(0), hi_lim = limit(ROWS - 1);
        const float rs0 = s_rs[g], rs1 = HL ? rs0 : s_rs[(g + 8) & (ROWS - 1)];
        float qs0[NG], qs1[NG];
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) qs0[gi] = s_qs[g][gi], qs1[gi] = HL ? 0.0f : s_qs[(g + 8) & (ROWS - 1)][gi];
        float o[NG][8][4], corr0[NG], corr1[NG], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float ref0 = -INFINITY, ref1 = -INFINITY;
        int ev = -40;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
            corr0[gi] = corr1[gi] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[gi][i][0] = o[gi][i][1] = o[gi][i][2] = o[gi][i][3] = 0.0f;
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
            // ---- scores: sc[n-tile][row g: columns 2t, 2t + 1 | row g + 8]
            float sc[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                uint4 A[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) A[x] = qf[(gi * 4 + x) * 32 + lane];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) {
                    const uint8_t *rc = rec[nt >> 1];
                    const int line = gi * a.l.bs + pl[nt >> 1] + (nt & 1) * 8;
                    const uint2 w = *(const uint2 *)(rc + (line + tk) * 32 + t * 8);
                    float acc[4] = {qs0[gi], qs0[gi], qs1[gi], qs1[gi]};
                    ka_mma(acc, A[0], w.x & 0x000f000fu, w.x & 0x00f000f0u);
                    ka_mma(acc, A[1], (w.x >> 8) & 0x000f000fu, (w.x >> 8) & 0x00f000f0u);
                    ka_mma(acc, A[2], w.y & 0x000f000fu, w.y & 0x00f000f0u);
                    ka_mma(acc, A[3], (w.y >> 8) & 0x000f000fu, (w.y >> 8) & 0x00f000f0u);
                    uint32_t dw = *(const uint32_t *)(rc + 2 * a.l.kb + (line + tp) * 2);
                    if (swap) dw = __byte_perm(dw, 0, 0x1032);
                    const float2 d = ka_unpack(dw);
                    if constexpr (HL) {
                        sc[nt][0] += (acc[0] + acc[2]) * d.x;
                        sc[nt][1] += (acc[1] + acc[3]) * d.y;
                    } else {
                        sc[nt][0] += acc[0] * d.x;
                        sc[nt][1] += acc[1] * d.y;
                        sc[nt][2] += acc[2] * d.x;
                        sc[nt][3] += acc[3] * d.y;
                    }
                }
            }
            // ---- V scales of this lane's tokens, and the largest exponent among the warp's
            uint32_t dv[4][NG];
            __half2 dmax = __float2half2_rn(0.0f);
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const int b = t0 + nt * 8;
                uint32_t keep = 0xffffffffu;
                if (masked) {
                    const bool there = valid >> ((half * 32 + nt * 8) / a.l.bs) & 1u;
                    keep = (there && b + tv0 < hi_lim ? 0xffffu : 0u) | (there && b + tv1 < hi_lim ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    uint32_t w = *(const uint32_t *)(rec[nt >> 1] + 2 * a.l.kb + a.l.sb + (gi * a.l.bs + pl[nt >> 1] + (nt & 1) * 8 + tp) * 2);
                    if (swap) w = __byte_perm(w, 0, 0x1032);
                    w &= keep;
                    dv[nt][gi] = w;
                    dmax = __hmax2(dmax, __habs2(*(const __half2 *)&w));
                }
            }
            float dm = fmaxf(__low2float(dmax), __high2float(dmax));
            dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, 1));
            dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, 2));
            ev = max(ev, (int)(__float_as_uint(dm) >> 23) - 127);
            // ---- running softmax in base 2
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                sc[nt][0] *= rs0;
                sc[nt][1] *= rs0;
                if constexpr (!HL) {
                    sc[nt][2] *= rs1;
                    sc[nt][3] *= rs1;
                }
                if (masked) {
                    const int b = t0 + nt * 8;
                    const bool there = valid >> ((half * 32 + nt * 8) / a.l.bs) & 1u;
                    if (!there || b + tv0 >= lim0) sc[nt][0] = -INFINITY;
                    if (!there || b + tv1 >= lim0) sc[nt][1] = -INFINITY;
                    if constexpr (!HL) {
                        if (!there || b + tv0 >= lim1) sc[nt][2] = -INFINITY;
                        if (!there || b + tv1 >= lim1) sc[nt][3] = -INFINITY;
                    }
                }
                m0 = fmaxf(m0, fmaxf(sc[nt][0], sc[nt][1]));
                if constexpr (!HL) m1 = fmaxf(m1, fmaxf(sc[nt][2], sc[nt][3]));
            }
            m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
            m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
            if constexpr (!HL) {
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
            }
            const float n0 = m0 + (float)(ev - 11), n1 = m1 + (float)(ev - 11);
            const bool moved = n0 != ref0 || (!HL && n1 != ref1);
            const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;
            if (__any_sync(0xffffffffu, moved)) {
                const float f0 = ka_exp2(ref0 - z0), f1 = HL ? f0 : ka_exp2(ref1 - z1);
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    corr0[gi] *= f0;
                    corr1[gi] *= f1;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[gi][i][0] *= f0;
                        o[gi][i][1] *= f0;
                        o[gi][i][2] *= f1;
                        o[gi][i][3] *= f1;
                    }
                }
                ref0 = n0;
                ref1 = n1;
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                sc[nt][0] = ka_exp2(sc[nt][0] - z0);
                sc[nt][1] = ka_exp2(sc[nt][1] - z0);
                l0 += sc[nt][0] + sc[nt][1];
                if constexpr (!HL) {
                    sc[nt][2] = ka_exp2(sc[nt][2] - z1);
                    sc[nt][3] = ka_exp2(sc[nt][3] - z1);
                    l1 += sc[nt][2] + sc[nt][3];
                }
            }
            // ---- out += (p dv) c, 16 tokens at a time
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    const float2 da = ka_unpack(dv[2 * b][gi]), db = ka_unpack(dv[2 * b + 1][gi]);
                    const float(&sa)[4] = sc[2 * b], (&sb)[4] = sc[2 * b + 1];
                    // a token that a row does not see weighs nothing whatever its scale is (NaN)
                    auto weigh = [&](float p, float d) { return masked && p == 0.0f ? 0.0f : p * d; };
                    const float x0 = weigh(sa[0], da.x), x1 = weigh(sa[1], da.y), x2 = weigh(sb[0], db.x), x3 = weigh(sb[1], db.y);
                    uint4 A;
                    A.x = ka_pack(x0, x1);
                    A.z = ka_pack(x2, x3);
                    corr0[gi] += (x0 + x1) + (x2 + x3);
                    if constexpr (HL) {
                        const float2 h0 = ka_unpack(A.x), h1 = ka_unpack(A.z);
                        A.y = ka_pack(x0 - h0.x, x1 - h0.y);
                        A.w = ka_pack(x2 - h1.x, x3 - h1.y);
                    } else {
                        const float y0 = weigh(sa[2], da.x), y1 = weigh(sa[3], da.y), y2 = weigh(sb[2], db.x), y3 = weigh(sb[3], db.y);
                        A.y = ka_pack(y0, y1);
                        A.w = ka_pack(y2, y3);
                        corr1[gi] += (y0 + y1) + (y2 + y3);
                    }
                    const uint8_t *vc = rec[b] + a.l.kb + (gi * a.l.bs + pl[b]) * 32 + g * 4;
                    const uint32_t w0 = *(const uint32_t *)(vc + tv0 * 32), w1 = *(const uint32_t *)(vc + tv1 * 32);
                    const uint32_t w2 = *(const uint32_t *)(vc + (8 + tv0) * 32), w3 = *(const uint32_t *)(vc + (8 + tv1) * 32);
#pragma unroll
                    for (int by = 0; by < 4; ++by) {
                        const uint32_t sel = (uint32_t)(by | by << 4 | (4 + by) << 8 | (4 + by) << 12);
                        const uint32_t x = __byte_perm(w0, w1, sel), y = __byte_perm(w2, w3, sel);
                        ka_mma(o[gi][2 * by], A, x & 0x000f000fu, y & 0x000f000fu);
                        ka_mma(o[gi][2 * by + 1], A, x & 0x00f000f0u, y & 0x00f000f0u);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ka_arrive(&empty[sl]);
        }
        // ---- merge the four warps: one reference per row, sums added quarter by quarter in a fixed order
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            l1 += __shfl_xor_sync(0xffffffffu, l1, x);
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                corr0[gi] += __shfl_xor_sync(0xffffffffu, corr0[gi], x);
                corr1[gi] += __shfl_xor_sync(0xffffffffu, corr1[gi], x);
            }
        }
        if (t == 0) {
            s_ref[warp][g] = ref0;
            s_l[warp][g] = l0;
            if constexpr (!HL) {
                s_ref[warp][g + 8] = ref1;
                s_l[warp][g + 8] = l1;
            }
        }
        if (ka_bar_or(!alive)) return;  // a wait gave up: all warps leave here together
        auto top = [&](int i) { return fmaxf(fmaxf(s_ref[0][i], s_ref[1][i]), fmaxf(s_ref[2][i], s_ref[3][i])); };
        const float t0 = top(g), t1 = HL ? t0 : top(g + 8);
        // a warp without a key has nothing; a row whose scores are all NaN keeps them through the reference 0
        const float f0 = ka_exp2((ref0 == -INFINITY ? (t0 == -INFINITY ? 0.0f : -INFINITY) : ref0 - t0));
        const float f1 = HL ? f0 : ka_exp2((ref1 == -INFINITY ? (t1 == -INFINITY ? 0.0f : -INFINITY) : ref1 - t1));
        if (tid < ROWS) {
            const float tt = top(tid);
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < KA_CONS; ++w)
                l += s_l[w][tid] * ka_exp2(s_ref[w][tid] == -INFINITY ? (tt == -INFINITY ? 0.0f : -INFINITY) : s_ref[w][tid] - tt);
            s_mref[tid] = tt;
            s_ml[tid] = l;
        }
        for (int round = 0; round < 4; ++round) {
#pragma unroll
            for (int qd = 0; qd < 4; ++qd) {
                if (((warp + round) & 3) != qd) continue;
#pragma unroll
                for (int x = qd * NG * 2; x < (qd + 1) * NG * 2; ++x) {  // 8 NG products of 8 columns, a quarter of them
                    const int gi = x >> 3, i = x & 7;
                    const float up = i & 1 ? 1048576.0f : 16777216.0f;
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        const int d = gi * KV4_GROUP + 8 * (2 * t + cc) + i;
                        const float v0 = ((HL ? o[gi][i][cc] + o[gi][i][2 + cc] : o[gi][i][cc]) * up - 8.0f * corr0[gi]) * f0;
                        float *p = ob + g * HD + d;
                        *p = round ? *p + v0 : v0;
                        if constexpr (!HL) {
                            const float v1 = (o[gi][i][2 + cc] * up - 8.0f * corr1[gi]) * f1;
                            p += 8 * HD;
                            *p = round ? *p + v1 : v1;
                        }
                    }
                }
            }
            ka_bar();
        }
        // the row tile's output, from sums and weights of any place
        auto emit = [&](auto sums, auto weight) {
            for (int e = tid; e < nrow * HD; e += 32 * KA_CONS) {
                const int i = e / HD, d = e - i * HD, f = tile * ROWS + i, tok = f / a.group, h = kv * a.group + f - tok * a.group;
                const int64_t row = rq.first + tok;
                float y = 0.0f;
                if (limit(i) > 0) {
                    y = sums(i, d) / weight(i);
                    if (a.gate) y *= sigm(ka_f<T>(((const T *)after_wait(a.gate))[row * a.gt + h * a.gh + d]));
                }
                ((T *)a.out)[row * a.ot + (int64_t)h * HD + d] = (T)y;
            }
        };
        if (k == 0 && kend == rq.tiles) {
            emit([&](int i, int d) { return ob[i * HD + d]; }, [&](int i) { return s_ml[i]; });
        } else {
            // ---- a part of a row tile: into the workspace; the last CTA of 16 joins them, the last of those the rest
            const long long first = u - k;  // the row tile's first unit (of this run's numbering)
            const int c0 = (int)(first / per), c1 = (int)((first + rq.tiles - 1) / per), c = blockIdx.x;
            auto slot = [&](int cta) {  // a CTA's part lies at its run's start (0) or after it (1)
                return a.part + ((size_t)cta * 2 + (cta == c0 && first != c0 * per)) * KA_PART_MAX;
            };
            float *my = slot(c);
            for (int e = tid * 4; e < ROWS * HD; e += 32 * KA_CONS * 4) __stcg((float4 *)(my + e), *(const float4 *)(ob + e));
            if (tid < ROWS) {
                __stcg(my + ROWS * HD + tid, s_mref[tid]);
                __stcg(my + ROWS * HD + ROWS + tid, s_ml[tid]);
            }
            // joins `count` parts at CTAs b, b + step, ..; into ob / s_mref / s_ml
            auto join = [&](int b, int step, int count) {
                if (tid < ROWS) {
                    float m = -INFINITY, l = 0.0f;
                    for (int x = 0; x < count; ++x) m = fmaxf(m, __ldcg(slot(b + x * step) + ROWS * HD + tid));
                    for (int x = 0; x < count; ++x) {
                        const float *p = slot(b + x * step) + ROWS * HD;
                        const float rf = __ldcg(p + tid);
                        l += __ldcg(p + ROWS + tid) * ka_exp2(rf == -INFINITY ? (m == -INFINITY ? 0.0f : -INFINITY) : rf - m);
                    }
                    s_mref[tid] = m;
                    s_ml[tid] = l;
                }
                ka_bar();
                for (int e = tid * 4; e < ROWS * HD; e += 32 * KA_CONS * 4) {
                    const float m = s_mref[e / HD];
                    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int x = 0; x < count; ++x) {
                        const float *p = slot(b + x * step);
                        const float rf = __ldcg(p + ROWS * HD + e / HD);
                        const float f = ka_exp2(rf == -INFINITY ? (m == -INFINITY ? 0.0f : -INFINITY) : rf - m);
                        const float4 v = __ldcg((const float4 *)(p + e));
                        y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
                    }
                    *(float4 *)(ob + e) = y;
                }
                ka_bar();
            };
            // true for the last of `count` arrivals (all of this CTA's stores before it are visible to that one)
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
            if (mineis) {
                join(gb, 1, gn);
                if (parts > KA_FAN) {
                    float *to = slot(gb);
                    for (int e = tid * 4; e < ROWS * HD; e += 32 * KA_CONS * 4) __stcg((float4 *)(to + e), *(const float4 *)(ob + e));
                    if (tid < ROWS) {
                        __stcg(to + ROWS * HD + tid, s_mref[tid]);
                        __stcg(to + ROWS * HD + ROWS + tid, s_ml[tid]);
                    }
                    const int groups = (parts + KA_FAN - 1) / KA_FAN;
                    mineis = last_of(a.cnt + 2 * KA_MAX_GRID + c0, groups);
                    if (mineis) join(c0, KA_FAN, groups);
                }
            }
            if (mineis) emit([&](int i, int d) { return ob[i * HD + d]; }, [&](int i) { return s_ml[i]; });
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

template <int HD, bool HL> static cudaError_t attn_go(const Kv4AttnArgs &a, int grid, cudaStream_t s) {
    const cudaError_t e = allow_max_dynamic_smem(k_kv4_attn<HD, HL>);
    if (e != cudaSuccess) return e;
    return launch_k(k_kv4_attn<HD, HL>, dim3(grid), dim3(KA_THREADS), KaCfg<HD, HL>::SMEM, s, a);
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
        // no more CTAs than there can be pairs of units
        const long long tiles = ((long long)max_pages * c->page_size + KA_TOK - 1) / KA_TOK;
        const long long rt = ((long long)std::min(max_new, rows) * a.group + (f32 ? 7 : 15)) / (f32 ? 8 : 16);
        const long long most = std::max(1ll, (long long)n * c->nkv * rt * tiles / 2);
        const int grid = (int)std::min(most, (long long)std::min(num_sms() * KA_CTAS, KA_MAX_GRID));
        cudaError_t e;
        const cudaStream_t s = (cudaStream_t)stream;
        if (c->hd == 64) e = f32 ? attn_go<64, true>(a, grid, s) : attn_go<64, false>(a, grid, s);
        else if (c->hd == 128) e = f32 ? attn_go<128, true>(a, grid, s) : attn_go<128, false>(a, grid, s);
        else e = f32 ? attn_go<256, true>(a, grid, s) : attn_go<256, false>(a, grid, s);
        if (e != cudaSuccess) return fail(std::string("kv4 attn launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
