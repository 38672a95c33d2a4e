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
// bits below its nominal size; so both first halves are whole numbers up to 2^11 (q scaled per row by a power of two, p dv
// by one per row and block): all their products and sums are multiples of one unit, and exact. Floating halves lost 2.5e-6
// of the output where this form loses 3e-7. Sums over more than 32 tokens are added in fp32 outside the tensor core, whose
// own accumulation cuts instead of rounding (bf16 rows: where a CTA may have many tokens of a row, KA_LONG). The softmax runs in
// base 2 with the running maximum of a row's scores as its reference; p dv is scaled by the exponent of the largest |dv| that the row has
// seen in the same 64 dims, so that it uses fp16's range whatever the size of V is, there, in other blocks, and in tokens that the row
// does not see. (That scale, looked at for every 32 tokens, costs 2 to 5 % of the time beside one scale for the whole row tile; fp32
// rows' weights beside the largest of their own 32 tokens, and the sum of the rounded ones, another 1.5 %: errors against 64 bits 5.8e-7 ->
// 3.8e-7 at 77 tokens, 1.7e-6 -> 5.2e-7 at 100 thousand.)
//
// Work. A unit is 64 tokens of one kv head for one row tile (8 or 16 rows: the heads of a group, token after token). All
// units of the call in a row are cut into equal runs, one per CTA, whatever request they belong to: each CTA finds its run
// from the lengths by a prefix sum, so nothing about the lengths is known on the host and a captured call serves any.
// A row tile whose units lie in several CTAs leaves a partial result in each; a second small kernel joins them in the order
// of the CTAs, so the result does not depend on timing (joining in the CTA that finishes last cost 20 us of latency chains
// for 147 parts, where the second kernel takes 6 to 8).
//
// What bounds it, and measured (device time): one request of 131071 tokens, bf16, 16 heads over 2 kv heads of 256 (71 MB) 29.3 us,
// of which some 16 us in the page loop (4.4 TB/s); 32 requests of 65 to 4096 tokens, fp32 26.0 us; 64 requests of 100 to 8192 tokens,
// bf16, 32 heads over 8 of 128 (298 MB) 79.5 us (3.7 TB/s, issue of the page loop); one request of 77 tokens 9.0 us, a chain of round
// trips to memory.
//
// A CTA: one warp copies pages into a ring (one bulk copy per page and head: codes and scales of K and V), four warps
// compute, two on each 64-token stage, 32 tokens each, with their own running softmax; they merge at the end of a run.
#include "fn_kv4_attn.cuh"

namespace fn {

constexpr int KA_CONS = 4;                    // computing warps
// 64-token tiles that a CTA may have of one row from which bf16 rows take the LONG form. The tensor core's accumulation cuts: t tiles lose
// up to t 2^-24 of the sum of |c p dv|, which may be twice the output and more; 2^21 tokens (32768 tiles) lost 0.6 % of it on average, so
// 512 lose 1e-4, beside 2e-3 of the output's own rounding. The LONG form costs 3 to 4 % of the time.
constexpr int KA_LONG = 512;
// registers of the wide form: 256 threads x 128 at launch; the copying warpgroup gives up what the computing one takes
// (40 + 216 = 2 x 128)
constexpr int KA_REG_COPY = 40, KA_REG_COMP = 216;

__device__ __forceinline__ void ka_mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of halves, row g columns 2t, 2t + 1 in lane 4 g + t, turned
__device__ __forceinline__ uint32_t ka_turn(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
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
template <int HD, bool HL, int NT> struct KaCfg {
    using T = std::conditional_t<HL, float, __nv_bfloat16>;
    static constexpr int NG = HD / KV4_GROUP, ROWS = 8 * NT;
    // CTAs per SM: three of 4 + 1 warps with 128 registers, or two with 216 for the computing warps where the sums are many
    static constexpr bool WIDE = HD * NT >= 256;
    static constexpr int CTAS = WIDE ? 2 : 3, THREADS = WIDE ? 256 : 160;
    static constexpr int OS = HD + 1;                         // floats between rows of the merged sums (banks)
    static constexpr uint32_t STAGE = KA_TOK * HD / 16 * 17;  // bytes of 64 tokens of one head
    static constexpr uint32_t QF = NT * NG * 4 * 32 * (HL ? 16 : 8);  // q as B operands: [n-tile][group][step][lane]
    static constexpr uint32_t OB = (ROWS * OS * 4 + 127) / 128 * 128;
    // the merged sums share their place with q, which is rebuilt for the next row tile
    static constexpr uint32_t Q_OFF = 1024, ST_OFF = Q_OFF + (QF > OB ? QF : OB);
    static constexpr uint32_t SMEM_MAX = (WIDE ? 112 : 73) * 1024;  // 228 KB / CTAS, less static memory and 1 KB
    // stages, an even number: a slot then always belongs to the same pair of warps, whose waits see each of its phases
    static constexpr int S = (SMEM_MAX - ST_OFF) / STAGE > 16 ? 16 : (SMEM_MAX - ST_OFF) / STAGE / 2 * 2;
    static constexpr uint32_t SMEM = ST_OFF + S * STAGE;
};
constexpr int KA_PART_MAX = 16 * 256 + 32;

// LONG: bf16 rows' sums leave the tensor core after every 32 tokens, as fp32 rows' always do
template <int HD, bool HL, int NT, bool LONG> __global__ void __launch_bounds__(KaCfg<HD, HL, NT>::THREADS, KaCfg<HD, HL, NT>::CTAS)
    k_kv4_attn(const __grid_constant__ Kv4AttnArgs a) {
    using C = KaCfg<HD, HL, NT>;
    using T = typename C::T;
    constexpr int NG = C::NG, ROWS = C::ROWS, S = C::S, OS = C::OS, THREADS = C::THREADS;
    using QF = std::conditional_t<HL, uint4, uint2>;
    extern __shared__ __align__(128) uint8_t sm_ka[];
    __shared__ long long red[THREADS / 32], s_off;
    __shared__ int s_req;
    __shared__ KaReq s_rq;
    __shared__ volatile int s_fail;
    __shared__ __align__(8) float s_rs[ROWS], s_qs[2][NG][ROWS];
    __shared__ float s_ref[KA_CONS][ROWS], s_l[KA_CONS][ROWS], s_mref[ROWS], s_ml[ROWS];
    __shared__ uint32_t s_valid[S];
    uint64_t *full = (uint64_t *)sm_ka, *empty = full + S;
    uint8_t *s_up = sm_ka + 512;  // [warp][group][row]
    static_assert(2 * S * 8 <= 512 && KA_CONS * NG * ROWS <= 512);
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
    const int per_t = (a.n + THREADS - 1) / THREADS, r0 = min(tid * per_t, a.n), r1 = min(r0 + per_t, a.n);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) {
        const KaReq q = ka_req<ROWS>(a, r);
        mine += (long long)q.rt * a.l.nkv * (q.tiles + KA_EXTRA);
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
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += red[w];
        units += red[w];
    }
    const long long per = max((units + gridDim.x - 1) / gridDim.x, 2ll + KA_EXTRA);
    const long long u0 = blockIdx.x * per, u1 = min(u0 + per, units);
    if (u0 < u1 && u0 >= before && u0 < before + mine) {
        long long at = before;
        for (int r = r0; r < r1; ++r) {
            const KaReq q = ka_req<ROWS>(a, r);
            const long long w = (long long)q.rt * a.l.nkv * (q.tiles + KA_EXTRA);
            if (u0 < at + w) {
                s_req = r;
                s_rq = q;
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
        for (long long i = (long long)blockIdx.x * THREADS + tid; i < left; i += (long long)gridDim.x * THREADS) {
            const long long row = i / (a.nh * HD);
            ((T *)a.out)[(live + row) * a.ot + (i - row * a.nh * HD)] = (T)0.0f;
        }
    }
    if (tid == 0) a.split[blockIdx.x].parts = 0;
    __syncthreads();
    if (u0 >= u1) return;

    int r = s_req;
    KaReq rq = s_rq;
    // the run is at place `off` of a row tile's units: its own follow KA_EXTRA that only count
    int item = (int)(s_off / (rq.tiles + KA_EXTRA)), off = (int)(s_off - (long long)item * (rq.tiles + KA_EXTRA));
    long long u = u0;
    int k, kend;  // the tiles that the run has of the row tile (none: k = kend)
    auto here = [&]() {
        k = max(off - KA_EXTRA, 0);
        kend = max((int)min((long long)(rq.tiles + KA_EXTRA), off + (u1 - u)) - KA_EXTRA, 0);
    };
    // to the next row tile of the run, if there is one
    auto next = [&]() {
        u += rq.tiles + KA_EXTRA - off;
        off = 0;
        if (u >= u1 || ++item < rq.rt * a.l.nkv) return;
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
    const int ppt = KA_TOK >> a.l.lbs;  // pages of a stage

    if (warp >= KA_CONS) {
        if constexpr (C::WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KA_REG_COPY));
        if (warp > KA_CONS) return;
        // ---- copies: lane p fetches page p of a stage; a lane holds one entry of the next 32 pages' ids
        int it = 0;
        for (; u < u1; next()) {
            here();
            const int kv = item / rq.rt;
            const int pages = (rq.len + a.l.bs - 1) >> a.l.lbs;
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
        }
    drained:
        // a CTA must not leave with copies into its shared memory in flight: the computing warps may give up after this warp is done, so
        // it always stays until its last copies have landed
        if (lane == 0)
            for (int i = max(it - S, 0); i < it; ++i) mbar_park(&full[i % S], (uint32_t)(i / S) & 1u);
        return;
    }

    // ---- compute
    if constexpr (C::WIDE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KA_REG_COMP));
    const int g = lane >> 2, t = lane & 3, half = warp & 1, pair = warp >> 1;
    // index n of 8 tokens is token n ^ (n >> 2): with it both the K reads (8 bytes of 8 tokens x 4 lanes, 16 lanes at a
    // time) and the V reads (4 bytes of 4 tokens x 8 words) touch 32 different banks
    const int tk = g ^ (g >> 2);
    const int tv0 = (2 * t) ^ (t >> 1), tv1 = (2 * t + 1) ^ (t >> 1);
    int it = 0;
    for (; u < u1; next()) {
        here();
        if (k == kend) continue;
        const int kv = item / rq.rt, tile = item - kv * rq.rt;
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
                    s_qs[0][gi][i] = sum * (-8.0f / 16777216.0f);
                    if (HL) s_qs[1][gi][i] = sum_lo * (-8.0f / 16777216.0f);
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
        float o[NT][NG][4][4];
        float2 corr[NT][NG], m[NT], l[NT];
        // p dv is scaled by ug = 2^(10 - e) of the largest |dv| that the row has seen in a group, the same for all rows until the tiles that
        // some see a part of; from there on (own) each row's is in s_up, by its exponent. -24 is the least e of an fp16 number.
        float ug[NG];
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) ug[gi] = 17179869184.0f;
        bool own = false;
        auto inverse = [](float a) { return __uint_as_float(0x7f000000u - __float_as_uint(a)); };  // of a power of two
        auto row_up = [&](int n, int gi) {
            if (!own) return make_float2(ug[gi], ug[gi]);
            const uint8_t *e = s_up + (warp * NG + gi) * ROWS + 8 * n + 2 * t;
            return make_float2(__uint_as_float((uint32_t)e[0] << 23), __uint_as_float((uint32_t)e[1] << 23));
        };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            lim[n][0] = limit(8 * n + 2 * t);
            lim[n][1] = limit(8 * n + 2 * t + 1);
            m[n] = make_float2(-INFINITY, -INFINITY);
            l[n] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                corr[n][gi] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int by = 0; by < 4; ++by) o[n][gi][by][0] = o[n][gi][by][1] = o[n][gi][by][2] = o[n][gi][by][3] = 0.0f;
            }
        }
        // 32 tokens of a stage; M: some of them are hidden from some rows
        auto step = [&](auto mk, const uint8_t *st, int t0, uint32_t valid) {
            constexpr bool M = decltype(mk)::value;
            // the run's first 16 tokens, and how far its second 16 are
            const int at = half * 32, pg = at >> a.l.lbs, pl = at & (a.l.bs - 1);
            const uint8_t *rec = st + pg * a.l.rec;
            const uint32_t code2 = a.l.bs == 16 ? a.l.rec : 512, scale2 = a.l.bs == 16 ? a.l.rec : 32;
            const uint32_t cstep = a.l.bs * 32, sstep = a.l.bs * 2;  // to the next 64 dims
            const uint8_t *kp = rec + (pl + tk) * 32 + t * 8, *ks = rec + 2 * a.l.kb + (pl + tk) * 2;
            auto hidden = [&](int b, int h, int lm) {
                return !(valid >> ((at + b * 16 + h * 8 >> a.l.lbs)) & 1u) || t0 + b * 16 + h * 8 + tk >= lm;
            };
            // ---- scores of tokens tk, tk + 8 of both runs
            float2 sc[NT][2][2] = {};
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                QF B[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) B[n][x] = qf[((n * NG + gi) * 4 + x) * 32 + lane];
                uint4 A[2][4];
                float d[2][2], acc[NT][2][4];
                [[maybe_unused]] float low[NT][2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint8_t *c = kp + gi * cstep + b * code2, *s = ks + gi * sstep + b * scale2;
                    const uint2 w = *(const uint2 *)c, v = *(const uint2 *)(c + 256);
                    d[b][0] = ka_half(s), d[b][1] = ka_half(s + 16);
                    const uint32_t w8 = w.x >> 8, v8 = v.x >> 8, x8 = w.y >> 8, y8 = v.y >> 8;
                    A[b][0] = make_uint4(w.x & 0x000f000fu, v.x & 0x000f000fu, w.x & 0x00f000f0u, v.x & 0x00f000f0u);
                    A[b][1] = make_uint4(w8 & 0x000f000fu, v8 & 0x000f000fu, w8 & 0x00f000f0u, v8 & 0x00f000f0u);
                    A[b][2] = make_uint4(w.y & 0x000f000fu, v.y & 0x000f000fu, w.y & 0x00f000f0u, v.y & 0x00f000f0u);
                    A[b][3] = make_uint4(x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 i0 = *(const float2 *)&s_qs[0][gi][8 * n + 2 * t];
                        acc[n][b][0] = acc[n][b][2] = i0.x, acc[n][b][1] = acc[n][b][3] = i0.y;
                        if constexpr (HL) {
                            const float2 i1 = *(const float2 *)&s_qs[1][gi][8 * n + 2 * t];
                            low[n][b][0] = low[n][b][2] = i1.x, low[n][b][1] = low[n][b][3] = i1.y;
                        }
                    }
                }
                // the sums of both runs (and halves) side by side: an instruction does not wait for the one before it
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            ka_mma(acc[n][b], A[b][x], B[n][x].x, B[n][x].y);
                            if constexpr (HL) ka_mma(low[n][b], A[b][x], B[n][x].z, B[n][x].w);
                        }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float2 s = make_float2(acc[n][b][2 * h], acc[n][b][2 * h + 1]);
                            if constexpr (HL) s = __fadd2_rn(s, make_float2(low[n][b][2 * h], low[n][b][2 * h + 1]));
                            sc[n][b][h] = __ffma2_rn(s, make_float2(d[b][h], d[b][h]), sc[n][b][h]);
                        }
            }
            // ---- V scales of this lane's tokens
            float dv[2][2][NG];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) dv[b][h][gi] = ka_half(ks + a.l.sb + gi * sstep + b * scale2 + h * 16);
            // the largest of a group that a row below `lm` sees (what it does not see counts for nothing, whatever is there)
            auto largest = [&](int gi, int lm) {
                float d = 0.0f;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (!M || !hidden(b, h, lm)) d = fmaxf(d, fabsf(dv[b][h][gi]));
                return d;
            };
            // ---- running softmax in base 2: p = exp2(s - maximum), |p dv up| < 2^11. fp32 rows: the maximum of these 32 tokens, so that
            // their weights have all of their bits beside one another, whatever came before; the sums of the 32 come to the running
            // maximum's unit as they are added (100k tokens: 1.7e-6 off 64 bits otherwise)
            float2 mx[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 rs = *(const float2 *)&s_rs[8 * n + 2 * t];
                mx[n] = HL ? make_float2(-INFINITY, -INFINITY) : m[n];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2 s = __fmul2_rn(sc[n][b][h], rs);
                        if constexpr (M) {
                            if (hidden(b, h, lim[n][0])) s.x = -INFINITY;
                            if (hidden(b, h, lim[n][1])) s.y = -INFINITY;
                        }
                        sc[n][b][h] = s;
                        mx[n].x = fmaxf(mx[n].x, s.x);
                        mx[n].y = fmaxf(mx[n].y, s.y);
                    }
            }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mx[n].x = fmaxf(mx[n].x, __shfl_xor_sync(0xffffffffu, mx[n].x, x));
                    mx[n].y = fmaxf(mx[n].y, __shfl_xor_sync(0xffffffffu, mx[n].y, x));
                }
            }
            [[maybe_unused]] float2 up[M ? NT : 1][M ? NG : 1];
            if constexpr (M) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) up[n][gi] = row_up(n, gi);
            }
            bool moved = false, grown = false;
            float2 z[NT];  // minus the maximum (0 for a row that has seen nothing)
            [[maybe_unused]] float2 unit[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if constexpr (HL) {
                    const float2 here = mx[n];
                    mx[n] = make_float2(fmaxf(m[n].x, here.x), fmaxf(m[n].y, here.y));
                    unit[n] = make_float2(here.x == -INFINITY ? 0.0f : ka_exp2(here.x - mx[n].x), here.y == -INFINITY ? 0.0f : ka_exp2(here.y - mx[n].y));
                    z[n] = make_float2(here.x == -INFINITY ? 0.0f : -here.x, here.y == -INFINITY ? 0.0f : -here.y);
                }
                moved |= mx[n].x != m[n].x || mx[n].y != m[n].y;
                if constexpr (!HL) z[n] = make_float2(mx[n].x == -INFINITY ? 0.0f : -mx[n].x, mx[n].y == -INFINITY ? 0.0f : -mx[n].y);
            }
            if constexpr (M) {
#pragma unroll
                for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                    for (int n = 0; n < NT; ++n) grown |= largest(gi, hi_lim) * fmaxf(up[n][gi].x, up[n][gi].y) >= 2048.0f;
            } else {
                float d = 0.0f;
#pragma unroll
                for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            dv[b][h][gi] *= ug[gi];
                            d = fmaxf(d, fabsf(dv[b][h][gi]));
                        }
                grown = d >= 2048.0f;
            }
            // (what is rare is short too: the code of a step that runs once is fetched for it, and a part has some seven steps a warp)
            if (__any_sync(0xffffffffu, moved | grown)) {
                float2 f[NT][NG];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 fm = make_float2(m[n].x == -INFINITY ? 0.0f : ka_exp2(m[n].x - mx[n].x), m[n].y == -INFINITY ? 0.0f : ka_exp2(m[n].y - mx[n].y));
                    l[n] = __fmul2_rn(l[n], fm);
                    m[n] = mx[n];
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) f[n][gi] = fm;
                }
                if (__any_sync(0xffffffffu, grown)) {
                    // u where d fits it, else the power that d asks for
                    auto scaled = [](float u, float d) { return d * u < 2048.0f ? u : __uint_as_float(264u - (__float_as_uint(d) >> 23) << 23); };
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) {
                        if constexpr (M) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                auto over = [&](float d) {  // of the warp's tokens
#pragma unroll
                                    for (int x = 4; x < 32; x <<= 1) d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, x));
                                    return fminf(d, 65504.0f);
                                };
                                const float2 u = make_float2(scaled(up[n][gi].x, over(largest(gi, lim[n][0]))), scaled(up[n][gi].y, over(largest(gi, lim[n][1]))));
                                f[n][gi] = __fmul2_rn(f[n][gi], make_float2(u.x * inverse(up[n][gi].x), u.y * inverse(up[n][gi].y)));
                                up[n][gi] = u;
                                uint8_t *e = s_up + (warp * NG + gi) * ROWS + 8 * n + 2 * t;
                                e[0] = (uint8_t)(__float_as_uint(u.x) >> 23), e[1] = (uint8_t)(__float_as_uint(u.y) >> 23);
                            }
                            ug[gi] = up[NT - 1][gi].y;  // (all rows' where whole pages are missing, and whole tiles come after it)
                        } else {  // the same tokens, and factors, in all rows
                            const float d = fminf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest(gi, 0)))), 65504.0f * ug[gi]);
                            const float r = scaled(1.0f, d);
#pragma unroll
                            for (int n = 0; n < NT; ++n) f[n][gi] = __fmul2_rn(f[n][gi], make_float2(r, r));
                            ug[gi] *= r;
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int h = 0; h < 2; ++h) dv[b][h][gi] *= r;
                        }
                    }
                    own = M;
                    __syncwarp();
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi) {
                        corr[n][gi] = __fmul2_rn(corr[n][gi], f[n][gi]);
#pragma unroll
                        for (int by = 0; by < 4; ++by)
#pragma unroll
                            for (int x = 0; x < 4; x += 2) {
                                const float2 y = __fmul2_rn(make_float2(o[n][gi][by][x], o[n][gi][by][x + 1]), f[n][gi]);
                                o[n][gi][by][x] = y.x, o[n][gi][by][x + 1] = y.y;
                            }
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = __fadd2_rn(sc[n][b][h], z[n]);
                        sc[n][b][h] = make_float2(ka_exp2(x.x), ka_exp2(x.y));
                    }
                const float2 sum = __fadd2_rn(__fadd2_rn(sc[n][0][0], sc[n][0][1]), __fadd2_rn(sc[n][1][0], sc[n][1][1]));
                l[n] = HL ? __ffma2_rn(sum, unit[n], l[n]) : __fadd2_rn(l[n], sum);
            }
            if constexpr (M) {
                // (below, what weighs nothing counts for nothing, hidden NaN scales among it; a NaN that a row sees counts)
                bool odd = false;
#pragma unroll
                for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) odd |= !(fabsf(dv[b][h][gi]) < INFINITY) && !hidden(b, h, hi_lim);
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    const float none = dv[b][h][gi] * 0.0f;
                                    if (!hidden(b, h, lim[n][0])) corr[n][gi].x += none;
                                    if (!hidden(b, h, lim[n][1])) corr[n][gi].y += none;
                                }
                }
            }
            // ---- out += c (p dv)
            const uint8_t *vp0 = rec + a.l.kb + (pl + tv0) * 32 + g * 4, *vp1 = vp0 + (tv1 - tv0) * 32;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                uint32_t P[NT][2][2];  // B operands: tokens 2t, 2t + 1 (+ 8) of row g
                [[maybe_unused]] uint32_t Q[NT][2][2];  // their second halves
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float2 add[2][2];
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float d = dv[b][h][gi];
                            float2 x = make_float2(d, d);
                            if constexpr (M) x = __fmul2_rn(x, up[n][gi]);
                            x = __fmul2_rn(sc[n][b][h], x);
                            // a token that a row does not see weighs nothing whatever its scale is (NaN)
                            if constexpr (M) x = make_float2(sc[n][b][h].x == 0.0f ? 0.0f : x.x, sc[n][b][h].y == 0.0f ? 0.0f : x.y);
                            // (the sum is of the rounded weights, so that the 8 of a code cancels and their rounding counts c - 8 times, not c)
                            if constexpr (HL) {
                                const float2 big = make_float2(12582912.0f, 12582912.0f);  // 1.5 2^23: rounds to whole numbers
                                const float2 w = __fadd2_rn(__fadd2_rn(x, big), make_float2(-12582912.0f, -12582912.0f));
                                const float2 r = __ffma2_rn(w, make_float2(-1.0f, -1.0f), x);
                                const uint32_t rest = ka_pack(r.x, r.y);
                                P[n][b][h] = ka_turn(ka_pack(w.x, w.y));
                                Q[n][b][h] = ka_turn(rest);
                                add[b][h] = __fadd2_rn(w, ka_unpack(rest));
                            } else {
                                const uint32_t w = ka_pack(x.x, x.y);
                                add[b][h] = ka_unpack(w);
                                P[n][b][h] = ka_turn(w);
                            }
                        }
                    const float2 sum = __fadd2_rn(__fadd2_rn(add[0][0], add[0][1]), __fadd2_rn(add[1][0], add[1][1]));
                    corr[n][gi] = HL ? __ffma2_rn(sum, unit[n], corr[n][gi]) : __fadd2_rn(corr[n][gi], sum);
                }
                uint4 A[4][2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint8_t *c0 = vp0 + gi * cstep + b * code2, *c1 = vp1 + gi * cstep + b * code2;
                    const uint32_t w0 = *(const uint32_t *)c0, w1 = *(const uint32_t *)c1;
                    const uint32_t w2 = *(const uint32_t *)(c0 + 256), w3 = *(const uint32_t *)(c1 + 256);
#pragma unroll
                    for (int by = 0; by < 4; ++by) {
                        const uint32_t sel = (uint32_t)(by | by << 4 | (4 + by) << 8 | (4 + by) << 12);
                        const uint32_t x = __byte_perm(w0, w1, sel), y = __byte_perm(w2, w3, sel);
                        A[by][b] = make_uint4(x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (HL || LONG) {
                        float acc[4][4] = {};
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int by = 0; by < 4; ++by) ka_mma(acc[by], A[by][b], P[n][b][0], P[n][b][1]);
                        if constexpr (HL) {
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int by = 0; by < 4; ++by) ka_mma(acc[by], A[by][b], Q[n][b][0], Q[n][b][1]);
                        }
#pragma unroll
                        for (int by = 0; by < 4; ++by)
#pragma unroll
                            for (int x = 0; x < 4; x += 2) {
                                const float2 a2 = make_float2(acc[by][x], acc[by][x + 1]), o2 = make_float2(o[n][gi][by][x], o[n][gi][by][x + 1]);
                                const float2 y = HL ? __ffma2_rn(a2, unit[n], o2) : __fadd2_rn(o2, a2);
                                o[n][gi][by][x] = y.x, o[n][gi][by][x + 1] = y.y;
                            }
                    } else {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int by = 0; by < 4; ++by) ka_mma(o[n][gi][by], A[by][b], P[n][b][0], P[n][b][1]);
                    }
                }
            }
        };
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
            if (t0 + 32 > lo_lim || valid != (1u << ppt) - 1u) step(std::true_type{}, st, t0, valid);
            else step(std::false_type{}, st, t0, valid);
            __syncwarp();
            if (lane == 0) ka_arrive(&empty[sl]);
        }

        // ---- merge the four warps: one reference per row, sums added quarter by quarter in a fixed order
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                l[n].x += __shfl_xor_sync(0xffffffffu, l[n].x, x);
                l[n].y += __shfl_xor_sync(0xffffffffu, l[n].y, x);
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) {
                    corr[n][gi].x += __shfl_xor_sync(0xffffffffu, corr[n][gi].x, x);
                    corr[n][gi].y += __shfl_xor_sync(0xffffffffu, corr[n][gi].y, x);
                }
            }
        if (g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s_ref[warp][8 * n + 2 * t] = m[n].x, s_ref[warp][8 * n + 2 * t + 1] = m[n].y;
                s_l[warp][8 * n + 2 * t] = l[n].x, s_l[warp][8 * n + 2 * t + 1] = l[n].y;
            }
        }
        if (ka_bar_or(!alive)) return;  // a wait gave up: all warps leave here together
        auto top = [&](int i) { return fmaxf(fmaxf(s_ref[0][i], s_ref[1][i]), fmaxf(s_ref[2][i], s_ref[3][i])); };
        float2 wf[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
            wf[n] = make_float2(ka_weight(m[n].x, top(8 * n + 2 * t)), ka_weight(m[n].y, top(8 * n + 2 * t + 1)));
        // with the sums' own scales (2^-24 and 2^-20 of the codes are taken back below)
        float2 back[NT][NG];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
                const float2 u = row_up(n, gi);
                back[n][gi] = make_float2(wf[n].x * inverse(u.x), wf[n].y * inverse(u.y));
            }
        if (tid < ROWS) {
            const float tt = top(tid);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < KA_CONS; ++w) sum += s_l[w][tid] * ka_weight(s_ref[w][tid], tt);
            s_mref[tid] = tt;
            s_ml[tid] = sum;
        }
        // (the quarter is a constant in each branch: as a variable index it would put the sums into local memory)
        auto quarter = [&](auto q, int round) {
            constexpr int by = decltype(q)::value;
            float old[NT][NG][4];  // read together, then written together
            auto at = [&](int n, int gi, int x) { return ob + (8 * n + 2 * t + (x & 1)) * OS + gi * KV4_GROUP + 8 * g + 2 * by + (x >> 1); };
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                    for (int x = 0; x < 4; ++x) old[n][gi][x] = round ? *at(n, gi, x) : 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        *at(n, gi, x) = old[n][gi][x] + (o[n][gi][by][x] * (x >= 2 ? 1048576.0f : 16777216.0f) - 8.0f * (x & 1 ? corr[n][gi].y : corr[n][gi].x)) * (x & 1 ? back[n][gi].y : back[n][gi].x);
        };
        for (int round = 0; round < 4; ++round) {
            const int q = (warp + round) & 3;
            if (q == 0) quarter(std::integral_constant<int, 0>{}, round);
            else if (q == 1) quarter(std::integral_constant<int, 1>{}, round);
            else if (q == 2) quarter(std::integral_constant<int, 2>{}, round);
            else quarter(std::integral_constant<int, 3>{}, round);
            ka_bar();
        }
        const bool starts = k == 0, ends = kend == rq.tiles;
        if (starts && ends) {
            // the row tile's output: a warp takes a row at a time
            for (int i = warp; i < nrow; i += KA_CONS) {
                const float inv = 1.0f / s_ml[i];
                ka_emit<T, HD>(a, rq, kv, tile * ROWS + i, lane, limit(i) > 0, [&](int d) { return ob[i * OS + d] * inv; });
            }
        } else {
            // a part of a row tile: its start (1), or what goes on from the run before (0)
            float *to = a.part + ((size_t)blockIdx.x * 2 + starts) * a.stride;
            for (int e = tid; e < nrow * HD; e += 32 * KA_CONS) to[e] = ob[e / HD * OS + e % HD];
            if (tid < ROWS) {
                to[ROWS * HD + tid] = s_mref[tid];
                to[ROWS * HD + ROWS + tid] = s_ml[tid];
            }
            if (tid == 0 && starts)
                a.split[blockIdx.x] = KaSplit{(int)((u - off + KA_EXTRA + rq.tiles - 1) / per) - (int)blockIdx.x + 1, kv, tile, rq};
        }
    }
}

}  // namespace fn

using namespace fn;

// every CTA's split row tile and note, then its two partial results
constexpr size_t KA_HEAD = KA_MAX_GRID * (sizeof(KaSplit) + sizeof(int));
static_assert(KA_HEAD % 256 == 0);
FN_API uint64_t fn_kv4_attn_workspace(void) {
    const uint64_t few = (uint64_t)std::min(num_sms() * 3, KA_MAX_GRID) * 2 * KA_PART_MAX * 4;
    return KA_HEAD + std::max(few, kv4_prompt_workspace());
}

template <int HD, bool HL, int NT> static cudaError_t attn_launch(const Kv4AttnArgs &a, int max_new, long long items, long long tiles, cudaStream_t s) {
    // no more CTAs than pairs of units there can be
    const long long units = items * tiles;
    const int grid = (int)std::min(std::max(units / 2, 1ll), (long long)std::min(num_sms() * KaCfg<HD, HL, NT>::CTAS, KA_MAX_GRID));
    cudaError_t e;
    auto go = [&](auto kernel) {
        e = allow_max_dynamic_smem(kernel);
        if (e == cudaSuccess) e = launch_k(kernel, dim3(grid), dim3(KaCfg<HD, HL, NT>::THREADS), KaCfg<HD, HL, NT>::SMEM, s, a);
    };
    if (!HL && std::min(tiles, units / grid) > KA_LONG) go(k_kv4_attn<HD, HL, NT, !HL>);
    else go(k_kv4_attn<HD, HL, NT, false>);
    // one request of at most two tiles: its row tiles weigh the same, 2 + KA_EXTRA units at most, which is the shortest run, so
    // none is split (if there are no more of them than max_new says: a caller's bound is not trusted here)
    if (e != cudaSuccess || (a.n == 1 && max_new >= a.rows && tiles <= 2 && grid == units / 2)) return e;
    using C = KaCfg<HD, HL, NT>;
    using T = typename C::T;
    // few row tiles may have many parts, many have few
    if (items <= KJ_GRID)
        return launch_k(k_kv4_join_few<T, HD, C::ROWS>, dim3(std::min(grid, KJ_GRID), C::ROWS), dim3(32 * KJ_WARPS), 0, s, a, grid);
    return launch_k(k_kv4_join<T, HD, C::ROWS>, dim3(grid, C::ROWS / 8), dim3(256), 0, s, a);
}
// Rows of a request (the largest, by max_new) from which the prompts' kernel takes the call. Measured with 128 dims, 8 heads to each of 4 kv
// heads, fp32 (bf16), this kernel against the prompts': 16 requests of 2000 tokens, 64 rows 49 against 51 us (37 against 42), 80 rows 58
// against 51 (44 against 43). It looks at rows alone: one request of 2000 tokens takes 19 against 34 us (16 against 29) at 64 rows and 29 against
// 38 at 192, one of 16384 is equal at 128 (53 us), so single requests of 64 to some 128 rows get the slower kernel, and so do decoding
// requests beside a prompt in the same call.
constexpr int KP_FROM = 64;

template <int HD> static cudaError_t attn_go(const Kv4AttnArgs &a, bool f32, int max_new, cudaStream_t s) {
    const long long rows = (long long)std::min(max_new, a.rows) * a.group;
    if (rows >= KP_FROM) return launch_kv4_prompt(a, f32, max_new, s);
    // requests whose rows fill one column tile of 8 take the narrow form
    const int nt = rows <= 8 ? 1 : 2;
    // the most row tiles, and units of one, that there can be
    const long long tiles = ((long long)a.max_pages * a.l.bs + KA_TOK - 1) / KA_TOK;
    const long long items = (long long)a.n * a.l.nkv * std::max((rows + 8 * nt - 1) / (8 * nt), 1ll);
    if (nt == 1) return f32 ? attn_launch<HD, true, 1>(a, max_new, items, tiles, s) : attn_launch<HD, false, 1>(a, max_new, items, tiles, s);
    return f32 ? attn_launch<HD, true, 2>(a, max_new, items, tiles, s) : attn_launch<HD, false, 2>(a, max_new, items, tiles, s);
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
        if ((long long)rows * (nh / c->nkv) > INT32_MAX - 256) return fail("kv4 attn: too many rows");
        if ((long long)max_pages * c->page_size > INT32_MAX - 256) return fail("kv4 attn: table too wide");
        if (rows == 0) return 0;
        if ((uintptr_t)q % (type == T_F32 ? 4 : 2) || (uintptr_t)out % (type == T_F32 ? 4 : 2) || (uintptr_t)gate % (type == T_F32 ? 4 : 2))
            return fail("kv4 attn: rows must be aligned to their type");
        if (!q || !out || !cu || !kv_len || !table || !ws) return fail("kv4 attn: null pointer");
        if (ws_bytes < fn_kv4_attn_workspace() || (uintptr_t)ws % 256) return fail("kv4 attn: workspace too small or unaligned");
        a.n = n, a.rows = rows, a.nh = nh, a.max_pages = max_pages;
        a.q = q, a.gate = gate, a.out = out;
        a.qt = q_token, a.qh = q_head, a.gt = gate_token, a.gh = gate_head, a.ot = out_token;
        a.cu = cu, a.kv_len = kv_len, a.table = table;
        a.scale = scale;
        a.err = dev_error_ptr();
        a.group = nh / c->nkv;
        a.split = (KaSplit *)ws;
        a.stride = KA_PART_MAX;
        a.far = (int *)((uint8_t *)ws + KA_MAX_GRID * sizeof(KaSplit));
        a.part = (float *)((uint8_t *)ws + KA_HEAD);
        const bool f32 = type == T_F32;
        const int64_t size = f32 ? 4 : 2;
        a.vec = (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && q_token * size % 16 == 0 && q_head * size % 16 == 0 && out_token * size % 16 == 0 &&
                (!gate || ((uintptr_t)gate % 16 == 0 && gate_token * size % 16 == 0 && gate_head * size % 16 == 0));
        a.always = kv4_rows_meet(out, out_token, c->hd, q, q_token, q_head, rows, nh, c->hd, size) ||
                   (gate && kv4_rows_meet(out, out_token, c->hd, gate, gate_token, gate_head, rows, nh, c->hd, size));
        const cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e = c->hd == 64 ? attn_go<64>(a, f32, max_new, s)
                            : c->hd == 128 ? attn_go<128>(a, f32, max_new, s)
                                           : attn_go<256>(a, f32, max_new, s);
        if (e != cudaSuccess) return fail(std::string("kv4 attn launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
