// Attention over the paged 4-bit KV cache for prompts: many query rows per request (fn_kv4_attn.cu has few).
//
// A row tile is 128 rows of one kv head (the heads of its group, token after token), one per tensor-memory lane. Per 64
// tokens the tensor cores (tcgen05, fp16 operands, fp32 sums in tensor memory) form S = Q K^T (128 x 64) and O = P V
// (128 x hd). Here K and V are dequantised, once per 128 rows: 8192 products per code pay for it.
//
// Roles of the CTA's 16 warps, one CTA per SM:
//   * warp 0 copies pages into rings (K and V parts apart: they are consumed at different times);
//   * warp 2 (only in the long form, below) looks at each tile's scales: K's and V's exponents, and which of V's are not finite;
//   * warp 1 issues the MMAs: S of tile j + 1 before O of tile j, so the softmax of one runs beside the products of the other;
//   * warps 4..7 (a row a lane): scores out of tensor memory, running softmax, P back into tensor memory in S's place;
//   * warps 8..15: Q into tensor memory, K and V codes into the MMAs' operands in shared memory, and the running output:
//     each tile's O is read out of tensor memory and added in registers, o = o 2^.. + O, half a row a lane. So the sums
//     over tokens are rounded fp32 additions, where the tensor core's own accumulation over a long context cuts, and a new
//     maximum needs no pass over tensor memory.
//
// Scales. Codes become (c - 8) d in fp16 as they are. The product has 15 bits, the last of them d's last, and that is 2^-24 or more, fp16's
// own: at the small end nothing is lost, however small K and V are, so neither needs a scale of its own (dividing them by 8 lost
// bits of keys below 4e-3; normalising V by its tile's largest lost those of everything 2^14 below it). At the large end 8 d fits up
// to d = 8188. Weights are 2^10 exp2(s - maximum), 22 bits (11 for bf16 rows) of each down to 2^-12 of the largest and to 2^-35 of it
// beyond, so that values which a row does not see, or hardly weighs, cost it nothing. Rows of q are scaled by a power of two.
// bf16 rows: one product each; q is exact, K, P and V are rounded to 11 bits. fp32 rows: q, K, P and V are fp16 pairs (22
// bits, K's and V's exact), three products each, the small ones first, so that the sum's cut bits are few.
//
// The long form (FAR) is for what that does not serve: scales past 8188, scales that are not finite, scores past 2^20 (beside which the
// weights' 2^10 would be rounded). It is a kernel of its own, the same code with more in it: in one kernel every call paid for it (the
// roles' loops share the instruction cache: 8 bf16 prompts 963 us instead of 607). The first kernel notes whether it met any such thing;
// the second, launched behind it, returns at once (2 us) or does the call again. There:
//   * K's and V's codes of a tile become (c - 8) d 2^(11 - e), e the exponent of the tile's largest finite |d|; K's e goes into the scores'
//     unit, V's into the weights: P = 2^10 2^(s + e - r), a row's reference r the running maximum of s + e. Scales down to 2^-25 of
//     the largest keep all their bits.
//   * Where a tile's K scales lie further apart each token takes its own e. Where its V scales lie more than 2^12 apart no e serves all:
//     the weights stay fp32, and the workers add p v on the CUDA cores instead of the tensor core's O (some 15 times as slow).
//   * What no row of the tile sees becomes 0 in V, whatever its scale is. A visible token whose V scale is not finite also becomes 0
//     and is noted: the rows that see it turn NaN in its 64 dims, the others must not (0 x NaN in the product).
//
// What bounds it, and measured: 2048 new of 4096 tokens, fp32, 16 heads over 2 kv heads of 256 423 us (244 TFLOP/s of the case's
// products, three times that in the tensor cores): the workers, whose one operand buffer makes V wait for the O before it; 8
// prompts, bf16, 32 heads over 8 of 128 607 us (327 TFLOP/s): issue and instruction fetch of softmax and workers, some 2400 cycles per 64
// tokens beside 512 of products.
//
// Work is cut into runs of 64-token units as in fn_kv4_attn.cu, one run per CTA; partial row tiles are joined after it.
#include "fn_kv4_attn.cuh"
#include "fn_umma.cuh"

namespace fn {

constexpr int KP_ROWS = 128, KP_THREADS = 512;
constexpr int KP_EXTRA = 8;  // units that a row tile counts beside its own, for its start and end
constexpr int KP_W_SM = 4, KP_W_WORK = 8;
constexpr int KP_POLLS = 1 << 17;         // of a wait before it gives up, 20 us at most each
constexpr uint32_t KP_FIXED = 5120;       // bytes before the operands (KpShared)
// long form: binades between the K, or the V scales of a tile from which its tokens take their own exponents, or are added in fp32. The
// operands are exact up to 25; but V's e stands for every token and block of the tile, and P keeps 22 bits down to 12 below the largest
constexpr int KP_FAR_K = 25, KP_FAR_V = 12;
constexpr uint32_t KP_MOST = 0x6fff;  // 8188 as a half: the scale of which 8 are fp16's largest number

template <int HD, bool HL, bool FAR> struct KpCfg {
    using T = std::conditional_t<HL, float, __nv_bfloat16>;
    static constexpr int NG = HD / KV4_GROUP, TERMS = HL ? 2 : 1;
    static constexpr int NB = HL && HD == 256 ? 1 : 2;      // operand buffers of K and of V
    static constexpr int RK = 2, RV = NB;                    // stages of the copies
    static constexpr uint32_t KT = KA_TOK * HD * 2;          // K operand: [dim / 8][token] x 16 bytes
    // V operand: [token / 8][dim] x 16 bytes, the token groups 16 bytes further apart (banks of the stores)
    static constexpr uint32_t VG = HD * 16 + 16, VT = 8 * VG;
    // 64 tokens' codes and scales of V, and of K (FAR: with V's scales beside its own, as both are looked at before K is made)
    static constexpr uint32_t RAW = KA_TOK * (HD / 2 + HD / KV4_GROUP * 2), RAWK = RAW + FAR * KA_TOK * HD / KV4_GROUP * 2;
    static constexpr uint32_t QL = HL ? KP_ROWS * HD * 2 : 0;  // second halves of q: [dim / 8][row] x 16 bytes
    static constexpr uint32_t K_OFF = KP_FIXED, V_OFF = K_OFF + NB * TERMS * KT, Q_OFF = V_OFF + NB * TERMS * VT;
    static constexpr uint32_t RK_OFF = Q_OFF + QL, RV_OFF = RK_OFF + RK * RAWK, SMEM = RV_OFF + RV * RAW;
    // registers by warpgroup: IO + SM + 2 WORK <= 4 x 128 at launch; the workers hold HD / 2 sums
    static constexpr int REG_IO = HD == 256 ? 56 : 72, REG_SM = HD == 256 ? 120 : 128, REG_WORK = HD == 256 ? 168 : 152;
    static_assert(REG_IO + REG_SM + 2 * REG_WORK <= 512);
    static constexpr int PART = KP_ROWS * HD + 2 * KP_ROWS;
    // tensor memory: O, then q's first halves, then S / P twice (64 columns: of 16 tokens' scores,
    // P's first halves take 8 and its second halves 8)
    static constexpr uint32_t TM_O = 0, TM_Q = HD, TM_S = HD + HD / 2;
    static_assert(SMEM <= 227 * 1024 && TM_S + 128 <= 512);
};

// the fixed part of shared memory
struct KpShared {
    uint64_t rkf[2], rke[2], rvf[2], rve[2], kf[2], ke[2], vf[2], sf[2], pf[2], xf[8], of, oe, qf, qe, lf, done;
    long long red[KP_THREADS / 32], off;
    uint32_t tmem, valid[8];  // pages there of tile & 7; bit 31: all of them, and every token seen by some row
    int req, fail, met;  // met: what only the long form serves
    // rings as long as the fastest role can be ahead of the slowest reader
    float f[4][KP_ROWS], l[KP_ROWS], rs[KP_ROWS];
    // long form
    float ev[8], ek[8];  // e of V, 2^(e - 11) of K: the scores' unit
    uint32_t bad[8][4][2];  // tokens whose V scale is not finite: [tile & 7][group][token / 32]
    uint8_t any_bad[8], kfar[8], vfar[8];
    uint8_t kexp[8][KA_TOK];  // kfar: exponents by token (biased by 127)
};
static_assert(sizeof(KpShared) <= KP_FIXED);

// true in one lane of the warp
__device__ __forceinline__ bool kp_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// whether a phase has completed, after a wait of up to 20 us in the hardware
__device__ __forceinline__ bool kp_try(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
                 : "memory");
    return done != 0;
}
// the workers' barrier, and whether any of them brought `p`
__device__ __forceinline__ bool kp_bar_work_or(bool p) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 2, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"((uint32_t)p)
        : "memory");
    return any != 0;
}
// tcgen05.ld without its wait; kp_tmem_got makes the values of a load usable after tmem_wait_ld
__device__ __forceinline__ void kp_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void kp_tmem_st8(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void kp_tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void kp_tmem_got(uint32_t (&r)[16]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ float2 kp_pair(const uint32_t (&r)[16], int i) {
    return make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}
__device__ __forceinline__ float kp_tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;\n" : "=r"(r) : "r"(taddr) : "memory");
    return __uint_as_float(r);
}
__device__ __forceinline__ void kp_arrive2(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 2;\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void kp_bar_work() { asm volatile("bar.sync 2, 256;" ::: "memory"); }
__device__ __forceinline__ float kp_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t kp_hsub2(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ uint32_t kp_hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ uint32_t kp_hmax2(uint32_t a, uint32_t b) {  // NaN where either is
    const __half2 r = __hmax2_nan(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ uint32_t kp_hzero2(uint32_t a) { return __heq2_mask(*(const __half2 *)&a, __half2half2(__ushort_as_half(0))); }
__device__ __forceinline__ uint32_t kp_hmin2(uint32_t a, uint32_t b) {
    const __half2 r = __hmin2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
// a b - c, rounded once
__device__ __forceinline__ uint32_t kp_hrest2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*(const __half2 *)&a, *(const __half2 *)&b, __hneg2(*(const __half2 *)&c));
    return *(const uint32_t *)&r;
}
// the nibbles under 0x000f000f and 0x00f000f0 of w as halves c - 8
__device__ __forceinline__ uint32_t kp_low(uint32_t w) { return kp_hsub2((w & 0x000f000fu) | 0x64006400u, 0x64086408u); }
__device__ __forceinline__ uint32_t kp_high(uint32_t w) { return kp_hsub2((w & 0x00f000f0u) | 0x54005400u, 0x54805480u); }

// N adjacent values of a row (zeros unless `there`); vec: 16-byte aligned
template <typename T, int N> __device__ __forceinline__ void kp_load(const T *p, bool there, bool vec, float (&x)[N]) {
    if (!there) {
#pragma unroll
        for (int d = 0; d < N; ++d) x[d] = 0.0f;
    } else if (!vec) {
#pragma unroll
        for (int d = 0; d < N; ++d) x[d] = ka_f<T>(p[d]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int d = 0; d < N; d += 4) {
            const float4 v = *(const float4 *)(p + d);
            x[d] = v.x, x[d + 1] = v.y, x[d + 2] = v.z, x[d + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int d = 0; d < N; d += 8) {
            const uint4 v = *(const uint4 *)(p + d);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) x[d + 2 * y] = __uint_as_float(w[y] << 16), x[d + 2 * y + 1] = __uint_as_float(w[y] & 0xffff0000u);
        }
    }
}

// tiles of 64 tokens that row tile i of a request sees
__device__ __forceinline__ int kp_tiles(const KaReq &q, int group, int i) {
    const int last = min((int)min((long long)(i + 1) * KP_ROWS, (long long)q.fresh * group) - 1, INT32_MAX - 1) / group;
    const int lim = min(max(q.len - q.fresh + last + 1, 0), q.len);
    return max((lim + KA_TOK - 1) / KA_TOK, 1);
}
__device__ __forceinline__ KaReq kp_req(const Kv4AttnArgs &a, int r) { return ka_req<KP_ROWS>(a, r); }

// FAR: the long form, for a call in which the other met what it does not serve (it notes that in a.far, a place for each CTA)
template <int HD, bool HL, bool FAR> __global__ void __launch_bounds__(KP_THREADS, 1) k_kv4_prompt(const __grid_constant__ Kv4AttnArgs a) {
    using C = KpCfg<HD, HL, FAR>;
    using T = typename C::T;
    constexpr int NG = C::NG, NB = C::NB;
    extern __shared__ __align__(1024) uint8_t sm_kp[];
    KpShared &sh = *(KpShared *)sm_kp;
    volatile int *const s_fail = &sh.fail;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.rkf[i], 1), mbar_init(&sh.rke[i], FAR ? 5 : 4), mbar_init(&sh.rvf[i], 1), mbar_init(&sh.rve[i], 8);
            mbar_init(&sh.kf[i], 4), mbar_init(&sh.ke[i], 1), mbar_init(&sh.vf[i], 4);
            mbar_init(&sh.sf[i], 1), mbar_init(&sh.pf[i], 4);
        }
        mbar_init(&sh.of, 1), mbar_init(&sh.oe, 8), mbar_init(&sh.qf, 8), mbar_init(&sh.qe, 1), mbar_init(&sh.lf, 4);
        mbar_init(&sh.done, 1);
        for (int i = 0; i < 8; ++i) mbar_init(&sh.xf[i], 1);
        mbar_fence_init();
        sh.fail = 0;
        sh.met = 0;
    }
    if constexpr (FAR) {
        pdl_wait();
        pdl_trigger();
        if (!__syncthreads_or(a.always || (tid < gridDim.x && after_wait(a.far)[tid]))) return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if constexpr (!FAR) {
        pdl_wait();
        pdl_trigger();
    }

    // ---- this CTA's run of units
    const int per_t = (a.n + KP_THREADS - 1) / KP_THREADS, r0 = min(tid * per_t, a.n), r1 = min(r0 + per_t, a.n);
    auto weight = [&](int r) {
        const KaReq q = kp_req(a, r);
        long long w = 0;
        for (int i = 0; i < q.rt; ++i) w += kp_tiles(q, a.group, i) + KP_EXTRA;
        return w * a.l.nkv;
    };
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += weight(r);
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) sh.red[warp] = incl;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    long long before = incl - mine, units = 0;
    for (int w = 0; w < KP_THREADS / 32; ++w) {
        if (w < warp) before += sh.red[w];
        units += sh.red[w];
    }
    const long long per = max((units + gridDim.x - 1) / gridDim.x, 2ll + KP_EXTRA);
    const long long u0 = blockIdx.x * per, u1 = min(u0 + per, units);
    if (u0 < u1 && u0 >= before && u0 < before + mine) {
        long long at = before;
        for (int r = r0; r < r1; ++r) {
            const long long w = weight(r);
            if (u0 < at + w) {
                sh.req = r;
                sh.off = u0 - at;
                break;
            }
            at += w;
        }
    }
    // rows that belong to no request
    {
        const int live = min(max(after_wait(a.cu)[a.n], 0), a.rows);
        const long long left = (long long)(a.rows - live) * a.nh * HD;
        for (long long i = (long long)blockIdx.x * KP_THREADS + tid; i < left; i += (long long)gridDim.x * KP_THREADS) {
            const long long row = i / (a.nh * HD);
            ((T *)a.out)[(live + row) * a.ot + (i - row * a.nh * HD)] = (T)0.0f;
        }
    }
    if (tid == 0) a.split[blockIdx.x].parts = 0;
    __syncthreads();
    const uint32_t tmem = sh.tmem;

    // the walk over the run's row tiles, the same in every role
    int r = 0, tile = 0, kv = 0, tiles = 0, off = 0, k = 0, kend = 0;
    long long u = u0;
    KaReq rq{};
    auto next = [&]() {
        u += tiles + KP_EXTRA - off;
        off = 0;
        if (u >= u1 || ++kv < a.l.nkv) return;
        kv = 0;
        if (++tile >= rq.rt) {
            tile = 0;
            do rq = kp_req(a, ++r);
            while (rq.rt == 0);
        }
        tiles = kp_tiles(rq, a.group, tile);
    };
    auto here = [&]() {
        k = max(off - KP_EXTRA, 0);
        kend = max((int)min((long long)(tiles + KP_EXTRA), off + (u1 - u)) - KP_EXTRA, 0);
        return k < kend;
    };
    if (u0 < u1) {
        r = sh.req;
        rq = kp_req(a, r);
        long long at = sh.off;
        for (;; ++tile) {
            tiles = kp_tiles(rq, a.group, tile);
            const long long w = (long long)a.l.nkv * (tiles + KP_EXTRA);
            if (at < w) break;
            at -= w;
        }
        kv = (int)(at / (tiles + KP_EXTRA));
        off = (int)(at - (long long)kv * (tiles + KP_EXTRA));
    }
    // rows of the tile see tokens below their limit; rows past its last see what the last sees (results dropped)
    auto limit = [&](int i) {
        const int nrow = (int)min((long long)KP_ROWS, (long long)rq.fresh * a.group - (long long)tile * KP_ROWS);
        const int f = tile * KP_ROWS + min(i, nrow - 1);
        return min(max(rq.len - rq.fresh + f / a.group + 1, 0), rq.len);
    };
    // (few instructions, as it stands in every loop of every role: with a time limit by the clock each place had some 30 more, and the
    // loops lost their places in the instruction cache)
    auto wt = [&](uint64_t *bar, int phase) {
#pragma unroll 1
        for (int i = 0; i < KP_POLLS; ++i) {
            if (kp_try(bar, (uint32_t)phase & 1u)) return true;
            if (*s_fail) return false;
        }
        *s_fail = 1;
        dev_fail(a.err, DEV_WAIT_TIMEOUT);
        return false;
    };
    const int ppt = KA_TOK >> a.l.lbs;  // pages of a tile
    const uint32_t praw = a.l.kb + a.l.sb, prawk = praw + FAR * a.l.sb;  // bytes of a page's V part in a stage, of its K part
    int gt = 0, gi = 0;  // tiles and row tiles done by this role

    if (warp < KP_W_SM) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_IO));
        if (warp == 0) {
            // ---- copies: lane p fetches page p of a tile
            bool ok = true;
            int begun[2] = {};  // stages of K, of V
            for (; u < u1 && ok; next()) {
                if (!here()) continue;
                const int pages = (rq.len + a.l.bs - 1) >> a.l.lbs, hi_lim = limit(KP_ROWS - 1);
                const int *tab = after_wait(a.table) + (size_t)r * a.max_pages;
                int ahead = lane < ppt && k * ppt + lane < pages ? tab[k * ppt + lane] : -1;
                for (int j = k; j < kend && ok; ++j, ++gt) {
                    const int pg = j * ppt + lane, id = ahead;
                    const bool want = lane < ppt && pg < pages, good = want && id >= 0 && id < a.l.n_pages;
                    ahead = lane < ppt && pg + ppt < pages ? tab[pg + ppt] : -1;
                    if (want && !good) dev_fail(a.err, DEV_BAD_ARG);
                    const uint32_t m = __ballot_sync(0xffffffffu, good);
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int R = v ? C::RV : C::RK, sl = gt % R;
                        uint64_t *full = v ? &sh.rvf[sl] : &sh.rkf[sl], *empty = v ? &sh.rve[sl] : &sh.rke[sl];
                        if (lane == 0) {
                            ok = gt < R || wt(empty, gt / R - 1);
                            if (ok) {
                                if (v == 0) sh.valid[gt & 7] = m | (m == (1u << ppt) - 1u && (j + 1) * KA_TOK <= hi_lim ? 0x80000000u : 0u);
                                mbar_arrive_tx(full, (uint32_t)__popc(m) * (v ? praw : prawk));
                            }
                        }
                        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
                        if (!ok) break;
                        ++begun[v];
                        if (good) {
                            const uint8_t *rec = a.l.pages + ((int64_t)id * a.l.nkv + kv) * (int64_t)a.l.rec;
                            uint8_t *to = sm_kp + (v ? C::RV_OFF + sl * C::RAW + lane * praw : C::RK_OFF + sl * C::RAWK + lane * prawk);
                            bulk_g2s(to, rec + v * a.l.kb, a.l.kb, full);
                            bulk_g2s(to + a.l.kb, rec + 2 * a.l.kb + v * a.l.sb, FAR && !v ? 2 * a.l.sb : a.l.sb, full);
                        }
                    }
                }
            }
            // a CTA must not leave with copies into its shared memory in flight: other warps may give up after this one is done, so it always
            // stays until its last copies have landed
            if (lane == 0)
                for (int v = 0; v < 2; ++v) {
                    const int R = v ? C::RV : C::RK;
                    for (int i = max(begun[v] - R, 0); i < begun[v]; ++i)
                        mbar_wait(v ? &sh.rvf[i % R] : &sh.rkf[i % R], (uint32_t)(i / R) & 1u, 1u << 16);
                }
        } else if (FAR && warp == 2) {
            // ---- scales of a tile: the exponents of the largest finite K and V scale, which of V's are not finite, and whether K's
            // lie so far apart that each token takes its own exponent
            bool ok = true;
            for (; u < u1 && ok; next()) {
                if (!here()) continue;
                const int hi_lim = limit(KP_ROWS - 1);
                for (int j = k; j < kend && ok; ++j, ++gt) {
                    ok = __all_sync(0xffffffffu, wt(&sh.rkf[gt % C::RK], gt / C::RK));
                    if (!ok) break;
                    const uint8_t *raw = sm_kp + C::RK_OFF + (gt % C::RK) * C::RAWK + a.l.kb;
                    const uint32_t valid = sh.valid[gt & 7];
                    auto here_ = [&](int tok) { return (valid >> (tok >> a.l.lbs) & 1u) && j * KA_TOK + tok < hi_lim; };
                    auto place = [&](int tok) { return raw + (tok >> a.l.lbs) * prawk + (tok & (a.l.bs - 1)) * 2; };
                    // two tokens a lane, as halves (positive ones order as their bits do); zeros set no exponent
                    const uint8_t *at = place(2 * lane);
                    const uint32_t mask = (here_(2 * lane) ? 0x7fffu : 0u) | (here_(2 * lane + 1) ? 0x7fff0000u : 0u);
                    uint32_t kn = 0x7bff7bffu, vn = kn, kmax = 0, vmax = 0;
#pragma unroll
                    for (int x = 0; x < NG; ++x) {
                        const uint32_t dk = *(const uint32_t *)(at + x * a.l.bs * 2) & mask, dv = *(const uint32_t *)(at + a.l.sb + x * a.l.bs * 2) & mask;
                        kn = kp_hmin2(kn, dk | (kp_hzero2(dk) & 0x7bff7bffu));
                        vn = kp_hmin2(vn, dv | (kp_hzero2(dv) & 0x7bff7bffu));
                    }
                    const uint32_t kmin = __reduce_min_sync(0xffffffffu, min(kn & 0xffffu, kn >> 16));
                    const uint32_t vmin = __reduce_min_sync(0xffffffffu, min(vn & 0xffffu, vn >> 16));
                    auto exponent = [](uint32_t h) { return (int)(__float_as_uint(__half2float(__ushort_as_half((unsigned short)h))) >> 23); };
                    // a closer look, a token a lane: what is not finite sets no exponent either
                    bool any = false;
                    uint32_t own[2] = {};  // the token's largest K scale
#pragma unroll 1
                    for (int x = 0; x < NG; ++x)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint8_t *p = place(lane + 32 * h) + x * a.l.bs * 2;
                            const bool in = here_(lane + 32 * h);
                            const uint32_t dk = *(const uint16_t *)p & 0x7fffu, dv = *(const uint16_t *)(p + a.l.sb) & 0x7fffu;
                            if (in && dk < 0x7c00u) own[h] = max(own[h], dk);
                            if (in && dv < 0x7c00u) vmax = max(vmax, dv);
                            const uint32_t bad = __ballot_sync(0xffffffffu, in && dv >= 0x7c00u);
                            if (lane == 0) sh.bad[gt & 7][x][h] = bad;
                            any |= bad != 0;
                        }
                    kmax = __reduce_max_sync(0xffffffffu, max(own[0], own[1]));
                    vmax = __reduce_max_sync(0xffffffffu, vmax);
#pragma unroll
                    for (int h = 0; h < 2; ++h) sh.kexp[gt & 7][lane + 32 * h] = (uint8_t)exponent(own[h] ? own[h] : kmax);
                    const bool vfar = vmax && exponent(vmax) > exponent(vmin) + KP_FAR_V;
                    if (vfar) vmax = vmin;  // what is added in fp32 raises no reference
                    if (lane == 0) {
                        sh.any_bad[gt & 7] = any;
                        sh.kfar[gt & 7] = kmax && exponent(kmax) > exponent(kmin) + KP_FAR_K;
                        sh.vfar[gt & 7] = vfar;
                        sh.ev[gt & 7] = vmax ? (float)(exponent(vmax) - 127) : 0.0f;
                        sh.ek[gt & 7] = kmax ? kp_pow2(exponent(kmax) - 138) : 1.0f;
                    }
                    __syncwarp();
                    if (lane == 0) {
                        tc_arrive(&sh.xf[gt & 7]);
                        tc_arrive(&sh.rke[gt % C::RK]);
                    }
                }
            }
        } else if (warp == 1) {
            // ---- MMAs. The whole warp runs this and one elected lane issues: the operands' descriptors then live in uniform
            // registers. (As one lane's own values each MMA took 120 cycles and more, whatever its size; so it takes what its size
            // asks, 32 cycles at 64 columns.)
            constexpr uint32_t id_s = umma_idesc_f16(128, KA_TOK), id_o = umma_idesc_f16(128, HD);
            const uint64_t kd0 = umma_desc(smem_u32(sm_kp + C::K_OFF), 1024u, 128u), qd = umma_desc(smem_u32(sm_kp + C::Q_OFF), 2048u, 128u);
            const uint64_t vd0 = umma_desc(smem_u32(sm_kp + C::V_OFF), C::VG, 128u);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), tq = tm + C::TM_Q, to = tm + C::TM_O;
            auto scores = [&](int g) {  // S of tile g
                const uint32_t ts = tm + C::TM_S + (uint32_t)(g & 1) * 64u;
                const uint64_t kd = kd0 + (uint64_t)((g % NB) * (C::TERMS * C::KT >> 4));
                if constexpr (HL) {
#pragma unroll
                    for (int x = 0; x < HD / 16; ++x) umma_f16_smem_a(ts, qd + x * 256u, kd + x * 128u, id_s, x > 0);
#pragma unroll
                    for (int x = 0; x < HD / 16; ++x) umma_bf16_tmem_a(ts, tq + 8u * x, kd + (C::KT >> 4) + x * 128u, id_s, 1u);
                }
#pragma unroll
                for (int x = 0; x < HD / 16; ++x) umma_bf16_tmem_a(ts, tq + 8u * x, kd + x * 128u, id_s, HL || x > 0);
            };
            auto outputs = [&](int g) {  // O of tile g
                const uint32_t tp = tm + C::TM_S + (uint32_t)(g & 1) * 64u;
                const uint64_t vd = vd0 + (uint64_t)((g % NB) * (C::TERMS * C::VT >> 4));
                if constexpr (HL) {
#pragma unroll
                    for (int x = 0; x < KA_TOK / 16; ++x) umma_bf16_tmem_a(to, tp + 8u + 16u * x, vd + x * (C::VG >> 3), id_o, x > 0);
#pragma unroll
                    for (int x = 0; x < KA_TOK / 16; ++x) umma_bf16_tmem_a(to, tp + 16u * x, vd + (C::VT >> 4) + x * (C::VG >> 3), id_o, 1u);
                }
#pragma unroll
                for (int x = 0; x < KA_TOK / 16; ++x) umma_bf16_tmem_a(to, tp + 16u * x, vd + x * (C::VG >> 3), id_o, HL || x > 0);
            };
            auto wtw = [&](uint64_t *bar, int phase) { return __all_sync(0xffffffffu, wt(bar, phase)) != 0; };
            bool ok = true;
            for (; u < u1 && ok; next()) {
                if (!here()) continue;
                ok = wtw(&sh.qf, gi);
                const int n = kend - k, g0 = gt;
                for (int j = 0; j <= n && ok; ++j) {
                    if (j < n) {
                        const int g = g0 + j;
                        // S takes the place of P of tile g - 2, which the workers may still read. (Not where that is of the row tile before: q came
                        // after it had been added, and its phase of oe, two ago by now, would look like the one to come.)
                        ok = wtw(&sh.kf[g % NB], g / NB) && (!FAR || j < 2 || !sh.vfar[(g - 2) & 7] || wtw(&sh.oe, g - 2));
                        if (!ok) break;
                        tc_fence_after();
                        if (kp_elect()) {
                            scores(g);
                            umma_commit(&sh.sf[g & 1]);
                            umma_commit(&sh.ke[g % NB]);
                            if (j == n - 1) umma_commit(&sh.qe);
                        }
                        __syncwarp();
                    }
                    if (j > 0) {
                        const int g = g0 + j - 1;
                        ok = wtw(&sh.pf[g & 1], g >> 1) && wtw(&sh.vf[g % NB], g / NB) && (g == 0 || wtw(&sh.oe, g - 1));
                        if (!ok) break;
                        tc_fence_after();
                        if (kp_elect()) {
                            if (!FAR || !sh.vfar[g & 7]) outputs(g);
                            umma_commit(&sh.of);
                        }
                        __syncwarp();
                    }
                }
                gt = g0 + n;
                ++gi;
            }
            // every MMA issued has finished before the CTA gives its memory back
            if (kp_elect()) umma_commit(&sh.done);
            __syncwarp();
            mbar_park(&sh.done, 0);
        }
        __syncwarp();
    } else if (warp < KP_W_WORK) {
        // ---- softmax: row 32 (warp % 4) + lane
        if constexpr (C::REG_SM < 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_SM));
        const int row = tid - 32 * KP_W_SM;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + C::TM_S;
        bool ok = true;
        for (; u < u1 && ok; next()) {
            if (!here()) continue;
            const int lim = limit(row);
            // the reference, as the score and the exponent that it came of: a large score would swallow the exponent
            float sref = -INFINITY, eref = 0.0f, l = 0.0f, rs = 0.0f;
            [[maybe_unused]] bool met = false;
            for (int j = k; j < kend; ++j, ++gt) {
                const int b = gt & 1;
                ok = wt(&sh.sf[b], gt >> 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                // (what warps 0 and 2 and the workers left for this tile is there: they came before the K and q of these scores)
                if (j == k) rs = sh.rs[row];
                const uint32_t valid = sh.valid[gt & 7], ts = tl + (uint32_t)b * 64u;
                const int left = lim - j * KA_TOK;  // tokens of the tile that the row sees
                const bool masked = left < KA_TOK || !(valid >> 31);
                const float ev = FAR ? sh.ev[gt & 7] : 0.0f;
                float rsj = FAR ? rs * sh.ek[gt & 7] : rs;
                if (FAR && sh.kfar[gt & 7]) {  // every column by its own unit
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t s[16];
                        kp_tmem_ld16(ts + 16u * c, s);
                        kp_tmem_wait_ld();
                        kp_tmem_got(s);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[i] = __float_as_uint(__uint_as_float(s[i]) * (rs * kp_pow2((int)sh.kexp[gt & 7][16 * c + i] - 138)));
                        tmem_st16(ts + 16u * c, s);
                        tmem_wait_st();
                    }
                    rsj = 1.0f;
                }
                // (16 columns at a time, read twice: a short loop stays in the instruction cache beside the other roles' loops,
                // where 64 columns unrolled had every role wait for instructions)
                auto hide = [&](uint32_t(&s)[16], int c) {
                    if (masked) {
                        const int n = valid >> (16 * c >> a.l.lbs) & 1u ? left - 16 * c : 0;  // a page is 16 tokens or more
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (i >= n) s[i] = 0xff800000u;  // -inf
                    }
                };
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t s[16];
                    kp_tmem_ld16(ts + 16u * c, s);
                    kp_tmem_wait_ld();
                    kp_tmem_got(s);
                    hide(s, c);
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx[i & 1] = fmaxf(mx[i & 1], __uint_as_float(s[i]));
                }
                // rs > 0: the maximum may be taken before the scaling
                const float top = fmaxf(mx[0], mx[1]) * rsj;
                const bool higher = FAR ? top - sref > eref - ev : top > sref;  // (never so for -inf beside -inf)
                const float ns = higher ? top : sref, ne = FAR && higher ? ev : eref;
                const float fac = sref == -INFINITY ? 0.0f : ka_exp2((sref - ns) + (eref - ne));
                sref = ns, eref = ne;
                // P = 2^10 exp2(s (+ e) - reference): fp16 keeps 11 bits down to 2^-24 of the largest. Beside a reference of 2^20 and more
                // the 10 would be rounded, and at 2^27 a weight could pass fp16: the long form takes the exact difference to the best score
                // first.
                const float z0 = ns == -INFINITY ? 0.0f : -ns, z1 = 10.0f + ev - ne, z = z0 + z1;
                // (one at a time: the packed product and sum would become one, and the rounding of the best score differ)
                [[maybe_unused]] auto apart = [&](uint32_t x) { return __fadd_rn(__fadd_rn(__fmul_rn(__uint_as_float(x), rsj), z0), z1); };
                if constexpr (!FAR) met |= fabsf(ns) > 1048576.0f && ns != -INFINITY;
                sh.f[gt & 3][row] = fac;
                const float2 rs2 = make_float2(rsj, rsj), z2 = make_float2(z, z);
                float2 ls = make_float2(0.0f, 0.0f);
                if (FAR && sh.vfar[gt & 7]) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t s[16];
                        kp_tmem_ld16(ts + 16u * c, s);
                        kp_tmem_wait_ld();
                        kp_tmem_got(s);
                        hide(s, c);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float p = ka_exp2(apart(s[i]));
                            ls.x += p;
                            s[i] = __float_as_uint(p);
                        }
                        tmem_st16(ts + 16u * c, s);
                    }
                }
#pragma unroll 1
                for (int c = FAR && sh.vfar[gt & 7] ? 4 : 0; c < 4; ++c) {
                    uint32_t s[16], p16[16];
                    kp_tmem_ld16(ts + 16u * c, s);
                    kp_tmem_wait_ld();
                    kp_tmem_got(s);
                    hide(s, c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float2 x;
                        if constexpr (FAR) x = make_float2(apart(s[2 * i]), apart(s[2 * i + 1]));
                        else x = __ffma2_rn(kp_pair(s, i), rs2, z2);
                        const float2 p = make_float2(ka_exp2(x.x), ka_exp2(x.y));
                        ls = __fadd2_rn(ls, p);
                        p16[i] = ka_pack(p.x, p.y);
                        if constexpr (HL) {
                            const float2 h = ka_unpack(p16[i]);
                            p16[8 + i] = ka_pack(p.x - h.x, p.y - h.y);
                        }
                    }
                    if constexpr (HL) tmem_st16(ts + 16u * c, p16);
                    else kp_tmem_st8(ts + 16u * c, p16);
                }
                l = l * fac + (FAR ? (ls.x + ls.y) * kp_pow2(11 - (int)ev) : ls.x + ls.y);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&sh.pf[b]);
            }
            if (!ok) break;
            if constexpr (!FAR)
                if (met) sh.met = 1;
            if (k == 0 && kend == tiles) {
                sh.l[row] = l;
            } else {
                float *to = a.part + ((size_t)blockIdx.x * 2 + (k == 0)) * a.stride + KP_ROWS * HD;
                to[row] = sref + eref;
                to[KP_ROWS + row] = l;
                if (tid == 32 * KP_W_SM && k == 0)
                    a.split[blockIdx.x] = KaSplit{(int)((u - off + KP_EXTRA + tiles - 1) / per) - (int)blockIdx.x + 1, kv, tile, rq};
            }
            __syncwarp();
            if (lane == 0) tc_arrive(&sh.lf);
        }
    } else {
        // ---- workers: q, K, V into operands; the running output, dims [half HD / 2, + HD / 2) of row 32 (warp % 4) + lane
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_WORK));
        const int wtid = tid - 32 * KP_W_WORK, half = (warp - KP_W_WORK) >> 2, row = 32 * (warp & 3) + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        constexpr int HH = HD / 2, NH = HH >= KV4_GROUP ? HH / KV4_GROUP : 1;  // this half's dims, and its 64-dim groups
        const int g0 = half * HH / KV4_GROUP;
        bool ok = true;
        [[maybe_unused]] uint32_t seen = 0;  // the largest scales (NaN: one of them is)
        // Warps 8..11 make K, 12..15 V. A thread takes 16 bytes of codes (32 dims) of token k_tok at a time, from quarter k_q on,
        // or word v_wd (8 dims) of tokens v_tok .. + 7: places in the stages and operands
        constexpr int KU = NG, VU = HD >= 128 ? HD / 128 : 1;
        const int gtid = wtid & 127;
        const int k_tok = gtid & 63, k_q = gtid >> 6, k_line = k_tok & (a.l.bs - 1);
        const uint32_t k_src = (k_tok >> a.l.lbs) * prawk + k_line * 32 + k_q * 16, k_dst = k_q * 4096 + k_tok * 16;
        const uint32_t k_sc = (k_tok >> a.l.lbs) * prawk + a.l.kb + k_line * 2;
        const int v_tok = (gtid & 7) * 8, v_wd = gtid >> 3, v_line = (v_wd >> 3) * a.l.bs + (v_tok & (a.l.bs - 1));
        const uint32_t v_page = (v_tok >> a.l.lbs) * praw, v_src = v_page + v_line * 32 + (v_wd & 7) * 4, v_sc = v_page + a.l.kb + v_line * 2;
        const uint32_t v_dst = (gtid & 7) * C::VG + v_wd * 128;
        // a wait by all lanes, with one answer
        auto wtw = [&](uint64_t *bar, int phase) { return __all_sync(0xffffffffu, wt(bar, phase)) != 0; };
        for (; u < u1; next()) {
            if (!here()) continue;
            // a warp whose wait gave up goes on to this barrier, where all leave together
            if (ok && gi > 0) ok = wtw(&sh.qe, gi - 1);
            if (kp_bar_work_or(!ok)) break;
            const int lim = limit(row), hi_lim = limit(KP_ROWS - 1);
            const long long flat = (long long)tile * KP_ROWS + row;
            const bool live = flat < (long long)rq.fresh * a.group;
            const int tok_row = live ? (int)(flat / a.group) : 0, head = kv * a.group + (live ? (int)(flat - (long long)tok_row * a.group) : 0);
            // ---- q: scaled so that the row's largest value is 2^10..2^11, dims in the order of the codes' nibbles
            {
                const T *src = (const T *)after_wait(a.q) + (int64_t)(rq.first + tok_row) * a.qt + (int64_t)head * a.qh + half * HH;
                float mx = 0.0f;
#pragma unroll 2
                for (int d = 0; d < HH; d += 16) {
                    float x[16];
                    kp_load<T, 16>(src + d, live, a.vec, x);
#pragma unroll
                    for (int y = 0; y < 16; ++y) mx = fmaxf(mx, fabsf(x[y]));
                }
                // both halves of the row agree on its exponent (K's place is free before the row tile's first K)
                float *sx = (float *)(sm_kp + C::K_OFF);
                sx[half * KP_ROWS + row] = mx;
                kp_bar_work();
                mx = fmaxf(mx, sx[(half ^ 1) * KP_ROWS + row]);
                const int e = min(max(10 - ((int)(__float_as_uint(mx) >> 23) - 127), -90), 120);
                const float up = a.scale < 0.0f ? -kp_pow2(e) : kp_pow2(e);
                // scores in base 2: undo the scaling; positive also for a scale of zero (beside K's unit, 2^-35 or more, too)
                if (half == 0) sh.rs[row] = fmaxf(fabsf(a.scale) * 1.44269504f * kp_pow2(-e), 1e-26f);
                kp_bar_work();
#pragma unroll 1
                for (int d = 0; d < HH; d += 32) {
                    float x[32];
                    kp_load<T, 32>(src + d, live, a.vec, x);
                    uint32_t hi[16];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t lo[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const float x0 = x[8 * w + y] * up, x1 = x[8 * w + y + 4] * up;
                            hi[4 * w + y] = ka_pack(x0, x1);
                            const float2 h = ka_unpack(hi[4 * w + y]);
                            lo[y] = ka_pack(x0 - h.x, x1 - h.y);
                        }
                        if constexpr (HL)
                            *(uint4 *)(sm_kp + C::Q_OFF + ((half * HH + d) / 8 + w) * 2048 + row * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                    tmem_st16(tl + C::TM_Q + (uint32_t)(half * HH + d) / 2u, hi);
                }
                tmem_wait_st();
                tc_fence_before();
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) tc_arrive(&sh.qf);
            }
            float2 o[HH / 2];
#pragma unroll
            for (int c = 0; c < HH / 2; ++c) o[c] = make_float2(0.0f, 0.0f);
            auto there = [&](int g, int j, int tok) { return (sh.valid[g & 7] >> (tok >> a.l.lbs) & 1u) && j * KA_TOK + tok < hi_lim; };
            // K of tile g (the row tile's j): 16 bytes of codes (32 dims of a token) at a time
            auto make_k = [&](int g, int j) {
                if (!wtw(&sh.rkf[g % C::RK], g / C::RK) || (FAR && !wtw(&sh.xf[g & 7], g >> 3))) return false;
                if (g >= NB && !wtw(&sh.ke[g % NB], g / NB - 1)) return false;
                const uint8_t *raw = sm_kp + C::RK_OFF + (g % C::RK) * C::RAWK;
                uint8_t *to = sm_kp + C::K_OFF + (g % NB) * C::TERMS * C::KT + k_dst;
                const bool all = sh.valid[g & 7] >> 31;
                const bool keep = all || there(g, j, k_tok);
                [[maybe_unused]] float up;  // 2^(11 - e)
                if constexpr (FAR) up = __uint_as_float(sh.kfar[g & 7] ? 265u - sh.kexp[g & 7][k_tok] << 23 : 0x7f000000u - __float_as_uint(sh.ek[g & 7]));
#pragma unroll 1
                for (int x = 0; x < KU; ++x) {  // a 64-dim group each
                    const uint4 w4 = *(const uint4 *)(raw + k_src + x * a.l.bs * 32);
                    uint32_t dd = *(const uint16_t *)(raw + k_sc + x * a.l.bs * 2) * 0x10001u;
                    if constexpr (FAR) {
                        const float d = ka_unpack(dd).x * up;
                        dd = ka_pack(d, d);
                    }
                    if (!keep) dd = 0;
                    if constexpr (!FAR) seen = kp_hmax2(seen, dd & 0x7fff7fffu);
                    const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t w = ws[y], w8 = w >> 8, c0 = kp_low(w), c1 = kp_high(w), c2 = kp_low(w8), c3 = kp_high(w8);
                        const uint32_t h0 = kp_hmul2(c0, dd), h1 = kp_hmul2(c1, dd), h2 = kp_hmul2(c2, dd), h3 = kp_hmul2(c3, dd);
                        uint8_t *at = to + (x * 8 + y) * 1024;
                        *(uint4 *)at = make_uint4(h0, h1, h2, h3);
                        if constexpr (HL)
                            *(uint4 *)(at + C::KT) = make_uint4(kp_hrest2(c0, dd, h0), kp_hrest2(c1, dd, h1), kp_hrest2(c2, dd, h2), kp_hrest2(c3, dd, h3));
                    }
                }
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    tc_arrive(&sh.kf[g % NB]);
                    tc_arrive(&sh.rke[g % C::RK]);
                }
                return true;
            };
            // V of tile g: 8 tokens x 8 dims at a time, turned. Its buffer's last reader came before an O that has been added.
            auto make_v = [&](int g, int j) {
                if (!wtw(&sh.rvf[g % C::RV], g / C::RV) || (FAR && !wtw(&sh.xf[g & 7], g >> 3))) return false;
                const uint8_t *raw = sm_kp + C::RV_OFF + (g % C::RV) * C::RAW;
                [[maybe_unused]] const float up = FAR ? kp_pow2(11 - (int)sh.ev[g & 7]) : 1.0f;
                const bool all = (sh.valid[g & 7] >> 31) && !(FAR && sh.any_bad[g & 7]), far = FAR && sh.vfar[g & 7];
#pragma unroll 1
                for (int un = 0; un < VU; ++un) {
                    if (far || (HD < 128 && v_wd >= HD / 8)) break;
                    const uint8_t *src = raw + v_src + un * 2 * a.l.bs * 32;  // 16 words on: two groups
                    const uint4 s4 = *(const uint4 *)(raw + v_sc + un * 2 * a.l.bs * 2);
                    const uint32_t ss[4] = {s4.x, s4.y, s4.z, s4.w};
                    uint32_t w[8], dd[4];
#pragma unroll
                    for (int y = 0; y < 8; ++y) w[y] = *(const uint32_t *)(src + y * 32);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int tok = v_tok + 2 * y;
                        if constexpr (FAR) {
                            float2 d = __fmul2_rn(ka_unpack(ss[y]), make_float2(up, up));
                            if (!all) {
                                if (!(there(g, j, tok) && fabsf(d.x) < INFINITY)) d.x = 0.0f;
                                if (!(there(g, j, tok + 1) && fabsf(d.y) < INFINITY)) d.y = 0.0f;
                            }
                            dd[y] = ka_pack(d.x, d.y);
                        } else {
                            dd[y] = ss[y];
                            if (!all) dd[y] &= (there(g, j, tok) ? 0xffffu : 0u) | (there(g, j, tok + 1) ? 0xffff0000u : 0u);
                            seen = kp_hmax2(seen, dd[y] & 0x7fff7fffu);
                        }
                    }
                    uint8_t *at = sm_kp + C::V_OFF + (g % NB) * C::TERMS * C::VT + v_dst + un * 2048;
#pragma unroll 1
                    for (int by = 0; by < 4; ++by) {
                        const uint32_t sel = 0x4400u + 0x1111u * (uint32_t)by;  // byte `by` of two tokens
                        uint32_t h[2][4];
                        [[maybe_unused]] uint32_t lo[2][4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const uint32_t x = __byte_perm(w[2 * y], w[2 * y + 1], sel), c0 = kp_low(x), c1 = kp_high(x);
                            h[0][y] = kp_hmul2(c0, dd[y]), h[1][y] = kp_hmul2(c1, dd[y]);
                            if constexpr (HL) lo[0][y] = kp_hrest2(c0, dd[y], h[0][y]), lo[1][y] = kp_hrest2(c1, dd[y], h[1][y]);
                        }
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            *(uint4 *)(at + (2 * by + x) * 16) = make_uint4(h[x][0], h[x][1], h[x][2], h[x][3]);
                            if constexpr (HL) *(uint4 *)(at + C::VT + (2 * by + x) * 16) = make_uint4(lo[x][0], lo[x][1], lo[x][2], lo[x][3]);
                        }
                    }
                }
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    tc_arrive(&sh.vf[g % NB]);
                    if (!far) kp_arrive2(&sh.rve[g % C::RV]);
                }
                return true;
            };
            // step j: K of tile j + 1 by half of the warps, V of tile j by the other half, then all add O of tile j - 1. (Every part
            // appears once: the instruction cache holds the loop.)
            for (int j = k - 1; j <= kend && ok; ++j) {
                const int g = gt + j - k;
                const bool adds = j > k;
                // a tile whose V scales lie far apart: o = o f + p v in fp32, a token at a time. First of all, since the stage that it gives
                // back may be the only one, and the next copies wait behind it.
                const bool far = FAR && adds && sh.vfar[(g - 1) & 7];
                if (far) {
                    const int gp = g - 1;
                    if (!wtw(&sh.rvf[gp % C::RV], gp / C::RV) || !wtw(&sh.pf[gp & 1], gp >> 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const float f = sh.f[gp & 3][row], up = kp_pow2(11 - (int)sh.ev[gp & 7]);
#pragma unroll
                    for (int c = 0; c < HH / 2; ++c) o[c].x *= f, o[c].y *= f;
#pragma unroll 1
                    for (int tok = 0; tok < KA_TOK; ++tok) {
                        const float p = kp_tmem_ld1(tl + C::TM_S + (uint32_t)(gp & 1) * 64u + tok);
                        const uint8_t *raw = sm_kp + C::RV_OFF + (gp % C::RV) * C::RAW + (tok >> a.l.lbs) * praw;
                        const int line = tok & (a.l.bs - 1);
                        const bool in = there(gp, j - 1, tok);
#pragma unroll
                        for (int w = 0; w < HH / 8; ++w) {
                            const int at = (half * HH + 8 * w) / KV4_GROUP * a.l.bs + line;
                            const float d = ka_half(raw + a.l.kb + at * 2), pd = in && fabsf(d) < INFINITY ? p * (d * up) : 0.0f;
                            const uint32_t c = *(const uint32_t *)(raw + at * 32 + (half * HH / 8 + w) % 8 * 4);
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                o[4 * w + x].x = fmaf((float)(int)(c >> (8 * x) & 15u) - 8.0f, pd, o[4 * w + x].x);
                                o[4 * w + x].y = fmaf((float)(int)(c >> (8 * x + 4) & 15u) - 8.0f, pd, o[4 * w + x].y);
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) tc_arrive(&sh.rve[gp % C::RV]);
                }
                if (half == 0) {
                    if (j + 1 < kend) ok = make_k(g + 1, j + 1);
                } else if (NB == 2 && j >= k && j < kend) {
                    ok = make_v(g, j);
                }
                if (!ok) break;
                if (adds && !wtw(&sh.of, g - 1)) {
                    ok = false;
                    break;
                }
                // with one buffer V has to wait for the O before it
                if (NB == 1 && half == 1 && j >= k && j < kend) {
                    ok = make_v(g, j);
                    if (!ok) break;
                }
                const uint32_t to = tl + C::TM_O + (uint32_t)(half * HH);
                if (adds) {  // o = o f + O
                    const int gp = (g - 1) & 7;
                    const float f = sh.f[gp & 3][row];
                    const float2 f2 = make_float2(f, f);
                    uint32_t x[2][16];
                    tc_fence_after();
                    if (!far) {
#pragma unroll
                        for (int c = 0; c < HH; c += 32) {
                            kp_tmem_ld16(to + c, x[0]);
                            kp_tmem_ld16(to + c + 16u, x[1]);
                            kp_tmem_wait_ld();
                            kp_tmem_got(x[0]);
                            kp_tmem_got(x[1]);
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int y = 0; y < 8; ++y) o[c / 2 + h * 8 + y] = __ffma2_rn(o[c / 2 + h * 8 + y], f2, kp_pair(x[h], y));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc_arrive(&sh.oe);
                    if (FAR && sh.any_bad[gp]) {
                        const int left = lim - (j - 1) * KA_TOK;  // tokens of the tile that the row sees
                        const uint32_t m0 = left <= 0 ? 0u : left >= 32 ? 0xffffffffu : (1u << left) - 1u;
                        const uint32_t m1 = left <= 32 ? 0u : left >= 64 ? 0xffffffffu : (1u << (left - 32)) - 1u;
                        const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
                        for (int y = 0; y < NH; ++y)
                            if ((sh.bad[gp][g0 + y][0] & m0) | (sh.bad[gp][g0 + y][1] & m1))
#pragma unroll
                                for (int c = y * 32; c < (y + 1) * 32 && c < HH / 2; ++c) o[c] = make_float2(nan, nan);
                    }
                }
            }
            gt += kend - k;
            ok = ok && wtw(&sh.lf, gi);
            ++gi;
            if (!ok) continue;
            if (k == 0 && kend == tiles) {
                if (live) {
                    const float inv = lim > 0 ? 1.0f / sh.l[row] : 0.0f;
                    const int64_t at = rq.first + tok_row;
                    T *dst = (T *)a.out + at * a.ot + (int64_t)head * HD + half * HH;
                    const T *gate = a.gate ? (const T *)after_wait(a.gate) + at * a.gt + (int64_t)head * a.gh + half * HH : nullptr;
#pragma unroll
                    for (int c = 0; c < HH; c += 8) {
                        float y[8];
#pragma unroll
                        for (int x = 0; x < 4; ++x) y[2 * x] = lim > 0 ? o[c / 2 + x].x * inv : 0.0f, y[2 * x + 1] = lim > 0 ? o[c / 2 + x].y * inv : 0.0f;
                        if (gate) {
                            float gx[8];
                            kp_load<T, 8>(gate + c, true, a.vec, gx);
#pragma unroll
                            for (int x = 0; x < 8; ++x) y[x] *= ka_gate(gx[x]);
                        }
                        if (a.vec) {
                            if constexpr (HL) {
                                *(float4 *)(dst + c) = make_float4(y[0], y[1], y[2], y[3]);
                                *(float4 *)(dst + c + 4) = make_float4(y[4], y[5], y[6], y[7]);
                            } else {
                                uint32_t w[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * x], y[2 * x + 1]);
                                    w[x] = *(const uint32_t *)&h;
                                }
                                *(uint4 *)(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 8; ++x) dst[c + x] = (T)y[x];
                        }
                    }
                }
            } else {
                float *to = a.part + ((size_t)blockIdx.x * 2 + (k == 0)) * a.stride + (size_t)row * HD + half * HH;
#pragma unroll
                for (int c = 0; c < HH / 2; c += 2) *(float4 *)(to + 2 * c) = make_float4(o[c].x, o[c].y, o[c + 1].x, o[c + 1].y);
            }
        }
        if constexpr (!FAR)
            if ((seen & 0xffffu) > KP_MOST || (seen >> 16) > KP_MOST) sh.met = 1;
    }
    // ---- everybody is here (the copies and MMAs of a CTA that gave up as well)
    tc_fence_before();
    __syncthreads();
    if (!FAR && tid == 0) a.far[blockIdx.x] = sh.met;
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
}

uint64_t kv4_prompt_workspace() {
    return (uint64_t)std::min(num_sms(), KA_MAX_GRID) * 2 * KpCfg<256, true, false>::PART * 4;
}

template <int HD, bool HL> static cudaError_t prompt_go(Kv4AttnArgs a, int max_new, cudaStream_t s) {
    using C = KpCfg<HD, HL, false>;
    cudaError_t e = allow_max_dynamic_smem(k_kv4_prompt<HD, HL, false>);
    if (e == cudaSuccess) e = allow_max_dynamic_smem(k_kv4_prompt<HD, HL, true>);
    if (e != cudaSuccess) return e;
    a.stride = C::PART;
    const long long rt = ((long long)std::min(max_new, a.rows) * a.group + KP_ROWS - 1) / KP_ROWS;
    const long long tiles = ((long long)a.max_pages * a.l.bs + KA_TOK - 1) / KA_TOK;
    const long long units = (long long)a.n * a.l.nkv * std::max(rt, 1ll) * tiles;
    const int grid = (int)std::min(std::max(units / 2, 1ll), (long long)std::min(num_sms(), KA_MAX_GRID));
    // outputs over q or gate could not be made twice
    if (!a.always) e = launch_k(k_kv4_prompt<HD, HL, false>, dim3(grid), dim3(KP_THREADS), C::SMEM, s, a);
    if (e == cudaSuccess) e = launch_k(k_kv4_prompt<HD, HL, true>, dim3(grid), dim3(KP_THREADS), KpCfg<HD, HL, true>::SMEM, s, a);
    if (e != cudaSuccess || grid == 1) return e;
    return launch_k(k_kv4_join<typename C::T, HD, KP_ROWS>, dim3(grid, KP_ROWS / 8), dim3(256), 0, s, a);
}

cudaError_t launch_kv4_prompt(Kv4AttnArgs a, bool f32, int max_new, cudaStream_t s) {
    switch (a.l.hd) {
        case 64: return f32 ? prompt_go<64, true>(a, max_new, s) : prompt_go<64, false>(a, max_new, s);
        case 128: return f32 ? prompt_go<128, true>(a, max_new, s) : prompt_go<128, false>(a, max_new, s);
        default: return f32 ? prompt_go<256, true>(a, max_new, s) : prompt_go<256, false>(a, max_new, s);
    }
}

}  // namespace fn
