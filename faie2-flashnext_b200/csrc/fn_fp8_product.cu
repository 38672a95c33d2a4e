// Product of 8-bit rows and an 8-bit weight on the 5th-generation tensor cores (tcgen05, kind::f8f6f4):
//
//   out[m][n] = sum_g xs[m][g] ws[n / 128][g] sum_{k in group g} x[m][k] w[n][k]  (+ add[m][n])
//
// The inner sum of a group of 128 is what the tensor core adds up, in its fp32 accumulators in tensor memory; the outer sum is fp32
// in registers, where each group's sum takes its two scales (their product is rounded once to fp32). The reference's k_tgemv
// (engine/faie2fn.cu:734-955) takes up to 8 rows on CUDA cores and no 8-bit floating point.
//
// Rows of the weight lie on the 128 lanes (operand A), rows of x on the columns (operand B, N = 16 .. 128): few rows of x waste none
// of the weight's bandwidth, and a warp stores adjacent columns of an output row. A tile takes `height` (a multiple of 8 up to 128)
// rows of the weight, chosen so that the tiles fill whole waves of SMs: the MMA has 128 lanes whatever the height, but with few rows of
// x it is not what bounds the call, and an idle SM is bandwidth not used. Lanes past the height multiply whatever the ring holds
// there, and nothing reads them.
//
// One CTA per SM and roles that meet only at mbarriers: a warp that issues the TMA copies, one that issues the MMAs, two that
// bring the scales 8 groups at a time, four or eight that read the accumulators back, scale and add them and store a tile.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "fn_fp8.h"
#include "fn_umma.cuh"

namespace fn {

constexpr int FP_RING = 32, FP_ACC = 4, FP_CHUNK = 8;  // ring stages at most; accumulators; groups per chunk of scales

struct Fp8Args {
    CUtensorMap tw, tx;  // codes of the weight, of x: boxes of 128 columns x height, x NT rows
    const float *ws, *xs;
    int m, n, groups, height, tiles_m, tiles, stages;
    int wide;  // 1: rows of out and add in whole 16-byte words
    const void *add;
    int64_t adds;
    void *out;
    int64_t outs;
    uint32_t *err;
};

__device__ __forceinline__ bool fp_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ bool fp_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity), "r"(20000u)
                 : "memory");
    return done != 0;
}
// The whole warp waits until two phases have completed, for about a second at most; ends at once when another role gave up. By
// votes, so that the warp stays together.
__device__ __forceinline__ bool fp_wait_body(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int *fail, uint32_t *err) {
    const uint64_t t0 = global_ns();
    for (;;) {
        if (__all_sync(0xffffffffu, fp_try(bar, parity) && fp_try(bar2, parity2))) return true;
        const bool late = global_ns() - t0 > 1000000000ull;
        if (__any_sync(0xffffffffu, late)) {
            *fail = 1;
            dev_fail(err, DEV_WAIT_TIMEOUT);
            return false;
        }
        if (__any_sync(0xffffffffu, *fail != 0)) return false;
    }
}
// Out of line: the loops that wait are chains of a few dozen dependent instructions, and what lies between them shows in a call's time.
__device__ __noinline__ bool fp_wait_long(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int *fail, uint32_t *err) {
    return fp_wait_body(bar, parity, bar2, parity2, fail, err);
}
// A barrier's phase n (0, 1, ..) has parity n & 1; parity 1 of a new barrier counts as complete, so that what waits for a slot to be
// emptied waits for parity (turn & 1) ^ 1 from the first turn on.
__device__ __forceinline__ bool fp_wait(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int *fail, uint32_t *err) {
    const bool a = fp_try(bar, parity), b = fp_try(bar2, parity2);
    if (__all_sync(0xffffffffu, a && b)) return true;
    return fp_wait_long(bar, parity, bar2, parity2, fail, err);
}
__device__ __forceinline__ bool fp_wait(uint32_t bar, uint32_t parity, volatile int *fail, uint32_t *err) {
    if (__all_sync(0xffffffffu, fp_try(bar, parity))) return true;
    return fp_wait_long(bar, parity, bar, parity, fail, err);
}
__device__ __forceinline__ void fp_tma(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst), "l"(map),
        "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fp_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fp_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fp_prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}
// rows of 128 bytes, swizzled over 8 of them (1024-byte groups, the next 8 rows 1024 bytes on)
__device__ __forceinline__ uint64_t fp_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, e4m3 A and B, both K-major
__host__ __device__ constexpr uint32_t fp_idesc(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void fp_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// N (8, 16 or 32) fp32 columns of this warp's 32 tensor-memory lanes on their way into v; fp_ld_wait before they are used
template <int N> __device__ __forceinline__ void fp_ld(uint32_t taddr, float *v) {
    if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "r"(taddr));
    else if constexpr (N == 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
              "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
            : "r"(taddr));
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
            "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
              "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
              "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
              "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
            : "r"(taddr));
}
// every fp_ld of this warp has arrived; the N values of v are not used before it
template <int N> __device__ __forceinline__ void fp_ld_wait(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

struct Fp8Shared {
    uint64_t full[FP_RING], empty[FP_RING];  // ring stages
    uint64_t af[FP_ACC], ae[FP_ACC];         // accumulators
    uint64_t sf[2], se[2];                   // chunks of scales
    uint64_t done;
    uint32_t tmem;
    int fail;
};

// warps that add: 4 up to 48 columns, else two sets of 4 with half the columns each
constexpr int fp_sets(int nt) { return nt > 48 ? 2 : 1; }

template <typename T, int NT> __global__ void __launch_bounds__(128 + 128 * fp_sets(NT), 1) k_fp8_product(const __grid_constant__ Fp8Args a) {
    constexpr uint32_t COLS = FP_ACC * NT <= 64 ? 64 : FP_ACC * NT <= 128 ? 128 : FP_ACC * NT <= 256 ? 256 : 512;
    constexpr int SETS = fp_sets(NT), NC = NT / SETS;  // columns of a thread
    extern __shared__ uint8_t sm_fp8[];
    __shared__ Fp8Shared sh;
    __shared__ __align__(16) float sc[2][FP_CHUNK][2][NT];  // of a group: the columns' scales times that of either block of the weight
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t a_bytes = (uint32_t)a.height * 128u, stage = a_bytes + NT * 128u;
    uint8_t *const ring = sm_fp8 + (1024 - (smem_u32(sm_fp8) & 1023)) % 1024;  // the swizzle counts from 1024-byte boundaries
    volatile int *const s_fail = &sh.fail;
    if (tid < FP_RING) mbar_init(&sh.full[tid], 1), mbar_init(&sh.empty[tid], 1);
    else if (tid < FP_RING + FP_ACC) mbar_init(&sh.af[tid - FP_RING], 1), mbar_init(&sh.ae[tid - FP_RING], 4 * SETS);
    else if (tid < FP_RING + FP_ACC + 2) mbar_init(&sh.sf[tid - FP_RING - FP_ACC], 64), mbar_init(&sh.se[tid - FP_RING - FP_ACC], 4 * SETS);
    else if (tid == FP_RING + FP_ACC + 2) mbar_init(&sh.done, 1), sh.fail = 0;
    else if (tid == FP_RING + FP_ACC + 3) fp_prefetch_map(&a.tw), fp_prefetch_map(&a.tx);
    if (tid < 64) mbar_fence_init();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();
    pdl_trigger();
    const uint32_t full = smem_u32(sh.full), empty = smem_u32(sh.empty), af = smem_u32(sh.af), ae = smem_u32(sh.ae), base = smem_u32(ring);
    // Warps 0 and 1 run as a whole and one elected lane issues: descriptors and addresses then live in uniform registers (one lane's
    // own MMAs take some 100 cycles each to issue)
    if (warp == 0) {
        const bool lead = fp_elect();
        int i = 0;
        uint32_t s = 0, turn = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % a.tiles_m * NT, n0 = tile / a.tiles_m * a.height;
            for (int g = 0; g < a.groups; ++g, ++i) {
                ok = fp_wait(empty + 8 * s, (turn & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
                if (lead) {
                    fp_expect(full + 8 * s, stage);
                    fp_tma(base + s * stage, &a.tw, g * FP8_GROUP, n0, full + 8 * s);
                    fp_tma(base + s * stage + a_bytes, &a.tx, g * FP8_GROUP, m0, full + 8 * s);
                }
                if (++s == (uint32_t)a.stages) s = 0, ++turn;
            }
        }
        // what was issued has landed before the CTA gives its memory back
        if (!ok)
            for (int j = max(0, i - a.stages); j < i; ++j) mbar_park(&sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u);
    } else if (warp == 1) {
        constexpr uint32_t idesc = fp_idesc(128, NT);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t ad0 = fp_desc(base), bd0 = fp_desc(base + a_bytes);
        const int total = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * a.groups;
        const bool lead = fp_elect();
        uint32_t s = 0, turn = 0;
        for (int i = 0; i < total; ++i) {
            const uint32_t b = (uint32_t)i % FP_ACC;
            if (!fp_wait(full + 8 * s, turn & 1, ae + 8 * b, ((uint32_t)i / FP_ACC & 1) ^ 1, s_fail, a.err)) break;
            tc_fence_after();
            if (lead) {
                const uint32_t at = s * (stage >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) fp_mma(tm + b * NT, ad0 + at + 2u * k, bd0 + at + 2u * k, idesc, k > 0);
                fp_commit(empty + 8 * s);
                fp_commit(af + 8 * b);
            }
            __syncwarp();
            if (++s == (uint32_t)a.stages) s = 0, ++turn;
        }
        if (lead) umma_commit(&sh.done);
        __syncwarp();
        mbar_park(&sh.done, 0);
    } else if (warp < 4) {
        // scales: some groups of a tile at a time
        const int t64 = tid - 64;
        int c = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % a.tiles_m * NT, n0 = tile / a.tiles_m * a.height;
            const int b0 = n0 / FP8_GROUP, b1 = (min(n0 + a.height, a.n) - 1) / FP8_GROUP;
            for (int g0 = 0; g0 < a.groups; g0 += FP_CHUNK, ++c) {
                const int n = min(FP_CHUNK, a.groups - g0), j0 = lane & (FP_CHUNK - 1);
                const float w = a.ws[(int64_t)(lane < FP_CHUNK ? b0 : b1) * a.groups + g0 + min(j0, n - 1)];
                float x[(NT + 63) / 64][FP_CHUNK];
#pragma unroll
                for (int u = 0; u < (NT + 63) / 64; ++u) {
                    const float *p = a.xs + (int64_t)min(m0 + t64 + 64 * u, a.m - 1) * a.groups + g0;
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) x[u][j] = p[min(j, n - 1)];
                }
                ok = fp_wait(smem_u32(&sh.se[c & 1]), ((uint32_t)c / 2 & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < FP_CHUNK; ++j) {
                    const float w0 = __shfl_sync(0xffffffffu, w, j), w1 = __shfl_sync(0xffffffffu, w, FP_CHUNK + j);
#pragma unroll
                    for (int u = 0; u < (NT + 63) / 64; ++u)
                        if (t64 + 64 * u < NT) sc[c & 1][j][0][t64 + 64 * u] = x[u][j] * w0, sc[c & 1][j][1][t64 + 64 * u] = x[u][j] * w1;
                }
                tc_arrive(&sh.sf[c & 1]);
            }
        }
    } else {
        const int row = tid & 127, col = SETS > 1 ? (warp - 4) / 4 * NC : 0;  // this thread's lane of tensor memory, its first column
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)col;
        int i = 0, c = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % a.tiles_m * NT + col, n0 = tile / a.tiles_m * a.height, n = n0 + row;
            const int second = n / FP8_GROUP > n0 / FP8_GROUP;
            float sum[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) sum[j] = 0.0f;
            for (int g = 0; g < a.groups; ++g, ++i) {
                const int b = i % FP_ACC, gc = g % FP_CHUNK;
                ok = fp_wait(af + 8u * b, (uint32_t)i / FP_ACC & 1, smem_u32(&sh.sf[c & 1]), (uint32_t)c / 2 & 1, s_fail, a.err);
                if (!ok) break;
                tc_fence_after();
                float v[NC];
#pragma unroll
                for (int q = 0; q + 16 <= NC; q += 16) fp_ld<16>(tl + (uint32_t)(b * NT + q), v + q);
                if constexpr (NC % 16 != 0) fp_ld<8>(tl + (uint32_t)(b * NT + NC / 16 * 16), v + NC / 16 * 16);
                fp_ld_wait<NC>(v);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&sh.ae[b]);
                const float4 *f = (const float4 *)&sc[c & 1][gc][second][col];
#pragma unroll
                for (int j = 0; j < NC; j += 4) {
                    const float4 x = f[j / 4];
                    sum[j] = fmaf(v[j], x.x, sum[j]);
                    sum[j + 1] = fmaf(v[j + 1], x.y, sum[j + 1]);
                    sum[j + 2] = fmaf(v[j + 2], x.z, sum[j + 2]);
                    sum[j + 3] = fmaf(v[j + 3], x.w, sum[j + 3]);
                }
                if (gc == FP_CHUNK - 1 || g == a.groups - 1) {
                    __syncwarp();
                    if (lane == 0) tc_arrive(&sh.se[c & 1]);
                    ++c;
                }
            }
            if (!ok) break;
            if (row < a.height && n < a.n) {
                const int64_t first = (int64_t)m0 * a.outs + n, first_add = (int64_t)m0 * a.adds + n;
                const T *add = a.add ? (const T *)a.add + first_add : nullptr;
                T *out = (T *)a.out + first;
                constexpr int PER = NC % 16 ? 8 : 16;
                // not unrolled, for the instruction cache (the sums move down instead); loads before stores, which might be to the same place
#pragma unroll 1
                for (int left = min(NC, a.m - m0); left > 0; left -= PER) {
                    float x[PER];
#pragma unroll
                    for (int j = 0; j < PER; ++j) x[j] = add && j < left ? (float)add[j * a.adds] : 0.0f;
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        if (j < left) out[j * a.outs] = (T)(sum[j] + x[j]);
                    if (add) add += PER * a.adds;
                    out += PER * a.outs;
#pragma unroll
                    for (int j = 0; j + PER < NC; ++j) sum[j] = sum[j + PER];
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(COLS) : "memory");
}

// ---- many rows --------------------------------------------------------------------------------------------------------
// Pairs of SMs (cta_group::2) on tiles of 256 rows of x (operand A: 128 lanes of either SM) x 256 rows of the weight (operand B: each
// SM's shared memory holds half, both read all): a code that comes from L2 takes part in 256 products, where two single SMs would
// read each B tile twice. Rows of x on the lanes, so that a thread scales with two numbers a group: 8 warps add 128 columns each.
constexpr int FW_T = 384, FW_RING = 5, FW_PITCH = 36;  // FW_PITCH: floats from row to row of a warp's 32 x 32 values on their way out
constexpr uint32_t FW_OP = 128 * 128, FW_STAGE = 2 * FW_OP;  // bytes of an operand's half in one SM, of a ring stage

struct Fp8WideShared {
    uint64_t full[FW_RING], empty[FW_RING];
    uint64_t af[2][2], ae[2][2];  // accumulators: [columns of either set of adding warps][group parity]
    uint64_t sf[2], se[2];
    uint64_t done;
    uint32_t tmem;
    int fail;
    float xsc[2][FP_CHUNK][128], wsc[2][FP_CHUNK][2];
};

__device__ __forceinline__ uint32_t fw_leader(const void *p) {  // the address of the pair's first CTA
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}
__device__ __forceinline__ void fw_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void fw_tma(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fw_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void fw_commit(uint32_t bar) {  // arrives in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                     bar),
                 "h"((uint16_t)3)
                 : "memory");
}
// after tensor-memory loads and their fence, which order themselves: a release of the cluster would be a memory barrier (measured: half
// of the promoting warps' time)
__device__ __forceinline__ void fw_arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// V values (V > 1: 16 bytes of T) of rows r, r + step, .. < end at column n, from shared memory, plus those of `add`, rounded once. Four
// rows' loads come before their stores, which for all the compiler knows might be to the same place.
template <typename T, int V> __device__ __forceinline__ void fp_copy_out(const float *x, int step, const T *add, int64_t adds, T *out,
                                                                         int64_t outs, int r, int end, int n, int cols) {
    if (n >= cols) return;
    constexpr int B = 4;
    add = add ? add + (int64_t)r * adds + n : nullptr;
    out += (int64_t)r * outs + n;
#pragma unroll 1
    for (; r < end; r += B * step, x += B * step * FW_PITCH, out += B * step * outs, add = add ? add + B * step * adds : nullptr) {
        float v[B][V];
        uint4 w[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const bool in = r + b * step < end;
            if constexpr (V == 1) {
                v[b][0] = x[b * step * FW_PITCH];
                w[b].x = add && in ? __float_as_uint((float)add[b * step * adds]) : 0u;
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 4) *(float4 *)&v[b][j] = *(const float4 *)(x + b * step * FW_PITCH + j);
                w[b] = add && in ? *(const uint4 *)(add + b * step * adds) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (r + b * step >= end) break;
            if constexpr (V == 1) out[b * step * outs] = (T)(v[b][0] + __uint_as_float(w[b].x));
            else {
                uint32_t u[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (V == 4) u[j] = __float_as_uint(v[b][j] + __uint_as_float(u[j]));
                    else {
                        const __nv_bfloat162 z = __floats2bfloat162_rn(v[b][2 * j] + __uint_as_float(u[j] << 16),
                                                                       v[b][2 * j + 1] + __uint_as_float(u[j] & 0xffff0000u));
                        memcpy(&u[j], &z, 4);
                    }
                }
                *(uint4 *)(out + b * step * outs) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }
}

template <typename T> __global__ void __launch_bounds__(FW_T, 1) k_fp8_product_wide(const __grid_constant__ Fp8Args a) {
    extern __shared__ uint8_t sm_fp8[];
    __shared__ Fp8WideShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = blockIdx.x & 1;
    uint8_t *const ring = sm_fp8 + (1024 - (smem_u32(sm_fp8) & 1023)) % 1024;
    float *const stage = (float *)(ring + FW_RING * FW_STAGE);
    volatile int *const s_fail = &sh.fail;
    if (tid < FW_RING) mbar_init(&sh.full[tid], 1), mbar_init(&sh.empty[tid], 1);
    else if (tid < FW_RING + 4) mbar_init(&sh.af[0][0] + (tid - FW_RING), 1), mbar_init(&sh.ae[0][0] + (tid - FW_RING), 8);
    else if (tid < FW_RING + 6) mbar_init(&sh.sf[tid - FW_RING - 4], 64), mbar_init(&sh.se[tid - FW_RING - 4], 8);
    else if (tid == FW_RING + 6) mbar_init(&sh.done, 1), sh.fail = 0;
    else if (tid == FW_RING + 7) fp_prefetch_map(&a.tw), fp_prefetch_map(&a.tx);
    if (tid < 32) mbar_fence_init();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    fw_cluster_sync();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();
    pdl_trigger();
    const uint32_t full = smem_u32(sh.full), empty = smem_u32(sh.empty), af = smem_u32(sh.af), base = smem_u32(ring);
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    // registers: 384 threads of 168 at launch become 128 of 72 and 256 of 216
    if (warp == 0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // either CTA brings its own half of both operands; the copies complete on the first CTA's barrier
        const bool lead = fp_elect();
        const uint32_t full0 = fw_leader(sh.full);
        int i = 0;
        uint32_t s = 0, turn = 0;
        bool ok = true;
        for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
            const int m0 = tile % a.tiles_m * 256 + (int)rank * 128, n0 = tile / a.tiles_m * 256 + (int)rank * 64;
            for (int g = 0; g < a.groups; ++g, ++i) {
                ok = fp_wait(empty + 8 * s, (turn & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
                if (lead) {
                    const uint32_t dst = base + s * FW_STAGE, bar = full0 + 8 * s;
                    if (rank == 0) fp_expect(full + 8 * s, 2 * FW_STAGE);
                    fw_tma(dst, &a.tx, g * FP8_GROUP, m0, bar);
                    fw_tma(dst + FW_OP, &a.tw, g * FP8_GROUP, n0, bar);
                    fw_tma(dst + FW_OP + FW_OP / 2, &a.tw, g * FP8_GROUP, n0 + 128, bar);
                }
                if (++s == FW_RING) s = 0, ++turn;
            }
        }
        if (!ok && rank == 0)
            for (int j = max(0, i - FW_RING); j < i; ++j) mbar_park(&sh.full[j % FW_RING], (uint32_t)(j / FW_RING) & 1u);
    } else if (warp == 1) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (rank == 0) {
            // A group's two halves of 128 columns are accumulators of their own, each emptied by its own warps: an accumulator then has
            // the time of three halves, not of two, between its sums and the next, which the barriers' and the loads' latencies take
            constexpr uint32_t idesc = fp_idesc(256, 128);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), ae = smem_u32(sh.ae);
            const uint64_t ad0 = fp_desc(base), bd0 = fp_desc(base + FW_OP);
            const int total = (a.tiles - pair + pairs - 1) / pairs * a.groups;
            const bool lead = fp_elect();
            uint32_t s = 0, turn = 0;
            bool ok = true;
            for (int i = 0; i < total && ok; ++i) {
                const uint32_t b = (uint32_t)i & 1, at = s * (FW_STAGE >> 4), parity = ((uint32_t)i / 2 & 1) ^ 1;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ok = h ? fp_wait(ae + 16 + 8 * b, parity, s_fail, a.err) : fp_wait(full + 8 * s, turn & 1, ae + 8 * b, parity, s_fail, a.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            fw_mma(tm + b * 256 + h * 128, ad0 + at + 2u * k, bd0 + at + 512u * h + 2u * k, idesc, k > 0);
                        fw_commit(af + 16 * h + 8 * b);
                        if (h) fw_commit(empty + 8 * s);
                    }
                    __syncwarp();
                }
                if (++s == FW_RING) s = 0, ++turn;
            }
            if (lead) fw_commit(smem_u32(&sh.done));
            __syncwarp();
        }
        mbar_park(&sh.done, 0);  // in both CTAs: every MMA has read its operands
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int t64 = tid - 64;
        int c = 0;
        bool ok = true;
        for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
            const int m0 = tile % a.tiles_m * 256 + (int)rank * 128, b0 = tile / a.tiles_m * 2, b1 = min(b0 + 1, (a.n - 1) / FP8_GROUP);
            for (int g0 = 0; g0 < a.groups; g0 += FP_CHUNK, ++c) {
                const int n = min(FP_CHUNK, a.groups - g0), j0 = lane & (FP_CHUNK - 1);
                const float w = a.ws[(int64_t)(lane < FP_CHUNK ? b0 : b1) * a.groups + g0 + min(j0, n - 1)];
                float x[2][FP_CHUNK];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float *p = a.xs + (int64_t)min(m0 + t64 + 64 * u, a.m - 1) * a.groups + g0;
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) x[u][j] = p[min(j, n - 1)];
                }
                ok = fp_wait(smem_u32(&sh.se[c & 1]), ((uint32_t)c / 2 & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < FP_CHUNK; ++j) sh.xsc[c & 1][j][t64] = x[0][j], sh.xsc[c & 1][j][t64 + 64] = x[1][j];
                if (t64 < 2 * FP_CHUNK) sh.wsc[c & 1][j0][t64 / FP_CHUNK] = w;
                tc_arrive(&sh.sf[c & 1]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int row = 32 * (warp & 3) + lane, half = (warp - 4) >> 2;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)(half * 128);
        float *const out_stage = stage + (warp - 4) * (32 * FW_PITCH);
        const uint32_t ae = fw_leader(&sh.ae[half][0]);
        int i = 0, c = 0;
        bool ok = true;
        for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
            const int m0 = tile % a.tiles_m * 256 + (int)rank * 128, n0 = tile / a.tiles_m * 256 + half * 128;
            float sum[128], v[2][32];
#pragma unroll
            for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
            // the columns of a group 32 at a time, the next on their way while some are added, across groups too (but not across the
            // loop's end, where the compiler may move registers that are still to be written)
            auto begin = [&](int g) {  // group g's sums are there (and its scales): its first columns on their way
                const uint32_t full_at = af + 16u * half + 8u * (i & 1), scales_at = smem_u32(&sh.sf[c & 1]);
                const bool sums = fp_try(full_at, (uint32_t)i / 2 & 1), scales = fp_try(scales_at, (uint32_t)c / 2 & 1);
                ok = __all_sync(0xffffffffu, sums && scales) ||  // (a call would want the registers that the sums are in)
                     fp_wait_body(full_at, (uint32_t)i / 2 & 1, scales_at, (uint32_t)c / 2 & 1, s_fail, a.err);
                tc_fence_after();
                if (ok) fp_ld<32>(tl + (uint32_t)((i & 1) * 256), v[0]);
            };
            begin(0);
            fp_ld_wait<32>(v[0]);
            for (int g = 0; g < a.groups && ok; ++g) {
                const int gc = g % FP_CHUNK;
                const float f = sh.xsc[c & 1][gc][row] * sh.wsc[c & 1][gc][half];
                const uint32_t t = tl + (uint32_t)((i & 1) * 256);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (q) fp_ld_wait<32>(v[q & 1]);
                    if (q < 3) fp_ld<32>(t + 32u * (q + 1), v[(q + 1) & 1]);
                    else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            fw_arrive_at(ae + 8u * (uint32_t)(i & 1));
                            if (gc == FP_CHUNK - 1 || g == a.groups - 1) tc_arrive(&sh.se[c & 1]);
                        }
                        if (gc == FP_CHUNK - 1 || g == a.groups - 1) ++c;
                        ++i;
                        if (g + 1 < a.groups) begin(g + 1);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[q * 32 + j] = fmaf(v[q & 1][j], f, sum[q * 32 + j]);
                }
                fp_ld_wait<32>(v[0]);
            }
            if (!ok) break;
            // out by way of shared memory, 32 rows x 32 columns at a time, so that a warp stores whole lines. What is not unrolled here is
            // for the instruction cache: unrolled, a tile's end took 14 us, its code fetched once a tile.
            const T *add = (const T *)a.add;
            T *out = (T *)a.out;
            const int r0 = m0 + 32 * (warp & 3);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                float4 *mine = (float4 *)(out_stage + lane * FW_PITCH);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (q == u) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            mine[j] = make_float4(sum[u * 32 + 4 * j], sum[u * 32 + 4 * j + 1], sum[u * 32 + 4 * j + 2], sum[u * 32 + 4 * j + 3]);
                    }
                __syncwarp();
                const int nq = n0 + q * 32;
                if (a.wide) {
                    constexpr int V = 16 / sizeof(T), L = 32 / V, R = 32 / L;  // values a lane, lanes a row, rows at once
                    fp_copy_out<T, V>(out_stage + lane / L * FW_PITCH + lane % L * V, R, add, a.adds, out, a.outs, r0 + lane / L,
                                      min(a.m, r0 + 32), nq + lane % L * V, a.n);
                } else fp_copy_out<T, 1>(out_stage + lane, 1, add, a.adds, out, a.outs, r0, min(a.m, r0 + 32), nq + lane, a.n);
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    fw_cluster_sync();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

// ---- host: tensor maps, tiles, launch --------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled fp_encoder() {
    static EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return (EncodeTiled) nullptr;
        return (EncodeTiled)p;
    }();
    return f;
}
// codes [rows][cols], boxes of 128 columns (past the last: zeros) x `box` rows
static bool fp_map(CUtensorMap *map, const uint8_t *codes, int rows, int cols, int box) {
    const EncodeTiled enc = fp_encoder();
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols};
    const cuuint32_t bx[2] = {128, (cuuint32_t)box}, es[2] = {1, 1};
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)codes, dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int NT> static cudaError_t fp_launch(Fp8Args &a, cudaStream_t s) {
    auto *k = k_fp8_product<T, NT>;
    cudaError_t e = allow_max_dynamic_smem(k);
    if (e != cudaSuccess) return e;
    const uint32_t stage = (uint32_t)a.height * 128u + NT * 128u;
    // the last stage's operand A reaches 16 KiB from its start whatever its height
    const int room = 227 * 1024 - (int)sizeof(Fp8Shared) - 2 * FP_CHUNK * 2 * NT * 4 - 16 * 1024 - 2048;
    a.stages = std::min(FP_RING, room / (int)stage);
    return launch_k(k, dim3((unsigned)std::min(a.tiles, num_sms())), dim3(128 + 128 * fp_sets(NT)), (size_t)a.stages * stage + 17 * 1024, s, a);
}
template <typename T> static cudaError_t fp_launch_wide(Fp8Args &a, cudaStream_t s) {
    auto *k = k_fp8_product_wide<T>;
    const cudaError_t e = allow_max_dynamic_smem(k);
    if (e != cudaSuccess) return e;
    const size_t smem = FW_RING * FW_STAGE + 8 * 32 * FW_PITCH * sizeof(float) + 1024;
    return launch_kc(k, dim3((unsigned)(2 * std::min(a.tiles, num_sms() / 2))), dim3(FW_T), 2u, smem, s, a);
}
template <typename T> static cudaError_t fp_launch_nt(Fp8Args &a, int nt, cudaStream_t s) {
    switch (nt) {
        case 16: return fp_launch<T, 16>(a, s);
        case 32: return fp_launch<T, 32>(a, s);
        case 48: return fp_launch<T, 48>(a, s);
        case 64: return fp_launch<T, 64>(a, s);
        case 80: return fp_launch<T, 80>(a, s);
        case 96: return fp_launch<T, 96>(a, s);
        case 112: return fp_launch<T, 112>(a, s);
        default: return fp_launch<T, 128>(a, s);
    }
}

}  // namespace fn

using namespace fn;

FN_API int fn_fp8_product(const fn_fp8_t *w, const uint8_t *codes, const float *scales, int rows, uint32_t type, const void *add,
                          int64_t add_stride, void *out, int64_t out_stride, void *stream) {
    return kv4_entry("fp8 product", [&]() -> int {
        if (!w || !w->codes || !w->scales) return fail("fp8 product: no weight");
        if (w->rows < 1 || w->rows > 1 << 28 || w->cols < 16 || w->cols % 16 || w->cols > 1 << 24)
            return fail("fp8 product: bad weight sizes (columns: multiples of 16)");
        if (type != T_F32 && type != T_BF16) return fail("fp8 product: outputs must be F32 or BF16");
        if (rows < 0 || rows > 1 << 28) return fail("fp8 product: bad row count");
        if (rows == 0) return 0;
        if (!codes || !scales || !out) return fail("fp8 product: null pointer");
        if (((uintptr_t)w->codes | (uintptr_t)codes) % 16) return fail("fp8 product: codes must be 16-byte aligned");
        if (((uintptr_t)w->scales | (uintptr_t)scales) % 4 || ((uintptr_t)out | (uintptr_t)add) % (type == T_F32 ? 4 : 2))
            return fail("fp8 product: scales, add and out must be aligned to their types");
        Fp8Args a{};
        a.ws = w->scales, a.xs = scales;
        a.m = rows, a.n = w->rows, a.groups = fp8_groups(w->cols);
        a.add = add, a.adds = add_stride, a.out = out, a.outs = out_stride;
        a.err = dev_error_ptr();
        const int per = type == T_F32 ? 4 : 8;
        a.wide = (((uintptr_t)out | (uintptr_t)add) % 16 | (uint64_t)a.n % per | (uint64_t)out_stride % per | (uint64_t)add_stride % per) == 0;
        if (rows > 512) {
            a.tiles_m = (rows + 255) / 256;
            const int64_t tiles = (int64_t)a.tiles_m * ((a.n + 255) / 256);
            if (tiles * a.groups > INT32_MAX) return fail("fp8 product: too large");
            a.tiles = (int)tiles;
            if (!fp_map(&a.tw, w->codes, w->rows, w->cols, 64) || !fp_map(&a.tx, codes, rows, w->cols, 128))
                return fail("fp8 product: tensor map encoding failed");
            const cudaError_t e = type == T_F32 ? fp_launch_wide<float>(a, (cudaStream_t)stream) : fp_launch_wide<__nv_bfloat16>(a, (cudaStream_t)stream);
            if (e != cudaSuccess) return fail(std::string("fp8 product launch: ") + cudaGetErrorString(e));
            return 0;
        }
        // tiles of x of equal size, up to 128 rows; then the weight rows per tile that fill whole waves of SMs
        a.tiles_m = fp8_groups(rows);
        const int nt = ((rows + a.tiles_m - 1) / a.tiles_m + 15) / 16 * 16;
        const int64_t sms = num_sms(), waves = ((int64_t)fp8_groups(a.n) * a.tiles_m + sms - 1) / sms;
        const int64_t per_n = std::max<int64_t>(waves * sms / a.tiles_m, 1);
        a.height = (int)std::min<int64_t>(128, ((a.n + per_n - 1) / per_n + 7) / 8 * 8);
        const int64_t tiles = (int64_t)((a.n + a.height - 1) / a.height) * a.tiles_m;
        if (tiles * a.groups > INT32_MAX) return fail("fp8 product: too large");
        a.tiles = (int)tiles;
        if (!fp_map(&a.tw, w->codes, w->rows, w->cols, a.height) || !fp_map(&a.tx, codes, rows, w->cols, nt))
            return fail("fp8 product: tensor map encoding failed");
        const cudaError_t e = type == T_F32 ? fp_launch_nt<float>(a, nt, (cudaStream_t)stream) : fp_launch_nt<__nv_bfloat16>(a, nt, (cudaStream_t)stream);
        if (e != cudaSuccess) return fail(std::string("fp8 product launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
