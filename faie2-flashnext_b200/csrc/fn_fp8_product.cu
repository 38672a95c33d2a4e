// Product of 8-bit rows and an 8-bit weight on the 5th-generation tensor cores (tcgen05, kind::f8f6f4):
//
//   out[m][n] = sum_g xs[m][g] ws[n / 128][g] sum_{k in group g} x[m][k] w[n][k]  (+ add[m][n])
//
// The inner sum of a group of 128 is what the tensor core adds up, in its fp32 accumulators in tensor memory; the outer sum is fp32
// in registers, where each group's sum takes its two scales (their product is rounded once to fp32). The reference's k_tgemv
// (engine/faie2fn.cu:734-955) takes up to 8 rows on CUDA cores and no 8-bit floating point.
//
// Which operand lies on the 128 lanes (A) and which on the columns (B) goes by the rows of x:
//   up to 32   (and a large weight) the weight on the lanes, x on 16 or 32 columns, whose scales a thread reads from shared
//              memory, four bytes for each fused multiply-add; few columns to read back and add
//   more       x on the lanes, the weight on up to 128 columns: a thread's sums are of one row, whose scale is one number a group (with
//              128 columns of x their scales alone would take 512 cycles a group of shared memory, where the MMAs take 257)
//   many       as the second, by pairs of SMs on tiles of 256 x 256
// What is past the last row of a tile multiplies whatever the ring holds there, and nothing stores it: few rows cost MMAs, which are not
// what bounds them, but no memory traffic.
//
// Roles meet only at mbarriers: a warp that issues the TMA copies, one that issues the MMAs, two that bring the scales 8 groups at a
// time, four or eight that read the accumulators back, scale and add them and store a tile. The loops are rolled, two groups a step, and
// waits that have nothing to wait for are short: with few rows a call is a chain of such steps (a group took 700 cycles before, its 4
// MMAs 157).
//
// What bounds it: few rows of a large weight its bytes (32 x 151936, K 2048: 54 us, 6.1 TB/s; 1 x 12352: 5.5 us), few rows of a small one that
// chain and the operands from L2 (333 x 2048, K 4096: 11.3 us), many rows the reading back and adding of every group's sums (8192 x 12352, K 2048,
// bf16: 207 us, 2.0 PFLOP/s; 840 cycles a group, its MMAs 512).
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "fn_fp8.h"
#include "fn_umma.cuh"

namespace fn {

constexpr int FP_RING = 32, FP_CHUNK = 8, FP_STEP = 2;  // ring stages at most; groups per chunk of scales, per step of the single SMs

struct Fp8Args {
    CUtensorMap tw, tx;  // codes of the weight, of x: boxes of 128 columns
    const float *ws, *xs;
    int m, n, groups, tiles_m, tiles;
    int width, abox, bbox, stages;  // single SMs: rows of the weight in a tile, rows of A and B that are copied, ring stages
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
// (45 cycles on a completed phase; with a time limit of its own 82)
__device__ __forceinline__ bool fp_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}
// The whole warp waits until two phases have completed, for about a second at most; ends at once when another role gave up. By
// votes, so that the warp stays together.
__device__ __forceinline__ bool fp_wait_body(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int *fail, uint32_t *err) {
    const uint64_t t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 32; ++i)  // the timer is slow to read
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
// CALL false: in line also when it takes long (where registers are split, a call would want those that the sums are in).
template <bool CALL = true>
__device__ __forceinline__ bool fp_wait(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int *fail, uint32_t *err) {
    const bool a = fp_try(bar, parity), b = fp_try(bar2, parity2);
    if (__all_sync(0xffffffffu, a && b)) return true;
    if constexpr (CALL) return fp_wait_long(bar, parity, bar2, parity2, fail, err);
    return fp_wait_body(bar, parity, bar2, parity2, fail, err);
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
template <int N> __device__ __forceinline__ void fp_ld_cols(uint32_t taddr, float *v) {
    if constexpr (N >= 32) {
        fp_ld<32>(taddr, v);
        fp_ld_cols<N - 32>(taddr + 32, v + 32);
    } else if constexpr (N >= 16) {
        fp_ld<16>(taddr, v);
        fp_ld_cols<N - 16>(taddr + 16, v + 16);
    } else if constexpr (N >= 8) fp_ld<8>(taddr, v);
}
// every fp_ld of this warp has arrived; the N values of v are not used before it
template <int N> __device__ __forceinline__ void fp_ld_wait(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

constexpr int FP_PITCH = 36;  // floats from row to row of a warp's 32 x 32 values on their way out (rows 4 banks apart)

// columns n0 .. < end of row `row` of `add` on their way into L2 before their tile ends (8192 x 12352, K 2048, bf16: 303 -> 287 us, fp32 413 ->
// 384)
template <typename T> __device__ __forceinline__ void fp_add_ahead(const Fp8Args &a, int row, int n0, int end) {
    if (row >= a.m) return;
    const T *const p = (const T *)a.add + row * a.adds;
    for (int n = n0; n < end; n += 128 / (int)sizeof(T)) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p + n) : "memory");
}

// A warp's 32 rows x W columns, from row r0 and column n0 on, on their way out: V values a lane (V > 1: 16 bytes of T), B rows at R a time.
// `add` is read before the stores, which for all the compiler knows might be to the same place, for as many rows as registers hold: all of
// them in whole words, whose reads (begin) run while the sums go through shared memory.
template <typename T, int V, int W, bool ADD> struct FpOut {
    static constexpr int L = W / V, R = 32 / L, B = V == 1 ? 16 / R : 32 / R;  // lanes a row, rows at once, times that before stores
    uint4 w[ADD ? B : 1];
    int lane, rows;
    bool in;
    const T *add;
    T *out;
    __device__ __forceinline__ void begin(const Fp8Args &a, int r0, int n0, int end) {
        lane = threadIdx.x & 31;
        const int n = n0 + lane % L * V, r = r0 + lane / L;
        in = n < end && r < a.m;
        rows = a.m - r;  // from this lane's first one on
        out = (T *)a.out + (int64_t)r * a.outs + n;
        if (ADD) {
            add = (const T *)a.add + (int64_t)r * a.adds + n;
            if (V > 1 && in) read(a.adds, 0);
        }
    }
    __device__ __forceinline__ void read(int64_t adds, int at) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const T *p = add + (at + b * R < rows ? at + b * R : 0) * adds;
            if constexpr (V == 1) w[b].x = __float_as_uint((float)*p);
            else w[b] = *(const uint4 *)p;
        }
    }
    __device__ __forceinline__ void end(const Fp8Args &a, const float *stage) {
        if (!in) return;
        const float *x = stage + lane / L * FP_PITCH + lane % L * V;
#pragma unroll 1
        for (int at = 0; at < 32; at += B * R) {
            if (ADD && V == 1) read(a.adds, at);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                if (at + b * R >= rows) break;
                T *const to = out + (at + b * R) * a.outs;
                const float *from = x + (at + b * R) * FP_PITCH;
                if constexpr (V == 1) *to = (T)(*from + (ADD ? __uint_as_float(w[b].x) : 0.0f));
                else {
                    float v[V];
#pragma unroll
                    for (int j = 0; j < V; j += 4) *(float4 *)&v[j] = *(const float4 *)(from + j);
                    uint32_t u[4];
                    const uint32_t e[4] = {w[ADD ? b : 0].x, w[ADD ? b : 0].y, w[ADD ? b : 0].z, w[ADD ? b : 0].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (V == 4) u[j] = __float_as_uint(ADD ? v[j] + __uint_as_float(e[j]) : v[j]);
                        else {
                            if (ADD) v[2 * j] += __uint_as_float(e[j] << 16), v[2 * j + 1] += __uint_as_float(e[j] & 0xffff0000u);
                            const __nv_bfloat162 z = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                            memcpy(&u[j], &z, 4);
                        }
                    }
                    *(uint4 *)to = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        }
    }
};
// N sums a thread, its row's columns n0 .. < end of out, by way of shared memory, 32 rows x up to 32 words at a time, so that a warp stores
// whole lines. What is not unrolled here is for the instruction cache: unrolled, a tile's end took 14 us, its code fetched once a tile; kernels
// with and without `add` for the same reason (8192 x 12352, K 2048, bf16: 237 -> 228 us). WIDE: rows in whole 16-byte words, -1: as a.wide says.
template <typename T, int N, bool ADD, int WIDE = -1>
__device__ __forceinline__ void fp_tile_out(const Fp8Args &a, float *stage, const float (&sum)[N], int r0, int n0, int end) {
    if constexpr (!ADD && sizeof(T) == 2 && WIDE != 0) {
        if (WIDE > 0 || a.wide) {  // rounded before, two values a word: half the way through shared memory (228 -> 207 us)
            constexpr int M = N / 2, W = M % 32 == 0 ? 32 : M % 16 == 0 ? 16 : M % 8 == 0 ? 8 : 4, L = W / 4, R = 32 / L;  // words; lanes a row, rows at once
            const int lane = threadIdx.x & 31, rows = min(a.m - r0, 32);
            uint4 *mine = (uint4 *)(stage + lane * FP_PITCH);
            const uint4 *from = (const uint4 *)(stage + lane / L * FP_PITCH) + lane % L;
            T *out = (T *)a.out + (int64_t)(r0 + lane / L) * a.outs + n0 + lane % L * 8;
#pragma unroll 1
            for (int q = 0; q < M / W; ++q) {
#pragma unroll
                for (int u = 0; u < M / W; ++u)
                    if (q == u) {
#pragma unroll
                        for (int j = 0; j < L; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const __nv_bfloat162 z = __floats2bfloat162_rn(sum[2 * (u * W + 4 * j + k)], sum[2 * (u * W + 4 * j + k) + 1]);
                                memcpy(&w[k], &z, 4);
                            }
                            mine[j] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                __syncwarp();
                if (n0 + 2 * (q * W) + lane % L * 8 < end) {
#pragma unroll
                    for (int b = 0; b < L; ++b)
                        if (lane / L + b * R < rows) *(uint4 *)(out + 2 * (q * W) + b * R * a.outs) = from[b * R * (FP_PITCH / 4)];
                }
                __syncwarp();
            }
            return;
        }
    }
    auto go = [&]<int V>() {
        constexpr int W = N % 32 == 0 ? 32 : N % 16 == 0 ? 16 : 8;
        float4 *mine = (float4 *)(stage + (threadIdx.x & 31) * FP_PITCH);
#pragma unroll 1
        for (int q = 0; q < N / W; ++q) {
            FpOut<T, V, W, ADD> o;
            o.begin(a, r0, n0 + q * W, end);
#pragma unroll
            for (int u = 0; u < N / W; ++u)
                if (q == u) {
#pragma unroll
                    for (int j = 0; j < W / 4; ++j)
                        mine[j] = make_float4(sum[u * W + 4 * j], sum[u * W + 4 * j + 1], sum[u * W + 4 * j + 2], sum[u * W + 4 * j + 3]);
                }
            __syncwarp();
            o.end(a, stage);
            __syncwarp();
        }
    };
    if (WIDE < 0 ? a.wide : WIDE) go.template operator()<16 / (int)sizeof(T)>();
    else go.template operator()<1>();
}

// ---- single SMs -----------------------------------------------------------------------------------------------------
// FEW: up to N (16 or 32) rows of x, tiles of `width` rows of the weight. Else tiles of 128 rows of x by `width` rows of the weight. The
// width, a multiple of 8, is chosen so that the tiles fill whole waves of SMs (N: what the MMAs and the adding warps take, width or
// more); a tile may lie across two blocks of the weight.
constexpr int fp_sets(int n, bool few) { return !few && n > 32 ? 2 : 1; }  // sets of four warps that add, each its share of the columns
constexpr int fp_acc(int n) { return n > 64 ? 2 : 4; }                     // steps whose sums tensor memory holds
constexpr int fp_stage(int n) { return n > 64 ? 1 : 2; }                   // groups of a ring stage

template <int N, bool FEW> struct Fp8Shared {
    uint64_t full[FP_RING], empty[FP_RING];
    uint64_t af[4], ae[4];  // accumulators
    uint64_t sf[2], se[2];  // chunks of scales
    uint64_t done;
    uint32_t tmem;
    int fail;
    // scales: of the tile's rows of x and of its blocks of the weight, the first and the last; FEW: of either block times the rows'
    float xsc[2][FP_CHUNK][FEW ? 4 : 128], wsc[2][FP_CHUNK][2];
    alignas(16) float both[2][FP_CHUNK][2][FEW ? N : 4];
};

template <typename T, int N, bool FEW, bool ADD>
__global__ void __launch_bounds__(128 + 128 * fp_sets(N, FEW), 1) k_fp8_product(const __grid_constant__ Fp8Args a) {
    constexpr int SETS = fp_sets(N, FEW), NC = N / SETS, U = FP_STEP, G = fp_stage(N), ACC = fp_acc(N);  // NC: columns of a thread
    constexpr uint32_t USED = ACC * U * N, COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
    extern __shared__ uint8_t sm_fp8[];
    __shared__ Fp8Shared<N, FEW> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t a_bytes = (uint32_t)a.abox * 128u, group = a_bytes + (uint32_t)a.bbox * 128u, stage = G * group;
    uint8_t *const ring = sm_fp8 + (1024 - (smem_u32(sm_fp8) & 1023)) % 1024;  // the swizzle counts from 1024-byte boundaries
    volatile int *const s_fail = &sh.fail;
    if (tid < FP_RING) mbar_init(&sh.full[tid], 1), mbar_init(&sh.empty[tid], 1);
    else if (tid < FP_RING + 4) mbar_init(&sh.af[tid - FP_RING], 1), mbar_init(&sh.ae[tid - FP_RING], 4 * SETS);
    else if (tid < FP_RING + 6) mbar_init(&sh.sf[tid - FP_RING - 4], 64), mbar_init(&sh.se[tid - FP_RING - 4], 4 * SETS);
    else if (tid == FP_RING + 6) mbar_init(&sh.done, 1), sh.fail = 0;
    else if (tid == FP_RING + 7) fp_prefetch_map(&a.tw), fp_prefetch_map(&a.tx);
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
    const int steps = (a.groups + U - 1) / U;  // of a tile; past the last group there are zeros
    // Warps 0 and 1 run as a whole and one elected lane issues: descriptors and addresses then live in uniform registers (one lane's
    // own MMAs take some 100 cycles each to issue)
    if (warp == 0) {
        const bool lead = fp_elect();
        int i = 0;
        uint32_t s = 0, turn = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int a0 = FEW ? tile * a.width : tile % a.tiles_m * 128, b0 = FEW ? 0 : tile / a.tiles_m * a.width;
            for (int g = 0; g < steps * U; g += G, ++i) {
                ok = fp_wait(empty + 8 * s, (turn & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
                if (lead) {
                    fp_expect(full + 8 * s, stage);
#pragma unroll
                    for (int u = 0; u < G; ++u) {
                        const uint32_t dst = base + s * stage + u * group;
                        fp_tma(dst, FEW ? &a.tw : &a.tx, (g + u) * FP8_GROUP, a0, full + 8 * s);
                        fp_tma(dst + a_bytes, FEW ? &a.tx : &a.tw, (g + u) * FP8_GROUP, b0, full + 8 * s);
                    }
                }
                if (++s == (uint32_t)a.stages) s = 0, ++turn;
            }
        }
        // what was issued has landed before the CTA gives its memory back
        if (!ok)
            for (int j = max(0, i - a.stages); j < i; ++j) mbar_park(&sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u);
    } else if (warp == 1) {
        constexpr uint32_t idesc = fp_idesc(128, N);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t ad0 = fp_desc(base), bd0 = fp_desc(base + a_bytes);
        const int total = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * steps;
        const bool lead = fp_elect();
        uint32_t s = 0, turn = 0;
        bool ok = true;
        for (int i = 0; i < total && ok; ++i) {
            const uint32_t b = (uint32_t)i % ACC;
#pragma unroll
            for (int h = 0; h < U / G; ++h) {
                ok = h ? fp_wait(full + 8 * s, turn & 1, s_fail, a.err)
                       : fp_wait(full + 8 * s, turn & 1, ae + 8 * b, ((uint32_t)i / ACC & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
                tc_fence_after();
                if (lead) {
#pragma unroll
                    for (int u = 0; u < G; ++u) {
                        const uint32_t at = (s * stage + u * group) >> 4;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            fp_mma(tm + (b * U + h * G + u) * N, ad0 + at + 2u * k, bd0 + at + 2u * k, idesc, k > 0);
                    }
                    fp_commit(empty + 8 * s);
                    if (h == U / G - 1) fp_commit(af + 8 * b);
                }
                __syncwarp();
                if (++s == (uint32_t)a.stages) s = 0, ++turn;
            }
        }
        if (lead) umma_commit(&sh.done);
        __syncwarp();
        mbar_park(&sh.done, 0);
    } else if (warp < 4) {
        constexpr int R = FEW ? 1 : 2;  // rows of x a thread
        const int t = tid - 64;
        int c = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = FEW ? 0 : tile % a.tiles_m * 128, n0 = (FEW ? tile : tile / a.tiles_m) * a.width;
            const int64_t b0 = n0 / FP8_GROUP, b1 = (min(n0 + a.width, a.n) - 1) / FP8_GROUP;
            for (int g0 = 0; g0 < a.groups; g0 += FP_CHUNK, ++c) {
                const int n = min(FP_CHUNK, a.groups - g0), jw = t & (FP_CHUNK - 1);
                const float w = jw < n ? a.ws[(t & FP_CHUNK ? b1 : b0) * a.groups + g0 + jw] : 0.0f;
                float x[R][FP_CHUNK];
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const float *p = a.xs + (int64_t)min(m0 + t + 64 * u, a.m - 1) * a.groups + g0;
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) x[u][j] = j < n ? p[j] : 0.0f;
                }
                ok = fp_wait(smem_u32(&sh.se[c & 1]), ((uint32_t)c / 2 & 1) ^ 1, s_fail, a.err);
                if (!ok) break;
                if constexpr (FEW) {
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) {
                        const float w0 = __shfl_sync(0xffffffffu, w, j), w1 = __shfl_sync(0xffffffffu, w, FP_CHUNK + j);
                        if (t < N) sh.both[c & 1][j][0][t] = x[0][j] * w0, sh.both[c & 1][j][1][t] = x[0][j] * w1;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) sh.xsc[c & 1][j][t] = x[0][j], sh.xsc[c & 1][j][t + 64] = x[R - 1][j];
                    if (t < 2 * FP_CHUNK) sh.wsc[c & 1][jw][t / FP_CHUNK] = w;
                }
                tc_arrive(&sh.sf[c & 1]);
            }
        }
    } else {
        const int row = tid & 127, col = SETS > 1 ? (warp - 4) / 4 * NC : 0;  // this thread's lane of tensor memory, its first column
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)col;
        float *const out_stage = (float *)(ring + a.stages * stage) + (warp - 4) * (32 * FP_PITCH);
        int i = 0, c = 0;
        bool ok = true;
        auto add_ahead = [&](int tile) {  // a thread a row of x
            if (!ADD || tile >= a.tiles) return;
            const int n0 = (FEW ? tile : tile / a.tiles_m) * a.width + col, end = min(min(n0 + NC, n0 - col + a.width), a.n);
            if constexpr (FEW) {
                if (warp == 4) fp_add_ahead<T>(a, lane, n0, min(n0 + a.width, a.n));
            } else fp_add_ahead<T>(a, tile % a.tiles_m * 128 + row, n0, end);
        };
        add_ahead(blockIdx.x);
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            add_ahead(tile + gridDim.x);
            const int r0 = (FEW ? 0 : tile % a.tiles_m * 128) + 32 * (warp & 3), first = (FEW ? tile : tile / a.tiles_m) * a.width;
            const int edge = (first / FP8_GROUP + 1) * FP8_GROUP - first;  // the tile's rows of the weight from it on are of the second block
            const int end = min(first + a.width, a.n);
            const bool live = FEW ? 32 * (warp & 3) < a.width : r0 < a.m;
            float sum[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) sum[j] = 0.0f;
            for (int g = 0; g < steps; ++g, ++i) {
                const int b = i % ACC, gc = g * U % FP_CHUNK;
                const bool last = gc + U >= FP_CHUNK || g == steps - 1;  // of this chunk of scales
                ok = fp_wait(af + 8u * b, (uint32_t)i / ACC & 1, smem_u32(&sh.sf[c & 1]), (uint32_t)c / 2 & 1, s_fail, a.err);
                if (!ok) break;
                tc_fence_after();
                // a step's columns in P parts of Q: two parts in registers, one on its way while the other is added (or both, if that is all)
                constexpr int Q = NC > 32 ? NC / 2 : NC, P = U * NC / Q;
                float v[2][Q], f[U][2];
                if (live) {
                    constexpr int H = NC / Q;  // parts of a group
                    const uint32_t t = tl + (uint32_t)(b * U * N);
                    fp_ld_cols<Q>(t, v[0]);
                    if constexpr (P == 2) fp_ld_cols<Q>(t + (uint32_t)(1 / H * N + 1 % H * Q), v[1]);
                    if constexpr (!FEW) {
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const float x = sh.xsc[c & 1][gc + u][row];
                            f[u][0] = x * sh.wsc[c & 1][gc + u][0];
                            f[u][1] = x * sh.wsc[c & 1][gc + u][1];
                        }
                    }
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const int u = p / H, j0 = p % H * Q;
                        if (P == 2) {  // both at once
                            if (p == 0) fp_ld_wait<Q>(v[0]), fp_ld_wait<Q>(v[1]);
                        } else {
                            fp_ld_wait<Q>(v[p & 1]);
                            if (p + 1 < P) fp_ld_cols<Q>(t + (uint32_t)((p + 1) / H * N + (p + 1) % H * Q), v[(p + 1) & 1]);
                        }
                        if (P == 2 ? p == 0 : p == P - 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) tc_arrive(&sh.ae[b]);
                        }
                        if constexpr (FEW) {
                            const float4 *s = (const float4 *)&sh.both[c & 1][gc + u][row >= edge][j0];
#pragma unroll
                            for (int j = 0; j < Q; j += 4) {
                                const float4 x = s[j / 4];
                                sum[j0 + j] = fmaf(v[p & 1][j], x.x, sum[j0 + j]);
                                sum[j0 + j + 1] = fmaf(v[p & 1][j + 1], x.y, sum[j0 + j + 1]);
                                sum[j0 + j + 2] = fmaf(v[p & 1][j + 2], x.z, sum[j0 + j + 2]);
                                sum[j0 + j + 3] = fmaf(v[p & 1][j + 3], x.w, sum[j0 + j + 3]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < Q; ++j)
                                sum[j0 + j] = fmaf(v[p & 1][j], (j0 + j) / 8 * 8 < edge - col ? f[u][0] : f[u][1], sum[j0 + j]);
                        }
                    }
                } else if (lane == 0) tc_arrive(&sh.ae[b]);
                if (last) {
                    __syncwarp();
                    if (lane == 0) tc_arrive(&sh.se[c & 1]);
                    ++c;
                }
            }
            if (!ok) break;
            if constexpr (!FEW) {
                if (live) fp_tile_out<T, NC, ADD>(a, out_stage, sum, r0, first + col, end);
            } else if (first + row < end) {
                const T *add = ADD ? (const T *)a.add + first + row : nullptr;
                T *out = (T *)a.out + first + row;
                // 16 rows at a time, not unrolled, for the instruction cache (the sums move down instead); loads before the stores, which
                // for all the compiler knows might be to the same place
#pragma unroll 1
                for (int left = a.m; left > 0; left -= 16) {
                    float x[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = ADD && j < left ? (float)add[j * a.adds] : 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j < left) out[j * a.outs] = (T)(sum[j] + x[j]);
                    if (ADD) add += 16 * a.adds;
                    out += 16 * a.outs;
#pragma unroll
                    for (int j = 0; j + 16 < NC; ++j) sum[j] = sum[j + 16];
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
constexpr int FW_T = 384, FW_RING = 5;
constexpr uint32_t FW_OP = 128 * 128, FW_STAGE = 2 * FW_OP;  // bytes of an operand's half in one SM, of a ring stage

struct Fp8WideShared {
    uint64_t full[FW_RING], empty[FW_RING];
    uint64_t af[2], ae[2], sf[2], se[2];
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
__device__ __forceinline__ void fw_commit_here(uint32_t bar) {  // arrives in this CTA
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// after tensor-memory loads and their fence, which order themselves: a release of the cluster would be a memory barrier (measured: half
// of the promoting warps' time)
__device__ __forceinline__ void fw_arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
template <typename T, bool ADD, bool WIDE> __global__ void __launch_bounds__(FW_T, 1) k_fp8_product_wide(const __grid_constant__ Fp8Args a) {
    extern __shared__ uint8_t sm_fp8[];
    __shared__ Fp8WideShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = blockIdx.x & 1;
    uint8_t *const ring = sm_fp8 + (1024 - (smem_u32(sm_fp8) & 1023)) % 1024;
    float *const stage = (float *)(ring + FW_RING * FW_STAGE);
    volatile int *const s_fail = &sh.fail;
    if (tid < FW_RING) mbar_init(&sh.full[tid], 1), mbar_init(&sh.empty[tid], 1);
    else if (tid < FW_RING + 2) mbar_init(&sh.af[tid - FW_RING], 1), mbar_init(&sh.ae[tid - FW_RING], 16);
    else if (tid < FW_RING + 4) mbar_init(&sh.sf[tid - FW_RING - 2], 64), mbar_init(&sh.se[tid - FW_RING - 2], 8);
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
    // registers: 384 threads of 168 at launch become 128 of 72 and 256 of 216. All warps of a warpgroup change theirs by the same instruction
    // (PTX leaves anything else undefined), before their roles part.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            // either CTA brings its own half of both operands; the copies complete on the first CTA's barrier
            const bool lead = fp_elect();
            const uint32_t full0 = fw_leader(sh.full);
            int i = 0;
            uint32_t s = 0, turn = 0;
            bool ok = true;
            for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
                const int m0 = tile % a.tiles_m * 256 + (int)rank * 128, n0 = tile / a.tiles_m * 256 + (int)rank * 128;
                for (int g = 0; g < a.groups; ++g, ++i) {
                    ok = fp_wait(empty + 8 * s, (turn & 1) ^ 1, s_fail, a.err);
                    if (!ok) break;
                    if (lead) {
                        const uint32_t dst = base + s * FW_STAGE, bar = full0 + 8 * s;
                        if (rank == 0) fp_expect(full + 8 * s, 2 * FW_STAGE);
                        fw_tma(dst, &a.tx, g * FP8_GROUP, m0, bar);
                        fw_tma(dst + FW_OP, &a.tw, g * FP8_GROUP, n0, bar);
                    }
                    if (++s == FW_RING) s = 0, ++turn;
                }
            }
            if (!ok && rank == 0)
                for (int j = max(0, i - FW_RING); j < i; ++j) mbar_park(&sh.full[j % FW_RING], (uint32_t)(j / FW_RING) & 1u);
        } else if (warp == 1) {
            if (rank == 0) {
                constexpr uint32_t idesc = fp_idesc(256, 256);
                const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), ae = smem_u32(sh.ae);
                const uint64_t ad0 = fp_desc(base), bd0 = fp_desc(base + FW_OP);
                const int total = (a.tiles - pair + pairs - 1) / pairs * a.groups;
                const bool lead = fp_elect();
                uint32_t s = 0, turn = 0;
                bool ok = true;
                for (int i = 0; i < total && ok; ++i) {
                    const uint32_t b = (uint32_t)i & 1, at = s * (FW_STAGE >> 4), parity = ((uint32_t)i / 2 & 1) ^ 1;
                    ok = fp_wait(full + 8 * s, turn & 1, ae + 8 * b, parity, s_fail, a.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) fw_mma(tm + b * 256, ad0 + at + 2u * k, bd0 + at + 2u * k, idesc, k > 0);
                        fw_commit(af + 8 * b);
                        fw_commit(empty + 8 * s);
                    }
                    __syncwarp();
                    if (++s == FW_RING) s = 0, ++turn;
                }
                if (lead) fw_commit_here(smem_u32(&sh.done));
                __syncwarp();
                mbar_park(&sh.done, 0);  // every MMA has read its operands (the other CTA waits for this one at the end)
            }
        } else {
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
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int row = 32 * (warp & 3) + lane, half = (warp - 4) >> 2;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)(half * 128);
        float *const out_stage = stage + (warp - 4) * (32 * FP_PITCH);
        const uint32_t ae = fw_leader(sh.ae);
        int i = 0, c = 0;
        bool ok = true;
        for (int tile = pair; tile < a.tiles && ok; tile += pairs) {
            const int m0 = tile % a.tiles_m * 256 + (int)rank * 128, n0 = tile / a.tiles_m * 256 + half * 128;
            if (ADD) fp_add_ahead<T>(a, m0 + row, n0, min(n0 + 128, a.n));
            float sum[128], v[2][32];
#pragma unroll
            for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
            // the columns of a group 32 at a time, the next on their way while some are added, across groups too (but not across the
            // loop's end, where the compiler may move registers that are still to be written)
            auto begin = [&](int g) {  // group g's sums are there (and its scales): its first columns on their way
                ok = fp_wait<false>(af + 8u * (i & 1), (uint32_t)i / 2 & 1, smem_u32(&sh.sf[c & 1]), (uint32_t)c / 2 & 1, s_fail, a.err);
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
            fp_tile_out<T, 128, ADD, WIDE>(a, out_stage, sum, m0 + 32 * (warp & 3), n0, a.n);
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

template <typename T> static cudaError_t fp_launch_wide(Fp8Args &a, cudaStream_t s) {
    auto *k = a.add ? (a.wide ? k_fp8_product_wide<T, true, true> : k_fp8_product_wide<T, true, false>)
                    : (a.wide ? k_fp8_product_wide<T, false, true> : k_fp8_product_wide<T, false, false>);
    const cudaError_t e = allow_max_dynamic_smem(k);
    if (e != cudaSuccess) return e;
    const size_t smem = FW_RING * FW_STAGE + 8 * 32 * FP_PITCH * sizeof(float) + 1024;
    return launch_kc(k, dim3((unsigned)(2 * std::min(a.tiles, num_sms() / 2))), dim3(FW_T), 2u, smem, s, a);
}
template <typename T, int N, bool FEW> static cudaError_t fp_launch(Fp8Args &a, cudaStream_t s) {
    auto *k = a.add ? k_fp8_product<T, N, FEW, true> : k_fp8_product<T, N, FEW, false>;
    const cudaError_t e = allow_max_dynamic_smem(k);
    if (e != cudaSuccess) return e;
    constexpr int sets = fp_sets(N, FEW), out = FEW ? 0 : 4 * sets * 32 * FP_PITCH * (int)sizeof(float);
    const int stage = fp_stage(N) * (a.abox + a.bbox) * 128;
    // behind the ring the tile on its way out, and 16 KiB at least: either operand of a group reaches 16 KiB from its start, whatever
    // the rows that are copied
    const int tail = std::max(16 * 1024, out);
    a.stages = std::min(FP_RING, (227 * 1024 - (int)sizeof(Fp8Shared<N, FEW>) - tail - 2048) / stage);
    return launch_k(k, dim3((unsigned)std::min(a.tiles, num_sms())), dim3(128 + 128 * sets), (size_t)a.stages * stage + tail + 1024, s, a);
}
template <typename T> static cudaError_t fp_launch_n(Fp8Args &a, bool few, cudaStream_t s) {
    if (few) return a.m <= 16 ? fp_launch<T, 16, true>(a, s) : fp_launch<T, 32, true>(a, s);
    if (a.width <= 16) return fp_launch<T, 16, false>(a, s);
    if (a.width <= 32) return fp_launch<T, 32, false>(a, s);
    if (a.width <= 48) return fp_launch<T, 48, false>(a, s);
    if (a.width <= 64) return fp_launch<T, 64, false>(a, s);
    if (a.width <= 96) return fp_launch<T, 96, false>(a, s);
    return fp_launch<T, 128, false>(a, s);
}

}  // namespace fn

using namespace fn;

FN_API int fn_fp8_product(const fn_fp8_t *w, const uint8_t *codes, const float *scales, int rows, uint32_t type, const void *add,
                          int64_t add_stride, void *out, int64_t out_stride, void *stream) {
    return kv4_entry("fp8 product", [&]() -> int {
        if (!w || !w->codes || !w->scales) return fail("fp8 product: no weight");
        if (w->rows < 1 || w->rows > 1 << 28 || w->cols < 16 || w->cols % 16 || w->cols > FP8_MAX_COLS)
            return fail("fp8 product: bad weight sizes (columns: multiples of 16)");
        if (type != T_F32 && type != T_BF16) return fail("fp8 product: outputs must be F32 or BF16");
        if (rows < 0 || rows > 1 << 28) return fail("fp8 product: bad row count");
        if (rows == 0) return 0;
        if (!codes || !scales || !out) return fail("fp8 product: null pointer");
        if (((uintptr_t)w->codes | (uintptr_t)codes) % 16) return fail("fp8 product: codes must be 16-byte aligned");
        if (((uintptr_t)w->scales | (uintptr_t)scales) % 4 || ((uintptr_t)out | (uintptr_t)add) % (type == T_F32 ? 4 : 2))
            return fail("fp8 product: scales, add and out must be aligned to their types");
        const int size = type == T_F32 ? 4 : 2;
        if (rows > 1 && out_stride < w->rows) return fail("fp8 product: rows of out overlap");
        if (rows_mixed(out, out_stride, add, add_stride, rows, w->rows, size))
            return fail("fp8 product: out lies over other rows of add");
        const int64_t groups = fp8_groups(w->cols);
        auto meets = [&](const void *q, int64_t n) { return rows_meet_bytes(out, out_stride * size, rows, (int64_t)w->rows * size, q, n); };
        if (meets(codes, (int64_t)rows * w->cols) || meets(scales, rows * groups * 4) || meets(w->codes, (int64_t)w->rows * w->cols) ||
            meets(w->scales, fp8_groups(w->rows) * groups * 4))
            return fail("fp8 product: out lies over codes or scales");
        Fp8Args a{};
        a.ws = w->scales, a.xs = scales;
        a.m = rows, a.n = w->rows, a.groups = fp8_groups(w->cols);
        a.add = add, a.adds = add_stride, a.out = out, a.outs = out_stride;
        a.err = dev_error_ptr();
        const int per = type == T_F32 ? 4 : 8;
        a.wide = (((uintptr_t)out | (uintptr_t)add) % 16 | (uint64_t)a.n % per | (uint64_t)out_stride % per | (uint64_t)add_stride % per) == 0;
        const int64_t sms = num_sms(), tm = fp8_groups(rows), waves = (fp8_groups(a.n) * tm + sms - 1) / sms;  // of tiles of 128 x 128
        const int64_t wide_tiles = (int64_t)((rows + 255) / 256) * ((a.n + 255) / 256), wide_waves = (wide_tiles + sms / 2 - 1) / (sms / 2);
        // A group takes a pair of SMs 0.47 to 0.50 us for 256 x 256, a single one 0.33 us for 128 x 128 (K 4096 less K 2048): pairs where
        // their fewer waves save more than that. 768 x 12352, K 2048, fp32: 25.3 us by pairs, 30.1 by single SMs; 512 x 12352: 24.3 and
        // 23.0; 1024 x 2048, K 4096: 20.7 and 14.8; 2048 x 2048: 21.8 and 26.6.
        if (3 * wide_waves < 2 * waves && sms >= 2) {
            a.tiles_m = (rows + 255) / 256;
            if (wide_tiles * a.groups > INT32_MAX) return fail("fp8 product: too large");
            a.tiles = (int)wide_tiles;
            if (!fp_map(&a.tw, w->codes, w->rows, w->cols, 128) || !fp_map(&a.tx, codes, rows, w->cols, 128))
                return fail("fp8 product: tensor map encoding failed");
            const cudaError_t e = type == T_F32 ? fp_launch_wide<float>(a, (cudaStream_t)stream) : fp_launch_wide<__nv_bfloat16>(a, (cudaStream_t)stream);
            if (e != cudaSuccess) return fail(std::string("fp8 product launch: ") + cudaGetErrorString(e));
            return 0;
        }
        // the rows of the weight per tile that fill whole waves of SMs; the weight on the lanes where that is more of them than rows of x
        // (32 rows, K 2048: 7.3 us on the lanes, 9.3 on the columns for 12352 in tiles of 88, 6.9 and 5.5 for 2048 in tiles of 16)
        const int box = std::min(128, (rows + 7) / 8 * 8);
        a.tiles_m = (int)tm;
        const int64_t per_n = std::max<int64_t>(waves * sms / tm, 1);
        a.width = (int)std::min<int64_t>(128, ((a.n + per_n - 1) / per_n + 7) / 8 * 8);
        const bool few = rows <= 32 && a.width > 32;
        a.abox = few ? a.width : box, a.bbox = few ? box : a.width;
        const int64_t tiles = (int64_t)((a.n + a.width - 1) / a.width) * a.tiles_m;
        if (tiles * (a.groups + 1) > INT32_MAX) return fail("fp8 product: too large");
        a.tiles = (int)tiles;
        if (!fp_map(&a.tw, w->codes, w->rows, w->cols, a.width) || !fp_map(&a.tx, codes, rows, w->cols, box))
            return fail("fp8 product: tensor map encoding failed");
        const cudaError_t e = type == T_F32 ? fp_launch_n<float>(a, few, (cudaStream_t)stream) : fp_launch_n<__nv_bfloat16>(a, few, (cudaStream_t)stream);
        if (e != cudaSuccess) return fail(std::string("fp8 product launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
