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
// One CTA per SM and roles that meet only at mbarriers: a warp that issues the TMA copies, one that issues the MMAs, one that
// brings the scales 16 groups at a time, four that read the accumulators back, scale and add them and store a tile.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "fn_fp8.h"
#include "fn_umma.cuh"

namespace fn {

constexpr int FP_T = 256, FP_RING = 32, FP_ACC = 4, FP_CHUNK = 16;  // threads; ring stages at most; accumulators; groups per chunk of scales

struct Fp8Args {
    CUtensorMap tw, tx;  // codes of the weight, of x: boxes of 128 columns x height, x NT rows
    const float *ws, *xs;
    int m, n, groups, height, tiles_m, tiles, stages;
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
__device__ __forceinline__ bool fp_try(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ void fp_tma(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
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

struct Fp8Shared {
    uint64_t full[FP_RING], empty[FP_RING];  // ring stages
    uint64_t af[FP_ACC], ae[FP_ACC];         // accumulators
    uint64_t sf[2], se[2];                   // chunks of scales
    uint64_t done;
    uint32_t tmem;
    int fail;
};

template <typename T, int NT> __global__ void __launch_bounds__(FP_T, 1) k_fp8_product(const __grid_constant__ Fp8Args a) {
    constexpr uint32_t COLS = FP_ACC * NT <= 64 ? 64 : FP_ACC * NT <= 128 ? 128 : FP_ACC * NT <= 256 ? 256 : 512;
    extern __shared__ uint8_t sm_fp8[];
    __shared__ Fp8Shared sh;
    __shared__ __align__(16) float xsc[2][FP_CHUNK][NT], wsc[2][FP_CHUNK][2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t a_bytes = (uint32_t)a.height * 128u, stage = a_bytes + NT * 128u;
    uint8_t *const ring = sm_fp8 + (1024 - (smem_u32(sm_fp8) & 1023)) % 1024;  // the swizzle counts from 1024-byte boundaries
    volatile int *const s_fail = &sh.fail;
    if (tid == 0) {
        for (int i = 0; i < FP_RING; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        for (int i = 0; i < FP_ACC; ++i) mbar_init(&sh.af[i], 1), mbar_init(&sh.ae[i], 4);
        for (int i = 0; i < 2; ++i) mbar_init(&sh.sf[i], 32), mbar_init(&sh.se[i], 4);
        mbar_init(&sh.done, 1);
        mbar_fence_init();
        sh.fail = 0;
    }
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
    // a wait of about a second at most, that ends at once when another role gave up
    auto wt = [&](uint64_t *bar, uint32_t parity) {
        const uint64_t t0 = global_ns();
        while (!fp_try(bar, parity & 1u)) {
            if (*s_fail) return false;
            if (global_ns() - t0 > 1000000000ull) {
                *s_fail = 1;
                dev_fail(a.err, DEV_WAIT_TIMEOUT);
                return false;
            }
        }
        return true;
    };
    if (warp == 0) {
        if (lane == 0) {
            int i = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
                const int m0 = tile % a.tiles_m * NT, n0 = tile / a.tiles_m * a.height;
                for (int g = 0; g < a.groups; ++g, ++i) {
                    const int s = i % a.stages;
                    if (i >= a.stages && !(ok = wt(&sh.empty[s], (uint32_t)(i / a.stages - 1)))) break;
                    uint8_t *dst = ring + (size_t)s * stage;
                    mbar_arrive_tx(&sh.full[s], stage);
                    fp_tma(dst, &a.tw, g * FP8_GROUP, n0, &sh.full[s]);
                    fp_tma(dst + a_bytes, &a.tx, g * FP8_GROUP, m0, &sh.full[s]);
                }
            }
            // what was issued has landed before the CTA gives its memory back
            if (!ok)
                for (int j = max(0, i - a.stages); j < i; ++j) mbar_park(&sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u);
        }
    } else if (warp == 1) {
        // the whole warp runs this and one elected lane issues: descriptors then live in uniform registers
        constexpr uint32_t idesc = fp_idesc(128, NT);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), base = smem_u32(ring);
        int i = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x)
            for (int g = 0; g < a.groups; ++g, ++i) {
                const int s = i % a.stages, b = i % FP_ACC;
                ok = wt(&sh.full[s], (uint32_t)(i / a.stages)) && (i < FP_ACC || wt(&sh.ae[b], (uint32_t)(i / FP_ACC - 1)));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t ad = fp_desc(base + (uint32_t)s * stage), bd = fp_desc(base + (uint32_t)s * stage + a_bytes);
                if (fp_elect()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) fp_mma(tm + (uint32_t)(b * NT), ad + 2u * k, bd + 2u * k, idesc, k > 0);
                    umma_commit(&sh.empty[s]);
                    umma_commit(&sh.af[b]);
                }
                __syncwarp();
            }
        if (fp_elect()) umma_commit(&sh.done);
        __syncwarp();
        mbar_park(&sh.done, 0);
    } else if (warp == 2) {
        // scales: 16 groups of a tile at a time
        int c = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % a.tiles_m * NT, n0 = tile / a.tiles_m * a.height;
            const int b0 = n0 / FP8_GROUP, b1 = (min(n0 + a.height, a.n) - 1) / FP8_GROUP;
            for (int g0 = 0; g0 < a.groups; g0 += FP_CHUNK, ++c) {
                if (c >= 2) ok = wt(&sh.se[c & 1], (uint32_t)(c / 2 - 1));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int n = min(FP_CHUNK, a.groups - g0);
                for (int t = lane; t < NT; t += 32) {
                    const float *p = a.xs + (int64_t)min(m0 + t, a.m - 1) * a.groups + g0;
#pragma unroll
                    for (int j = 0; j < FP_CHUNK; ++j) xsc[c & 1][j][t] = j < n ? p[j] : 0.0f;
                }
                const int j = lane & 15;
                if (j < n) wsc[c & 1][j][lane >> 4] = a.ws[(int64_t)(lane < 16 ? b0 : b1) * a.groups + g0 + j];
                tc_arrive(&sh.sf[c & 1]);
            }
        }
    } else if (warp >= 4) {
        const int row = tid - 128;  // of the tile: this thread's lane of tensor memory
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        int i = 0, c = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % a.tiles_m * NT, n0 = tile / a.tiles_m * a.height, n = n0 + row;
            const int second = n / FP8_GROUP > n0 / FP8_GROUP;
            float sum[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) sum[j] = 0.0f;
            for (int g = 0; g < a.groups; ++g, ++i) {
                const int b = i % FP_ACC, gc = g % FP_CHUNK;
                if (gc == 0) ok = wt(&sh.sf[c & 1], (uint32_t)(c / 2));
                ok = ok && wt(&sh.af[b], (uint32_t)(i / FP_ACC));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const float w = wsc[c & 1][gc][second];
#pragma unroll
                for (int q = 0; q < NT; q += 16) {
                    float v[16];
                    tmem_ld16(tl + (uint32_t)(b * NT + q), v);
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 x = *(const float4 *)&xsc[c & 1][gc][q + j];
                        sum[q + j] = fmaf(v[j], x.x * w, sum[q + j]);
                        sum[q + j + 1] = fmaf(v[j + 1], x.y * w, sum[q + j + 1]);
                        sum[q + j + 2] = fmaf(v[j + 2], x.z * w, sum[q + j + 2]);
                        sum[q + j + 3] = fmaf(v[j + 3], x.w * w, sum[q + j + 3]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&sh.ae[b]);
                if (gc == FP_CHUNK - 1 || g == a.groups - 1) {
                    if (lane == 0) tc_arrive(&sh.se[c & 1]);
                    ++c;
                }
            }
            if (!ok) break;
            if (row < a.height && n < a.n) {
                const T *add = a.add ? (const T *)a.add + n : nullptr;
                T *out = (T *)a.out + n;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (m0 + j >= a.m) break;
                    const float x = add ? (float)add[(int64_t)(m0 + j) * a.adds] : 0.0f;
                    out[(int64_t)(m0 + j) * a.outs] = (T)(sum[j] + x);
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
    const int room = 227 * 1024 - (int)sizeof(Fp8Shared) - 2 * FP_CHUNK * (NT + 2) * 4 - 16 * 1024 - 2048;
    a.stages = std::min(FP_RING, room / (int)stage);
    return launch_k(k, dim3((unsigned)std::min(a.tiles, num_sms())), dim3(FP_T), (size_t)a.stages * stage + 17 * 1024, s, a);
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
