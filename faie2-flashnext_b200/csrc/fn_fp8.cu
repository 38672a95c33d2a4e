// Rows and weights in 8 bits: e4m3 codes with a scale for each 128 columns of a row, or each 128 x 128 block of a weight; for rows
// the residual's addition and RMSNorm in the same pass. The reference launches k_groupnorm (engine/faie2fn.cu:1222-1235) on fp32
// rows and has no 8-bit activations.
//
//   h = x + add (rounded to its type), y = h (mean h^2 + eps)^-1/2 w, a = max(|y|, 2^-116) over a group, scale = a (1 / 448),
//   code = e4m3(y (448 (1 / a))), to nearest, ties to even; products and reciprocals in fp32
//
// 448 is e4m3's largest number; 2^-116 keeps 448 / a and a / 448 normal numbers (a group of zeros has codes 0). A NaN in a group
// makes its scale NaN, an infinity its scale infinite and its codes NaN: both read back as NaN.
//
// What bounds it is memory: every input is read once and kept in registers between the row's sum and its codes (rows up to 8192
// columns; longer ones are read again, from L2). The sum of squares is held in 64 bits: an fp32 sum's last bits would move codes
// that lie next to a border, and squares of fp32 values leave that type's range.
#include <cuda_bf16.h>

#include <algorithm>
#include <utility>

#include "fn_fp8.h"

namespace fn {

constexpr int F8_T = 256;
constexpr float F8_MAX = 448.0f, F8_TINY = 1.2037062152420224e-35f, F8_STEP = 1.0f / 448.0f;  // F8_TINY: 2^-116

struct F8RowArgs {
    const void *x, *add;
    int64_t xs, adds;  // elements from row to row
    const float *w;
    float eps;
    double per;  // 1 / cols
    int rows, cols, groups;
    void *total, *normed;
    int64_t totals, normeds;
    uint8_t *codes;
    float *scales;
    int tpr;  // threads of a row: 32, 64, 128 or 256
};

__device__ __forceinline__ float f8_max_nan(float a, float b) {
    float e;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(a), "f"(b));
    return e;
}
__device__ __forceinline__ float f8_amax(const float (&y)[8]) {
    float m = fabsf(y[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = f8_max_nan(m, fabsf(y[i]));
    return m;
}
// eight codes, lowest byte first
__device__ __forceinline__ uint2 f8_codes(const float (&y)[8], float inv) {
    uint16_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[i]) : "f"(y[2 * i + 1] * inv), "f"(y[2 * i] * inv));
    return make_uint2((uint32_t)p[0] | (uint32_t)p[1] << 16, (uint32_t)p[2] | (uint32_t)p[3] << 16);
}

// eight adjacent values as they are stored; WIDE: 16-byte aligned
template <typename T> struct F8Raw {
    uint4 w[sizeof(T) / 2];
};
template <typename T, bool WIDE> __device__ __forceinline__ void f8_fetch(const T *p, F8Raw<T> &r) {
    if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) r.w[j] = ((const uint4 *)p)[j];
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
        memcpy(&r, v, sizeof(r));
    }
}
template <typename T> __device__ __forceinline__ void f8_unpack(const F8Raw<T> &r, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        memcpy(v, &r, sizeof(r));
    } else {
        const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
template <typename T, bool WIDE> __device__ __forceinline__ void f8_load(const T *p, float (&v)[8]) {
    F8Raw<T> r;
    f8_fetch<T, WIDE>(p, r);
    f8_unpack<T>(r, v);
}
template <typename T, bool WIDE> __device__ __forceinline__ void f8_store(T *p, const float (&v)[8]) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (T)v[i];
    } else if constexpr (sizeof(T) == 4) {
        *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            memcpy(&u[i], &b, 4);
        }
        *(uint4 *)p = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
// rounded to T
template <typename T> __device__ __forceinline__ void f8_round(float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(__float2bfloat16_rn(v[i]));
    }
}

// v^-1/2 to well below a rounding of fp32: CUDA's approximation and a Newton step for v r^2 = 1 in 64 bits
__device__ __forceinline__ float f8_rsqrt(double v) {
    if (!(v > 1e-30 && v < 1e30)) return (float)rsqrt(v);
    const double r = rsqrtf((float)v);
    return (float)fma(0.5 * r, fma(-v * r, r, 1.0), r);
}

// 8 columns a thread, `tpr` threads a row, R rounds of them held in registers (0: any number, read twice if there is a norm). A CTA takes
// rows at a stride of the grid, the next one's words on their way while one is summed and coded (R up to 2).
template <typename T, int R, bool WIDE> __global__ void __launch_bounds__(F8_T, R == 1 ? 6 : R == 2 ? 4 : 2) k_fp8_rows(const F8RowArgs a) {
    constexpr bool AHEAD = R == 1 || R == 2;
    __shared__ double s_sum[2][F8_T / 32];
    const int t = threadIdx.x & (a.tpr - 1), warp = threadIdx.x >> 5, here = F8_T / a.tpr;  // rows a CTA at once
    const int span = a.tpr * 8, rounds = R ? R : (a.cols + span - 1) / span;
    pdl_wait();
    pdl_trigger();
    const T *x = (const T *)after_wait(a.x), *add = (const T *)after_wait(a.add);
    F8Raw<T> rx[AHEAD ? R : 1], ra[AHEAD ? R : 1];
    auto ahead = [&](int64_t row) {
        if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < (AHEAD ? R : 1); ++k) {
                const int c = k * span + t * 8;
                if (c < a.cols) {
                    f8_fetch<T, WIDE>(x + row * a.xs + c, rx[k]);
                    if (add) f8_fetch<T, WIDE>(add + row * a.adds + c, ra[k]);
                }
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * here;
    int64_t row = (int64_t)blockIdx.x * here + threadIdx.x / a.tpr;
    if constexpr (AHEAD) ahead(row);
    for (int turn = 0; row - threadIdx.x / a.tpr < a.rows; row += step, turn ^= 1) {
        const bool live = row < a.rows;
        T *total = a.total ? (T *)a.total + row * a.totals : nullptr, *normed = a.normed ? (T *)a.normed + row * a.normeds : nullptr;
        uint8_t *codes = a.codes ? a.codes + row * a.cols : nullptr;
        float h[R ? R : 1][8] = {};
        // the row's sum h in columns c .. c + 7
        auto fetch = [&](int c, float (&v)[8], const F8Raw<T> &wx, const F8Raw<T> &wa) {
            f8_unpack<T>(wx, v);
            if (add) {
                float b[8];
                f8_unpack<T>(wa, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += b[i];
                f8_round<T>(v);
            }
        };
        auto read = [&](int c, float (&v)[8]) {
            F8Raw<T> wx, wa;
            f8_fetch<T, WIDE>(x + row * a.xs + c, wx);
            if (add) f8_fetch<T, WIDE>(add + row * a.adds + c, wa);
            fetch(c, v, wx, wa);
        };
        float r = 1.0f;
        if (R || a.w) {
            double ss = 0.0;
#pragma unroll
            for (int k = 0; k < rounds; ++k) {
                const int c = k * span + t * 8;
                float(&v)[8] = h[R ? k : 0];
                if (live && c < a.cols) {
                    if constexpr (AHEAD) fetch(c, v, rx[k], ra[k]);
                    else read(c, v);
                    if (total) f8_store<T, WIDE>(total + c, v);
                    if (a.w) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) ss = fma((double)v[i], (double)v[i], ss);
                    }
                }
            }
            if constexpr (AHEAD) ahead(row + step);
            if (a.w) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (a.tpr > 32) {
                    if ((threadIdx.x & 31) == 0) s_sum[turn][warp] = ss;
                    __syncthreads();
                    const int warps = a.tpr / 32;
                    ss = s_sum[turn][(warp & ~(warps - 1)) + (threadIdx.x & (warps - 1))];
                    for (int o = 1; o < warps; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                }
                r = f8_rsqrt(fma(ss, a.per, (double)a.eps));
            }
        }
#pragma unroll
        for (int k = 0; k < rounds; ++k) {
            const int c = k * span + t * 8;
            const bool in = live && c < a.cols;
            float(&v)[8] = h[R ? k : 0];
            if (!R && in) {
                if (a.w && total) f8_load<T, WIDE>(total + c, v);  // (x may be total: its sum is there already)
                else read(c, v);
                if (!a.w && total) f8_store<T, WIDE>(total + c, v);
            }
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = in ? v[i] : 0.0f;
            if (a.w && in) {
                float w[8];
                f8_load<float, true>(a.w + c, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
            }
            if (normed && in) f8_store<T, WIDE>(normed + c, y);
            if (!codes) continue;
            float m = f8_amax(y);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = f8_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            m = f8_max_nan(m, F8_TINY);
            if (!in) continue;
            *(uint2 *)(codes + c) = f8_codes(y, F8_MAX * __frcp_rn(m));
            if (t % 16 == 0) a.scales[row * a.groups + c / FP8_GROUP] = m * F8_STEP;
        }
    }
}

struct F8BlockArgs {
    const void *w;
    int64_t ws;
    int rows, cols, groups;
    uint8_t *codes;
    float *scales;
};

// one CTA per 128 x 128 block, its values in registers (as they are stored) between the maximum and the codes; 16 threads a row, 8
// columns each, four rows a thread
constexpr int F8_BT = 512;
template <typename T, bool WIDE> __global__ void __launch_bounds__(F8_BT, 2) k_fp8_blocks(const F8BlockArgs a) {
    __shared__ float s_max[F8_BT / 32];
    const int c = blockIdx.x * FP8_GROUP + (threadIdx.x & 15) * 8;
    const int64_t row0 = (int64_t)blockIdx.y * FP8_GROUP + (threadIdx.x >> 4);
    pdl_wait();
    pdl_trigger();
    const T *w = (const T *)after_wait(a.w) + c;
    T raw[4][8];
    float m = F8_TINY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t row = row0 + 32 * k;
        const bool in = row < a.rows && c < a.cols;
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                ((uint4 *)raw[k])[j] = in ? ((const uint4 *)(w + row * a.ws))[j] : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) raw[k][j] = in ? w[row * a.ws + j] : (T)0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)raw[k][j];
        m = f8_max_nan(m, f8_amax(v));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = f8_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
    m = s_max[threadIdx.x & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = f8_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float inv = F8_MAX * __frcp_rn(m);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t row = row0 + 32 * k;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)raw[k][j];
        if (row < a.rows && c < a.cols) *(uint2 *)(a.codes + row * a.cols + c) = f8_codes(v, inv);
    }
    if (threadIdx.x == 0) a.scales[(int64_t)blockIdx.y * a.groups + blockIdx.x] = m * F8_STEP;
}

template <typename T, bool WIDE> static cudaError_t launch_rows(const F8RowArgs &a, dim3 grid, cudaStream_t s) {
    const int per = a.tpr * 8;
    if (a.cols <= per) return launch_k(k_fp8_rows<T, 1, WIDE>, grid, dim3(F8_T), 0, s, a);
    if (a.cols <= 2 * per) return launch_k(k_fp8_rows<T, 2, WIDE>, grid, dim3(F8_T), 0, s, a);
    if (a.cols <= 4 * per) return launch_k(k_fp8_rows<T, 4, WIDE>, grid, dim3(F8_T), 0, s, a);
    return launch_k(k_fp8_rows<T, 0, WIDE>, grid, dim3(F8_T), 0, s, a);
}

}  // namespace fn

using namespace fn;

FN_API int fn_fp8_rows(uint32_t type, const void *x, int64_t x_stride, const void *add, int64_t add_stride, const float *weight, float eps,
                       int rows, int cols, void *total, int64_t total_stride, void *normed, int64_t normed_stride, uint8_t *codes,
                       float *scales, void *stream) {
    return kv4_entry("fp8 rows", [&]() -> int {
        if (type != T_F32 && type != T_BF16) return fail("fp8 rows: rows must be F32 or BF16");
        if (rows < 0 || cols < 16 || cols % 16 || cols > FP8_MAX_COLS)
            return fail("fp8 rows: bad row count, or columns that are no multiple of 16");
        if (rows == 0) return 0;
        if (!x || !codes != !scales) return fail("fp8 rows: null pointer");
        if (!codes && !total && !normed) return fail("fp8 rows: nothing to write");
        const int size = type == T_F32 ? 4 : 2;
        if (((uintptr_t)x | (uintptr_t)add | (uintptr_t)total | (uintptr_t)normed) % size)
            return fail("fp8 rows: rows must be aligned to their type");
        if ((uintptr_t)weight % 16 || (uintptr_t)codes % 16 || (uintptr_t)scales % 4)
            return fail("fp8 rows: weight and codes must be 16-byte aligned");
        const int64_t bytes = (int64_t)cols * size;
        if (rows > 1 && ((total && total_stride < cols) || (normed && normed_stride < cols))) return fail("fp8 rows: rows that are written overlap");
        for (const auto &[p, ps] : {std::pair(x, x_stride), std::pair(add, add_stride)})
            if (fp8_mixed(total, total_stride * size, p, ps * size, rows, bytes) || fp8_mixed(normed, normed_stride * size, p, ps * size, rows, bytes))
                return fail("fp8 rows: rows that are written lie over other rows that are read");
        if (normed && (normed == total || fp8_mixed(total, total_stride * size, normed, normed_stride * size, rows, bytes)))
            return fail("fp8 rows: total and normed lie over one another");
        const bool wide = ((uintptr_t)x | (uintptr_t)add | (uintptr_t)total | (uintptr_t)normed | (uint64_t)(x_stride * size) |
                           (uint64_t)(add_stride * size) | (uint64_t)(total_stride * size) | (uint64_t)(normed_stride * size)) % 16 == 0;
        int tpr = 32;
        while (tpr < F8_T && tpr * 8 < cols) tpr *= 2;
        // as many CTAs as the SMs hold (6 of 256 threads where a row's 8 columns a thread are one round, 4 else)
        const int64_t grid = std::min<int64_t>(((int64_t)rows * tpr + F8_T - 1) / F8_T, (int64_t)num_sms() * (cols <= 8 * tpr ? 6 : 4));
        const F8RowArgs a{x, add, x_stride, add_stride, weight, eps, 1.0 / cols, rows, cols, fp8_groups(cols), total, normed, total_stride,
                          normed_stride, codes, scales, tpr};
        const dim3 g((unsigned)grid);
        const cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e = type == T_F32 ? (wide ? launch_rows<float, true>(a, g, s) : launch_rows<float, false>(a, g, s))
                                            : (wide ? launch_rows<__nv_bfloat16, true>(a, g, s) : launch_rows<__nv_bfloat16, false>(a, g, s));
        if (e != cudaSuccess) return fail(std::string("fp8 rows launch: ") + cudaGetErrorString(e));
        return 0;
    });
}

FN_API int fn_fp8_blocks(uint32_t type, const void *w, int64_t stride, int rows, int cols, uint8_t *codes, float *scales, void *stream) {
    return kv4_entry("fp8 blocks", [&]() -> int {
        if (type != T_F32 && type != T_BF16) return fail("fp8 blocks: weights must be F32 or BF16");
        if (rows < 0 || cols < 16 || cols % 16 || cols > FP8_MAX_COLS)
            return fail("fp8 blocks: bad row count, or columns that are no multiple of 16");
        if (rows == 0) return 0;
        if (!w || !codes || !scales) return fail("fp8 blocks: null pointer");
        const int size = type == T_F32 ? 4 : 2;
        if ((uintptr_t)w % size || (uintptr_t)codes % 16 || (uintptr_t)scales % 4)
            return fail("fp8 blocks: weights must be aligned to their type, codes to 16 bytes");
        if (fp8_groups(rows) > 65535) return fail("fp8 blocks: too many rows");
        const F8BlockArgs a{w, stride, rows, cols, fp8_groups(cols), codes, scales};
        const dim3 g((unsigned)a.groups, (unsigned)fp8_groups(rows));
        const bool wide = ((uintptr_t)w | (uint64_t)(stride * size)) % 16 == 0;
        const cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e = type == T_F32 ? (wide ? launch_k(k_fp8_blocks<float, true>, g, dim3(F8_BT), 0, s, a)
                                                    : launch_k(k_fp8_blocks<float, false>, g, dim3(F8_BT), 0, s, a))
                                            : (wide ? launch_k(k_fp8_blocks<__nv_bfloat16, true>, g, dim3(F8_BT), 0, s, a)
                                                    : launch_k(k_fp8_blocks<__nv_bfloat16, false>, g, dim3(F8_BT), 0, s, a));
        if (e != cudaSuccess) return fail(std::string("fp8 blocks launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
