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
// What bounds it is memory, and close to it instruction issue (70%): every input is read once and kept in registers between the row's sum and
// its codes (rows up to 8192 columns; longer ones are read again, from L2). 8192 x 4096 in bf16 with a residual: 40.2 us, 5.9 TB/s. The sum of
// squares is held in 64 bits: an fp32 sum's last bits would move codes that lie next to a border, and squares of fp32 values leave that type's
// range.
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

// the larger magnitude of three numbers; NaN if one is
__device__ __forceinline__ float f8_max_nan(float a, float b, float c) {
    float e;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(e) : "f"(a), "f"(b), "f"(c));
    return e;
}
__device__ __forceinline__ float f8_max_nan(float a, float b) {
    float e;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(a), "f"(b));
    return e;
}
__device__ __forceinline__ float f8_amax(const float (&y)[8]) {
    const float m = f8_max_nan(y[0], y[1], y[2]), n = f8_max_nan(y[3], y[4], y[5]);
    return f8_max_nan(f8_max_nan(m, y[6], y[7]), n);
}
// y *= b, two numbers an instruction
__device__ __forceinline__ void f8_mul2(float &y0, float &y1, float b0, float b1) {
    asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n mul.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}\n"
        : "+f"(y0), "+f"(y1)
        : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void f8_scale(float (&y)[8], float b) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) f8_mul2(y[i], y[i + 1], b, b);
}
// eight codes of y inv, lowest byte first
__device__ __forceinline__ uint2 f8_codes(float (&y)[8], float inv) {
    uint16_t p[4];
    f8_scale(y, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[i]) : "f"(y[2 * i + 1]), "f"(y[2 * i]));
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
// rounded to T
template <typename T> __device__ __forceinline__ void f8_pack(const float (&v)[8], F8Raw<T> &r) {
    if constexpr (sizeof(T) == 4) memcpy(&r, v, sizeof(r));
    else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            memcpy(&u[i], &b, 4);
        }
        r.w[0] = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
template <typename T, bool WIDE> __device__ __forceinline__ void f8_store(T *p, const F8Raw<T> &r) {
    if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) ((uint4 *)p)[j] = r.w[j];
    } else {
        T v[8];
        memcpy(v, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
}

// v^-1/2 to well below a rounding of fp32: CUDA's approximation and a Newton step for v r^2 = 1 in 64 bits
__device__ __forceinline__ float f8_rsqrt(double v) {
    if (!(v > 1e-30 && v < 1e30)) return (float)rsqrt(v);
    const double r = rsqrtf((float)v);
    return (float)fma(0.5 * r, fma(-v * r, r, 1.0), r);
}

// rounds of 8 columns a thread that are on their way while others are worked on: 64 bytes a thread of x, and of add
constexpr bool f8_ahead(int rounds, int size) { return rounds && rounds * size <= 8; }
// CTAs that an SM holds, by the registers they need without spilling much (five in place of four, 8192 x 4096 bf16: 57 us in place of 51; more
// rounds at once in place of more CTAs are slower too, see launch_rows)
constexpr int f8_ctas(int rounds, int size) { return !f8_ahead(rounds, size) ? 2 : rounds * size <= 2 ? 6 : rounds * size == 4 ? 4 : 3; }

// 8 columns a thread, `tpr` threads a row, R rounds of them held in registers (0: any number, read twice if there is a norm). A CTA takes
// rows at a stride of the grid, the next one's words on their way while one is summed and coded. F: whether there is something to add (1) and
// a norm (2), or -1 for whatever there is. What lies past the last column or row reads the last ones' place, counts as zeros and is not
// stored: with branches around it all a row of two rounds took a warp 537 instructions instead of 448.
template <typename T, int R, bool WIDE, int F> __global__ void __launch_bounds__(F8_T, f8_ctas(R, sizeof(T))) k_fp8_rows(const F8RowArgs a) {
    constexpr bool AHEAD = f8_ahead(R, sizeof(T));
    const bool adds = F < 0 ? a.add != nullptr : F & 1, norm = F < 0 ? a.w != nullptr : F & 2;
    __shared__ double s_sum[2][F8_T / 32];
    const int t = threadIdx.x & (a.tpr - 1), warp = threadIdx.x >> 5, here = F8_T / a.tpr;  // rows a CTA at once
    const int span = a.tpr * 8, rounds = R ? R : (a.cols + span - 1) / span;
    pdl_wait();
    pdl_trigger();
    const T *x = (const T *)after_wait(a.x), *add = (const T *)after_wait(a.add);
    auto fetch = [&](uint32_t row, int c, F8Raw<T> &wx, F8Raw<T> &wa) {
        const int64_t at = min(row, (uint32_t)a.rows - 1);
        const int cc = min(c, a.cols - 8);
        f8_fetch<T, WIDE>(x + at * a.xs + cc, wx);
        if (adds) f8_fetch<T, WIDE>(add + at * a.adds + cc, wa);
    };
    F8Raw<T> rx[AHEAD ? R : 1], ra[AHEAD ? R : 1];
    auto ahead = [&](uint32_t row) {
#pragma unroll
        for (int k = 0; k < (AHEAD ? R : 1); ++k) fetch(row, k * span + t * 8, rx[k], ra[k]);
    };
    const uint32_t step = gridDim.x * here, rows = a.rows;
    uint32_t row0 = blockIdx.x * here;
    if constexpr (AHEAD) ahead(row0 + threadIdx.x / a.tpr);
    for (int turn = 0; row0 < rows; row0 += step, turn ^= 1) {
        const uint32_t row32 = row0 + threadIdx.x / a.tpr;
        const int64_t row = row32;
        const int cols = row32 < rows ? a.cols : 0;
        T *const total = (T *)a.total + row * a.totals, *const normed = (T *)a.normed + row * a.normeds;
        F8Raw<T> h[R ? R : 1];  // the row's sum, rounded to T
        auto sum = [&](const F8Raw<T> &wx, const F8Raw<T> &wa, bool in) {
            F8Raw<T> r = wx;
            if (adds) {
                float v[8], b[8];
                f8_unpack<T>(wx, v);
                f8_unpack<T>(wa, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += b[i];
                f8_pack<T>(v, r);
            }
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                if (!in) r.w[j] = make_uint4(0, 0, 0, 0);
            return r;
        };
        auto read = [&](int c) {
            F8Raw<T> wx, wa;
            fetch(row32, c, wx, wa);
            return sum(wx, wa, c < cols);
        };
        float r = 1.0f;
        if (R || norm) {
            double ss = 0.0;
#pragma unroll
            for (int k = 0; k < rounds; ++k) {
                const int c = k * span + t * 8;
                F8Raw<T> &w = h[R ? k : 0];
                if constexpr (AHEAD) w = sum(rx[k], ra[k], c < cols);
                else w = read(c);
                if (a.total && c < cols) f8_store<T, WIDE>(total + c, w);
                if (norm) {
                    float v[8];
                    f8_unpack<T>(w, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fma((double)v[i], (double)v[i], ss);
                }
            }
            if constexpr (AHEAD)
                if (row0 + step < rows) ahead(row32 + step);
            if (norm) {
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
            const bool in = c < cols;
            if (!R) {
                if (norm && a.total) {  // (x may be total: its sum is there already)
                    if (in) f8_fetch<T, WIDE>(total + c, h[0]);
                } else h[0] = read(c);
                if (!norm && a.total && in) f8_store<T, WIDE>(total + c, h[0]);
            }
            float y[8];
            f8_unpack<T>(h[R ? k : 0], y);
            if (norm) {
                F8Raw<float> w;
                f8_fetch<float, true>(a.w + min(c, a.cols - 8), w);
                float v[8];
                f8_unpack<float>(w, v);
                f8_scale(y, r);
#pragma unroll
                for (int i = 0; i < 8; i += 2) f8_mul2(y[i], y[i + 1], v[i], v[i + 1]);
            }
            if (a.normed && in) {
                F8Raw<T> w;
                f8_pack<T>(y, w);
                f8_store<T, WIDE>(normed + c, w);
            }
            if (!a.codes) continue;
            float m = in ? f8_amax(y) : 0.0f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = f8_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            m = f8_max_nan(m, F8_TINY);
            const uint2 codes = f8_codes(y, F8_MAX * __frcp_rn(m));
            if (in) *(uint2 *)(a.codes + row * a.cols + c) = codes;
            if (in && t % 16 == 0) a.scales[row * a.groups + c / FP8_GROUP] = m * F8_STEP;
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
// columns each, four rows a thread. Memory bounds it (12352 x 2048 bf16: 13.6 us, 5.6 TB/s).
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

template <typename T, bool WIDE> static cudaError_t launch_rows(F8RowArgs a, cudaStream_t s) {
    // As many threads a row as there are: 32 columns a thread and fewer threads a row take fewer instructions, but hold fewer CTAs (8192 x 4096
    // bf16: 48.5 us, so 40.2).
    a.tpr = 32;
    while (a.tpr < F8_T && a.tpr * 8 < a.cols) a.tpr *= 2;
    const int per = a.tpr * 8;
    auto grid = [&](int rounds) {
        return std::min<int64_t>(((int64_t)a.rows * a.tpr + F8_T - 1) / F8_T, (int64_t)num_sms() * f8_ctas(rounds, sizeof(T)));
    };
    auto launch = [&](auto *k, int rounds) { return launch_k(k, dim3((unsigned)grid(rounds)), dim3(F8_T), 0, s, a); };
    if constexpr (WIDE) {
        if (a.cols <= 2 * per) {
            switch ((a.add ? 1 : 0) + (a.w ? 2 : 0)) {
            case 0: return a.cols <= per ? launch(k_fp8_rows<T, 1, true, 0>, 1) : launch(k_fp8_rows<T, 2, true, 0>, 2);
            case 1: return a.cols <= per ? launch(k_fp8_rows<T, 1, true, 1>, 1) : launch(k_fp8_rows<T, 2, true, 1>, 2);
            case 2: return a.cols <= per ? launch(k_fp8_rows<T, 1, true, 2>, 1) : launch(k_fp8_rows<T, 2, true, 2>, 2);
            default: return a.cols <= per ? launch(k_fp8_rows<T, 1, true, 3>, 1) : launch(k_fp8_rows<T, 2, true, 3>, 2);
            }
        }
    } else {
        if (a.cols <= per) return launch(k_fp8_rows<T, 1, false, -1>, 1);
        if (a.cols <= 2 * per) return launch(k_fp8_rows<T, 2, false, -1>, 2);
    }
    if (a.cols <= 4 * per) return launch(k_fp8_rows<T, 4, WIDE, -1>, 4);
    return launch(k_fp8_rows<T, 0, WIDE, -1>, 0);
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
        if (rows > 1 && ((total && total_stride < cols) || (normed && normed_stride < cols))) return fail("fp8 rows: rows that are written overlap");
        for (const auto &[p, ps] : {std::pair(x, x_stride), std::pair(add, add_stride)})
            if (rows_mixed(total, total_stride, p, ps, rows, cols, size) || rows_mixed(normed, normed_stride, p, ps, rows, cols, size))
                return fail("fp8 rows: rows that are written lie over other rows that are read");
        if (normed && (normed == total || rows_mixed(total, total_stride, normed, normed_stride, rows, cols, size)))
            return fail("fp8 rows: total and normed lie over one another");
        const int64_t bytes = (int64_t)cols * size, n_codes = (int64_t)rows * cols, n_scales = (int64_t)rows * fp8_groups(cols) * 4, n_weight = (int64_t)cols * 4;
        auto meets = [&](const void *q, int64_t n) {
            return rows_meet_bytes(total, total_stride * size, rows, bytes, q, n) || rows_meet_bytes(normed, normed_stride * size, rows, bytes, q, n);
        };
        auto read = [&](const void *q, int64_t n) {
            return rows_meet_bytes(x, x_stride * size, rows, bytes, q, n) || rows_meet_bytes(add, add_stride * size, rows, bytes, q, n) ||
                   rows_meet_bytes(weight, 0, 1, n_weight, q, n);
        };
        if (meets(codes, n_codes) || meets(scales, n_scales) || read(codes, n_codes) || read(scales, n_scales) || meets(weight, n_weight) ||
            rows_meet_bytes(codes, 0, 1, n_codes, scales, n_scales))
            return fail("fp8 rows: codes, scales, weight and rows share memory");
        const bool wide = ((uintptr_t)x | (uintptr_t)add | (uintptr_t)total | (uintptr_t)normed | (uint64_t)(x_stride * size) |
                           (uint64_t)(add_stride * size) | (uint64_t)(total_stride * size) | (uint64_t)(normed_stride * size)) % 16 == 0;
        const F8RowArgs a{x, add, x_stride, add_stride, weight, eps, 1.0 / cols, rows, cols, fp8_groups(cols), total, normed, total_stride,
                          normed_stride, codes, scales, 0};
        const cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e = type == T_F32 ? (wide ? launch_rows<float, true>(a, s) : launch_rows<float, false>(a, s))
                                            : (wide ? launch_rows<__nv_bfloat16, true>(a, s) : launch_rows<__nv_bfloat16, false>(a, s));
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
        const int64_t n_codes = (int64_t)rows * cols, n_scales = (int64_t)fp8_groups(rows) * fp8_groups(cols) * 4;
        if (rows_meet_bytes(w, stride * size, rows, (int64_t)cols * size, codes, n_codes) ||
            rows_meet_bytes(w, stride * size, rows, (int64_t)cols * size, scales, n_scales) || rows_meet_bytes(codes, 0, 1, n_codes, scales, n_scales))
            return fail("fp8 blocks: codes, scales and the weight share memory");
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
