// q / k head RMSNorm and RoPE for rows at positions of their own (requests of different lengths): what k_attn_qkv
// (fn_model.cu) does at one position for all, without its cache. Reference: k_qk_norm_rope, engine/faie2fn.cu:1452-1478.
//
// One warp per head of a row, 8 of the 256 dims a lane. The rotated pairs (i, i + 32) of the first 64 dims lie in lanes 4
// apart, so the rotation is one exchange. Angles are formed and reduced in double, as in fn_model.cu: they reach thousands of
// radians.
#include "fn_engine.h"

namespace fn {

struct QkRopeArgs {
    const float *x[2], *w[2];  // q, k; their head norms [256]
    int64_t token[2], head[2];
    float *y[2];
    const float *inv_freq;
    const int *positions;
    int rows, nh, nkv;
    float eps;
};

__global__ void __launch_bounds__(128) k_qk_rope_rows(const QkRopeArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, heads = a.nh + a.nkv;
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (u >= (int64_t)a.rows * heads) return;
    const int64_t row = u / heads;
    const int j = (int)(u - row * heads), part = j >= a.nh, h = j - part * a.nh;
    const int pos = after_wait(a.positions)[row];
    float *out = a.y[part] + (row * (part ? a.nkv : a.nh) + h) * 256 + lane * 8;
    float x[8] = {};
    if (pos >= 0) {
        const float *src = after_wait(a.x[part]) + row * a.token[part] + h * a.head[part] + lane * 8, *w = a.w[part] + lane * 8;
        const float4 v0 = *(const float4 *)src, v1 = *(const float4 *)(src + 4);
        x[0] = v0.x, x[1] = v0.y, x[2] = v0.z, x[3] = v0.w, x[4] = v1.x, x[5] = v1.y, x[6] = v1.z, x[7] = v1.w;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss / 256.0f + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, x[i], 4);  // dim +- 32
            if (lane < 8) {
                double sd, cd;
                sincos((double)pos * (double)a.inv_freq[(lane & 3) * 8 + i], &sd, &cd);
                x[i] = lane < 4 ? x[i] * (float)cd - other * (float)sd : x[i] * (float)cd + other * (float)sd;
            }
        }
    }
    *(float4 *)out = make_float4(x[0], x[1], x[2], x[3]);
    *(float4 *)(out + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

}  // namespace fn

using namespace fn;

FN_API int fn_qk_rope_rows(const float *q, int64_t q_token, int64_t q_head, const float *k, int64_t k_token, int64_t k_head,
                           const float *wq, const float *wk, const float *inv_freq, const int *positions, int rows, int nh,
                           int nkv, float *q_out, float *k_out, float eps, void *stream) {
    if (rows < 0 || nh < 1 || nkv < 1) return fail("qk rope: bad row / head counts");
    if (rows == 0) return 0;
    if (!q || !k || !wq || !wk || !inv_freq || !positions || !q_out || !k_out) return fail("qk rope: null pointer");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out) % 16 || (q_token | q_head | k_token | k_head) % 4)
        return fail("qk rope: rows must be 16-byte aligned");
    const int64_t grid = ((int64_t)rows * (nh + nkv) + 3) / 4;
    if (grid > INT32_MAX) return fail("qk rope: too many rows");
    const QkRopeArgs a{{q, k}, {wq, wk}, {q_token, k_token}, {q_head, k_head}, {q_out, k_out}, inv_freq, positions, rows, nh, nkv, eps};
    const cudaError_t e = launch_k(k_qk_rope_rows, dim3((unsigned)grid), dim3(128), 0, (cudaStream_t)stream, a);
    if (e != cudaSuccess) return fail(std::string("qk rope launch: ") + cudaGetErrorString(e));
    return 0;
}
