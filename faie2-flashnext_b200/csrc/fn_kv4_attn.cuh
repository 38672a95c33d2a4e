// What the two attention kernels over the paged 4-bit cache share (fn_kv4_attn.cu: few rows per request, fn_kv4_prompt.cu:
// prompts): arguments, the requests' share of the work, a row's output, the join of partial results.
#pragma once

#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "fn_kv4.h"

namespace fn {

constexpr int KA_TOK = 64;                    // tokens of a unit
constexpr int KA_EXTRA = 4;                   // units that a row tile counts beside its own, for its start and end
constexpr int KA_MAX_GRID = 512;              // CTAs at most

struct Kv4AttnArgs {
    Kv4Lay l;
    int n, rows, nh, group, max_pages, vec;
    const void *q, *gate;
    int64_t qt, qh, gt, gh, ot;
    void *out;
    const int *cu, *kv_len, *table;
    float scale;
    float *part;     // [CTA][2]: a row tile's sums [rows][hd], references [rows], sums of weights [rows]
    int64_t stride;  // floats of a partial result's place
    struct KaSplit *split;  // [CTA]: the row tile that starts in the CTA's run and goes on past it
    int *far;    // prompts [CTA]: whether its run met what only the kernel's long form serves
    int always;  // prompts: only the long form runs
    uint32_t *err;
};

// a request's share of the work
struct KaReq {
    int first, fresh, len, tiles, rt;  // first row, rows, tokens, 64-token tiles, row tiles
};
struct KaSplit {
    int parts;  // CTAs it lies in (0: there is none)
    int kv, tile;
    KaReq rq;
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

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// sigmoid to a few 2^-23 of itself (the exact quotient is some 30 instructions, for every output)
__device__ __forceinline__ float ka_gate(float x) { return __fdividef(1.0f, 1.0f + ka_exp2(x * -1.44269504f)); }
__device__ __forceinline__ uint32_t ka_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ float2 ka_unpack(uint32_t w) { return __half22float2(*(const __half2 *)&w); }
__device__ __forceinline__ float ka_half(const uint8_t *p) { return __half2float(*(const __half *)p); }
// the weight of a part whose reference is `ref` beside the common one; a part without a key has none, and a row that has
// nothing but NaN scores keeps them through the reference 0
__device__ __forceinline__ float ka_weight(float ref, float common) {
    return ka_exp2(ref == -INFINITY ? (common == -INFINITY ? 0.0f : -INFINITY) : ref - common);
}
template <typename T> __device__ __forceinline__ float ka_f(T x);
template <> __device__ __forceinline__ float ka_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float ka_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// a row's output by one warp: value(d), gated
template <typename T, int HD, typename V>
__device__ __forceinline__ void ka_emit(const Kv4AttnArgs &a, const KaReq &rq, int kv, int flat, int lane, bool sees, V value) {
    const int tok = flat / a.group, h = kv * a.group + flat - tok * a.group;
    const int64_t row = rq.first + tok;
    float gate[HD / 32];
#pragma unroll
    for (int x = 0; x < HD / 32; ++x)
        gate[x] = a.gate && sees ? ka_f<T>(((const T *)after_wait(a.gate))[row * a.gt + h * a.gh + lane + 32 * x]) : 0.0f;
#pragma unroll
    for (int x = 0; x < HD / 32; ++x) {
        float y = sees ? value(lane + 32 * x) : 0.0f;
        if (a.gate) y *= ka_gate(gate[x]);
        ((T *)a.out)[row * a.ot + (int64_t)h * HD + lane + 32 * x] = (T)y;
    }
}

// ---- the join of row tiles that lie in several runs: the parts of the one that starts in run c are [ROWS][HD] sums, [ROWS]
// references (base 2) and [ROWS] sums of weights, a.stride floats apart, two to a run. Always in the order of the runs.
template <int HD, int W> struct KjShared {
    float w[KA_MAX_GRID], red[2][W], sum[W][HD];
};

// Row i of the tile by W warps: each takes every W-th part, the first of them loaded before the weights are known; their sums are
// added in the order of the warps.
template <typename T, int HD, int ROWS, int W>
__device__ __forceinline__ void ka_join_row(const Kv4AttnArgs &a, int c, const KaSplit &sp, int i, KjShared<HD, W> &sh) {
    constexpr int PER = HD / 32, U = 8, N = (KA_MAX_GRID + 32 * W - 1) / (32 * W);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long flat = (long long)sp.tile * ROWS + i;
    if (flat >= (long long)sp.rq.fresh * a.group) return;
    auto slot = [&](int x) { return after_wait(a.part) + ((size_t)(c + x) * 2 + (x == 0)) * a.stride; };
    float y[PER] = {}, v[U][PER];
    auto fetch = [&](int x0) {
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const bool in = x0 + W * x < sp.parts;
            const float *p = slot(in ? x0 + W * x : 0) + i * HD + lane;
#pragma unroll
            for (int d = 0; d < PER; ++d) v[x][d] = in ? p[32 * d] : 0.0f;
        }
    };
    fetch(warp);
    float rf[N], l[N], mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int q = tid + 32 * W * x;
        rf[x] = q < sp.parts ? slot(q)[ROWS * HD + i] : -INFINITY;
        l[x] = q < sp.parts ? slot(q)[ROWS * HD + ROWS + i] : 0.0f;
        mx = fmaxf(mx, rf[x]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sh.red[0][warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, sh.red[0][w]);
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int q = tid + 32 * W * x;
        if (q < sp.parts) {
            const float f = ka_weight(rf[x], mx);
            sh.w[q] = f;
            sum += f * l[x];
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.red[1][warp] = sum;
    __syncthreads();
    for (int x0 = warp; x0 < sp.parts; x0 += W * U) {
        if (x0 != warp) fetch(x0);
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const float w = x0 + W * x < sp.parts ? sh.w[x0 + W * x] : 0.0f;
#pragma unroll
            for (int d = 0; d < PER; ++d) y[d] += w * v[x][d];
        }
    }
#pragma unroll
    for (int d = 0; d < PER; ++d) sh.sum[warp][lane + 32 * d] = y[d];
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += sh.red[1][w];
    const bool sees = sp.rq.len - sp.rq.fresh + flat / a.group + 1 > 0 && sp.rq.len > 0;
    const float inv = 1.0f / sum;
    if (warp == 0)
        ka_emit<T, HD>(a, sp.rq, sp.kv, (int)flat, lane, sees, [&](int d) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += sh.sum[w][d];
            return s * inv;
        });
    __syncthreads();
}

// few row tiles, perhaps of many parts: CTA (x, row) takes the runs x, x + gridDim.x, ..
constexpr int KJ_WARPS = 16, KJ_GRID = 32;
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(32 * KJ_WARPS) k_kv4_join_few(const __grid_constant__ Kv4AttnArgs a, int runs) {
    __shared__ KjShared<HD, KJ_WARPS> sh;
    pdl_wait();
    pdl_trigger();
    const KaSplit *split = after_wait(a.split);
    for (int base = blockIdx.x; base < runs; base += 32 * gridDim.x) {
        const int mine = base + (threadIdx.x & 31) * gridDim.x;
        uint32_t todo = __ballot_sync(0xffffffffu, mine < runs && split[mine].parts != 0);
        for (; todo; todo &= todo - 1) {
            const int c = base + (__ffs(todo) - 1) * gridDim.x;
            ka_join_row<T, HD, ROWS, KJ_WARPS>(a, c, split[c], blockIdx.y, sh);
        }
    }
}

// many row tiles, mostly of few parts: CTA (c, eight rows), a warp a row, part after part; a row tile of many parts is taken row
// after row by all eight warps
template <typename T, int HD, int ROWS> __global__ void __launch_bounds__(256) k_kv4_join(const __grid_constant__ Kv4AttnArgs a) {
    constexpr int PER = HD / 32, U = 4, ALONE = 24;
    __shared__ KjShared<HD, 8> sh;
    pdl_wait();
    pdl_trigger();
    const int c = blockIdx.x, lane = threadIdx.x & 31, i = blockIdx.y * 8 + (threadIdx.x >> 5);
    const KaSplit sp = after_wait(a.split)[c];
    if (sp.parts == 0) return;
    if (sp.parts > ALONE) {
        for (int x = 0; x < 8; ++x) ka_join_row<T, HD, ROWS, 8>(a, c, sp, blockIdx.y * 8 + x, sh);
        return;
    }
    const long long flat = (long long)sp.tile * ROWS + i;
    if (flat >= (long long)sp.rq.fresh * a.group) return;
    auto slot = [&](int x) { return after_wait(a.part) + ((size_t)(c + x) * 2 + (x == 0)) * a.stride; };
    // a part's reference and sum of weights a lane
    const float rf = lane < sp.parts ? slot(lane)[ROWS * HD + i] : -INFINITY;
    const float l = lane < sp.parts ? slot(lane)[ROWS * HD + ROWS + i] : 0.0f;
    float v[U][PER], y[PER] = {};
    auto fetch = [&](int x0) {
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const bool in = x0 + x < sp.parts;
            const float *p = slot(in ? x0 + x : 0) + i * HD + lane;
#pragma unroll
            for (int d = 0; d < PER; ++d) v[x][d] = in ? p[32 * d] : 0.0f;
        }
    };
    fetch(0);
    float mx = rf;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float w = lane < sp.parts ? ka_weight(rf, mx) : 0.0f;
    float sum = w * l;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    for (int x0 = 0; x0 < sp.parts; x0 += U) {
        if (x0) fetch(x0);
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const float f = __shfl_sync(0xffffffffu, w, x0 + x);
#pragma unroll
            for (int d = 0; d < PER; ++d) y[d] += f * v[x][d];
        }
    }
    const bool sees = sp.rq.len - sp.rq.fresh + flat / a.group + 1 > 0 && sp.rq.len > 0;
    const float inv = 1.0f / sum;
    ka_emit<T, HD>(a, sp.rq, sp.kv, (int)flat, lane, sees, [&](int d) {
        float r = 0.0f;
#pragma unroll
        for (int x = 0; x < PER; ++x)
            if (d == lane + 32 * x) r = y[x];
        return r * inv;
    });
}

// host: prompts' kernel (fn_kv4_prompt.cu), and its share of the workspace
cudaError_t launch_kv4_prompt(Kv4AttnArgs a, bool f32, int max_new, cudaStream_t s);
uint64_t kv4_prompt_workspace();

}  // namespace fn
