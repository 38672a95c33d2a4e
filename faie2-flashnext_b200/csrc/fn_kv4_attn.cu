// Attention over the paged 4-bit KV cache (fn_kv4.h): softmax(scale q k^T) v per query row, causal, grouped heads.
// The reference's attention reads dense fp32 caches at one position for all (k_attn_split + k_attn_combine,
// engine/faie2fn.cu:1598-1690).
//
// First form: one CTA per row and query head, four warps over the tokens, each with a running maximum and sum (one pass),
// merged at the end. Right for every case; reads the cache once per query head and row.
#include <cuda_bf16.h>

#include "fn_kv4.h"

namespace fn {

struct Kv4AttnArgs {
    Kv4Lay l;
    int n, rows, nh, max_pages;
    const void *q, *gate;
    int64_t qt, qh, gt, gh, ot;
    void *out;
    const int *cu, *kv_len, *table;
    float scale;
    uint32_t *err;
};

template <typename T, int HD> __global__ void __launch_bounds__(128) k_kv4_attn_rows(const Kv4AttnArgs a) {
    constexpr int PER = HD / 32;  // dims a lane
    __shared__ float so[4][HD], sml[4][2];
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv = h / (a.nh / a.l.nkv);
    const int *cu = after_wait(a.cu);
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (cu[m] <= i) lo = m;
        else hi = m;
    }
    const int r = lo, len = min(max(after_wait(a.kv_len)[r], 0), a.max_pages * a.l.bs);
    const int see = i >= cu[r] && i < cu[r + 1] ? min(len, len - (cu[r + 1] - cu[r]) + i - cu[r] + 1) : 0;
    float q[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) q[j] = (float)((const T *)after_wait(a.q))[i * a.qt + h * a.qh + lane * PER + j] * a.scale;
    const uint32_t grp = lane * PER / KV4_GROUP, in = lane * PER % KV4_GROUP;
    for (int t = warp; t < see; t += 4) {
        const int page = after_wait(a.table)[(size_t)r * a.max_pages + t / a.l.bs], place = t % a.l.bs;
        if (page < 0 || page >= a.l.n_pages) {
            dev_fail(a.err, DEV_BAD_ARG);
            continue;
        }
        const uint8_t *rec = after_wait(a.l.pages) + ((int64_t)page * a.l.nkv + kv) * a.l.rec;
        const uint32_t line = grp * a.l.bs + place;
        const float dk = __half2float(*(const __half *)(rec + 2 * a.l.kb + line * 2));
        const float dv = __half2float(*(const __half *)(rec + 2 * a.l.kb + a.l.sb + line * 2));
        const uint8_t *kc = rec + line * 32 + in / 2, *vc = kc + a.l.kb;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j) s += q[j] * (float)((kc[j / 2] >> (4 * (j & 1)) & 15) - 8);
        s *= dk;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m, s), f = mn == -INFINITY ? 1.0f : expf(m - mn), p = mn == -INFINITY ? 0.0f : expf(s - mn);
        m = mn;
        l = l * f + p;
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] = o[j] * f + p * dv * (float)((vc[j / 2] >> (4 * (j & 1)) & 15) - 8);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) so[warp][lane * PER + j] = o[j];
    if (lane == 0) sml[warp][0] = m, sml[warp][1] = l;
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f, f[4];
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][0]);
    for (int w = 0; w < 4; ++w) {
        f[w] = sml[w][0] == -INFINITY && sml[w][1] == 0.0f ? 0.0f : expf(sml[w][0] - mm);
        ll += f[w] * sml[w][1];
    }
    for (int d = tid; d < HD; d += 128) {
        float y = 0.0f;
        for (int w = 0; w < 4; ++w) y += f[w] * so[w][d];
        y = see <= 0 ? 0.0f : y / ll;  // a NaN score leaves no sum: 0 / 0
        if (a.gate && see > 0) y *= sigm((float)((const T *)after_wait(a.gate))[i * a.gt + h * a.gh + d]);
        ((T *)a.out)[i * a.ot + (int64_t)h * HD + d] = (T)y;
    }
}

}  // namespace fn

using namespace fn;

FN_API uint64_t fn_kv4_attn_workspace(void) { return 256; }

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
        cudaError_t e = cudaSuccess;
        auto go = [&](auto k) { e = launch_k(k, dim3(rows, nh), dim3(128), 0, (cudaStream_t)stream, a); };
        const bool f32 = type == T_F32;
        if (c->hd == 64) f32 ? go(k_kv4_attn_rows<float, 64>) : go(k_kv4_attn_rows<__nv_bfloat16, 64>);
        else if (c->hd == 128) f32 ? go(k_kv4_attn_rows<float, 128>) : go(k_kv4_attn_rows<__nv_bfloat16, 128>);
        else f32 ? go(k_kv4_attn_rows<float, 256>) : go(k_kv4_attn_rows<__nv_bfloat16, 256>);
        if (e != cudaSuccess) return fail(std::string("kv4 attn launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
