// Paged KV cache in 4 bits: planning a step of many requests on the GPU, storing rows into their slots, loading them back.
// The attention that reads the pages is in fn_kv4_attn.cu, the page layout in fn_kv4.h. The reference keeps one dense
// fp32 cache per layer (k_qk_norm_rope appends to it, engine/faie2fn.cu:1452-1478); it has no counterpart of these.
#include <cuda_bf16.h>

#include "fn_kv4.h"

namespace fn {

// ---- planning ------------------------------------------------------------------------------------------------------
// Request r holds ctx[r] tokens in have = ceil(ctx / bs) pages and brings add[r] new ones: it needs ceil((ctx + add) / bs)
// - have further pages. Prefix sums over the requests give each its rows and its share of the free stack, so one CTA
// with the requests' offsets in shared memory does all of it; the flat loops (returned pages, taken pages, rows) find
// their request by bisection, so a prompt of thousands of rows spreads over all threads like many single tokens do.
// Nothing but latency bounds it: 3.9 us for 32 requests of a token, 9.9 us for 256 requests with 7284 rows (two launches).
struct PlanArgs {
    int n, max_pages, bs, n_pages, max_tokens;
    const int *ctx, *add;
    int *table, *free_ids;
    const int *free_in;
    int *free_out, *cu, *kv_len, *positions, *requests, *status;
    int64_t *slots;
    int *next;      // the lengths that requests go on with (may be null)
    int rows_here;  // 1: this kernel writes the rows; 0: k_kv4_rows does
};

constexpr int PLAN_T = 1024, PLAN_SMALL = 128;  // threads; the small form for steps of few requests and rows
constexpr int PLAN_PER = KV4_MAX_REQ / PLAN_T;

// exclusive prefix sum of v over the CTA's T threads, and the total
template <int T> __device__ __forceinline__ long long plan_scan(long long v, long long *red, long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    if (lane == 31) red[warp] = s;
    __syncthreads();
    long long w = lane < T / 32 ? red[lane] : 0, t = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
    }
    total = __shfl_sync(0xffffffffu, t, 31);
    const long long before = __shfl_sync(0xffffffffu, t - w, warp);
    __syncthreads();
    return before + s - v;
}

// the last r in 0..n-1 with off[r] <= i (off[0] = 0, not decreasing, i < off[n])
__device__ __forceinline__ int plan_find(const int *off, int n, int i) {
    int lo = 0, hi = n;  // off[lo] <= i < off[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (off[m] <= i) lo = m;
        else hi = m;
    }
    return lo;
}

__device__ __forceinline__ int plan_pages(long long tokens, int bs) { return (int)((tokens + bs - 1) / bs); }

__device__ __forceinline__ void plan_row(const PlanArgs &a, const int *cu, int served_len, int r, int i) {
    const int pos = max(a.ctx[r], 0) + i - cu[r];
    const bool ok = served_len > 0;  // a request with rows and no length was refused
    a.slots[i] = ok ? (int64_t)a.table[(size_t)r * a.max_pages + pos / a.bs] * a.bs + pos % a.bs : -1;
    a.positions[i] = ok ? pos : -1;
    a.requests[i] = r;
}

template <int T> __global__ void __launch_bounds__(T) k_kv4_plan(const PlanArgs a) {
    extern __shared__ int sm_plan[];
    __shared__ long long red[32];
    __shared__ int s_taken, s_refused;
    int *cu = sm_plan, *need0 = cu + a.n + 1, *back0 = need0 + a.n + 1, *len = back0 + a.n + 1;
    const int tid = threadIdx.x, per = (a.n + T - 1) / T, r0 = tid * per;
    if (tid == 0) s_taken = s_refused = 0;
    pdl_wait();
    pdl_trigger();
    const int top0 = min(max(*after_wait(a.free_in), 0), a.n_pages);
    long long ctx[PLAN_PER], fresh[PLAN_PER], sum = 0, total;
    int add[PLAN_PER];
#pragma unroll
    for (int k = 0; k < PLAN_PER; ++k) {
        const int r = r0 + k;
        const bool in = k < per && r < a.n;
        ctx[k] = in ? max(after_wait(a.ctx)[r], 0) : 0;
        add[k] = in ? after_wait(a.add)[r] : 0;
        fresh[k] = max(add[k], 0);
        sum += fresh[k];
    }
    long long end = plan_scan<T>(sum, red, total);
    // rows: offsets clipped to max_tokens; a request whose rows or pages do not fit its arrays takes nothing
    int need[PLAN_PER], back[PLAN_PER];
    bool fits[PLAN_PER];
    long long needs = 0, backs = 0;
#pragma unroll
    for (int k = 0; k < PLAN_PER; ++k) {
        const int r = r0 + k;
        if (k < per && r < a.n) cu[r] = (int)min(end, (long long)a.max_tokens);
        end += fresh[k];
        const long long want = (ctx[k] + fresh[k] + a.bs - 1) / a.bs;
        const int have = plan_pages(ctx[k], a.bs);
        fits[k] = fresh[k] == 0 || (want <= a.max_pages && end <= a.max_tokens);
        need[k] = fresh[k] > 0 && fits[k] ? (int)want - have : 0;
        back[k] = add[k] < 0 ? min(have, a.max_pages) : 0;
        needs += need[k];
        backs += back[k];
    }
    if (tid == 0) cu[a.n] = (int)min(total, (long long)a.max_tokens);
    long long nb = plan_scan<T>(needs, red, total), bb, back_total;
    if (tid == 0) need0[a.n] = (int)min(total, (long long)INT32_MAX);
    bb = plan_scan<T>(backs, red, back_total);
    const int returned = (int)min(back_total, (long long)(a.n_pages - top0)), top = top0 + returned;
    if (tid == 0) back0[a.n] = (int)min(back_total, (long long)INT32_MAX);
    int refused = 0, taken = 0;
#pragma unroll
    for (int k = 0; k < PLAN_PER; ++k) {
        const int r = r0 + k;
        if (k >= per || r >= a.n) continue;
        need0[r] = (int)min(nb, (long long)INT32_MAX);
        back0[r] = (int)min(bb, (long long)INT32_MAX);
        nb += need[k];
        bb += back[k];
        const bool ok = fits[k] && (need[k] == 0 || nb <= top);
        if (ok && need[k]) taken = (int)nb;  // the requests that get pages come before those that find none left
        refused += !ok;
        const int l = add[k] < 0 || !ok ? 0 : (int)min(ctx[k] + fresh[k], (long long)INT32_MAX);
        len[r] = l;
        a.kv_len[r] = l;
        if (a.next) a.next[r] = ok ? l : (int)ctx[k];  // a refused request stands where it stood
    }
    if (taken) atomicMax(&s_taken, taken);
    if (refused) atomicAdd(&s_refused, refused);
    // the pages of finished requests go on top of the stack, in request order
    __syncthreads();
    for (int j = tid; j < returned; j += T) {
        const int r = plan_find(back0, a.n, j);
        a.free_ids[top0 + j] = a.table[(size_t)r * a.max_pages + j - back0[r]];
    }
    for (int r = tid; r <= a.n; r += T) a.cu[r] = cu[r];
    if (tid == 0) {
        *a.free_out = top - s_taken;
        *a.status = s_refused;
    }
    __syncthreads();
    // the new pages come from the top
    for (int j = tid; j < s_taken; j += T) {
        const int r = plan_find(need0, a.n, j);
        a.table[(size_t)r * a.max_pages + plan_pages(max(a.ctx[r], 0), a.bs) + j - need0[r]] = a.free_ids[top - 1 - j];
    }
    if (!a.rows_here) return;
    __syncthreads();
    for (int i = tid; i < a.max_tokens; i += T) {
        if (i < cu[a.n]) {
            const int r = plan_find(cu, a.n, i);
            plan_row(a, cu, len[r], r, i);
        } else {
            a.slots[i] = -1;
            a.positions[i] = a.requests[i] = -1;
        }
    }
}

// the rows of a large step, after k_kv4_plan: one thread a row, the offsets in shared memory (a bisection in global memory
// took 8 round trips)
__global__ void __launch_bounds__(256) k_kv4_rows(const PlanArgs a) {
    extern __shared__ int sm_plan[];
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x * 256 + threadIdx.x;
    for (int r = threadIdx.x; r <= a.n; r += 256) sm_plan[r] = after_wait(a.cu)[r];
    __syncthreads();
    if (i >= a.max_tokens) return;
    if (i < sm_plan[a.n]) {
        const int r = plan_find(sm_plan, a.n, i);
        plan_row(a, sm_plan, after_wait(a.kv_len)[r], r, i);
    } else {
        a.slots[i] = -1;
        a.positions[i] = a.requests[i] = -1;
    }
}

// ---- store / load --------------------------------------------------------------------------------------------------
// A unit is 64 dims of one head of one token (K or V); eight lanes hold eight values each, so a warp covers four units:
// reads of 32 (16) bytes a lane, codes written as one word a lane, 32 adjacent bytes a unit. A thread takes four units, whose
// loads are all under way before the first is used; blockIdx.y is the head of K or V, so that no index is divided.
// Measured: 8192 rows of bf16, 8 heads of 128, store 20 and load 14 us (42 MB each; bound by instruction issue); 32 rows 3 us each.
// d = m / -8 with m the value of largest magnitude (of two opposite ones the positive), c = clamp(trunc(x / d + 8.5), 0,
// 15), so that m itself is the code 0 and all 16 codes are used; d is rounded to fp16 after the codes are chosen.
template <typename T> __device__ __forceinline__ void load8(const T *p, bool vec, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float>(const float *p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, bool vec, float (&x)[8]) {
    if (vec) {
        const uint4 a = *(const uint4 *)p;
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
}

struct Kv4RowArgs {
    Kv4Lay l;
    const void *x[2];          // k, v (store)
    int64_t token[2], head[2];  // their strides in elements
    void *y[2];                // k, v (load): [nt][nkv][hd]; either may be null
    const int64_t *slots;
    int nt, vec;
    uint32_t *err;
};

constexpr int ROW_UNITS = 4;  // of a thread

// unit x of a thread -> token and group; false past the end
__device__ __forceinline__ bool kv4_unit(const Kv4RowArgs &a, int x, int &t, int &g) {
    const int64_t u = ((int64_t)blockIdx.x * ROW_UNITS + x) * 32 + (threadIdx.x >> 3);
    const int lg = a.l.ng >> 1;  // log2 of 1, 2, 4
    g = (int)(u & (a.l.ng - 1));
    t = (int)(u >> lg);
    return (u >> lg) < a.nt;
}
// a slot's record, and the line of a group's codes and scale in it
__device__ __forceinline__ uint8_t *kv4_place(const Kv4Lay &l, int64_t slot, int h, int g, uint32_t &line) {
    line = (uint32_t)(g * l.bs) + (uint32_t)(slot & (l.bs - 1));
    return l.pages + ((slot >> l.lbs) * l.nkv + h) * (int64_t)l.rec;
}

template <typename T> __global__ void __launch_bounds__(256) k_kv4_store(const Kv4RowArgs a) {
    pdl_wait();
    pdl_trigger();
    const int part = blockIdx.y >= a.l.nkv, h = blockIdx.y - part * a.l.nkv, lane = threadIdx.x & 7;
    float v[ROW_UNITS][8];
    int64_t slot[ROW_UNITS];
#pragma unroll
    for (int x = 0; x < ROW_UNITS; ++x) {
        int t, g;
        const bool in = kv4_unit(a, x, t, g);
        slot[x] = in ? after_wait(a.slots)[t] : -1;
        if (in) load8<T>((const T *)after_wait(a.x[part]) + t * a.token[part] + h * a.head[part] + g * KV4_GROUP + lane * 8, a.vec, v[x]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[x][i] = 0.0f;
    }
#pragma unroll
    for (int x = 0; x < ROW_UNITS; ++x) {
        int t, g;
        kv4_unit(a, x, t, g);
        // fminf / fmaxf would drop a NaN, so what is not finite shows in a sum of zeros
        float big = v[x][0], small = v[x][0], zeros = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            big = fmaxf(big, v[x][i]);
            small = fminf(small, v[x][i]);
            zeros = fmaf(v[x][i], 0.0f, zeros);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            small = fminf(small, __shfl_xor_sync(0xffffffffu, small, o));
        }
        const bool bad = (__ballot_sync(0xffffffffu, zeros != 0.0f) >> (threadIdx.x & 24) & 255u) != 0;
        if (slot[x] >= (int64_t)a.l.n_pages * a.l.bs) dev_fail(a.err, DEV_BAD_ARG);
        else if (slot[x] >= 0) {
            const float d = (big >= -small ? big : small) * -0.125f;
            const float inv = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
            uint32_t w = 0, line;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // x / d + 8.5 is 0.5 .. 16.5: adding 2^23 cut towards zero leaves its whole part in the low bits (a conversion would
                // go through the slow pipe)
                const float t = __fadd_rn(__fmul_rn(v[x][i], inv), 8.5f);
                w |= min(__float_as_uint(__fadd_rz(t, 8388608.0f)) & 31u, 15u) << (4 * i);
            }
            uint8_t *rec = kv4_place(a.l, slot[x], h, g, line);
            *(uint32_t *)(rec + part * a.l.kb + line * 32 + lane * 4) = w;
            if (lane == 0) {
                // a block that holds a NaN or an infinity, or whose scale passes fp16, reads back as NaN
                const bool over = bad || fabsf(d) > 65504.0f;
                *(__half *)(rec + 2 * a.l.kb + part * a.l.sb + line * 2) = over ? __ushort_as_half(0x7fffu) : __float2half_rn(d);
            }
        }
    }
}

template <typename T> __global__ void __launch_bounds__(256) k_kv4_load(const Kv4RowArgs a) {
    pdl_wait();
    pdl_trigger();
    const int part = blockIdx.y >= a.l.nkv, h = blockIdx.y - part * a.l.nkv, lane = threadIdx.x & 7;
    if (!a.y[part]) return;
    uint32_t w[ROW_UNITS];
    float d[ROW_UNITS];
#pragma unroll
    for (int x = 0; x < ROW_UNITS; ++x) {
        int t, g;
        int64_t slot = kv4_unit(a, x, t, g) ? after_wait(a.slots)[t] : -1;
        if (slot >= (int64_t)a.l.n_pages * a.l.bs) {
            dev_fail(a.err, DEV_BAD_ARG);
            slot = -1;
        }
        w[x] = 0x88888888u, d[x] = 0.0f;
        if (slot >= 0) {
            uint32_t line;
            const uint8_t *rec = after_wait(kv4_place(a.l, slot, h, g, line));
            w[x] = *(const uint32_t *)(rec + part * a.l.kb + line * 32 + lane * 4);
            d[x] = __half2float(*(const __half *)(rec + 2 * a.l.kb + part * a.l.sb + line * 2));
        }
    }
#pragma unroll
    for (int x = 0; x < ROW_UNITS; ++x) {
        int t, g;
        if (!kv4_unit(a, x, t, g)) continue;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)  // c as the float 2^23 + c, less 2^23 + 8
            y[i] = (__uint_as_float((w[x] >> (4 * i) & 15u) | 0x4b000000u) - 8388616.0f) * d[x];
        T *o = (T *)a.y[part] + ((int64_t)t * a.l.nkv + h) * a.l.hd + g * KV4_GROUP + lane * 8;
        if constexpr (sizeof(T) == 4) {
            *(float4 *)o = make_float4(y[0], y[1], y[2], y[3]);
            *(float4 *)(o + 4) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                b[i] = *(const uint32_t *)&p;
            }
            *(uint4 *)o = make_uint4(b[0], b[1], b[2], b[3]);
        }
    }
}

static int rows_grid(const Kv4RowArgs &a, dim3 &grid) {
    const int64_t g = ((int64_t)a.nt * a.l.ng + 32 * ROW_UNITS - 1) / (32 * ROW_UNITS);
    if (g > INT32_MAX) return -1;
    grid = dim3((unsigned)g, 2 * a.l.nkv);
    return 0;
}

}  // namespace fn

using namespace fn;

FN_API int fn_kv4_plan(int n, const int *ctx, const int *add, int *table, int max_pages, int page_size, int *free_ids,
                       int n_pages, const int *free_in, int *free_out, int max_tokens, int *cu, int *kv_len,
                       int64_t *slots, int *positions, int *requests, int *status, void *stream) {
    return fn_kv4_plan_next(n, ctx, add, table, max_pages, page_size, free_ids, n_pages, free_in, free_out, max_tokens, cu, kv_len, slots,
                            positions, requests, status, nullptr, stream);
}

FN_API int fn_kv4_plan_next(int n, const int *ctx, const int *add, int *table, int max_pages, int page_size, int *free_ids,
                            int n_pages, const int *free_in, int *free_out, int max_tokens, int *cu, int *kv_len,
                            int64_t *slots, int *positions, int *requests, int *status, int *next, void *stream) {
    return kv4_entry("kv4 plan", [&]() -> int {
        if (n < 1 || n > KV4_MAX_REQ) return fail("kv4 plan: requests out of range (1..4096)");
        if (page_size != 16 && page_size != 32 && page_size != 64) return fail("kv4 plan: page size must be 16, 32 or 64");
        if (max_pages < 1 || n_pages < 1 || max_tokens < 0) return fail("kv4 plan: bad page / row counts");
        if (!ctx || !add || !table || !free_ids || !free_in || !free_out || !cu || !kv_len || !status ||
            (max_tokens && (!slots || !positions || !requests)))
            return fail("kv4 plan: null pointer");
        if (ctx == kv_len || add == kv_len) return fail("kv4 plan: kv_len must be an array of its own");
        if (next && (next == ctx || next == add || next == kv_len)) return fail("kv4 plan: next must be an array of its own");
        PlanArgs a{n, max_pages, page_size, n_pages, max_tokens, ctx, add, table, free_ids, free_in, free_out, cu,
                   kv_len, positions, requests, status, slots, next, 0};
        // few rows: the planning CTA writes them itself; many: a second grid
        a.rows_here = max_tokens <= 4 * PLAN_T;
        const size_t smem = (size_t)4 * (n + 1) * sizeof(int);
        cudaError_t e = allow_max_dynamic_smem(k_kv4_plan<PLAN_T>);
        if (e == cudaSuccess && n <= PLAN_SMALL && max_tokens <= 4 * PLAN_SMALL)
            e = launch_k(k_kv4_plan<PLAN_SMALL>, dim3(1), dim3(PLAN_SMALL), smem, (cudaStream_t)stream, a);
        else if (e == cudaSuccess)
            e = launch_k(k_kv4_plan<PLAN_T>, dim3(1), dim3(PLAN_T), smem, (cudaStream_t)stream, a);
        if (e == cudaSuccess && !a.rows_here)
            e = launch_k(k_kv4_rows, dim3((max_tokens + 255) / 256), dim3(256), (size_t)(n + 1) * sizeof(int), (cudaStream_t)stream, a);
        if (e != cudaSuccess) return fail(std::string("kv4 plan launch: ") + cudaGetErrorString(e));
        return 0;
    });
}

FN_API int fn_kv4_store(const fn_kv4_t *c, uint32_t type, const void *k, int64_t k_token, int64_t k_head, const void *v,
                        int64_t v_token, int64_t v_head, const int64_t *slots, int nt, void *stream) {
    return kv4_entry("kv4 store", [&]() -> int {
        Kv4RowArgs a{};
        if (kv4_layout(c, a.l, "kv4 store")) return -1;
        if (type != T_F32 && type != T_BF16) return fail("kv4 store: rows must be F32 or BF16");
        if (nt < 0) return fail("kv4 store: bad row count");
        if (nt == 0) return 0;
        if (!k || !v || !slots) return fail("kv4 store: null pointer");
        const int size = type == T_F32 ? 4 : 2;
        if ((uintptr_t)k % size || (uintptr_t)v % size) return fail("kv4 store: rows must be aligned to their type");
        a.x[0] = k, a.x[1] = v;
        a.token[0] = k_token, a.token[1] = v_token, a.head[0] = k_head, a.head[1] = v_head;
        a.slots = slots;
        a.nt = nt;
        a.err = dev_error_ptr();
        a.vec = 1;
        for (int i = 0; i < 2; ++i)
            a.vec &= (uintptr_t)a.x[i] % 16 == 0 && a.token[i] * size % 16 == 0 && a.head[i] * size % 16 == 0;
        dim3 grid;
        if (rows_grid(a, grid)) return fail("kv4 store: too many rows");
        const cudaError_t e = type == T_F32 ? launch_k(k_kv4_store<float>, grid, dim3(256), 0, (cudaStream_t)stream, a)
                                            : launch_k(k_kv4_store<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, a);
        if (e != cudaSuccess) return fail(std::string("kv4 store launch: ") + cudaGetErrorString(e));
        return 0;
    });
}

FN_API int fn_kv4_load(const fn_kv4_t *c, uint32_t type, const int64_t *slots, int nt, void *k, void *v, void *stream) {
    return kv4_entry("kv4 load", [&]() -> int {
        Kv4RowArgs a{};
        if (kv4_layout(c, a.l, "kv4 load")) return -1;
        if (type != T_F32 && type != T_BF16) return fail("kv4 load: rows must be F32 or BF16");
        if (nt < 0) return fail("kv4 load: bad row count");
        if (nt == 0) return 0;
        if ((!k && !v) || !slots) return fail("kv4 load: null pointer");
        if ((uintptr_t)k % 16 || (uintptr_t)v % 16) return fail("kv4 load: rows must be 16-byte aligned");
        a.y[0] = k, a.y[1] = v;
        a.slots = slots;
        a.nt = nt;
        a.err = dev_error_ptr();
        dim3 grid;
        if (rows_grid(a, grid)) return fail("kv4 load: too many rows");
        const cudaError_t e = type == T_F32 ? launch_k(k_kv4_load<float>, grid, dim3(256), 0, (cudaStream_t)stream, a)
                                            : launch_k(k_kv4_load<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, a);
        if (e != cudaSuccess) return fail(std::string("kv4 load launch: ") + cudaGetErrorString(e));
        return 0;
    });
}
