// Paged KV cache in 4 bits: the page layout that fn_kv4.cu (planning, store, load) and fn_kv4_attn.cu (attention) share.
//
// A record holds page_size tokens of one kv head: K codes [hd / 64][page_size][32 bytes], V codes likewise, K scales
// fp16 [hd / 64][page_size], V scales likewise. 64 dims of a token share a scale d; dim i of them is nibble i of its 32
// bytes (low nibble first), a code c that stands for d (c - 8). One record is one contiguous run, so a kernel fetches
// a page of a head with one bulk copy; inside it the 32 bytes of consecutive tokens are adjacent, which is what makes the
// attention kernel's fragment reads of shared memory free of bank conflicts (token-major rows of hd / 2 bytes would put
// eight tokens into the same banks).
#pragma once

#include "fn_engine.h"
#include "fn_rows.h"
#include "faie2fn.h"

namespace fn {

constexpr int KV4_GROUP = 64;       // dims that share a scale
constexpr int KV4_MAX_REQ = 4096;   // requests per call (the planning CTA's offsets live in its shared memory)

struct Kv4Lay {
    uint8_t *pages;
    int n_pages, bs, lbs, nkv, hd, ng;  // lbs = log2 bs, ng = hd / 64
    uint32_t kb, sb, rec;           // bytes of a record's K codes (= V codes), of its K scales (= V scales), of all
};

__host__ __device__ __forceinline__ uint32_t kv4_record(int hd, int bs) {
    return 2u * (uint32_t)bs * (uint32_t)(hd / 2 + hd / KV4_GROUP * 2);
}

// 0, or -1 with the message set
inline int kv4_layout(const fn_kv4_t *c, Kv4Lay &l, const char *who) {
    if (!c || !c->pages) return fail(std::string(who) + ": no cache");
    if (c->hd != 64 && c->hd != 128 && c->hd != 256) return fail(std::string(who) + ": head dim must be 64, 128 or 256");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64)
        return fail(std::string(who) + ": page size must be 16, 32 or 64");
    if (c->nkv < 1 || c->nkv > 1024 || c->n_pages < 1) return fail(std::string(who) + ": bad head / page counts");
    if ((uintptr_t)c->pages % 16) return fail(std::string(who) + ": pages must be 16-byte aligned");
    l.pages = c->pages;
    l.n_pages = c->n_pages;
    l.bs = c->page_size;
    l.lbs = l.bs == 16 ? 4 : l.bs == 32 ? 5 : 6;
    l.nkv = c->nkv;
    l.hd = c->hd;
    l.ng = c->hd / KV4_GROUP;
    l.kb = (uint32_t)l.bs * l.hd / 2;
    l.sb = (uint32_t)l.bs * l.ng * 2;
    l.rec = 2 * (l.kb + l.sb);
    return 0;
}

// a C entry must not let an exception pass
template <typename F> int kv4_entry(const char *who, F f) {
    try {
        return f();
    } catch (...) {
        try {
            return fail(std::string(who) + ": out of host memory");
        } catch (...) {
            return -1;
        }
    }
}

}  // namespace fn
