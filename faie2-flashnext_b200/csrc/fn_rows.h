// Rows of heads in memory (host).
#pragma once

#include <algorithm>
#include <cstdint>

namespace fn {

// Whether values of a, rows x nh x hd with token and head strides, may lie where values of b do: not if their bytes are apart, nor if both
// are columns of the same wider rows and those are apart. (Elements of `size` bytes, aligned to it.)
inline bool kv4_rows_meet(const void *a, int64_t a_token, int64_t a_head, const void *b, int64_t b_token, int64_t b_head, int64_t rows,
                          int64_t nh, int64_t hd, int64_t size) {
    struct Span {
        int64_t lo, hi;  // elements
    };
    auto span = [&](const void *p, int64_t token, int64_t head, int64_t tokens) {
        const int64_t at = (int64_t)((uintptr_t)p / (uintptr_t)size), t = (tokens - 1) * token, h = (nh - 1) * head;
        return Span{at + std::min<int64_t>(t, 0) + std::min<int64_t>(h, 0), at + std::max<int64_t>(t, 0) + std::max<int64_t>(h, 0) + hd};
    };
    const Span x = span(a, a_token, a_head, rows), y = span(b, b_token, b_head, rows);
    if (x.lo >= y.hi || y.lo >= x.hi) return false;
    const Span p = span(a, a_token, a_head, 1), q = span(b, b_token, b_head, 1);  // one row each
    if (a_token != b_token || a_token < p.hi - p.lo || a_token < q.hi - q.lo) return true;
    const int64_t from = ((p.lo - q.lo) % a_token + a_token) % a_token;  // where a's columns begin, counted from b's
    return from < q.hi - q.lo || from + (p.hi - p.lo) > a_token;
}

}  // namespace fn
