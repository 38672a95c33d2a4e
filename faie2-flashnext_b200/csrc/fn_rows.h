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

// The same for rows of `cols` values (strides of either sign, in elements), but for rows that are the same ones in the same order, which a
// kernel that reads an element before it writes it allows.
inline bool rows_mixed(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int64_t rows, int64_t cols, int64_t size) {
    if (!a || !b || (a == b && (a_stride == b_stride || rows == 1))) return false;
    return kv4_rows_meet(a, a_stride, 0, b, b_stride, 0, rows, 1, cols, size);
}

// Whether rows of `bytes` bytes, a step of `stride` bytes (of either sign) apart, share memory with the n bytes from q on. Null pointers
// share none.
inline bool rows_meet_bytes(const void *p, int64_t stride, int64_t rows, int64_t bytes, const void *q, int64_t n) {
    if (!p || !q || rows < 1 || bytes < 1 || n < 1) return false;
    int64_t at = (int64_t)((uintptr_t)q - (uintptr_t)p);  // where they begin, counted from the lowest row
    if (stride < 0) at -= (rows - 1) * stride, stride = -stride;
    if (stride == 0 || at < bytes) return at < bytes && at + n > 0;
    const int64_t i = (at - bytes) / stride + 1;  // the first row that ends behind there
    return i < rows && i * stride < at + n;
}

}  // namespace fn
