// 8-bit rows and weights: what fn_fp8.cu (quantising) and fn_fp8_product.cu (their product) share.
//
// A row's codes are e4m3 numbers, one byte each, with an fp32 scale for each 128 adjacent columns (the last group of a row may be
// shorter); a weight's have one for each 128 x 128 block. A code c stands for c * scale.
#pragma once

#include "fn_engine.h"
#include "fn_kv4.h"

namespace fn {

constexpr int FP8_GROUP = 128;

constexpr int FP8_MAX_COLS = 1 << 24;

inline int fp8_groups(int n) { return n / FP8_GROUP + (n % FP8_GROUP != 0); }

// Two matrices of `rows` rows of `bytes` bytes, p's a step of `ps` >= bytes bytes apart, q's of `qs`: whether they share memory in any way
// other than as the same rows (the same place and step), which a kernel that reads an element before it writes it allows. Columns of one
// buffer side by side do not.
inline bool fp8_mixed(const void *p, int64_t ps, const void *q, int64_t qs, int64_t rows, int64_t bytes) {
    if (!p || !q) return false;
    if (rows == 1) ps = qs = bytes;
    const int64_t d = (int64_t)((uintptr_t)q - (uintptr_t)p);
    if (ps == qs && d == 0) return false;
    if (d >= (rows - 1) * ps + bytes || -d >= (rows - 1) * qs + bytes) return false;
    if (ps != qs) return true;
    const int64_t at = (d % ps + ps) % ps;
    return at < bytes || at > ps - bytes;
}

}  // namespace fn
