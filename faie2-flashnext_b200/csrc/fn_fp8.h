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

}  // namespace fn
