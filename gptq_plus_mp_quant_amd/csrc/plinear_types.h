// The products with packed weights by element type: each type's kernels (one for every bit width) are a
// translation unit of their own.
#pragma once
#include "packed_bits.h"

template <typename TX>
void rq_linear_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, int nbits, const TX* bias, TX* y, int64_t ldy,
                    hipStream_t s);
template <typename TX>
void rq_linear_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, float* part, TX* dx, int64_t ldx,
                    hipStream_t s);

// How the gradient's sum over rows is split: parts of steps_per steps of 32 rows.
struct RqColSplit {
  int parts, steps_per;
};
constexpr int RQ_COL_TOKENS = 64;           // tokens per launch of the gradient
inline RqColSplit rq_col_split(int T, int R, int C) {
  const int tiles = (C + 127) / 128 * ((T + 63) / 64), steps = (R + 31) / 32;
  // 512 workgroups, each of 16 steps at least (two for each of its waves)
  int parts = (512 + tiles - 1) / tiles;
  parts = parts < (steps + 15) / 16 ? parts : (steps + 15) / 16;
  const int per = (steps + parts - 1) / parts;
  return RqColSplit{(steps + per - 1) / per, per};
}

// The gradient's parts [sp.parts, T, C] of T <= RQ_COL_TOKENS tokens, to be joined by the caller in their order.
template <typename TX>
void rq_cols_parts(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                   hipStream_t s);
