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

// The split where a launch takes up to RQ_COL_WIDE tokens and the caller joins the parts with work of its own: as many
// workgroups as run at once, none left over for a second round (128 tokens of 4096 x 14336: 5 parts for each 64 make
// 560 workgroups of 512 that run, 41 us a launch), of one step for each wave at least.
constexpr int RQ_COL_WIDE = 256;
inline RqColSplit rq_col_split_wide(int T, int64_t steps, int C) {
  const int tiles = (C + 127) / 128 * (T > 32 ? (T + 63) / 64 : 1), at_once = T > 16 && T <= 32 ? 256 : 512;
  int64_t parts = at_once / tiles, most = (steps + 7) / 8;
  parts = parts < most ? parts : most;
  parts = parts > 1 ? parts : 1;
  const int per = (int)((steps + parts - 1) / parts);
  return RqColSplit{(int)((steps + per - 1) / per), per};
}
// Floats of the parts of every launch of T tokens.
inline int64_t rq_col_parts_floats(int T, int64_t steps, int C) {
  int64_t floats = 0;
  for (const int n : {T < RQ_COL_WIDE ? T : RQ_COL_WIDE, T % RQ_COL_WIDE}) {     // a shorter last launch
    const int64_t need = n ? (int64_t)rq_col_split_wide(n, steps, C).parts * n * C : 0;
    floats = need > floats ? need : floats;
  }
  return floats;
}
inline int64_t rq_col_steps(int R) { return (R + 31) / 32; }

// The gradient's parts [sp.parts, T, C] of T <= RQ_COL_WIDE tokens, to be joined by the caller in their order.
template <typename TX>
void rq_cols_parts(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                   hipStream_t s);
// The same of dy W0 + (dy + plane) W1, two weights of one shape that agree in bits and kind of groups, with sp over the
// steps of both.
void rq_cols_parts2(const float* dy, int T, int64_t ldy, int64_t plane, const RqPacked& w0, const RqPacked& w1, int nbits,
                    const RqColSplit& sp, float* part, hipStream_t s);
// Which kernel serves the gradient of a weight: 128 columns' groups are one, 8 columns' are, or any.
inline int rq_cols_mode_of(const RqPacked& w) {
  return rq_runs_of(w, 128) ? 0 : w.groupsize > 0 && w.groupsize % 8 == 0 ? 1 : 2;
}
inline bool rq_cols_together(const RqPacked& w0, int nbits0, const RqPacked& w1, int nbits1) {
  return nbits0 == nbits1 && rq_cols_mode_of(w0) == rq_cols_mode_of(w1);
}
