// Low-rank adapters beside a packed weight: what the launches share.  Each element type's kernels are a translation
// unit of their own.
#pragma once
#include "packed_dot.h"
#include "plinear_types.h"

constexpr int LORA_MAX_RANK = 256;

// n adapters of rank r: a [n, r, C], b [n, R, r], both contiguous.  Token t's is ids[t] (below 0: none; n or more: one
// that does not exist, whose results are NaN), or the first where there are no ids.
template <typename TX>
struct RqLora {
  const TX* a;
  const TX* b;
  const int64_t* ids;
  const float* scaling;     // [n] or NULL: scale for all
  float scale;
  int n, r;
  __device__ __forceinline__ int of(int64_t t) const {
    if (!ids) return 0;
    const int64_t i = ids[t];
    return i < 0 ? -1 : i < n ? (int)i : n;
  }
  __device__ __forceinline__ float scale_of(int i) const { return scaling ? scaling[i] : scale; }
};

// What a token's adapter makes of its row: [parts, T, ranks], ranks past the last 0; rows of tokens without an adapter
// are not written.  Each part sums RQ_LORA_COLS columns.
struct RqLow {
  float* u;
  int parts, T, ranks;
  __device__ __forceinline__ int64_t at(int p, int64_t t) const { return ((int64_t)p * T + t) * ranks; }
};
constexpr int RQ_LORA_COLS = 2048;
inline RqLow rq_low(float* u, int T, int cols, int r) {
  return RqLow{u, (cols - 1) / RQ_LORA_COLS + 1, T, (r + 31) / 32 * 32};
}
inline int64_t rq_low_floats(const RqLow& l) { return (int64_t)l.parts * l.T * l.ranks; }

// One of low = A x_t (rows: x [T, C] with lora.a) and low = B^T x_t (x [T, R] with lora.b).
template <typename TX>
struct RqDown {
  const TX* x;
  int64_t ldx;
  int cols, rows;
  RqLow low;
};
// One or two of them (z >= zfirst: the second), of the same tokens; z = 0: none.
template <typename TX>
struct RqDownJobs {
  RqDown<TX> first, second;
  RqLora<TX> lora;
  int tiles, adapters, zfirst, z;
};
template <typename TX>
inline RqDownJobs<TX> rq_down_jobs(const RqDown<TX>& first, const RqDown<TX>* second, const RqLora<TX>& lora) {
  const int z0 = first.low.ranks / 16 * first.low.parts, z1 = second ? second->low.ranks / 16 * second->low.parts : 0;
  return RqDownJobs<TX>{first, second ? *second : first, lora, (first.low.T + 15) / 16, lora.ids ? (lora.n < 16 ? lora.n : 16) : 1, z0,
                        z0 + z1};
}
// Beside them: the first's x as RqArranged has it.
struct RqArrange {
  void* out;
  bool paired;
};
template <typename TX>
void rq_lora_down(const RqDownJobs<TX>& jobs, void* arranged, int nbits, hipStream_t s);
inline bool rq_lora_arranged(int T, const RqPacked& w) { return T > 16 && rq_whole_mode_of(w) == RQ_RUNS; }
// The gradient's parts of T <= RQ_COL_WIDE tokens as rq_cols_parts has them, and in the same launch the jobs.
template <typename TX>
void rq_lora_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                  const RqDownJobs<TX>& jobs, hipStream_t s);
// Rows of the grid that the jobs take there; 0: too many, they need a launch of their own.
template <typename TX>
inline int rq_jobs_rows(const RqDownJobs<TX>& jobs, int T, int C) {
  const int64_t row = (int64_t)((C + 127) / 128) * ((T + 63) / 64);
  const int64_t rows = ((int64_t)jobs.tiles * jobs.adapters * jobs.z + row - 1) / row;
  return rows <= 4096 ? (int)rows : 0;
}
// Whether the workgroups make u for themselves: one or two tokens, 16 ranks, and little enough of A for all of them
// together.  One token of 4096 x 4096 with 16 ranks: 13.0 us a call, 17.1 with a launch that makes u first.  That is
// the host's time: replayed in a graph it is 12.0 for 10.4, with few long rows more (2048 x 8192 19.7 for 13.0), and only for
// small weights less (1024 x 1024 7.1 for 7.8).
inline bool rq_lora_own(int T, int R, int C, int r, int bytes) {
  return T <= 2 && r <= 16 && (int64_t)((R + 15) / 16) * T * r * C * bytes <= 40 << 20;
}
// y = x W^T (+ bias) + s B u (low.u NULL: made there); arranged: x once more, where rq_lora_arranged says so.
template <typename TX>
void rq_lora_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, int nbits, const TX* bias, const RqLora<TX>& lora,
                  const RqLow& low, const void* arranged, TX* y, int64_t ldy, hipStream_t s);
// dx (NULL: none) of tokens t0..t0+T-1 = the sum of part [parts, T, C] + s A^T v, and with da (else NULL) da [n, r, C] =
// s sum_t v_t x_t^T and db [n, R, r] = s sum_t dy_t u_t^T over each adapter's tokens of all T.
template <typename TX>
struct RqLoraDx {
  const float* part;
  int parts, t0, T;
  TX* dx;                   // token t0's
  int64_t ldx;
};
template <typename TX>
void rq_lora_grads(const RqLoraDx<TX>& g, const TX* x, int64_t ldx, int C, const TX* dy, int64_t ldy, int R, int T,
                   const RqLora<TX>& lora, const RqLow& u, const RqLow& v, TX* da, TX* db, hipStream_t s);
