// A mixture-of-experts layer for a few tokens: what its launches share.  Each element type's kernels (one
// for every bit width) are a translation unit of their own.
#pragma once
#include "packed_dot.h"

constexpr int MOE_MAX_E = 1024, MOE_MAX_K = 64;
constexpr int MOE_TOKENS = 64;            // tokens per pass over the experts

// The experts' weights: expert e's entry is w with its pointers moved by e strides.
struct RqExperts {
  RqPacked w;
  int64_t sq, ss, sg;                     // strides of q, scales, g_idx from one expert to the next
};
__device__ __forceinline__ RqPacked rq_expert(const RqExperts& x, int e) {
  RqPacked w = x.w;
  w.q += x.sq * e;
  w.scales += x.ss * e;
  if (w.g_idx) w.g_idx += x.sg * e;
  return w;
}

// Up to 16 tokens of one expert: what a tile of the matrix cores takes.  pairs: token * K + place among the
// token's experts, ascending; past n the first again.  Units past the last have n = 0.
struct RqUnit {
  int expert, n, pairs[16];
};
// Units that T tokens with K experts each can make at most.
inline int rq_units(int T, int E, int K) {
  const int pairs = T * K, all = E + pairs / 16;
  return pairs < all ? pairs : all;
}

// Pieces of the activation between the two products: fp32 in bf16 planes, two where the result is rounded
// to 16 bits (2^-16 is lost), three for fp32 (exact).
template <typename TX>
constexpr int rq_moe_pieces() { return sizeof(TX) == 4 ? 3 : 2; }

// How down is read: h may be filled up to whole chunks, so RUNS needs no ragged end as long as rows are whole
// words of 32 columns; other rows go 8 columns at a time.
inline int rq_moe_out_mode(const RqPacked& down) {
  const int mode = rq_mode_of(down);
  return mode == RQ_RUNS && down.C % 32 ? RQ_SMALL : mode;
}

struct RqMoe {
  int T, D, I, E, K, norm;
  const int* nunits;                      // 1
  const RqUnit* units;                    // rq_units
  const float* weights;                   // T * K
  float* gate;                            // T * K * I: the gate's product where up has other bits or groups
  __hip_bfloat16* h;                      // pieces planes of T * K * ldh
  int ldh;                                // I; where h lies arranged (rq_arranged, for a down of RUNS), whole chunks
  bool arranged;
  float* parts;                           // rq_moe_parts planes of T * D
};
// The product with down for many pairs takes four row tiles a wave for a load of h, which is several times the
// weights' bytes where an expert has many tokens; workgroups share rows until there is one for every CU, and a launch
// of its own adds them up.  From 32 pairs on that is faster (one row tile / four, the whole layer: 8 experts of 4096 x
// 7168 at 5 bits, 2 of them a token, 8 tokens 172 / 178 us, 16 tokens 206 / 193, 64 tokens 340 / 286; 128 of 2048 x 768
// at 4 bits, 8 a token, 4 tokens 63 / 58, 16 tokens 134 / 108), as long as the sums of all tokens fit LDS.
constexpr int MOE_OUT_WAVES = 8, MOE_OUT_ROWS = 4;
inline int rq_moe_parts(int D) {
  const int tiles = (D + 16 * MOE_OUT_ROWS - 1) / (16 * MOE_OUT_ROWS), parts = (256 + tiles - 1) / tiles;
  return parts < 8 ? parts : 8;
}
inline int rq_moe_out_lds(const RqMoe& m, int rows) {
  return MOE_OUT_WAVES * m.T * 64 * rows + rq_units(m.T, m.E, m.K) * (int)sizeof(RqUnit);
}
inline bool rq_moe_dense(const RqMoe& m) {
  return m.T * m.K >= 32 && rq_moe_out_lds(m, MOE_OUT_ROWS) <= 160 * 1024;
}

// LDS for the scales of groups that are no runs of columns (bytes, 0 where there are too many groups): gate's and up's of a
// workgroup's rows, and down's of each wave's expert.  Gathered from memory they cost several times the product.
__host__ __device__ inline int rq_moe_in_lds(const RqPacked& gate, const RqPacked& up) {
  const int most = gate.ngroups > up.ngroups ? gate.ngroups : up.ngroups;
  return most < 256 ? (most + 1) * 128 : 0;
}
inline int rq_moe_out_scales(const RqPacked& down) { return down.ngroups < 64 ? (down.ngroups + 1) * 64 * MOE_OUT_WAVES : 0; }

// h = weight * silu(gate x) * (up x) of every pair, in pieces.
template <typename TX>
void rq_moe_in(const TX* x, int64_t ldx, const RqExperts& gate, int gate_bits, const RqExperts& up, int up_bits,
               const RqMoe& m, hipStream_t s);
// y = the sum over a token's pairs of down h.
template <typename TX>
void rq_moe_out(const RqExperts& down, int bits, const RqMoe& m, TX* y, int64_t ldy, hipStream_t s);
