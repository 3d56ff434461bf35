// A mixture-of-experts layer for a few tokens: what its launches share.  Each element type's kernels (one
// for every bit width) are a translation unit of their own.
#pragma once
#include "packed_dot.h"

constexpr int MOE_MAX_E = 1024, MOE_MAX_K = 64;
constexpr int MOE_TOKENS = 64;            // tokens per pass over the experts
constexpr int MOE_CHOICE = 4;             // times 64: experts of one token that the first product chooses from

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

__device__ __forceinline__ float rq_wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ int rq_lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// The K experts of one token's logits; a wave, lane i with experts i, 64 + i, ...  The K-th largest order key is
// found bit by bit from the number of experts that reach a value; all above it are taken, and of those equal to
// it the first: whatever the logits hold, exactly K.
template <int EL>
struct RqChoice {
  float v[EL], m;
  uint32_t key[EL];
  uint64_t taken[EL];                     // of experts 64 u..64 u + 63
  int used;                               // ceil(E / 64)
};
template <int EL>
__device__ __forceinline__ void rq_choose(const float* l, int E, int K, RqChoice<EL>& c) {
  const int lane = threadIdx.x & 63;
  c.used = (E + 63) / 64;
  c.m = -INFINITY;
#pragma unroll
  for (int u = 0; u < EL; ++u) {
    c.taken[u] = 0;
    c.v[u] = -INFINITY;
    c.key[u] = 0;
    if (u >= c.used) continue;
    const int e = 64 * u + lane;
    const float logit = l[min(e, E - 1)];
    c.v[u] = e < E ? logit : -INFINITY;
    c.key[u] = e < E ? rq_order_key(logit) : 0;      // below every logit's
    c.m = rq_nan_max(c.m, c.v[u]);
  }
  uint32_t least = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t tried = least | (1u << bit);
    int reach = 0;
#pragma unroll
    for (int u = 0; u < EL; ++u)
      if (u < c.used) reach += __popcll(__ballot(c.key[u] >= tried));
    if (reach >= K) least = tried;
    if (reach == K) break;
  }
  int above = 0, equal = 0;
#pragma unroll
  for (int u = 0; u < EL; ++u)
    if (u < c.used) above += __popcll(__ballot(c.key[u] > least));
#pragma unroll
  for (int u = 0; u < EL; ++u) {
    if (u >= c.used) continue;
    const uint64_t eq = __ballot(c.key[u] == least);
    c.taken[u] = __ballot(c.key[u] > least || (c.key[u] == least && equal + rq_lanes_before(eq) < K - above));
    equal += __popcll(eq);
  }
  for (int o = 32; o; o >>= 1) c.m = rq_nan_max(c.m, __shfl_xor(c.m, o));
}

// Pieces of the activation between the two products: an fp32 number in three bf16 planes, exactly, whatever x's type
// (kept in fp32 and cut where it is loaded it takes two thirds of the bytes, and longer: 128 experts of 2048 x 768, 1
// token 30.2 us for 27.0, 8 of 4096 x 7168, 8 tokens 190 for 178).
constexpr int MOE_PIECES = 3;

// How down is read: h may be filled up to whole chunks, so RUNS needs no ragged end as long as rows are whole
// words of 32 columns; other rows go 8 columns at a time.
inline int rq_moe_out_mode(const RqPacked& down) {
  const int mode = rq_mode_of(down);
  return mode == RQ_RUNS && down.C % 32 ? RQ_SMALL : mode;
}

struct RqMoe {
  int T, D, I, E, K, norm;
  int* nunits;                            // 1
  RqUnit* units;                          // rq_units
  const float* weights;                   // T * K
  float* gate;                            // T * K * I: the gate's product where up has other bits or groups
  __hip_bfloat16* h;                      // MOE_PIECES planes of T * K * ldh
  int ldh;                                // I; where h lies arranged (rq_arranged, for a down of RUNS), whole chunks
  bool arranged;
  float* parts;                           // rq_moe_parts planes of T * D
  const float* logits;                    // of the one token whose experts the first product chooses, or NULL
  int* ids_out;                           // then: NULL or K
  float* weights_out;
};
// The product with down for many pairs takes four row tiles a wave for a load of h, which is several times the
// weights' bytes where an expert has many tokens; workgroups share rows until there is one for every CU, and a launch
// of its own adds them up.  From 96 pairs' chunks of 128 columns on that is faster, as long as the sums of all tokens fit
// LDS (one row tile / four, the whole layer in us: 8 experts of 4096 x 7168 at 5 bits, 2 of them a token, 1 token 62.3 /
// 59.1, 8 tokens 179 / 155, 64 tokens 384 / 280; 128 of 2048 x 768 at 4 bits, 8 a token, 1 token 26.8 / 28.8, 2 tokens
// 41.0 / 39.2, 16 tokens 144 / 105; 16 of 512 x 1024 at 8 bits, 2 a token, 4 tokens 29.5 / 35.6).
constexpr int MOE_OUT_WAVES = 8, MOE_OUT_ROWS = 4, MOE_DENSE_CHUNKS = 96;
inline int rq_moe_parts(int D) {
  const int tiles = (D + 16 * MOE_OUT_ROWS - 1) / (16 * MOE_OUT_ROWS), parts = (256 + tiles - 1) / tiles;
  return parts < 8 ? parts : 8;
}
inline int rq_moe_out_lds(const RqMoe& m, int rows) {
  return MOE_OUT_WAVES * m.T * 64 * rows + rq_units(m.T, m.E, m.K) * (int)sizeof(RqUnit);
}
inline bool rq_moe_dense(const RqMoe& m) {
  return (int64_t)m.T * m.K * ((m.I + 127) / 128) >= MOE_DENSE_CHUNKS && rq_moe_out_lds(m, MOE_OUT_ROWS) <= 160 * 1024;
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
