// Reading a packed weight: rows of nbits-wide fields (pack.hip's format), and the scale of a column.
#pragma once
#include <type_traits>

#include "rq_common.h"

// A packed weight as the operators see it.  groupsize > 0: column c belongs to scale group
// c / groupsize; groupsize == 0: to g_idx[c].  One group needs neither.
struct RqPacked {
  const uint32_t* q;      // [R, ldp] words
  int64_t ldp;
  const float* scales;    // [ngroups, lds], row r's scale of group g at scales[g * lds + r]
  int64_t lds;
  const int32_t* g_idx;   // [C] or NULL
  int R, C, ngroups, groupsize;
  uint32_t run_magic;     // ceil(2^32 / (groupsize / 32)) for rq_run_group; 0: one group, 1: groups of 32
};

// The groups are runs of a multiple of n columns (n of 32), and rq_run_group may be asked for them.
inline bool rq_runs_of(const RqPacked& w, int n) {
  if (w.ngroups == 1) return true;
  return w.groupsize > 0 && w.groupsize % n == 0 && (int64_t)(w.C / 32 + 1) * (w.groupsize / 32 + 1) < 1ll << 32;
}

// The weight an entry point was given.  run_magic divides by groupsize / 32 (group sizes that are multiples of
// 32): n * magic >> 32 is n / d while n * d < 2^32.
inline RqPacked rq_packed(const uint32_t* q, int64_t ldp, const float* scales, int64_t lds, const int32_t* g_idx, int R,
                          int C, int ngroups, int groupsize) {
  const uint32_t d = ngroups > 1 && groupsize > 0 && groupsize % 32 == 0 ? (uint32_t)groupsize / 32 : 0;
  const uint32_t magic = d == 0 ? 0 : d == 1 ? 1 : (uint32_t)(((1ull << 32) + d - 1) / d);
  return RqPacked{q, ldp, scales, lds, g_idx, R, C, ngroups, groupsize, magic};
}

// The group of column c, ngroups where g_idx names none (its scale then reads as NaN, never out of bounds).
__device__ __forceinline__ uint32_t rq_group_of(const RqPacked& w, int c) {
  if (w.ngroups == 1) return 0;
  return min((uint32_t)(w.groupsize > 0 ? c / w.groupsize : w.g_idx[c]), (uint32_t)w.ngroups);
}
__device__ __forceinline__ float rq_scale_of(const RqPacked& w, uint32_t g, int r) {
  const float s = w.scales[(int64_t)(g < (uint32_t)w.ngroups ? g : 0) * w.lds + r];
  return g < (uint32_t)w.ngroups ? s : __builtin_nanf("");
}

// The nc <= 8 codes of columns [c, c + nc), c a multiple of 8; the rest read as 0.  No word past the last of these
// fields is read (row's first where nc <= 0 and c = 0): the loads are moved back, not masked.
template <int NB>
__device__ __forceinline__ void rq_codes8(const uint32_t* __restrict__ row, int c, int nc, int (&code)[8]) {
  constexpr int half = 1 << (NB - 1);
  constexpr uint32_t mask = (1u << NB) - 1u;
  constexpr int NW = (24 + 8 * NB + 31) / 32;
  const int64_t bit = (int64_t)c * NB;
  const uint32_t* p = row + (bit >> 5);
  const int off = (int)(bit & 31);                       // 0, 8, 16 or 24
  const int nw = (off + nc * NB + 31) >> 5;
  uint32_t w[NW + 1];
#pragma unroll
  for (int k = 0; k < NW; ++k) w[k] = p[max(min(k, nw - 1), 0)];
  w[NW] = 0u;
#pragma unroll
  for (int k = 0; k < NW; ++k) w[k] = (uint32_t)((((uint64_t)w[k + 1] << 32) | w[k]) >> off);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int b = k * NB, i = b >> 5, o = b & 31;
    const uint32_t hi = i + 1 < NW ? w[i + 1] : 0u;
    const int v = (int)((uint32_t)((((uint64_t)hi << 32) | w[i]) >> o) & mask) - half;
    code[k] = k < nc ? v : 0;
  }
}

// f(std::integral_constant<int, nbits>) for a run-time nbits in [2, 9]: 8-bit codes take 8 bits, or 9
// when the quantizer was asymmetric.
constexpr int RQ_PACKED_MAXBITS = 9;
template <typename F>
inline void rq_with_nbits(int nbits, F&& f) {
  switch (nbits) {
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 5: f(std::integral_constant<int, 5>{}); break;
    case 6: f(std::integral_constant<int, 6>{}); break;
    case 7: f(std::integral_constant<int, 7>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    default: f(std::integral_constant<int, 9>{}); break;
  }
}

// f(a null pointer of the element type) for a dtype code; false if there is no such type.
template <typename F>
inline bool rq_with_dtype(int dtype, F&& f) {
  if (dtype == RQ_F16) f((__half*)nullptr);
  else if (dtype == RQ_BF16) f((__hip_bfloat16*)nullptr);
  else if (dtype == RQ_F32) f((float*)nullptr);
  else return false;
  return true;
}

inline int rq_packed_check(const RqPacked& w, int nbits) {
  if (!w.q || !w.scales || w.R <= 0 || w.C <= 0 || w.ngroups <= 0 || w.lds < w.R || w.groupsize < 0) return RQ_EINVAL;
  if (nbits < 2 || nbits > RQ_PACKED_MAXBITS) return RQ_EINVAL;
  if (w.ldp < ((int64_t)w.C * nbits + 31) / 32) return RQ_EINVAL;
  if (w.ngroups > 1) {
    if (w.groupsize == 0 && !w.g_idx) return RQ_EINVAL;
    if (w.groupsize > 0 && (w.C - 1) / w.groupsize >= w.ngroups) return RQ_EINVAL;
  }
  return RQ_OK;
}
