// Rows of a packed weight times tokens on the matrix cores: 16 rows x 16 tokens a tile, no LDS on the
// way.
//
// v_mfma_f32_16x16x32: lane l = 16 q + i holds A[i][8q..8q+7] and B[8q..8q+7][i] and receives
// D[4q..4q+3][i].  A row of A is a row of the weight, a column of B a token.  Which columns of the weight
// the 32 k of a step stand for is free as long as A and B agree, so a lane takes whole words:
//   RUNS   a lane owns 32 consecutive columns (nbits words, one wide load) of each 128-column chunk, and
//          step s multiplies its codes 8s..8s+7.  All four steps of a chunk share one scale group (group
//          sizes that are multiples of 128, or one group): the codes, exact in 16 bits, are multiplied
//          as they are and the chunk's sums take the scale, four fp32 FMAs a lane.
//   SMALL  step s covers 32 consecutive columns, 8 a lane, for group sizes that are multiples of 32:
//          the scale joins after every step.
//   ANY    every weight s * q is formed in fp32 and multiplied on v_mfma_f32_16x16x4_f32 (lane 16 q + i:
//          A[i][q], B[q][i]): any groups, any type.  The workgroup's scales lie in LDS.
// fp32 x is cut into three bf16 pieces (8 + 8 + 8 bits: exact), one product each, with RUNS and SMALL.
#pragma once
#include "packed_bits.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx8 __attribute__((ext_vector_type(8)));

enum { RQ_RUNS = 0, RQ_SMALL = 1, RQ_ANY = 2 };

constexpr int RQ_CHUNK = 128;

// What the matrix cores multiply for an activation type: fp16 as it is, bf16 as it is, fp32 in pieces.
template <typename TX> struct RqOperand;
template <> struct RqOperand<__half> {
  typedef half8 raw;
  typedef half8 vec;
  static constexpr int pieces = 1;
};
template <> struct RqOperand<__hip_bfloat16> {
  typedef bf16x8 raw;
  typedef bf16x8 vec;
  static constexpr int pieces = 1;
};
template <> struct RqOperand<float> {
  typedef floatx8 raw;
  typedef bf16x8 vec;
  static constexpr int pieces = 3;
};
__device__ __forceinline__ floatx4 rq_mfma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 rq_mfma(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Unaligned loads of n bytes (the address is a multiple of the element's size only).
template <typename V, typename T>
__device__ __forceinline__ V rq_load_as(const T* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}

// Small integers (|v| <= 256, exact in every type) to the operand's type.
__device__ __forceinline__ void rq_set2(half8& v, int k, float a, float b) {
  v[k] = (_Float16)a;
  v[k + 1] = (_Float16)b;
}
__device__ __forceinline__ void rq_set2(bf16x8& v, int k, float a, float b) {
  v[k] = (__bf16)a;
  v[k + 1] = (__bf16)b;
}

// Word k of the pattern that has the top bit of every field set: codes are stored offset by
// 2^(NB-1), and flipping that bit makes them two's complement.
template <int NB>
constexpr uint32_t rq_top_bits(int k) {
  uint32_t m = 0;
  for (int j = 0; j < 32; ++j) {
    const int b = j * NB + NB - 1;
    if (b >= 32 * k && b < 32 * k + 32) m |= 1u << (b - 32 * k);
  }
  return m;
}
template <int NB>
__device__ __forceinline__ void rq_to_signed(uint32_t (&w)[NB]) {
#pragma unroll
  for (int k = 0; k < NB; ++k) w[k] ^= rq_top_bits<NB>(k);
}
// Code j of 32 in NB words of two's complement fields.
template <int NB>
__device__ __forceinline__ int rq_signed_code(const uint32_t (&w)[NB], int j) {
  const int b = j * NB, i = b >> 5, o = b & 31;
  if (o + NB <= 32) return ((int)(w[i] << (32 - NB - o))) >> (32 - NB);
  const uint32_t v = (uint32_t)((((uint64_t)w[i + 1 < NB ? i + 1 : i] << 32) | w[i]) >> o);
  return ((int)(v << (32 - NB))) >> (32 - NB);
}
template <typename V, int NB>
__device__ __forceinline__ V rq_codes_operand(const uint32_t (&w)[NB], int s) {
  V v;
#pragma unroll
  for (int k = 0; k < 8; k += 2)
    rq_set2(v, k, (float)rq_signed_code<NB>(w, 8 * s + k), (float)rq_signed_code<NB>(w, 8 * s + k + 1));
  return v;
}

// Eight x of a token as they are loaded (FULL: all eight exist; else the first n, the rest 0), and the
// operand's pieces made of them.
template <bool FULL>
__device__ __forceinline__ half8 rq_load_x(const __half* p, int n) {
  if (FULL) return rq_load_as<half8>(p);
  half8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? rq_load_as<_Float16>(p + k) : (_Float16)0.0f;
  return v;
}
template <bool FULL>
__device__ __forceinline__ bf16x8 rq_load_x(const __hip_bfloat16* p, int n) {
  if (FULL) return rq_load_as<bf16x8>(p);
  bf16x8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? rq_load_as<__bf16>(p + k) : (__bf16)0.0f;
  return v;
}
template <bool FULL>
__device__ __forceinline__ floatx8 rq_load_x(const float* p, int n) {
  if (FULL) return rq_load_as<floatx8>(p);
  floatx8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? p[k] : 0.0f;
  return v;
}
__device__ __forceinline__ void rq_operand(half8 x, half8 (&v)[1]) { v[0] = x; }
__device__ __forceinline__ void rq_operand(bf16x8 x, bf16x8 (&v)[1]) { v[0] = x; }
// fp32 in bf16 pieces.  Three: cut off by truncation, 8 + 8 + 8 bits, exact (canonicalising keeps a NaN's
// mark in its upper half).  Two: the first rounded to nearest, so the second leaves at most 2^-16 of the
// value.  An infinite first piece leaves 0 over.
template <int P>
__device__ __forceinline__ void rq_operand(floatx8 x, bf16x8 (&v)[P]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (P == 2) {
      v[0][k] = (__bf16)x[k];
      const float hi = (float)v[0][k];
      v[1][k] = (__bf16)(__builtin_fabsf(hi) == INFINITY ? 0.0f : x[k] - hi);
    } else {
      float r = __builtin_canonicalizef(x[k]);
      const bool inf = __builtin_fabsf(r) == INFINITY;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const uint32_t b = __float_as_uint(r) & 0xFFFF0000u;
        const uint16_t top = (uint16_t)(b >> 16);
        __bf16 h;
        __builtin_memcpy(&h, &top, 2);
        v[p][k] = h;
        r -= __uint_as_float(b);
        if (p == 0 && inf) r = 0.0f;
      }
    }
  }
}

// A lane's tokens, one for each of NT tiles: rows of x.
template <typename TX, int NT>
struct RqTokens {
  typedef typename RqOperand<TX>::raw raw;
  typedef typename RqOperand<TX>::vec vec;
  static constexpr int tiles = NT, pieces = RqOperand<TX>::pieces;
  const TX* p[NT];
  template <bool FULL>
  __device__ __forceinline__ raw load(int b, int c, int n) const { return rq_load_x<FULL>(p[b] + c, n); }
  __device__ __forceinline__ float element(int b, int c) const { return rq_load_elem(p[b] + c); }
};
// The same for fp32 values that were stored as P bf16 pieces, `plane` elements from one piece to the next.
template <int P>
struct RqPieceRow {
  bf16x8 v[P];
};
template <int P>
__device__ __forceinline__ void rq_operand(const RqPieceRow<P>& x, bf16x8 (&v)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) v[p] = x.v[p];
}
template <int P>
struct RqPieces {
  typedef RqPieceRow<P> raw;
  typedef bf16x8 vec;
  static constexpr int tiles = 1, pieces = P;
  const __hip_bfloat16* p;
  int64_t plane;
  template <bool FULL>
  __device__ __forceinline__ raw load(int, int c, int n) const {
    raw r;
#pragma unroll
    for (int k = 0; k < P; ++k) r.v[k] = rq_load_x<FULL>(p + k * plane + c, n);
    return r;
  }
  __device__ __forceinline__ float element(int, int c) const {
    float f = rq_load_elem(p + c);
#pragma unroll
    for (int k = 1; k < P; ++k) f += rq_load_elem(p + k * plane + c);
    return f;
  }
};

// The scales of group g and rows r..r+3, without a branch: a load that would pass the table's end is moved
// back and its values shifted up (rows past the weight get some scale, and are never stored).  The table
// holds at least four (rq_mode_of).
__device__ __forceinline__ floatx4 rq_scales4(const RqPacked& w, int g, int r) {
  const int64_t at = (int64_t)g * w.lds + r, last = (int64_t)(w.ngroups - 1) * w.lds + w.R - 4;
  const floatx4 v = rq_load_as<floatx4>(w.scales + (at < last ? at : last));
  const int d = at > last ? (int)(at - last) : 0;
  return floatx4{d == 0 ? v[0] : d == 1 ? v[1] : d == 2 ? v[2] : v[3], d == 0 ? v[1] : d == 1 ? v[2] : v[3],
                 d == 0 ? v[2] : v[3], v[3]};
}

__device__ __forceinline__ int rq_run_group(const RqPacked& w, int c) { return w.ngroups == 1 ? 0 : c / w.groupsize; }

// What a lane needs of a chunk of 128 columns with RUNS: its words and scales, and its tokens' x.
template <int NB, int RT>
struct RqRunsW {
  uint32_t wd[RT][NB];
  floatx4 sc[RT];
};
template <bool FULL, int NB, int RT>
__device__ __forceinline__ void rq_load_runs(const RqPacked& w, const uint32_t* const (&row)[RT], int r0, int ch,
                                             RqRunsW<NB, RT>& f) {
  const int q = (threadIdx.x & 63) >> 4, c = ch * RQ_CHUNK + 32 * q;
  const int g = rq_run_group(w, ch * RQ_CHUNK);
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    const uint32_t* p = row[a] + (int64_t)(c >> 5) * NB;
    if (FULL) {
      __builtin_memcpy(f.wd[a], p, 4 * NB);
    } else {
      const int words = c < w.C ? (min(32, w.C - c) * NB + 31) >> 5 : 0;
#pragma unroll
      for (int k = 0; k < NB; ++k) f.wd[a][k] = k < words ? p[k] : 0u;
    }
    f.sc[a] = rq_scales4(w, g, r0 + 16 * a + 4 * q);
  }
}
template <bool FULL, typename X>
__device__ __forceinline__ void rq_load_tokens(const X& xs, int C, int ch, typename X::raw (&x)[X::tiles][4]) {
  const int c = ch * RQ_CHUNK + 32 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int b = 0; b < X::tiles; ++b)
#pragma unroll
    for (int s = 0; s < 4; ++s) x[b][s] = xs.template load<FULL>(b, c + 8 * s, C - c - 8 * s);
}
template <typename X, int NB, int RT>
__device__ __forceinline__ void rq_chunk_runs(RqRunsW<NB, RT>& f, const typename X::raw (&x)[X::tiles][4],
                                              floatx4 (&acc)[RT][X::tiles]) {
  typedef typename X::vec V;
  constexpr int NT = X::tiles, P = X::pieces;
  floatx4 part[RT][NT];
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    rq_to_signed<NB>(f.wd[a]);
#pragma unroll
    for (int b = 0; b < NT; ++b) part[a][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    V xo[NT][P];
#pragma unroll
    for (int b = 0; b < NT; ++b) rq_operand(x[b][s], xo[b]);
#pragma unroll
    for (int a = 0; a < RT; ++a) {
      const V codes = rq_codes_operand<V, NB>(f.wd[a], s);
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int p = 0; p < P; ++p) part[a][b] = rq_mfma(codes, xo[b][p], part[a][b]);
    }
  }
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[a][b][k] = __builtin_fmaf(f.sc[a][k], part[a][b][k], acc[a][b][k]);
}

// Chunks first, first + step, ... of rows [r0, r0 + 16 RT): acc[a][b] += the weight's rows
// r0 + 16 a + 4q.. times the lane's token of tile b.  A lane without a token is given any other's (its sums
// go nowhere).  lds: scales of the workgroup's rows for ANY, laid out by rq_stage_scales, or NULL.
template <int NB, int MODE, int RT, typename X>
__device__ __forceinline__ void rq_rows_tokens(const RqPacked& w, int r0, const X& xs, int first, int step,
                                               const float* lds, floatx4 (&acc)[RT][X::tiles]) {
  typedef typename X::vec V;
  constexpr int NT = X::tiles, P = X::pieces;
  const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint32_t* row[RT];
#pragma unroll
  for (int a = 0; a < RT; ++a) row[a] = w.q + (int64_t)min(r0 + 16 * a + i, w.R - 1) * w.ldp;
  const int nfull = w.C / RQ_CHUNK, nch = (w.C + RQ_CHUNK - 1) / RQ_CHUNK;
  int ch = first;
  if constexpr (MODE == RQ_RUNS) {
    // The words of D chunks and the tokens of DX are in flight, a chunk's place refilled as soon as it has
    // been used.
    constexpr int D = RT * (NB + 4) <= 18 ? 4 : 2, DX = NT == 1 && sizeof(typename X::raw) <= 16 ? 2 : 1;
    const int n = ch < nfull ? (nfull - ch + step - 1) / step : 0;     // full chunks of this wave
    RqRunsW<NB, RT> f[D];
    typename X::raw x[DX][NT][4];
#pragma unroll
    for (int u = 0; u < D; ++u)
      if (u < n) rq_load_runs<true>(w, row, r0, ch + u * step, f[u]);
    if constexpr (DX == 2) {
#pragma unroll
      for (int u = 0; u < DX; ++u)
        if (u < n) rq_load_tokens<true>(xs, w.C, ch + u * step, x[u]);
    }
    for (int k = 0; k < n; k += D) {
#pragma unroll
      for (int u = 0; u < D; ++u) {
        if (k + u < n) {
          if constexpr (DX == 1) rq_load_tokens<true>(xs, w.C, ch + (k + u) * step, x[0]);
          rq_chunk_runs<X, NB, RT>(f[u], x[u % DX], acc);
          if (DX == 2 && k + u + DX < n) rq_load_tokens<true>(xs, w.C, ch + (k + u + DX) * step, x[u % DX]);
          if (k + u + D < n) rq_load_runs<true>(w, row, r0, ch + (k + u + D) * step, f[u]);
        }
      }
    }
    if (nfull < nch && nfull >= first && (nfull - first) % step == 0) {       // the ragged end is this wave's
      rq_load_runs<false>(w, row, r0, nfull, f[0]);
      rq_load_tokens<false>(xs, w.C, nfull, x[0]);
      rq_chunk_runs<X, NB, RT>(f[0], x[0], acc);
    }
  } else if constexpr (MODE == RQ_SMALL) {
    for (; ch < nch; ch += step) {
      const int c0 = ch * RQ_CHUNK;
      int code[4][RT][8];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int a = 0; a < RT; ++a) {
          const int c = c0 + 32 * s + 8 * q;
          rq_codes8<NB>(row[a], c < w.C ? c : 0, c < w.C ? min(8, w.C - c) : 0, code[s][a]);
        }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int c = c0 + 32 * s + 8 * q;
        if (c0 + 32 * s >= w.C) break;
        const int g = rq_run_group(w, c0 + 32 * s);
        V x[NT][P];
#pragma unroll
        for (int b = 0; b < NT; ++b)
          rq_operand(c + 8 <= w.C ? xs.template load<true>(b, c, 8) : xs.template load<false>(b, c, w.C - c), x[b]);
#pragma unroll
        for (int a = 0; a < RT; ++a) {
          V codes;
#pragma unroll
          for (int k = 0; k < 8; k += 2) rq_set2(codes, k, (float)code[s][a][k], (float)code[s][a][k + 1]);
          const floatx4 sc = rq_scales4(w, g, r0 + 16 * a + 4 * q);
#pragma unroll
          for (int b = 0; b < NT; ++b) {
            floatx4 part = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < P; ++p) part = rq_mfma(codes, x[b][p], part);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[a][b][k] = __builtin_fmaf(sc[k], part[k], acc[a][b][k]);
          }
        }
      }
    }
  } else {
    for (; ch < nch; ch += step) {
      const int c = ch * RQ_CHUNK + 32 * q, n = min(32, w.C - c);     // the lane's columns (n <= 0: none)
      uint32_t wd[RT][NB];
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        const uint32_t* p = row[a] + (int64_t)(c >> 5) * NB;
        const int words = n > 0 ? (n * NB + 31) >> 5 : 0;
#pragma unroll
        for (int k = 0; k < NB; ++k) wd[a][k] = k < words ? p[k] : 0u;
        rq_to_signed<NB>(wd[a]);
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const int g = j < n ? rq_group_of(w, c + j) : 0;
        float xv[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) xv[b] = j < n ? xs.element(b, c + j) : 0.0f;
#pragma unroll
        for (int a = 0; a < RT; ++a) {
          const float s = lds ? lds[((unsigned)g < (unsigned)w.ngroups ? g : w.ngroups) * (16 * RT) + 16 * a + i]
                              : rq_scale_of(w, g, min(r0 + 16 * a + i, w.R - 1));
          const float wv = j < n ? s * (float)rq_signed_code<NB>(wd[a], j) : 0.0f;
#pragma unroll
          for (int b = 0; b < NT; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv, xv[b], acc[a][b], 0, 0, 0);
        }
      }
    }
  }
}

// The workgroup's scales for ANY, group by group, and a group of NaN for columns without one.  The caller
// waits at a barrier before they are read.
__device__ __forceinline__ void rq_stage_scales(const RqPacked& w, int r0, int rows, float* lds) {
  const int total = (w.ngroups + 1) * rows;
  for (int k = threadIdx.x; k < total; k += blockDim.x) {
    const int g = k / rows, r = r0 + k % rows;
    lds[k] = g == w.ngroups ? __builtin_nanf("") : w.scales[(int64_t)g * w.lds + min(r, w.R - 1)];
  }
}
constexpr int RQ_STAGED_GROUPS = 127;       // groups whose scales a workgroup stages (8 KB for 16 rows)

// Which of the three serves a weight.
inline int rq_mode_of(const RqPacked& w) {
  if ((int64_t)(w.ngroups - 1) * w.lds + w.R < 4) return RQ_ANY;
  if (w.ngroups == 1 || (w.groupsize > 0 && w.groupsize % RQ_CHUNK == 0)) return RQ_RUNS;
  return w.groupsize > 0 && w.groupsize % 32 == 0 ? RQ_SMALL : RQ_ANY;
}
