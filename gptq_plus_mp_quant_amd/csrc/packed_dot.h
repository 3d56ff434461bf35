// Rows of a packed weight times tokens on the matrix cores: 16 rows x 16 tokens a tile, words and tokens
// straight to registers (a weight is used once, and LDS would only add a trip).
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

// Codes over rq_unit (integers up to 256 or sixteenths up to 8: exact in every type) to the operand's type.
__device__ __forceinline__ void rq_convert(floatx8 f, half8& v) { v = __builtin_convertvector(f, half8); }
__device__ __forceinline__ void rq_convert(floatx8 f, bf16x8& v) { v = __builtin_convertvector(f, bf16x8); }

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
// 4-bit codes have an instruction of their own, a signed nibble over 16 at the low end of a byte: with the odd
// nibbles shifted down once, 14 instructions make eight operands (20 and more with bit fields).
template <int NB>
constexpr float rq_unit() { return NB == 4 ? 16.0f : 1.0f; }
__device__ __forceinline__ uint32_t rq_odd_nibbles(uint32_t w) {
  uint32_t y = w >> 4;
  asm("" : "+v"(y));               // or the shift is joined with the byte's again
  return y;
}
__device__ __forceinline__ float rq_nibble(uint32_t w, uint32_t odd, int n) {
  return __builtin_amdgcn_cvt_off_f32_i4((n & 1 ? odd : w) >> (8 * (n >> 1)));
}
// Codes 8s..8s+7 of 32 over rq_unit.
template <int NB>
__device__ __forceinline__ floatx8 rq_codes_of(const uint32_t (&w)[NB], int s) {
  floatx8 f;
  if constexpr (NB == 4) {
    const uint32_t odd = rq_odd_nibbles(w[s]);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = rq_nibble(w[s], odd, k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = (float)rq_signed_code<NB>(w, 8 * s + k);
  }
  return f;
}

// Eight x of a token as they are loaded (FULL: all eight exist; else the first n, which may be none, the rest 0),
// and the operand's pieces made of them.  Loads past the row's end are moved back to its last element, whose
// place is p[n - 1], and their values dropped: a mask for every element would take the scalar registers.
template <bool FULL>
__device__ __forceinline__ half8 rq_load_x(const __half* p, int n) {
  if (FULL) return rq_load_as<half8>(p);
  half8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const _Float16 e = rq_load_as<_Float16>(p + min(k, n - 1));
    v[k] = k < n ? e : (_Float16)0.0f;
  }
  return v;
}
template <bool FULL>
__device__ __forceinline__ bf16x8 rq_load_x(const __hip_bfloat16* p, int n) {
  if (FULL) return rq_load_as<bf16x8>(p);
  bf16x8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const __bf16 e = rq_load_as<__bf16>(p + min(k, n - 1));
    v[k] = k < n ? e : (__bf16)0.0f;
  }
  return v;
}
template <bool FULL>
__device__ __forceinline__ floatx8 rq_load_x(const float* p, int n) {
  if (FULL) return rq_load_as<floatx8>(p);
  floatx8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float e = p[min(k, n - 1)];
    v[k] = k < n ? e : 0.0f;
  }
  return v;
}
__device__ __forceinline__ void rq_operand(half8 x, half8 (&v)[1]) { v[0] = x; }
__device__ __forceinline__ void rq_operand(bf16x8 x, bf16x8 (&v)[1]) { v[0] = x; }
// fp32 in bf16 pieces, each cut off by truncation: three carry 8 + 8 + 8 bits, exactly; two an fp16 number's 11
// (canonicalising keeps a NaN's mark in its upper half).  An infinite first piece leaves 0 over.
template <int P>
__device__ __forceinline__ void rq_operand(floatx8 x, bf16x8 (&v)[P]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
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

// A lane's tokens, one for each of NT tiles: rows of x.
template <typename TX, int NT>
struct RqTokens {
  typedef typename RqOperand<TX>::raw raw;
  typedef typename RqOperand<TX>::vec vec;
  static constexpr int tiles = NT, pieces = RqOperand<TX>::pieces;
  static constexpr bool arranged = false;
  const TX* p[NT];
  template <bool FULL>
  __device__ __forceinline__ raw load(int b, int c, int n) const { return rq_load_x<FULL>(p[b] + c, n); }
};
// Where column c of a row lies when its chunks are arranged: columns 32q + 8s.. of a chunk at 32s + 8q.
__device__ __forceinline__ int rq_arranged(int c) { return (c & ~127) + (c >> 3 & 3) * 32 + (c >> 5 & 3) * 8 + (c & 7); }
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
// ARRANGED: within every chunk of 128 columns the 4 x 4 blocks of 8 lie transposed (rq_arranged), as the lanes
// of the codes want them, and the last chunk is filled up with zeros.
template <int P, bool ARRANGED>
struct RqPieces {
  typedef RqPieceRow<P> raw;
  typedef bf16x8 vec;
  static constexpr int tiles = 1, pieces = P;
  static constexpr bool arranged = ARRANGED;
  const __hip_bfloat16* p;
  int64_t plane;
  template <bool FULL>
  __device__ __forceinline__ raw load(int, int c, int n) const {
    raw r;
#pragma unroll
    for (int k = 0; k < P; ++k) r.v[k] = rq_load_x<FULL>(p + k * plane + c, n);
    return r;
  }
};

// A lane's eight x of any kind as fp32.
template <typename V>
__device__ __forceinline__ void rq_floats(const V& x, floatx8& f) { f = __builtin_convertvector(x, floatx8); }
template <int P>
__device__ __forceinline__ void rq_floats(const RqPieceRow<P>& x, floatx8& f) {
  rq_floats(x.v[0], f);
#pragma unroll
  for (int p = 1; p < P; ++p) {
    floatx8 more;
    rq_floats(x.v[p], more);
    f += more;
  }
}
// The groups of the first n (FULL: all eight) of columns c..c+7; past them that of the row's last column.
template <bool FULL>
__device__ __forceinline__ void rq_groups8(const RqPacked& w, int c, int n, uint32_t (&g)[8]) {
  if (w.ngroups > 1 && w.groupsize == 0) {
    if (FULL) {
      __builtin_memcpy(g, w.g_idx + c, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = (uint32_t)w.g_idx[c + min(j, n - 1)];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = min(g[j], (uint32_t)w.ngroups);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = rq_group_of(w, c + (FULL ? j : min(j, n - 1)));
  }
}

// The scales of group g and rows r..r+3 (rows past the weight get some scale, and are never stored).  A load
// that would pass the table's end is moved back, and rq_scales4_of shifts its values up; where R is a
// multiple of 4 only rows past the weight are ever moved.  The table holds at least four (rq_mode_of).
__device__ __forceinline__ floatx4 rq_load_scales4(const RqPacked& w, int g, int r) {
  const int64_t at = (int64_t)g * w.lds + r, last = (int64_t)(w.ngroups - 1) * w.lds + w.R - 4;
  return rq_load_as<floatx4>(w.scales + (at < last ? at : last));
}
__device__ __forceinline__ floatx4 rq_scales4_of(const RqPacked& w, int g, int r, floatx4 v) {
  if ((w.R & 3) == 0) return v;
  const int64_t d = (int64_t)g * w.lds + r - ((int64_t)(w.ngroups - 1) * w.lds + w.R - 4);
  return floatx4{d <= 0 ? v[0] : d == 1 ? v[1] : d == 2 ? v[2] : v[3], d <= 0 ? v[1] : d == 1 ? v[2] : v[3],
                 d <= 0 ? v[2] : v[3], v[3]};
}

// The group of column c where rq_runs_of(w, 32).
__device__ __forceinline__ int rq_run_group(const RqPacked& w, int c) {
  const uint32_t n = (uint32_t)c >> 5;
  return w.run_magic > 1 ? (int)__umulhi(n, w.run_magic) : w.run_magic ? (int)n : 0;
}

// The words of columns c..c+31 of a row (c a multiple of 32); the row's last word again where it has none there,
// for columns whose x is 0.
template <int NB>
__device__ __forceinline__ void rq_words(const uint32_t* row, int c, int C, uint32_t (&w)[NB]) {
  const int64_t first = (int64_t)(c >> 5) * NB, last = ((int64_t)C * NB + 31) / 32 - 1;
#pragma unroll
  for (int k = 0; k < NB; ++k) w[k] = row[first + k < last ? first + k : last];
}

// What a lane needs of a chunk of 128 columns with RUNS: its words and scales, and its tokens' x.  Row tiles
// go over NM weights of one shape, tile a being rows r0 + 16 (a / NM) of weight a mod NM.
template <int NB, int RT>
struct RqRunsW {
  uint32_t wd[RT][NB];
  floatx4 sc[RT];
};
template <bool FULL, int NB, int RT, int NM>
__device__ __forceinline__ void rq_load_runs(const RqPacked (&w)[NM], const uint32_t* const (&row)[RT], int r0, int ch,
                                             RqRunsW<NB, RT>& f) {
  const int q = (threadIdx.x & 63) >> 4, c = ch * RQ_CHUNK + 32 * q;
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    if (FULL) {
      __builtin_memcpy(f.wd[a], row[a] + (int64_t)(c >> 5) * NB, 4 * NB);
    } else {
      rq_words<NB>(row[a], c, w[0].C, f.wd[a]);
    }
    f.sc[a] = rq_load_scales4(w[a % NM], rq_run_group(w[a % NM], ch * RQ_CHUNK), r0 + 16 * (a / NM) + 4 * q);
  }
}
// Step s loads columns 32s + 8q of the chunk, 64 bytes (of a 16-bit type) in a row of each token, and rq_to_runs
// brings them to the lanes of the codes that they go with (columns 32q + 8s, which loaded as they are would
// touch four times as many lines of the cache).
template <bool FULL, typename X>
__device__ __forceinline__ void rq_load_tokens(const X& xs, int C, int ch, typename X::raw (&x)[X::tiles][4]) {
  const int q = (threadIdx.x & 63) >> 4, c = ch * RQ_CHUNK + 8 * q;
#pragma unroll
  for (int b = 0; b < X::tiles; ++b)
#pragma unroll
    for (int s = 0; s < 4; ++s) x[b][s] = xs.template load<FULL>(b, c + 32 * s, C - c - 32 * s);
}
// The 4 x 4 transpose of a step's quarter q of the wave and the step, 32 bits at a time.
template <typename T>
__device__ __forceinline__ void rq_to_runs(T (&x)[4]) {
  static_assert(sizeof(T) % 4 == 0);
  constexpr int N = sizeof(T) / 4;
  uint32_t r[4][N];
  __builtin_memcpy(r, x, sizeof(x));
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const auto a = __builtin_amdgcn_permlane32_swap(r[0][k], r[2][k], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(r[1][k], r[3][k], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    r[0][k] = c[0];
    r[1][k] = c[1];
    r[2][k] = d[0];
    r[3][k] = d[1];
  }
  __builtin_memcpy(x, r, sizeof(x));
}
template <typename X, int NB, int RT, int NM>
__device__ __forceinline__ void rq_chunk_runs(const RqPacked (&w)[NM], int r0, int ch, RqRunsW<NB, RT>& f,
                                              typename X::raw (&x)[X::tiles][4], floatx4 (&acc)[RT][X::tiles]) {
  typedef typename X::vec V;
  constexpr int NT = X::tiles, P = X::pieces;
  floatx4 part[RT][NT];
  if constexpr (!X::arranged) {
#pragma unroll
    for (int b = 0; b < NT; ++b) rq_to_runs(x[b]);
  }
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
      V codes;
      rq_convert(rq_codes_of<NB>(f.wd[a], s), codes);
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int p = 0; p < P; ++p) part[a][b] = rq_mfma(codes, xo[b][p], part[a][b]);
    }
  }
  const int r = r0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    const RqPacked& wa = w[a % NM];
    const floatx4 sc = rq_scales4_of(wa, rq_run_group(wa, ch * RQ_CHUNK), r + 16 * (a / NM), f.sc[a]) * rq_unit<NB>();
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[a][b][k] = __builtin_fmaf(sc[k], part[a][b][k], acc[a][b][k]);
  }
}

// The wave's index as a scalar: what is computed from it needs no exec mask.
__device__ __forceinline__ int rq_wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// A wave's LDS accesses before it are done and seen by the wave's later ones.
__device__ __forceinline__ void rq_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Chunks first, first + step, ...: acc[a][b] += rows 4q.. of row tile a times the lane's token of tile b.  A lane
// without a token is given any other's (its sums go nowhere).  lds: scales of the rows for ANY, laid out by
// rq_stage_scales, or NULL.
template <int NB, int MODE, int RT, int NM, typename X>
__device__ __forceinline__ void rq_rows_tokens(const RqPacked (&w)[NM], int r0, const X& xs, int first, int step,
                                               const float* lds, floatx4 (&acc)[RT][X::tiles]) {
  typedef typename X::vec V;
  constexpr int NT = X::tiles, P = X::pieces;
  const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const uint32_t* row[RT];
#pragma unroll
  for (int a = 0; a < RT; ++a) row[a] = w[a % NM].q + (int64_t)min(r0 + 16 * (a / NM) + i, w[a % NM].R - 1) * w[a % NM].ldp;
  const int C = w[0].C, nfull = C / RQ_CHUNK, nch = (C + RQ_CHUNK - 1) / RQ_CHUNK;
  int ch = first;
  if constexpr (MODE == RQ_RUNS) {
    // The words of D chunks and the tokens of DX are in flight, a chunk's place refilled as soon as it has
    // been used.  No load of the loop is conditional: a wait then counts the later loads that may stay
    // in flight, where a branch around one would make it wait for all of them.
    constexpr int D = NT * P * NM == 1 && NB <= 5 ? 4 : 2, DX = NT == 1 && sizeof(typename X::raw) <= 16 ? 2 : 1;
    const int n = ch < nfull ? (nfull - ch + step - 1) / step : 0;     // full chunks of this wave
    RqRunsW<NB, RT> f[D];
    typename X::raw x[DX][NT][4];
    auto words = [&](int k, RqRunsW<NB, RT>& to) { rq_load_runs<true>(w, row, r0, ch + k * step, to); };
    auto tokens = [&](int k, typename X::raw (&to)[NT][4]) { rq_load_tokens<true>(xs, C, ch + k * step, to); };
    auto compute = [&](int k, RqRunsW<NB, RT>& of, typename X::raw (&xk)[NT][4]) {
      if constexpr (DX == 1) tokens(k, xk);
      rq_chunk_runs<X, NB, RT, NM>(w, r0, ch + k * step, of, xk, acc);
    };
    int k = 0;
    if (n >= D) {
#pragma unroll
      for (int u = 0; u < D; ++u) words(u, f[u]);
      if constexpr (DX == 2) {
        tokens(0, x[0]);
        tokens(1, x[1]);
      }
      for (; k + 2 * D <= n; k += D) {
#pragma unroll
        for (int u = 0; u < D; ++u) {
          compute(k + u, f[u], x[u % DX]);
          if constexpr (DX == 2) tokens(k + u + 2, x[u % 2]);
          words(k + u + D, f[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < D; ++u) {
        compute(k + u, f[u], x[u % DX]);
        if (DX == 2 && u + 2 < D) tokens(k + u + 2, x[u % 2]);
      }
      k += D;
    }
#pragma unroll
    for (int u = 0; u < D - 1; ++u)
      if (k + u < n) words(k + u, f[u]);
#pragma unroll
    for (int u = 0; u < D - 1; ++u)
      if (k + u < n) {
        if constexpr (DX == 2) tokens(k + u, x[0]);
        compute(k + u, f[u], x[0]);
      }
    if (nfull < nch && nfull >= first && (nfull - first) % step == 0) {       // the ragged end is this wave's
      rq_load_runs<false>(w, row, r0, nfull, f[0]);
      rq_load_tokens<false>(xs, C, nfull, x[0]);
      rq_chunk_runs<X, NB, RT, NM>(w, r0, nfull, f[0], x[0], acc);
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
          rq_codes8<NB>(row[a], c < C ? c : 0, c < C ? min(8, C - c) : 0, code[s][a]);
        }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int c = c0 + 32 * s + 8 * q;
        if (c0 + 32 * s >= C) break;
        V x[NT][P];
#pragma unroll
        for (int b = 0; b < NT; ++b)
          rq_operand(c + 8 <= C ? xs.template load<true>(b, c, 8) : xs.template load<false>(b, c, C - c), x[b]);
#pragma unroll
        for (int a = 0; a < RT; ++a) {
          V codes;
          floatx8 f;
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = (float)code[s][a][k];
          rq_convert(f, codes);
          const RqPacked& wa = w[a % NM];
          const int g = rq_run_group(wa, c0 + 32 * s), r = r0 + 16 * (a / NM) + 4 * q;
          const floatx4 sc = rq_scales4_of(wa, g, r, rq_load_scales4(wa, g, r));
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
      const int c = ch * RQ_CHUNK + 32 * q;                         // the lane's 32 columns
      uint32_t wd[RT][NB];
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        rq_words<NB>(row[a], c, C, wd[a]);
        rq_to_signed<NB>(wd[a]);
      }
      auto columns = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;                // else columns past the last have w = x = 0
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int ck = c + 8 * k, nk = C - ck;                    // eight columns, or the nk that exist
          floatx8 xv[NT];
          uint32_t g[NM][8];
#pragma unroll
          for (int b = 0; b < NT; ++b) rq_floats(xs.template load<FULL>(b, ck, nk), xv[b]);
#pragma unroll
          for (int m = 0; m < NM; ++m) rq_groups8<FULL>(w[m], ck, nk, g[m]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int a = 0; a < RT; ++a) {
              const RqPacked& wa = w[a % NM];
              const uint32_t ga = g[a % NM][j];
              const float s = lds ? lds[ga * (16 * RT) + 16 * a + i]
                                  : rq_scale_of(wa, ga, min(r0 + 16 * (a / NM) + i, wa.R - 1));
              const float v = s * (float)rq_signed_code<NB>(wd[a], 8 * k + j), wv = FULL || j < nk ? v : 0.0f;
#pragma unroll
              for (int b = 0; b < NT; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv, xv[b][j], acc[a][b], 0, 0, 0);
            }
          }
        }
      };
      if ((ch + 1) * RQ_CHUNK <= C) columns(std::true_type{});
      else columns(std::false_type{});
    }
  }
}

// Scales for ANY in LDS, group by group, and a group of NaN for columns without one: rows r0..r0+15 of row tile
// `tile` of `tiles`, by the threads first, first + step, ...  The caller waits before they are read.
__device__ __forceinline__ void rq_stage_scales(const RqPacked& w, int r0, int tile, int tiles, int first, int step, float* lds) {
  for (int k = first; k < (w.ngroups + 1) * 16; k += step) {
    const int g = k >> 4, r = r0 + (k & 15);
    lds[g * 16 * tiles + 16 * tile + (k & 15)] = g == w.ngroups ? __builtin_nanf("") : w.scales[(int64_t)g * w.lds + min(r, w.R - 1)];
  }
}
constexpr int RQ_STAGED_GROUPS = 1023;      // groups whose scales a workgroup stages (64 KB for 16 rows)

// Which of the three serves a weight.
inline int rq_mode_of(const RqPacked& w) {
  if ((int64_t)(w.ngroups - 1) * w.lds + w.R < 4) return RQ_ANY;
  if (rq_runs_of(w, RQ_CHUNK)) return RQ_RUNS;
  return rq_runs_of(w, 32) ? RQ_SMALL : RQ_ANY;
}
