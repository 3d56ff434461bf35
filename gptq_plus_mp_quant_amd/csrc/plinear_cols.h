// dx = dy W with a packed weight: the kernels and their launches for one element type.
//
// A workgroup takes 128 columns and 16 NT tokens over a range of rows; its waves take steps of 32 rows
// in turn.  v_mfma_f32_16x16x32_bf16 with the tokens as A's rows (k: the step's rows) and the weight as
// B: lane 16 q + j holds columns 8j..8j+7 of rows 8q..8q+7 (8 codes of each of 8 rows, read as they lie),
// and product n of a step takes code n of each row, so that D's column j is the weight's column 8j + n.
// The scale of column and row cannot wait until after the sum over rows:
//   RUNS   all 128 columns are in one group: it multiplies dy, and the codes go in as they are
//   SMALL  a lane's 8 columns are in one group (sizes that are multiples of 8): it multiplies the codes
//   ANY    a scale for every weight
// What a scale multiplied is an fp32 number and is cut into three bf16 pieces, exactly, whatever dy's type: sums
// that cancel keep fp32's precision.  Where both sides are cut, products that come to at most 2^-22 of a term (2^-24
// mostly) are left out.
// Rows are split over workgroups until there are 512, whose sums a second launch joins in their order.
// Measured: 4096 x 4096 5-bit fp16, 8 tokens 9.2 + 4.0 us, latency; 14336 x 4096 4-bit bf16, 64 tokens 33 + 5.4 us (30.6 with
// two pieces): by the counters 13 us of vector issue, conversions of codes and of dy, and 9 us of matrix instructions
// (7.5 GFLOP for each piece), overlapped in part by two waves a SIMD, and waits for the one step that is ahead.
#pragma once
#include "packed_dot.h"

namespace {

// Pieces of dy and of the weight where each is cut (1: bf16 as it is).
template <typename TX, int MODE> struct ColPieces;
template <int MODE> struct ColPieces<__half, MODE> {
  static constexpr int dy = MODE == RQ_RUNS ? 3 : 2, w = MODE == RQ_RUNS ? 1 : 3;
};
template <int MODE> struct ColPieces<__hip_bfloat16, MODE> {
  static constexpr int dy = MODE == RQ_RUNS ? 3 : 1, w = MODE == RQ_RUNS ? 1 : 3;
};
template <int MODE> struct ColPieces<float, MODE> {
  static constexpr int dy = 3, w = MODE == RQ_RUNS ? 1 : 3;
};
constexpr int PIECES_KEPT = 3;             // products of pieces i and j with i + j below this

constexpr int COLS = 128, STEP = 32;

// Words that hold columns c..c+7 of a row, shifted down to bit 0 (c a multiple of 8).
template <int NB>
struct Col8 {
  static constexpr int NW = (24 + 8 * NB + 31) / 32, N = (8 * NB + 31) / 32;
  uint32_t w[NW];
};
template <int NB>
__device__ __forceinline__ int col_code(const uint32_t (&w)[Col8<NB>::NW], int n) {
  const int b = n * NB, i = b >> 5, o = b & 31;
  if (o + NB <= 32) return ((int)(w[i] << (32 - NB - o))) >> (32 - NB);
  const uint32_t v = (uint32_t)((((uint64_t)w[i + 1 < Col8<NB>::NW ? i + 1 : i] << 32) | w[i]) >> o);
  return ((int)(v << (32 - NB))) >> (32 - NB);
}
// Code n of each of 8 rows, over rq_unit (odd: the rows' odd nibbles, for 4 bits).
template <int NB>
__device__ __forceinline__ floatx8 col_codes(const uint32_t (&w)[8][Col8<NB>::NW], const uint32_t (&odd)[8], int n) {
  floatx8 f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (NB == 4) f[k] = rq_nibble(w[k][0], odd[k], n);
    else f[k] = (float)col_code<NB>(w[k], n);
  }
  return f;
}

__device__ __forceinline__ void fp32_of(half8 v, floatx8& f) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (float)v[k];
}
__device__ __forceinline__ void fp32_of(bf16x8 v, floatx8& f) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (float)v[k];
}
__device__ __forceinline__ void fp32_of(floatx8 v, floatx8& f) { f = v; }

constexpr int cols_waves(int nt) { return nt >= 4 ? 4 : 8; }

// Waves of a SIMD that the registers are cut for: with RUNS four token tiles fit 256 (14336 x 4096 4-bit bf16,
// 64 tokens, two pieces: 30 us, 37 with one wave a SIMD and 280); the other modes would spill (4096 x 4096 along an order: 54 for
// 45).
constexpr int cols_occupancy(int mode, int nt) { return mode == RQ_RUNS && nt >= 4 ? 2 : 1; }

template <typename TX, int NB, int MODE, int NT>
__global__ __launch_bounds__(64 * cols_waves(NT), cols_occupancy(MODE, NT)) void k_packed_cols(
    const TX* __restrict__ dy, int T, int64_t ldy, RqPacked w, int steps_per, float* __restrict__ part, TX* __restrict__ dx,
    int64_t ldx) {
  constexpr int W = cols_waves(NT);
  typedef ColPieces<TX, MODE> P;
  typedef typename RqOperand<TX>::raw Raw;
  __shared__ floatx4 join[W / 2][8 * NT][64];
  const int lane = threadIdx.x & 63, wave = rq_wave(), j = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.x * COLS, c = c0 + 8 * j, t0 = blockIdx.z * 16 * NT;
  const int nc = min(8, w.C - c);                                  // the lane's columns (<= 0: none)
  const int nsteps = (w.R + STEP - 1) / STEP;
  const int sa = blockIdx.y * steps_per, sb = min(nsteps, sa + steps_per);
  const int64_t bit = (int64_t)c * NB;
  const int off = (int)(bit & 31), nw = nc > 0 ? (off + nc * NB + 31) >> 5 : 0;
  // A lane past the last column reads the row's first word; words past a row's last field are not read.
  const uint32_t* col = w.q + (nc > 0 ? bit >> 5 : 0);
  uint32_t g[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    g[k] = MODE == RQ_RUNS ? rq_run_group(w, c0) : (MODE == RQ_SMALL && k) ? g[0] : k < nc ? rq_group_of(w, c + k) : 0;
  const TX* tok[NT];
#pragma unroll
  for (int b = 0; b < NT; ++b) tok[b] = dy + (int64_t)min(t0 + 16 * b + j, T - 1) * ldy;

  floatx4 acc[8][NT];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[n][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  struct Step {
    uint32_t wd[8][Col8<NB>::NW];
    Raw dy[NT];
    floatx8 sc;
  };
  // FULL: all 32 rows exist; else rows past the last read as dy = 0 and any row's words.
  auto load = [&](auto full, int st, Step& f) {
    constexpr bool FULL = decltype(full)::value;
    const int r = st * STEP + 8 * q;                               // the lane's rows r..r+7
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t* p = col + (int64_t)(FULL ? r + k : min(r + k, w.R - 1)) * w.ldp;
#pragma unroll
      for (int m = 0; m < Col8<NB>::NW; ++m) f.wd[k][m] = p[max(min(m, nw - 1), 0)];
    }
#pragma unroll
    for (int b = 0; b < NT; ++b) f.dy[b] = rq_load_x<FULL>(tok[b] + r, w.R - r);
    if (MODE != RQ_ANY) {
      const float* s = w.scales + (int64_t)g[0] * w.lds + r;
      if (FULL) {
        f.sc = rq_load_as<floatx8>(s);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f.sc[k] = r + k < w.R ? s[k] : 0.0f;
      }
    }
  };
  auto compute = [&](auto full, int st, Step& f) {
    constexpr bool FULL = decltype(full)::value;
    const int r = st * STEP + 8 * q;
    bf16x8 d[NT][P::dy];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      if constexpr (P::dy == 1) {
        __builtin_memcpy(&d[b][0], &f.dy[b], 16);
      } else {
        floatx8 v;
        fp32_of(f.dy[b], v);
        if (MODE == RQ_RUNS) v *= f.sc * rq_unit<NB>();
        rq_operand<P::dy>(v, d[b]);
      }
    }
    // an inf's product with a piece of 0 would be a NaN that the formula does not have
    bf16x8 low[NT];
    if constexpr (P::w > 1) {
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = (float)d[b][0][k];
          low[b][k] = __builtin_fabsf(v) == INFINITY ? (__bf16)0.0f : d[b][0][k];
        }
    }
    uint32_t odd[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {                                  // fields to bit 0, two's complement
#pragma unroll
      for (int m = 0; m < Col8<NB>::N; ++m) {
        const uint32_t hi = m + 1 < Col8<NB>::NW ? f.wd[k][m + 1] : 0u;
        const uint32_t v = NB % 4 == 0 ? f.wd[k][m] : (uint32_t)((((uint64_t)hi << 32) | f.wd[k][m]) >> off);
        f.wd[k][m] = v ^ rq_top_bits<NB>(m);
      }
      odd[k] = NB == 4 ? rq_odd_nibbles(f.wd[k][0]) : 0u;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const floatx8 codes = col_codes<NB>(f.wd, odd, n);
      bf16x8 v[P::w];
      if constexpr (P::w == 1) {
        rq_convert(codes, v[0]);
      } else {
        floatx8 sc = f.sc;
        if (MODE == RQ_ANY) {
#pragma unroll
          for (int k = 0; k < 8; ++k) sc[k] = rq_scale_of(w, g[n], FULL ? r + k : min(r + k, w.R - 1));
          if (!FULL) {
#pragma unroll
            for (int k = 0; k < 8; ++k) sc[k] = r + k < w.R ? sc[k] : 0.0f;
          }
        }
        rq_operand<P::w>(sc * rq_unit<NB>() * codes, v);
      }
#pragma unroll
      for (int pd = 0; pd < P::dy; ++pd)
#pragma unroll
        for (int pw = 0; pw < P::w; ++pw)
          if (pd + pw < PIECES_KEPT) {
#pragma unroll
            for (int b = 0; b < NT; ++b) {
              if constexpr (P::w > 1) acc[n][b] = rq_mfma(pd == 0 && pw ? low[b] : d[b][pd], v[pw], acc[n][b]);
              else acc[n][b] = rq_mfma(d[b][pd], v[pw], acc[n][b]);
            }
          }
    }
  };
  // A step's loads are in flight while the one before is computed.
  const int sf = min(sb, w.R / STEP);                              // up to here steps are full
  Step now, then;
  int st = sa + wave;
  if (st < sf) {
    load(std::true_type{}, st, now);
    for (; st + W < sf; st += W) {
      load(std::true_type{}, st + W, then);
      compute(std::true_type{}, st, now);
      now = then;
    }
    compute(std::true_type{}, st, now);
    st += W;
  }
  if (st < sb) {
    load(std::false_type{}, st, now);
    compute(std::false_type{}, st, now);
  }
  // The waves' sums, halved together: always in the same order.
#pragma unroll
  for (int half = W / 2; half; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int b = 0; b < NT; ++b) join[wave - half][n * NT + b][lane] = acc[n][b];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[n][b] += join[wave][n * NT + b][lane];
    }
    __syncthreads();
  }
  if (wave) return;
#pragma unroll
  for (int b = 0; b < NT; ++b)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + 16 * b + 4 * q + k;
      if (t >= T) continue;
      floatx8 v;
#pragma unroll
      for (int n = 0; n < 8; ++n) v[n] = acc[n][b][k];
      if (part) {
        float* to = part + ((int64_t)blockIdx.y * T + t) * w.C + c;
        if (nc >= 8) {
          __builtin_memcpy(to, &v, 32);
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n)
            if (n < nc) to[n] = v[n];
        }
      } else {
#pragma unroll
        for (int n = 0; n < 8; ++n)
          if (n < nc) dx[(int64_t)t * ldx + c + n] = rq_cast<TX>(v[n]);
      }
    }
}

template <typename TX>
__global__ __launch_bounds__(256) void k_packed_join(const float* __restrict__ part, int nparts, int T, int C,
                                                     TX* __restrict__ dx, int64_t ldx) {
  const int c = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (c >= C) return;
  float s = 0.0f;
  for (int p = 0; p < nparts; ++p) s += part[((int64_t)p * T + t) * C + c];
  dx[(int64_t)t * ldx + c] = rq_cast<TX>(s);
}

template <typename TX, int NB, int MODE, int NT>
void launch_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, const RqColSplit& sp, float* part, TX* dx, int64_t ldx,
                 hipStream_t s) {
  hipLaunchKernelGGL((k_packed_cols<TX, NB, MODE, NT>), dim3((w.C + COLS - 1) / COLS, sp.parts, (T + 16 * NT - 1) / (16 * NT)),
                     dim3(64 * cols_waves(NT)), 0, s, dy, T, ldy, w, sp.steps_per, part, dx, ldx);
}
template <typename TX, int NB, int MODE>
void linear_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, const RqColSplit& sp, float* part, TX* dx, int64_t ldx,
                 hipStream_t s) {
  constexpr int NT = RqOperand<TX>::pieces == 1 ? 4 : 2;        // fp32's pieces leave registers for two token tiles
  if (T <= 16) launch_cols<TX, NB, MODE, 1>(dy, T, ldy, w, sp, part, dx, ldx, s);
  else if (T <= 32) launch_cols<TX, NB, MODE, 2>(dy, T, ldy, w, sp, part, dx, ldx, s);
  else launch_cols<TX, NB, MODE, NT>(dy, T, ldy, w, sp, part, dx, ldx, s);
}
// T <= RQ_COL_TOKENS tokens to their parts [sp.parts, T, C], or, without parts, to dx.
template <typename TX>
void cols_of(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part, TX* dx,
             int64_t ldx, hipStream_t s) {
  rq_with_nbits(nbits, [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if (rq_runs_of(w, COLS)) linear_cols<TX, NB, RQ_RUNS>(dy, T, ldy, w, sp, part, dx, ldx, s);
    else if (w.groupsize > 0 && w.groupsize % 8 == 0) linear_cols<TX, NB, RQ_SMALL>(dy, T, ldy, w, sp, part, dx, ldx, s);
    else linear_cols<TX, NB, RQ_ANY>(dy, T, ldy, w, sp, part, dx, ldx, s);
  });
}

}  // namespace

template <typename TX>
void rq_cols_parts(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                   hipStream_t s) {
  cols_of<TX>(dy, T, ldy, w, nbits, sp, part, nullptr, 0, s);
}

template <typename TX>
void rq_linear_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, float* part, TX* dx, int64_t ldx,
                    hipStream_t s) {
  for (int64_t t0 = 0; t0 < T; t0 += RQ_COL_TOKENS) {
    const int n = (int)(T - t0 < RQ_COL_TOKENS ? T - t0 : RQ_COL_TOKENS);
    const RqColSplit sp = rq_col_split(n, w.R, w.C);
    TX* out = dx + t0 * ldx;
    cols_of<TX>(dy + t0 * ldy, n, ldy, w, nbits, sp, sp.parts > 1 ? part : nullptr, out, ldx, s);
    if (sp.parts > 1)
      hipLaunchKernelGGL(k_packed_join<TX>, dim3((w.C + 255) / 256, n), dim3(256), 0, s, part, sp.parts, n, w.C, out, ldx);
  }
}
