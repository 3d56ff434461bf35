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
// (7.5 GFLOP for each piece), overlapped in part by two waves a SIMD, and waits for the one step of loads that is ahead.
// With the parts left to the caller, 128 tokens of 4096 x 14336 in one launch: 58 us (66 with an adapter's jobs), of which 40
// are issue: on a SIMD 24 matrix instructions (480 cycles) and 96 vector ones (506) of two waves take 739 together.  Two
// weights of 14336 x 4096 from fp32, 64 tokens: 50 us.
#pragma once
#include "packed_dot.h"
#include "plora_down.h"

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

// Where a lane's 8 columns lie in a row of the weight: words from `col` on, of which nw hold its nc columns, shifted by
// off bits.  A lane past the last column reads the row's first word; words past a row's last field are not read.
template <int NB>
struct ColLane {
  int c, nc, off, nw;                                              // nc <= 0: none
  const uint32_t* col;
};
template <int NB>
__device__ __forceinline__ ColLane<NB> col_lane(const RqPacked& w) {
  ColLane<NB> l;
  l.c = blockIdx.x * COLS + 8 * (threadIdx.x & 15);
  l.nc = min(8, w.C - l.c);
  const int64_t bit = (int64_t)l.c * NB;
  l.off = (int)(bit & 31);
  l.nw = l.nc > 0 ? (l.off + l.nc * NB + 31) >> 5 : 0;
  l.col = w.q + (l.nc > 0 ? bit >> 5 : 0);
  return l;
}
// The words of rows r..r+7 (FULL: all exist; else the last row again).
template <bool FULL, int NB>
__device__ __forceinline__ void col_words(const RqPacked& w, const ColLane<NB>& l, int r, uint32_t (&wd)[8][Col8<NB>::NW]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t* p = l.col + (int64_t)(FULL ? r + k : min(r + k, w.R - 1)) * w.ldp;
#pragma unroll
    for (int m = 0; m < Col8<NB>::NW; ++m) wd[k][m] = p[max(min(m, l.nw - 1), 0)];
  }
}
template <bool FULL>
__device__ __forceinline__ floatx8 col_scales(const RqPacked& w, uint32_t g, int r) {
  const float* s = w.scales + (int64_t)g * w.lds + r;
  if (FULL) return rq_load_as<floatx8>(s);
  floatx8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = r + k < w.R ? s[k] : 0.0f;
  return v;
}
// Fields to bit 0, two's complement; odd: their odd nibbles, for 4 bits.
template <int NB>
__device__ __forceinline__ void col_fields(int off, uint32_t (&wd)[8][Col8<NB>::NW], uint32_t (&odd)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int m = 0; m < Col8<NB>::N; ++m) {
      const uint32_t hi = m + 1 < Col8<NB>::NW ? wd[k][m + 1] : 0u;
      const uint32_t v = NB % 4 == 0 ? wd[k][m] : (uint32_t)((((uint64_t)hi << 32) | wd[k][m]) >> off);
      wd[k][m] = v ^ rq_top_bits<NB>(m);
    }
    odd[k] = NB == 4 ? rq_odd_nibbles(wd[k][0]) : 0u;
  }
}
// Eight finite numbers in the three pieces of rq_operand; a number that is not makes its second piece NaN.
__device__ __forceinline__ void col_pieces(floatx8 x, bf16x8 (&v)[3]) {
  uint32_t o[3][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a = x[2 * k], b = x[2 * k + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t ba = __float_as_uint(a), bb = __float_as_uint(b);
      o[p][k] = __builtin_amdgcn_perm(bb, ba, 0x07060302u);        // the upper halves
      a -= __uint_as_float(ba & 0xFFFF0000u);
      b -= __uint_as_float(bb & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) __builtin_memcpy(&v[p], o[p], 16);
}

// Steps first, first + W, ... below sb of 32 rows, RUNS: acc[n][b] += tokens of tile b times code n of the lane's columns.
// A step's words become operands once and serve all token tiles; the next step's words are then loaded, and each
// tile's place is refilled with the tile after the next as soon as it has been cut into pieces.
// CAREFUL: infinities and NaN among the tokens give what the formula gives; without it, NaN.
template <typename TX, int NB, int NT, bool CAREFUL>
__device__ __forceinline__ void cols_runs(const TX* __restrict__ dy, int T, int64_t ldy, const RqPacked& w, int t0, int first, int sb,
                                          floatx4 (&acc)[8][NT]) {
  constexpr int W = cols_waves(NT);
  typedef typename RqOperand<TX>::raw Raw;
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  const ColLane<NB> l = col_lane<NB>(w);
  const uint32_t g = rq_run_group(w, blockIdx.x * COLS);
  const TX* tok[NT];
#pragma unroll
  for (int b = 0; b < NT; ++b) tok[b] = dy + (int64_t)min(t0 + 16 * b + j, T - 1) * ldy + 8 * q;
  auto operands = [&](uint32_t (&wd)[8][Col8<NB>::NW], bf16x8 (&v)[8]) {
    uint32_t odd[8];
    col_fields<NB>(l.off, wd, odd);
#pragma unroll
    for (int n = 0; n < 8; ++n) rq_convert(col_codes<NB>(wd, odd, n), v[n]);
  };
  auto multiply = [&](const Raw& raw, const floatx8& sc, const bf16x8 (&v)[8], int b) {
    floatx8 f;
    fp32_of(raw, f);
    bf16x8 d[3];
    if constexpr (CAREFUL) rq_operand<3>(f * sc, d);
    else col_pieces(f * sc, d);
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int n = 0; n < 8; ++n) acc[n][b] = rq_mfma(d[p], v[n], acc[n][b]);
  };
  const int sf = min(sb, w.R / STEP);                              // up to here steps are full
  int st = first;
  if (!CAREFUL && st < sf) {
    constexpr int AHEAD = 2;
    auto tile = [&](int item, int from) {                          // token tile item mod NT of its step
      const int s = min(from + item / NT * W, sf - 1);
      return rq_load_x<true>(tok[item % NT] + s * STEP, 8);
    };
    uint32_t wd[8][Col8<NB>::NW];
    col_words<true, NB>(w, l, st * STEP + 8 * q, wd);
    floatx8 sc = col_scales<true>(w, g, st * STEP + 8 * q);
    Raw raw[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) raw[k] = tile(k, st);
    // NT = 1 takes two steps a round, so that a tile's place is known
    auto step = [&](auto at) {
      constexpr int AT = decltype(at)::value;
      bf16x8 v[8];
      operands(wd, v);
      const floatx8 s8 = sc * rq_unit<NB>();
      const int next = min(st + W, sf - 1) * STEP + 8 * q;         // the last one again where there is none
      col_words<true, NB>(w, l, next, wd);
      sc = col_scales<true>(w, g, next);
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        constexpr int base = AT % AHEAD;
        const Raw now = raw[(base + b) % AHEAD];
        raw[(base + b) % AHEAD] = tile(b + AHEAD, st);
        multiply(now, s8, v, b);
      }
      st += W;
    };
    if constexpr (NT == 1) {
      for (;;) {
        step(std::integral_constant<int, 0>{});
        if (st >= sf) break;
        step(std::integral_constant<int, 1>{});
        if (st >= sf) break;
      }
    } else {
      while (st < sf) step(std::integral_constant<int, 0>{});
    }
  }
  for (; st < sb; st += W) {                                       // the last rows; CAREFUL: all
    const int r = st * STEP + 8 * q;
    uint32_t wd[8][Col8<NB>::NW];
    col_words<false, NB>(w, l, r, wd);
    const floatx8 s8 = col_scales<false>(w, g, r) * rq_unit<NB>();
    bf16x8 v[8];
    operands(wd, v);
#pragma unroll
    for (int b = 0; b < NT; ++b) multiply(rq_load_x<false>(tok[b] + st * STEP, w.R - r), s8, v, b);
  }
}

// The same with SMALL and ANY, where a scale multiplies the codes, and with RUNS for packed_linear_backward, whose waves
// have a few steps each, too few for the loads further ahead and the second pass of cols_runs to pay (64 tokens,
// 4096 x 4096 4-bit bf16: 19.3 us for 21.0; 14336 x 4096 34.5 for 35.3).  Infinities and NaN as the formula has them.
template <typename TX, int NB, int MODE, int NT>
__device__ __forceinline__ void cols_scaled(const TX* __restrict__ dy, int T, int64_t ldy, const RqPacked& w, int t0, int first, int sb,
                                            floatx4 (&acc)[8][NT]) {
  constexpr int W = cols_waves(NT);
  typedef ColPieces<TX, MODE> P;
  typedef typename RqOperand<TX>::raw Raw;
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  const ColLane<NB> l = col_lane<NB>(w);
  uint32_t g[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    g[k] = MODE == RQ_RUNS ? rq_run_group(w, blockIdx.x * COLS) : (MODE == RQ_SMALL && k) ? g[0] : k < l.nc ? rq_group_of(w, l.c + k) : 0;
  const TX* tok[NT];
#pragma unroll
  for (int b = 0; b < NT; ++b) tok[b] = dy + (int64_t)min(t0 + 16 * b + j, T - 1) * ldy;

  struct Step {
    uint32_t wd[8][Col8<NB>::NW];
    Raw dy[NT];
    floatx8 sc;
  };
  // FULL: all 32 rows exist; else rows past the last read as dy = 0 and any row's words.
  auto load = [&](auto full, int st, Step& f) {
    constexpr bool FULL = decltype(full)::value;
    const int r = st * STEP + 8 * q;                               // the lane's rows r..r+7
    col_words<FULL, NB>(w, l, r, f.wd);
#pragma unroll
    for (int b = 0; b < NT; ++b) f.dy[b] = rq_load_x<FULL>(tok[b] + r, w.R - r);
    if (MODE != RQ_ANY) f.sc = col_scales<FULL>(w, g[0], r);
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
    col_fields<NB>(l.off, f.wd, odd);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const floatx8 codes = col_codes<NB>(f.wd, odd, n);
      bf16x8 v[P::w];
      floatx8 sc = f.sc;
      if (MODE == RQ_ANY) {
        sc = col_scales<FULL>(w, g[n] < (uint32_t)w.ngroups ? g[n] : 0, r);
        if (g[n] >= (uint32_t)w.ngroups) {
#pragma unroll
          for (int k = 0; k < 8; ++k) sc[k] = FULL || r + k < w.R ? __builtin_nanf("") : 0.0f;
        }
      }
      if constexpr (P::w == 1) rq_convert(codes, v[0]);
      else rq_operand<P::w>(sc * rq_unit<NB>() * codes, v);
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
  int st = first;
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
}

// The waves' sums, halved together, always in the same order, and stored: to part [parts, T, C] or, without parts (PARTS:
// there are), to dx.
template <bool PARTS, typename TX, int NT>
__device__ __forceinline__ void cols_store(floatx4 (&acc)[8][NT], int y, int t0, int T, int C, float* __restrict__ part,
                                           TX* __restrict__ dx, int64_t ldx, floatx4 (*join)[8 * NT][64]) {
  constexpr int W = cols_waves(NT);
  const int lane = threadIdx.x & 63, wave = rq_wave(), q = lane >> 4;
  const int c = blockIdx.x * COLS + 8 * (lane & 15), nc = min(8, C - c);
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
      if (PARTS || part) {
        float* to = part + ((int64_t)y * T + t) * C + c;
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

// packed_linear_backward: grid (tiles of 128 columns, parts, tiles of 16 NT tokens).  A kernel of its own: the arguments of
// the next one's jobs and second weight cost groups of 64 up to 3 % (one token, 4096 x 4096 4-bit bf16: 11.5 us for 11.9).
template <typename TX, int NB, int MODE, int NT>
__global__ __launch_bounds__(64 * cols_waves(NT), cols_occupancy(MODE, NT)) void k_linear_cols(
    const TX* __restrict__ dy, int T, int64_t ldy, RqPacked w, int steps_per, float* __restrict__ part, TX* __restrict__ dx,
    int64_t ldx) {
  __shared__ floatx4 join[cols_waves(NT) / 2][8 * NT][64];
  const int t0 = blockIdx.z * 16 * NT, nsteps = (w.R + STEP - 1) / STEP, sa = blockIdx.y * steps_per;
  floatx4 acc[8][NT];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[n][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  cols_scaled<TX, NB, MODE, NT>(dy, T, ldy, w, t0, sa + rq_wave(), min(nsteps, sa + steps_per), acc);
  cols_store<false, TX, NT>(acc, blockIdx.y, t0, T, w.C, part, dx, ldx, join);
}

// Grid (tiles of 128 columns, rows of jobs and then parts, tiles of 16 NT tokens).  The jobs (of packed linears with
// adapters: what does not wait for this product) come first and spare a launch.  NM weights one after the other: dx = dy_0 W_0 + dy_1 W_1,
// dy_1 lying `plane` elements behind dy_0, and a part is a range of the steps of all.
template <typename TX, int NB, int MODE, int NT, int NM>
__global__ __launch_bounds__(64 * cols_waves(NT), cols_occupancy(MODE, NT)) void k_packed_cols(
    const TX* __restrict__ dy, int T, int64_t ldy, int64_t plane, RqPacked w0, RqPacked w1, RqDownJobs<TX> jobs,
    int job_rows, int steps_per, float* __restrict__ part) {
  constexpr int W = cols_waves(NT);
  __shared__ floatx4 join[W / 2][8 * NT][64];
  const int y = (int)blockIdx.y - job_rows;
  if (y < 0) {
    const int64_t id = ((int64_t)blockIdx.z * job_rows + blockIdx.y) * gridDim.x + blockIdx.x;
    const int z = (int)(id % jobs.z), nth = (int)(id / jobs.z % jobs.adapters);
    const int64_t tile = id / jobs.z / jobs.adapters;
    if (tile < jobs.tiles) rq_lora_down_job<TX, W>(jobs, (int)tile, nth, z, &join[0][0][0]);
    return;
  }
  const int wave = rq_wave(), t0 = blockIdx.z * 16 * NT;
  const int nsteps = (w0.R + STEP - 1) / STEP;
  const int sa = y * steps_per, sb = min(NM * nsteps, sa + steps_per);
  floatx4 acc[8][NT];
  auto run = [&](auto careful) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int b = 0; b < NT; ++b) acc[n][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int m = 0; m < NM; ++m) {
      const int from = max(sa - m * nsteps, 0) + wave, to = min(sb - m * nsteps, nsteps);
      const RqPacked& w = NM == 2 && m ? w1 : w0;
      if constexpr (MODE == RQ_RUNS) cols_runs<TX, NB, NT, decltype(careful)::value>(dy + m * plane, T, ldy, w, t0, from, to, acc);
      else cols_scaled<TX, NB, MODE, NT>(dy + m * plane, T, ldy, w, t0, from, to, acc);
    }
  };
  run(std::false_type{});
  if constexpr (MODE == RQ_RUNS) {
    bool nan = false;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int k = 0; k < 4; k += 2) nan |= __builtin_isunordered(acc[n][b][k], acc[n][b][k + 1]);
    if (__any(nan)) run(std::true_type{});
  }
  cols_store<true, TX, NT>(acc, y, t0, T, w0.C, part, nullptr, 0, join);
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

// dy times one weight (w1 NULL) or two: T tokens to part [sp.parts, T, C].
template <typename TX>
struct Cols {
  const TX* dy;
  int T;
  int64_t ldy, plane;
  const RqPacked* w1;
  RqColSplit sp;
  float* part;
  RqDownJobs<TX> jobs;      // z = 0: none
};
template <typename TX, int NB, int MODE, int NT, int NM>
void launch_cols(const Cols<TX>& a, const RqPacked& w, hipStream_t s) {
  const int rows = a.jobs.z ? rq_jobs_rows(a.jobs, a.T, w.C) : 0;      // for tiles of 64 tokens: smaller ones leave some idle
  hipLaunchKernelGGL((k_packed_cols<TX, NB, MODE, NT, NM>),
                     dim3((w.C + COLS - 1) / COLS, rows + a.sp.parts, (a.T + 16 * NT - 1) / (16 * NT)), dim3(64 * cols_waves(NT)), 0, s,
                     a.dy, a.T, a.ldy, a.plane, w, NM == 2 ? *a.w1 : w, a.jobs, rows, a.sp.steps_per, a.part);
}
// The mode that serves a weight, as a constant, and its number of bits.
template <typename F>
void with_cols_mode(const RqPacked& w, int nbits, F&& f) {
  rq_with_nbits(nbits, [&](auto nb) {
    switch (rq_cols_mode_of(w)) {
      case RQ_RUNS: f(nb, std::integral_constant<int, RQ_RUNS>{}); break;
      case RQ_SMALL: f(nb, std::integral_constant<int, RQ_SMALL>{}); break;
      default: f(nb, std::integral_constant<int, RQ_ANY>{});
    }
  });
}
template <typename TX, int NM>
void cols_of(const Cols<TX>& a, const RqPacked& w, int nbits, hipStream_t s) {
  with_cols_mode(w, nbits, [&](auto nb, auto mode) {
    constexpr int NB = decltype(nb)::value, MODE = decltype(mode)::value;
    // Where codes and fp32 tokens are both cut, registers are left for two token tiles; with RUNS four fit.
    constexpr int NT = RqOperand<TX>::pieces == 1 || MODE == RQ_RUNS ? 4 : 2;
    if (a.T <= 16) launch_cols<TX, NB, MODE, 1, NM>(a, w, s);
    else if (a.T <= 32) launch_cols<TX, NB, MODE, 2, NM>(a, w, s);
    else launch_cols<TX, NB, MODE, NT, NM>(a, w, s);
  });
}

}  // namespace

template <typename TX>
void rq_cols_parts(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                   hipStream_t s) {
  cols_of<TX, 1>(Cols<TX>{dy, T, ldy, 0, nullptr, sp, part, {}}, w, nbits, s);
}
template <typename TX>
void rq_lora_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, const RqColSplit& sp, float* part,
                  const RqDownJobs<TX>& jobs, hipStream_t s) {
  cols_of<TX, 1>(Cols<TX>{dy, T, ldy, 0, nullptr, sp, part, jobs}, w, nbits, s);
}

template <typename TX>
void rq_linear_cols(const TX* dy, int T, int64_t ldy, const RqPacked& w, int nbits, float* part, TX* dx, int64_t ldx,
                    hipStream_t s) {
  with_cols_mode(w, nbits, [&](auto nb, auto mode) {
    for (int64_t t0 = 0; t0 < T; t0 += RQ_COL_TOKENS) {
      const int n = (int)(T - t0 < RQ_COL_TOKENS ? T - t0 : RQ_COL_TOKENS);
      const RqColSplit sp = rq_col_split(n, w.R, w.C);
      TX* out = dx + t0 * ldx;
      auto launch = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        hipLaunchKernelGGL((k_linear_cols<TX, decltype(nb)::value, decltype(mode)::value, NT>),
                           dim3((w.C + COLS - 1) / COLS, sp.parts, (n + 16 * NT - 1) / (16 * NT)), dim3(64 * cols_waves(NT)), 0, s,
                           dy + t0 * ldy, n, ldy, w, sp.steps_per, sp.parts > 1 ? part : nullptr, out, ldx);
      };
      // fp32's pieces leave registers for two token tiles
      if (n <= 16) launch(std::integral_constant<int, 1>{});
      else if (n <= 32) launch(std::integral_constant<int, 2>{});
      else launch(std::integral_constant<int, RqOperand<TX>::pieces == 1 ? 4 : 2>{});
      if (sp.parts > 1)
        hipLaunchKernelGGL(k_packed_join<TX>, dim3((w.C + 255) / 256, n), dim3(256), 0, s, part, sp.parts, n, w.C, out, ldx);
    }
  });
}
