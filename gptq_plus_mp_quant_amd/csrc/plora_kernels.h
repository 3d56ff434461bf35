// The products with low-rank adapters, for one element type.
//
// A tile is 16 tokens, as with the packed weight, and goes once over every adapter that one of them has: the matrix
// cores' columns are tokens, so what another adapter makes of a token is dropped, not added as 0 (an adapter that holds an
// inf or NaN spoils its own tokens only).
#pragma once
#include "plora_types.h"
#include "plinear_rows.h"

namespace {

__device__ __forceinline__ floatx4 mfma4(float a, float b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// acc += A[.][32 k] B[32 k][.]: lane 16 q + i holds A[i][8q..8q+7] and B[8q..8q+7][i].
__device__ __forceinline__ floatx4 mfma32(half8 a, half8 b, floatx4 c) { return rq_mfma(a, b, c); }
__device__ __forceinline__ floatx4 mfma32(bf16x8 a, bf16x8 b, floatx4 c) { return rq_mfma(a, b, c); }
__device__ __forceinline__ floatx4 mfma32(floatx8 a, floatx8 b, floatx4 c) {
#pragma unroll
  for (int k = 0; k < 8; ++k) c = mfma4(a[k], b[k], c);
  return c;
}

// Four elements from p on as fp32, the first n of them (which may be none; the rest 0).
template <typename TX>
__device__ __forceinline__ floatx4 load4(const TX* p, int n) {
  floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n >= 4) {
    TX e[4];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = rq_load_elem(e + k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) v[k] = rq_load_elem(p + k);
  }
  return v;
}

// u = A x or B^T x.  Grid (tiles of 16 tokens, the tile's adapters in the order of their first tokens, rank tiles x
// parts); the waves take steps of 32 columns in turn and are joined through LDS in their order.
constexpr int DOWN_WAVES = 8;
template <typename TX, bool ROWS>
__global__ __launch_bounds__(64 * DOWN_WAVES) void k_lora_down(const TX* __restrict__ x, int64_t ldx, int cols, RqLora<TX> lora,
                                                               RqLow low) {
  typedef typename RqOperand<TX>::raw Raw;
  __shared__ floatx4 join[DOWN_WAVES][64];
  const int lane = threadIdx.x & 63, wave = rq_wave(), i = lane & 15, q = lane >> 4;
  const int64_t t = (int64_t)blockIdx.x * 16 + i;
  const int own = t < low.T ? lora.of(t) : -1;
  uint64_t pending = __ballot(lane < 16 && own >= 0 && own < lora.n);
  for (int k = 0; k < (int)blockIdx.y && pending; ++k)
    pending &= ~__ballot(own == __builtin_amdgcn_readlane(own, __ffsll((unsigned long long)pending) - 1));
  if (!pending) return;
  const int lead = __ffsll((unsigned long long)pending) - 1, a = __builtin_amdgcn_readlane(own, lead);
  const int tiles = low.ranks / 16, rank = (blockIdx.z % tiles) * 16, part = blockIdx.z / tiles;
  const int c0 = part * RQ_LORA_COLS, c1 = min(cols, c0 + RQ_LORA_COLS);
  const TX* xs = x + (own == a ? t : (int64_t)blockIdx.x * 16 + lead) * ldx;
  const int row = min(rank + i, lora.r - 1);
  const TX* as = ROWS ? lora.a + ((int64_t)a * lora.r + row) * cols : lora.b + (int64_t)a * cols * lora.r + row;
  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto step = [&](auto full, int c) {
    constexpr bool FULL = decltype(full)::value;
    const int n = c1 - c;                            // the lane's columns (may be none)
    const Raw xv = rq_load_x<FULL>(xs + c, n);
    Raw av;
    if constexpr (ROWS) {
      av = rq_load_x<FULL>(as + c, n);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        typename std::remove_reference<decltype(av[0])>::type e;
        __builtin_memcpy(&e, as + (int64_t)(c + (FULL ? k : min(k, n - 1))) * lora.r, sizeof(e));
        av[k] = FULL || k < n ? e : (decltype(e))0.0f;
      }
    }
    acc = mfma32(av, xv, acc);
  };
  int c = c0 + 32 * wave;
#pragma unroll 4
  for (; c + 32 <= c1; c += 32 * DOWN_WAVES) step(std::true_type{}, c + 8 * q);
  if (c < c1) step(std::false_type{}, c + 8 * q);
  join[wave][lane] = acc;
  __syncthreads();
  if (wave || own != a) return;
  for (int w = 1; w < DOWN_WAVES; ++w) acc += join[w][lane];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (rank + 4 * q + k >= lora.r) acc[k] = 0.0f;
  *reinterpret_cast<floatx4*>(low.u + low.at(part, t) + rank + 4 * q) = acc;
}

// Four ranks of a token, its parts joined in their order.
__device__ __forceinline__ floatx4 low4(const RqLow& low, int64_t t, int rank) {
  floatx4 v = *reinterpret_cast<const floatx4*>(low.u + low.at(0, t) + rank);
  for (int p = 1; p < low.parts; ++p) v += *reinterpret_cast<const floatx4*>(low.u + low.at(p, t) + rank);
  return v;
}

// s B u to the sums of a row tile: 16 ranks of an adapter at a time, dealt to the waves by adapter and rank alone, so that
// a token's bits do not depend on its companions.
template <typename TX>
struct RqLowRank {
  RqLora<TX> lora;
  RqLow low;
  template <int RT, int NT>
  __device__ __forceinline__ void add(int r0, int R, int t0, int T, int wave, int waves, floatx4 (&acc)[RT][NT]) const {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int mine = lane < 16 * NT && t0 + lane < T ? lora.of(t0 + lane) : -1;
    int own[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) own[b] = __shfl(mine, 16 * b + i);
    for (uint64_t pending = __ballot(mine >= 0 && mine < lora.n); pending;) {
      const int a = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)pending) - 1);
      pending &= ~__ballot(mine == a);
      const float s = lora.scale_of(a);
      int turn = wave - a % waves;                   // the first of its rank tiles that this wave takes
      for (int k0 = 16 * (turn < 0 ? turn + waves : turn); k0 < lora.r; k0 += 16 * waves) {
        const int k = k0 + 4 * q;
        floatx4 u[NT], part[RT][NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) u[b] = low4(low, min(t0 + 16 * b + i, T - 1), k);
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          const floatx4 w = load4(lora.b + ((int64_t)a * R + min(r0 + 16 * m + i, R - 1)) * lora.r + k, lora.r - k);
#pragma unroll
          for (int b = 0; b < NT; ++b) {
            part[m][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 4; ++j) part[m][b] = mfma4(w[j], u[b][j], part[m][b]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[m][b][j] = own[b] == a ? __builtin_fmaf(s, part[m][b][j], acc[m][b][j]) : acc[m][b][j];
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NT; ++b)
      if (own[b] == lora.n) {
#pragma unroll
        for (int m = 0; m < RT; ++m) acc[m][b] = floatx4{1.0f, 1.0f, 1.0f, 1.0f} * __builtin_nanf("");
      }
  }
};

// dx: the packed weight's parts and the adapter's term.
template <typename TX>
__global__ __launch_bounds__(256) void k_lora_dx(const float* __restrict__ part, int parts, int64_t t0, int T, int C,
                                                 RqLora<TX> lora, RqLow v, TX* __restrict__ dx, int64_t ldx) {
  __shared__ float low[LORA_MAX_RANK];
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int64_t t = t0 + blockIdx.y;
  const int a = lora.of(t);
  if (a >= 0 && a < lora.n) {
    for (int k = threadIdx.x; k < lora.r; k += 256) {
      float s = v.u[v.at(0, t) + k];
      for (int p = 1; p < v.parts; ++p) s += v.u[v.at(p, t) + k];
      low[k] = s * lora.scale_of(a);
    }
    __syncthreads();
  }
  if (c >= C) return;
  float s = 0.0f;
  for (int p = 0; p < parts; ++p) s += part[((int64_t)p * T + blockIdx.y) * C + c];
  if (a >= lora.n) s = __builtin_nanf("");
  else if (a >= 0) {
    const TX* w = lora.a + (int64_t)a * lora.r * C + c;
    for (int k = 0; k < lora.r; ++k) s = __builtin_fmaf(low[k], rq_load_elem(w + (int64_t)k * C), s);
  }
  dx[(int64_t)blockIdx.y * ldx + c] = rq_cast<TX>(s);
}

// da and db.  Grid (tiles of 128 columns of x, then of dy; rank tiles; adapters): the tokens of the adapter, four to a
// matrix instruction, to the waves in turn.  Lane 16 q + i holds columns 8i..8i+7 of token q, and product n takes
// the n-th of each, so that D's column i is column 8i + n.
constexpr int OUTER_WAVES = 4, WINDOW = 512;
template <typename TX>
__global__ __launch_bounds__(64 * OUTER_WAVES) void k_lora_outer(const TX* __restrict__ x, int64_t ldx, int C,
                                                                 const TX* __restrict__ dy, int64_t ldy, int R, int T,
                                                                 RqLora<TX> lora, RqLow u, RqLow v, TX* __restrict__ da,
                                                                 TX* __restrict__ db) {
  typedef typename RqOperand<TX>::raw Raw;
  __shared__ floatx4 join[OUTER_WAVES][8][64];
  __shared__ int list[WINDOW];
  __shared__ int count;
  const int lane = threadIdx.x & 63, wave = rq_wave(), i = lane & 15, q = lane >> 4;
  const int ctiles = (C + 127) / 128, a = blockIdx.z, rank = blockIdx.y * 16;
  const bool of_a = (int)blockIdx.x < ctiles;        // da: v with x; db: u with dy
  const int width = of_a ? C : R, col = (of_a ? blockIdx.x : blockIdx.x - ctiles) * 128 + 8 * i;
  const TX* src = of_a ? x : dy;
  const int64_t ld = of_a ? ldx : ldy;
  const RqLow low = of_a ? v : u;
  floatx4 acc[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) acc[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t w0 = 0; w0 < T; w0 += WINDOW) {
    if (wave == 0) {
      int n = 0;
      for (int k = 0; k < WINDOW && w0 + k < T; k += 64) {
        const bool is = w0 + k + lane < T && lora.of(w0 + k + lane) == a;
        const uint64_t mask = __ballot(is);
        if (is) list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = k + lane;
        n += __popcll(mask);
      }
      if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    for (int g = 4 * wave; g < n; g += 4 * OUTER_WAVES) {
      const bool is = g + q < n;
      const int64_t t = w0 + list[is ? g + q : 0];
      float m = low.u[low.at(0, t) + rank + i];
      for (int p = 1; p < low.parts; ++p) m += low.u[low.at(p, t) + rank + i];
      const Raw r = col + 8 <= width ? rq_load_x<true>(src + t * ld + col, 8) : rq_load_x<false>(src + t * ld + col, width - col);
      floatx8 f;
      rq_floats(r, f);
      if (!is) {
        m = 0.0f;
        f = floatx8{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = mfma4(m, f[k], acc[k]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) join[wave][n][lane] = acc[n];
  __syncthreads();
  const float s = lora.scale_of(a);
  if (of_a) {
    // wave w: rank 4q + w, eight columns
    const int k = rank + 4 * q + wave;
    if (k >= lora.r) return;
    TX* out = da + ((int64_t)a * lora.r + k) * C + col;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float o = 0.0f;
      for (int w = 0; w < OUTER_WAVES; ++w) o += join[w][n][lane][wave];
      if (col + n < C) out[n] = rq_cast<TX>(s * o);
    }
  } else {
    // wave w: rows 2w and 2w + 1 of the lane's eight, four ranks
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = 2 * wave + h, row = col + n;
      floatx4 o = join[0][n][lane];
      for (int w = 1; w < OUTER_WAVES; ++w) o += join[w][n][lane];
      if (row >= R) continue;
      TX* out = db + ((int64_t)a * R + row) * lora.r + rank + 4 * q;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (rank + 4 * q + k < lora.r) out[k] = rq_cast<TX>(s * o[k]);
    }
  }
}

}  // namespace

template <typename TX>
void rq_lora_down(const TX* x, int T, int64_t ldx, int cols, bool rows, const RqLora<TX>& lora, const RqLow& low, hipStream_t s) {
  const dim3 grid((T + 15) / 16, lora.ids ? (lora.n < 16 ? lora.n : 16) : 1, low.ranks / 16 * low.parts), block(64 * DOWN_WAVES);
  if (rows) hipLaunchKernelGGL((k_lora_down<TX, true>), grid, block, 0, s, x, ldx, cols, lora, low);
  else hipLaunchKernelGGL((k_lora_down<TX, false>), grid, block, 0, s, x, ldx, cols, lora, low);
}

template <typename TX>
void rq_lora_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, int nbits, const TX* bias, const RqLora<TX>& lora,
                  const RqLow& low, TX* y, int64_t ldy, hipStream_t s) {
  rq_with_nbits(nbits, [&](auto nb) {
    linear_rows<TX, decltype(nb)::value>(x, T, ldx, w, bias, y, ldy, RqLowRank<TX>{lora, low}, s);
  });
}

template <typename TX>
void rq_lora_dx(const float* part, int parts, int64_t t0, int T, int C, const RqLora<TX>& lora, const RqLow& v, TX* dx,
                int64_t ldx, hipStream_t s) {
  hipLaunchKernelGGL(k_lora_dx<TX>, dim3((C + 255) / 256, T), dim3(256), 0, s, part, parts, t0, T, C, lora, v, dx, ldx);
}

template <typename TX>
void rq_lora_outer(const TX* x, int64_t ldx, int C, const TX* dy, int64_t ldy, int R, int T, const RqLora<TX>& lora,
                   const RqLow& u, const RqLow& v, TX* da, TX* db, hipStream_t s) {
  hipLaunchKernelGGL(k_lora_outer<TX>, dim3((C + 127) / 128 + (R + 127) / 128, u.ranks / 16, lora.n), dim3(64 * OUTER_WAVES), 0, s,
                     x, ldx, C, dy, ldy, R, T, lora, u, v, da, db);
}
