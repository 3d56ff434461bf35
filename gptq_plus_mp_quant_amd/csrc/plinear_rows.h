// y = x W^T (+ bias) with a packed weight: the kernel and its launch for one element type.
#pragma once
#include "packed_dot.h"

namespace {

// --- y = x W^T ----------------------------------------------------------------------------------
// A workgroup of W waves takes 16 RT rows and 16 NT tokens; its waves take the chunks of 128 columns in
// turn (rows alone would leave most CUs without work) and are joined through LDS, in their order.
// Few tokens are bound by the weight's bytes.  Measured, 4 bits in groups of 128, bf16: 4096 x 4096 (8.9 MB), 1
// token 6.3 us, a launch and three trips to memory; 8192 x 28672 (125 MB), 1 / 16 tokens 35 / 48 us, 3.6 / 2.6 TB/s (with
// the words in a cache from the call before; from HBM 2 and 1 us more): 16 tokens' loads, twice the words' bytes, share
// the CU's load path with them, and vector instructions, mostly conversions, take 19 us.  Groups along an order (ANY)
// 223 us there, a scale from LDS and an fp32 product for every weight; 1026 x 1365 at 5 bits, fp32, 7 tokens 9.7 us, 65
// workgroups' latency.
// MORE adds what else a row tile's sums take (RqNothing, or the low-rank term of plora_kernels.h).
constexpr int rows_threads(int rt, int nt) { return rt * nt >= 2 ? 512 : 1024; }     // 256 or 128 registers a lane
struct RqNothing {
  static constexpr bool arranged = false, whole = false;
  static constexpr int staged_groups = RQ_STAGED_GROUPS;
  template <int RT, int NT>
  __device__ __forceinline__ void add(int, int, int, int, int, int, const float*, floatx4 (&)[RT][NT]) const {}
};
// ARRANGED (MORE::arranged, more than one token tile, RUNS): x lies as RqArranged has it, at more.arranged_x.
template <typename TX, int NB, int MODE, int RT, int NT, typename MORE>
__global__ __launch_bounds__(rows_threads(RT, NT)) void k_packed_rows(const TX* __restrict__ x, int T, int64_t ldx, RqPacked w,
                                                      const TX* __restrict__ bias, TX* __restrict__ y, int64_t ldy, MORE more) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & 63, wave = rq_wave(), waves = blockDim.x >> 6;
  const int r0 = blockIdx.x * 16 * RT, t0 = blockIdx.y * 16 * NT;
  constexpr bool ARRANGED = MORE::arranged && MODE == RQ_RUNS && NT > 1;
  typename std::conditional<ARRANGED, RqArranged<TX, NT, rq_pairs<TX>(NB)>,
                            typename std::conditional<MORE::whole, RqWholeTokens<TX, NT>, RqTokens<TX, NT>>::type>::type xs;
  if constexpr (ARRANGED) rq_arranged_tokens<TX>(more.arranged_x, T, w.C, t0, xs.p);
  else {
#pragma unroll
    for (int b = 0; b < NT; ++b) xs.p[b] = x + (int64_t)min(t0 + 16 * b + (lane & 15), T - 1) * ldx;
  }
  if constexpr (MORE::whole && NT == 1) more.prepare(x, T, ldx, w.C, wave, waves, lds);
  const bool staged = MODE == RQ_ANY && w.ngroups <= MORE::staged_groups;
  if (staged) {
    for (int a = 0; a < RT; ++a)
      rq_stage_scales(w, rq_tile_row<MORE::whole>(r0 + 16 * a, w.R), a, RT, threadIdx.x, blockDim.x, lds);
    __syncthreads();
  }
  floatx4 acc[RT][NT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  rq_rows_tokens<NB, MODE, RT, 1>({w}, r0, xs, wave, waves, staged ? lds : nullptr, acc);
  more.add(r0, w.R, t0, T, wave, waves, lds, acc);
  if (staged) __syncthreads();
  floatx4* out = reinterpret_cast<floatx4*>(lds);
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) out[((wave * RT + a) * NT + b) * 64 + lane] = acc[a][b];
  __syncthreads();
  for (int e = threadIdx.x; e < RT * NT * 64; e += blockDim.x) {
    const int l = e & 63, b = (e >> 6) % NT, a = (e >> 6) / NT;
    const int t = t0 + 16 * b + (l & 15), ra = r0 + 16 * a, r = rq_tile_row<MORE::whole>(ra, w.R) + 4 * (l >> 4);
    if (t >= T) continue;
    floatx4 v = out[e];
    for (int k = 1; k < waves; ++k) v += out[k * RT * NT * 64 + e];
    TX* dst = y + (int64_t)t * ldy + r;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < w.R && r + k >= ra) dst[k] = rq_cast<TX>(v[k] + (bias ? rq_load_elem(bias + r + k) : 0.0f));
  }
}

constexpr int TOKENS_PER_LAUNCH = 1 << 19;     // grid.y holds at most 65535 blocks of 16 tokens

// Waves per workgroup: enough that all of them together fill the GPU (8 a CU), no more than there are
// chunks to take, and their sums fit 64 KB of LDS.
inline int waves_for(int tiles, int chunks, int per_wave_kb, int most) {
  int waves = 4;
  while (waves < most && tiles * waves < 2048) waves *= 2;
  while (waves > 1 && (waves > chunks || waves * per_wave_kb > 64)) waves /= 2;
  return waves;
}

template <typename TX, int NB, int MODE, int RT, int NT, typename MORE>
void launch_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, const TX* bias, TX* y, int64_t ldy, const MORE& more,
                 hipStream_t s) {
  const int bx = (w.R + 16 * RT - 1) / (16 * RT), by = (T + 16 * NT - 1) / (16 * NT);
  int waves = waves_for(bx * by, (w.C + RQ_CHUNK - 1) / RQ_CHUNK, RT * NT, rows_threads(RT, NT) / 64);
  // Workgroups of eight waves go one to a CU there, in two rounds; of four two to a CU, in one: adapters of 24 / 48 / 64
  // tokens, 14336 x 4096, 29.1 / 37.3 / 43.3 us a call with eight, 26.1 / 32.8 / 39.5 with four.  (Without adapters the
  // sums stay as they are.)
  if (MORE::whole && RT * NT >= 4 && bx * by > 256 && bx * by <= 512 && waves > 4) waves = 4;
  size_t lds = (size_t)waves * RT * NT * 1024;
  if (MODE == RQ_ANY && w.ngroups <= MORE::staged_groups) {
    const size_t scales = (size_t)(w.ngroups + 1) * 16 * RT * 4;
    lds = lds > scales ? lds : scales;
  }
  MORE with = more;
  if constexpr (MORE::whole && NT == 1) lds = with.own_lds(lds);
  hipLaunchKernelGGL((k_packed_rows<TX, NB, MODE, RT, NT, MORE>), dim3(bx, by), dim3(64 * waves), lds, s, x, T, ldx, w,
                     bias, y, ldy, with);
}

template <typename TX, int NB, typename MORE>
void linear_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, const TX* bias, TX* y, int64_t ldy, const MORE& more,
                 hipStream_t s) {
  constexpr int R2 = RqOperand<TX>::pieces == 1 ? 2 : 1;      // fp32's pieces leave registers for one row tile
  switch (MORE::whole ? rq_whole_mode_of(w) : rq_mode_of(w)) {
    case RQ_RUNS:
      // Two row tiles a wave share their tokens' loads.  Up to 16 tokens they are taken where they still make a workgroup
      // for every CU (8192 x 28672 4-bit bf16, 1 / 16 tokens: 42 / 71 us with one, 35 / 49 with two); beyond, where a
      // CU holds one workgroup, as soon as one row tile makes more workgroups than there are CUs (24 / 64 tokens, one
      // and two: 4096 x 4096 11.0 / 19.7 and 12.0 / 21.9 us, 5120 x 4096 16.9 / 35.8 and 11.6 / 22.0, 8192 x 28672 98 / 216 and
      // 62 / 121).  Two token tiles up to 32 tokens: 4096 x 4096, 32 tokens 11.4 us for 14.5 with four.
      if (T <= 16 && w.R >= 8192) launch_rows<TX, NB, RQ_RUNS, 2, 1>(x, T, ldx, w, bias, y, ldy, more, s);
      else if (T <= 16) launch_rows<TX, NB, RQ_RUNS, 1, 1>(x, T, ldx, w, bias, y, ldy, more, s);
      else if (T <= 32 && w.R > 4096) launch_rows<TX, NB, RQ_RUNS, R2, 2>(x, T, ldx, w, bias, y, ldy, more, s);
      else if (T <= 32) launch_rows<TX, NB, RQ_RUNS, 1, 2>(x, T, ldx, w, bias, y, ldy, more, s);
      else if (MORE::whole && T <= 48) {
        // Three token tiles, with adapters: 33 / 48 tokens of 14336 x 4096 29.8 / 32.8 us a call for 32.7 / 35.9 with four,
        // 48 of 4096 x 4096 18.3 for 21.6.
        if constexpr (MORE::whole) {
          if (w.R > 4096) launch_rows<TX, NB, RQ_RUNS, R2, 3>(x, T, ldx, w, bias, y, ldy, more, s);
          else launch_rows<TX, NB, RQ_RUNS, 1, 3>(x, T, ldx, w, bias, y, ldy, more, s);
        }
      } else if (w.R > 4096) launch_rows<TX, NB, RQ_RUNS, R2, 4>(x, T, ldx, w, bias, y, ldy, more, s);
      else launch_rows<TX, NB, RQ_RUNS, 1, 4>(x, T, ldx, w, bias, y, ldy, more, s);
      break;
    case RQ_SMALL:
      // One row tile: with two 4096 x 4096 4-bit bf16 in groups of 64 takes 18.6 us for 11.2 (4 tokens), 29.1 for 21.9 (64).
      if (T <= 16) launch_rows<TX, NB, RQ_SMALL, 1, 1>(x, T, ldx, w, bias, y, ldy, more, s);
      else launch_rows<TX, NB, RQ_SMALL, 1, 4>(x, T, ldx, w, bias, y, ldy, more, s);
      break;
    default:
      if (T <= 16) launch_rows<TX, NB, RQ_ANY, 1, 1>(x, T, ldx, w, bias, y, ldy, more, s);
      else launch_rows<TX, NB, RQ_ANY, 1, 4>(x, T, ldx, w, bias, y, ldy, more, s);
  }
}

}  // namespace

template <typename TX>
void rq_linear_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, int nbits, const TX* bias, TX* y, int64_t ldy,
                    hipStream_t s) {
  rq_with_nbits(nbits, [&](auto nb) {
    for (int64_t t0 = 0; t0 < T; t0 += TOKENS_PER_LAUNCH)
      linear_rows<TX, decltype(nb)::value>(x + t0 * ldx, (int)(T - t0 < TOKENS_PER_LAUNCH ? T - t0 : TOKENS_PER_LAUNCH),
                                           ldx, w, bias, y + t0 * ldy, ldy, RqNothing{}, s);
  });
}
