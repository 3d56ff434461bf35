// u = A x and v = B^T dy: what a token's adapter makes of its rows.
#pragma once
#include "plora_types.h"

__device__ __forceinline__ floatx4 rq_mfma4(float a, float b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// acc += A[.][32 k] B[32 k][.]: lane 16 q + i holds A[i][8q..8q+7] and B[8q..8q+7][i].
__device__ __forceinline__ floatx4 rq_mfma32(half8 a, half8 b, floatx4 c) { return rq_mfma(a, b, c); }
__device__ __forceinline__ floatx4 rq_mfma32(bf16x8 a, bf16x8 b, floatx4 c) { return rq_mfma(a, b, c); }
__device__ __forceinline__ floatx4 rq_mfma32(floatx8 a, floatx8 b, floatx4 c) {
#pragma unroll
  for (int k = 0; k < 8; ++k) c = rq_mfma4(a[k], b[k], c);
  return c;
}

// A workgroup takes 16 tokens, one of their adapters (the nth in the order of their first tokens) and 16 ranks of one
// part of one of the jobs (z); its waves take steps of 32 columns in turn, four in flight, and are joined through LDS (64 for
// each wave) in their order.  Latency: a part of 2048 columns is one round of loads for 16 waves (one token of 4096
// columns 4.8 us, 7.7 with parts of 4096 for 8 waves).
template <typename TX, int WAVES>
__device__ __forceinline__ void rq_lora_down_job(const RqDownJobs<TX>& jobs, int tile, int nth, int z, floatx4* join) {
  typedef typename RqOperand<TX>::raw Raw;
  constexpr int STEPS = RQ_LORA_COLS / (32 * WAVES);
  const int lane = threadIdx.x & 63, wave = rq_wave(), i = lane & 15, q = lane >> 4;
  const bool one = z < jobs.zfirst;
  const RqDown<TX> d = one ? jobs.first : jobs.second;
  const RqLora<TX>& lora = jobs.lora;
  const RqLow& low = d.low;
  if (!one) z -= jobs.zfirst;
  const int64_t t = (int64_t)tile * 16 + i;
  const int own = t < low.T ? lora.of(t) : -1;
  uint64_t pending = __ballot(lane < 16 && own >= 0 && own < lora.n);
  for (int k = 0; k < nth && pending; ++k)
    pending &= ~__ballot(own == __builtin_amdgcn_readlane(own, __ffsll((unsigned long long)pending) - 1));
  if (!pending) return;
  const int lead = __ffsll((unsigned long long)pending) - 1, a = __builtin_amdgcn_readlane(own, lead);
  const int tiles = low.ranks / 16, rank = z % tiles * 16, part = z / tiles;
  const int c0 = part * RQ_LORA_COLS, c1 = min(d.cols, c0 + RQ_LORA_COLS);
  const TX* xs = d.x + (own == a ? t : (int64_t)tile * 16 + lead) * d.ldx;
  const int row = min(rank + i, lora.r - 1);
  const TX* as = d.rows ? lora.a + ((int64_t)a * lora.r + row) * d.cols : lora.b + (int64_t)a * d.cols * lora.r + row;
  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto load = [&](auto full, int c, Raw& xv, Raw& av) {
    constexpr bool FULL = decltype(full)::value;
    const int n = c1 - c;                            // the lane's columns (may be none)
    xv = rq_load_x<FULL>(xs + c, n);
    if (d.rows) {
      av = rq_load_x<FULL>(as + c, n);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        typename std::remove_reference<decltype(av[0])>::type e;
        __builtin_memcpy(&e, as + (int64_t)(c + (FULL ? k : min(k, n - 1))) * lora.r, sizeof(e));
        av[k] = FULL || k < n ? e : (decltype(e))0.0f;
      }
    }
  };
  if (rank >= lora.r) {
    // a tile of padding
  } else if (c0 + RQ_LORA_COLS <= c1) {
#pragma unroll 1
    for (int k0 = 0; k0 < STEPS; k0 += 4) {
      Raw xv[4], av[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) load(std::true_type{}, c0 + 32 * (wave + WAVES * (k0 + k)) + 8 * q, xv[k], av[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc = rq_mfma32(av[k], xv[k], acc);
    }
  } else {
    Raw xv, av;
    int c = c0 + 32 * wave;
    for (; c + 32 <= c1; c += 32 * WAVES) {
      load(std::true_type{}, c + 8 * q, xv, av);
      acc = rq_mfma32(av, xv, acc);
    }
    if (c < c1) {
      load(std::false_type{}, c + 8 * q, xv, av);
      acc = rq_mfma32(av, xv, acc);
    }
  }
  join[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave || own != a) return;
  for (int w = 1; w < WAVES; ++w) acc += join[w * 64 + lane];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (rank + 4 * q + k >= lora.r) acc[k] = 0.0f;
  *reinterpret_cast<floatx4*>(low.u + low.at(part, t) + rank + 4 * q) = acc;
}
