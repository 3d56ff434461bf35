// act(x Wg^T) * (x Wu^T) from packed weights, and what its gradient takes beside the gradient of a packed linear: the
// kernels for one element type.
#pragma once
#include "pgated_types.h"
#include "plinear_rows.h"

namespace {

enum { GATED_BOTH = 0, GATED_GATE = 1, GATED_UP = 2 };

// 16 RP rows of both weights and 16 NT tokens to a workgroup; the waves take the chunks of 128 columns in turn, multiply RP
// row tiles of gate and of up by the tokens they have loaded once, and are joined through LDS in their order.  GATE
// and UP (weights of different bits or groups): one of the two, the gate's product goes by way of pre.
// Bound by the weights' bytes and the path that brings them and the tokens to a CU.  Measured, 4-bit: 14336 x 4096 bf16, 1
// token 18.7 us (3.3 TB/s), 28672 x 8192 fp16, 24 tokens 84.7 us (2.8 TB/s).  With one row tile of each weight, a call there:
// 127 us with tokens as they lie, 97 to 100 with tokens laid out once (k_arrange, 5 us), codes to fp16 in 9 instructions and
// unguarded rows; of those 27 went without the tokens' loads, 45 without the words'.
template <typename TX, int NB, int MODE, int NM, int NT, int RP, bool DIRECT>
__global__ __launch_bounds__(rows_threads(2, NT)) void k_packed_gated(const TX* __restrict__ x, const void* __restrict__ xa, int T, int64_t ldx, RqPacked first,
                                                                      RqPacked second, int what, int act, bool staged,
                                                                      float* pre, TX* __restrict__ h, int64_t ldh) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & 63, wave = rq_wave(), waves = blockDim.x >> 6;
  const int I = first.R, r0 = blockIdx.x * 16 * RP, t0 = blockIdx.y * 16 * NT;
  constexpr int RT = NM * RP;
  constexpr bool ARRANGED = MODE == RQ_RUNS && NT > 1;
  typename std::conditional<ARRANGED, RqArranged<TX, NT, rq_pairs<TX>(NB)>,
                            typename std::conditional<DIRECT, RqDirect<TX, rq_pairs<TX>(NB)>, RqWholeTokens<TX, NT>>::type>::type xs;
  if constexpr (ARRANGED) rq_arranged_tokens<TX>(xa, T, first.C, t0, xs.p);
  else {
#pragma unroll
    for (int b = 0; b < NT; ++b) xs.p[b] = x + (int64_t)min(t0 + 16 * b + (lane & 15), T - 1) * ldx;
  }
  RqPacked w[NM];
  w[0] = first;
  if constexpr (NM == 2) w[1] = second;
  if (MODE == RQ_ANY && staged) {
#pragma unroll
    for (int a = 0; a < RT; ++a) rq_stage_scales(w[a % NM], rq_tile_row<true>(r0 + 16 * (a / NM), I), a, RT, threadIdx.x, blockDim.x, lds);
    __syncthreads();
  }
  floatx4 acc[RT][NT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  rq_rows_tokens<NB, MODE, RT, NM>(w, r0, xs, wave, waves, MODE == RQ_ANY && staged ? lds : nullptr, acc);
  if (MODE == RQ_ANY && staged) __syncthreads();
  floatx4* out = reinterpret_cast<floatx4*>(lds);
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) out[((wave * RT + a) * NT + b) * 64 + lane] = acc[a][b];
  __syncthreads();
  for (int e = threadIdx.x; e < RP * NT * 64; e += blockDim.x) {
    const int l = e & 63, b = (e >> 6) % NT, m = (e >> 6) / NT;      // row tiles m NM and m NM + NM - 1
    const int t = t0 + 16 * b + (l & 15), rm = r0 + 16 * m, r = rq_tile_row<true>(rm, I) + 4 * (l >> 4);
    if (t >= T) continue;
    const floatx4 *at = out + (m * NM * NT + b) * 64 + l, *up = at + (NM - 1) * NT * 64;
    floatx4 g = *at, u = *up;
    for (int k = 1; k < waves; ++k) {
      g += at[k * RT * NT * 64];
      u += up[k * RT * NT * 64];
    }
    float* p = pre ? pre + (int64_t)t * 2 * I + r : nullptr;
    TX* dst = h + (int64_t)t * ldh + r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (r + k >= I || r + k < rm) continue;
      if (what == GATED_UP) g[k] = p[k];
      if (p && what != GATED_UP) p[k] = g[k];
      if (what == GATED_GATE) continue;
      if (p) p[I + k] = u[k];
      dst[k] = rq_cast<TX>(rq_act(act, g[k]).f * u[k]);
    }
  }
}

template <typename TX>
__global__ __launch_bounds__(256) void k_arrange(const TX* __restrict__ x, int T, int64_t ldx, int C, bool paired, void* __restrict__ xa) {
  const int chunks = (C + RQ_CHUNK - 1) / RQ_CHUNK, per = (chunks + gridDim.y - 1) / gridDim.y;
  rq_arrange<TX>(x, T, ldx, C, blockIdx.x, min((int)blockIdx.y * per, chunks), min(((int)blockIdx.y + 1) * per, chunks), paired,
                 threadIdx.x, 256, xa);
}

template <typename TX, int NB, int MODE, int NM, int NT, int RP, bool DIRECT>
void launch_gated(const TX* x, void* xa, int T, int64_t ldx, const RqPacked& first, const RqPacked& second, int what, int act, float* pre,
                  TX* h, int64_t ldh, hipStream_t s) {
  constexpr int RT = NM * RP;
  const int bx = (first.R + 16 * RP - 1) / (16 * RP), by = (T + 16 * NT - 1) / (16 * NT);
  const int waves = waves_for(bx * by, (first.C + RQ_CHUNK - 1) / RQ_CHUNK, RT * NT, rows_threads(2, NT) / 64);
  size_t lds = (size_t)waves * RT * NT * 1024;
  const size_t scales = (size_t)((first.ngroups > second.ngroups ? first.ngroups : second.ngroups) + 1) * 16 * RT * 4;
  const bool staged = MODE == RQ_ANY && scales <= 65536;
  if (staged && lds < scales) lds = scales;
  hipLaunchKernelGGL((k_packed_gated<TX, NB, MODE, NM, NT, RP, DIRECT>), dim3(bx, by), dim3(64 * waves), lds, s, x, xa, T, ldx, first, second,
                     what, act, staged, pre, h, ldh);
}

template <typename TX, int NB, int MODE, int NM>
void gated_of(const TX* x, void* xa, int T, int64_t ldx, const RqPacked& first, const RqPacked& second, int what, int act, float* pre,
              TX* h, int64_t ldh, hipStream_t s) {
  constexpr int NT = RqOperand<TX>::pieces == 1 ? 4 : 2;
  auto launch = [&](auto nt, auto rp, auto direct) {
    launch_gated<TX, NB, MODE, NM, decltype(nt)::value, decltype(rp)::value, decltype(direct)::value>(x, xa, T, ldx, first, second, what,
                                                                                                     act, pre, h, ldh, s);
  };
  auto run = [&](auto nt, auto rp) { launch(nt, rp, std::false_type{}); };
  typedef std::integral_constant<int, 1> One;
  // 14336 x 4096 4-bit bf16, 1 / 4 tokens: 17.0 / 18.9 us a call, 18.6 / 20.3 without; 4096 x 4096 6.8 / 7.4 and 7.2 / 7.6.
  if constexpr (MODE == RQ_RUNS && NM == 2)
    if (T <= 4) return launch(One{}, One{}, std::true_type{});
  if (T <= 16) return run(One{}, One{});
  if constexpr (MODE == RQ_RUNS) {
    // 4-bit fp16, 24 tokens, one row tile of each weight a wave and two, us a call on the same weights: 28672 x 8192 73.4 and
    // 69.9, 20480 x 8192 53.6 and 51.7, 16384 x 8192 44.4 and 38.6.  With fewer rows it is how the workgroups fall on
    // the CUs that decides: 14336 x 8192 43.3 and 38.9, 11008 x 8192 34.1 and 37.8, 14336 x 4096 (32 tokens) 24.2 and 25.3.
    if constexpr (NM == 2 && NT == 4)
      if (T <= 32 && first.R >= 16384) return run(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
    if (T <= 32) return run(std::integral_constant<int, 2>{}, One{});
    if (NT == 4 && T <= 48) return run(std::integral_constant<int, NT == 4 ? 3 : NT>{}, One{});
  }
  run(std::integral_constant<int, NT>{}, One{});
}
template <typename TX, int NM>
void gated_one(const TX* x, void* xa, int T, int64_t ldx, const RqPacked& first, const RqPacked& second, int bits, int what, int act, float* pre,
               TX* h, int64_t ldh, hipStream_t s) {
  rq_with_nbits(bits, [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    switch (rq_whole_mode_of(first)) {
      case RQ_RUNS: gated_of<TX, NB, RQ_RUNS, NM>(x, xa, T, ldx, first, second, what, act, pre, h, ldh, s); break;
      case RQ_SMALL: gated_of<TX, NB, RQ_SMALL, NM>(x, xa, T, ldx, first, second, what, act, pre, h, ldh, s); break;
      default: gated_of<TX, NB, RQ_ANY, NM>(x, xa, T, ldx, first, second, what, act, pre, h, ldh, s);
    }
  });
}

template <typename TX>
__global__ __launch_bounds__(256) void k_gated_pre_grad(const TX* __restrict__ grad_h, int64_t ldg, int T, int I, int act,
                                                        const float* __restrict__ pre, float* __restrict__ d) {
  const int i = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (i >= I) return;
  const float g = rq_load_elem(grad_h + (int64_t)t * ldg + i);
  const float a = pre[(int64_t)t * 2 * I + i], b = pre[(int64_t)t * 2 * I + I + i];
  const RqAct v = rq_act(act, a);
  d[(int64_t)t * I + i] = g * b * v.df;
  d[((int64_t)T + t) * I + i] = g * v.f;
}

// Sixteen parts' loads in flight (they lie in other XCDs' caches or beyond); summed in their order.
template <typename TX>
__global__ __launch_bounds__(256) void k_gated_join(const float* __restrict__ part, int parts, int T, int C, TX* __restrict__ dx,
                                                    int64_t ldx) {
  const int c = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (c >= C) return;
  const float* p = part + (int64_t)t * C + c;
  const int64_t plane = (int64_t)T * C;
  float s = 0.0f;
  for (int m = 0; m < parts; m += 16) {
    float e[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) e[k] = p[min(m + k, parts - 1) * plane];
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (m + k < parts) s += e[k];
  }
  dx[(int64_t)t * ldx + c] = rq_cast<TX>(s);
}

}  // namespace

template <typename TX>
void rq_gated_rows(const TX* x, void* xa, int T, int64_t ldx, const RqPacked& gate, int gate_bits, const RqPacked& up, int up_bits,
                   int act, float* pre, TX* h, int64_t ldh, hipStream_t s) {
  auto arrange = [&](int bits) {
    const int chunks = (gate.C + RQ_CHUNK - 1) / RQ_CHUNK;
    hipLaunchKernelGGL(k_arrange<TX>, dim3((T + 15) / 16, chunks < 65535 ? chunks : 65535), dim3(256), 0, s, x, T, ldx, gate.C, rq_pairs<TX>(bits), xa);
  };
  if (rq_gated_together(gate, gate_bits, up, up_bits)) {
    if (rq_gated_arranged(T, gate)) arrange(gate_bits);
    return gated_one<TX, 2>(x, xa, T, ldx, gate, up, gate_bits, GATED_BOTH, act, pre, h, ldh, s);
  }
  if (rq_gated_arranged(T, gate)) arrange(gate_bits);
  gated_one<TX, 1>(x, xa, T, ldx, gate, gate, gate_bits, GATED_GATE, act, pre, h, ldh, s);
  if (rq_gated_arranged(T, up) && (!rq_gated_arranged(T, gate) || rq_pairs<TX>(gate_bits) != rq_pairs<TX>(up_bits))) arrange(up_bits);
  gated_one<TX, 1>(x, xa, T, ldx, up, up, up_bits, GATED_UP, act, pre, h, ldh, s);
}
template <typename TX>
void rq_gated_pre_grad(const TX* grad_h, int64_t ldg, int T, int I, int act, const float* pre, float* d, hipStream_t s) {
  hipLaunchKernelGGL(k_gated_pre_grad<TX>, dim3((I + 255) / 256, T), dim3(256), 0, s, grad_h, ldg, T, I, act, pre, d);
}
template <typename TX>
void rq_gated_join(const float* part, int parts, int T, int C, TX* dx, int64_t ldx, hipStream_t s) {
  hipLaunchKernelGGL(k_gated_join<TX>, dim3((C + 255) / 256, T), dim3(256), 0, s, part, parts, T, C, dx, ldx);
}
