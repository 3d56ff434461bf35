// The two products of a mixture-of-experts layer on the matrix cores (packed_dot.h), for one element type.
#pragma once
#include "packed_dot.h"
#include "pmoe_types.h"

namespace {

enum { MOE_BOTH = 0, MOE_GATE = 1, MOE_UP = 2 };

// Grid (row tiles, units).  BOTH: the first half of the waves takes 16 rows of gate, the second the same rows of
// up, chunks of 128 columns in turn; joined through LDS, in their order.  GATE leaves the gate's product in
// fp32, UP takes it from there (weights of different bits or groups).
template <typename TX, int NB, int MODE>
__global__ __launch_bounds__(512) void k_moe_in(const TX* __restrict__ x, int64_t ldx, RqExperts gate, RqExperts up,
                                                int what, RqMoe m) {
  __shared__ floatx4 join[8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if ((int)blockIdx.y >= *m.nunits) return;
  const RqUnit& u = m.units[blockIdx.y];
  const int r0 = blockIdx.x * 16, pair = u.pairs[lane & 15];
  RqTokens<TX, 1> xs;
  xs.p[0] = x + (int64_t)(pair / m.K) * ldx;
  const int each = what == MOE_BOTH ? waves / 2 : waves;
  const RqPacked w = rq_expert(what == MOE_UP || wave >= each ? up : gate, u.expert);
  floatx4 acc[1][1] = {{{0.0f, 0.0f, 0.0f, 0.0f}}};
  rq_rows_tokens<NB, MODE, 1>(w, r0, xs, wave % each, each, nullptr, acc);
  join[wave][lane] = acc[0][0];
  __syncthreads();
  if (wave || (lane & 15) >= u.n) return;
  floatx4 a = join[0][lane];
  for (int k = 1; k < each; ++k) a += join[k][lane];
  const int r = r0 + 4 * (lane >> 4);
  float* g = m.gate + (int64_t)pair * m.I + r;
  floatx4 b;
  if (what == MOE_GATE) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < m.I) g[k] = a[k];
    return;
  }
  if (what == MOE_BOTH) {
    b = join[each][lane];
    for (int k = 1; k < each; ++k) b += join[each + k][lane];
  } else {
    b = a;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = r + k < m.I ? g[k] : 0.0f;
  }
  constexpr int P = rq_moe_pieces<TX>();
  const int64_t plane = (int64_t)m.T * m.K * m.I;
  __hip_bfloat16* h = m.h + (int64_t)pair * m.I + r;
  const float p = m.weights[pair];
  floatx8 v = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = p * (a[k] / (1.0f + expf(-a[k])) * b[k]);
  bf16x8 o[P];
  rq_operand<P>(v, o);
#pragma unroll
  for (int q = 0; q < P; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < m.I) __builtin_memcpy(h + q * plane + k, (const char*)&o[q] + 2 * k, 2);
}

// Grid (row tiles): 16 rows of down for every unit.  Chunk c of expert e goes to wave (c + e) mod W, whatever else
// is in the batch, and a wave adds its units' sums to its own copy of the workgroup's results in LDS, in the
// order of the experts: a token's result does not depend on the other tokens.
template <typename TX, int NB, int MODE, int W>
__global__ __launch_bounds__(64 * W) void k_moe_out(RqExperts down, RqMoe m, TX* __restrict__ y, int64_t ldy) {
  constexpr int P = rq_moe_pieces<TX>();
  extern __shared__ __attribute__((aligned(16))) floatx4 sums[];       // [W][T][4]: 16 rows of a token
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int r0 = blockIdx.x * 16, n = *m.nunits;
  floatx4* mine = sums + wave * m.T * 4;
  for (int k = lane; k < m.T * 4; k += 64) mine[k] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int k = 0; k < n; ++k) {
    const RqUnit& u = m.units[k];
    const int pair = u.pairs[i];
    RqPieces<P> xs;
    xs.p = m.h + (int64_t)pair * m.I;
    xs.plane = (int64_t)m.T * m.K * m.I;
    floatx4 acc[1][1] = {{{0.0f, 0.0f, 0.0f, 0.0f}}};
    rq_rows_tokens<NB, MODE, 1>(rq_expert(down, u.expert), r0, xs, (wave + W - u.expert % W) % W, W, nullptr, acc);
    if (i < u.n) mine[pair / m.K * 4 + q] += acc[0][0];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < m.T * 4; e += 64 * W) {
    const int t = e >> 2, r = r0 + 4 * (e & 3);
    floatx4 v = sums[e];
    for (int k = 1; k < W; ++k) v += sums[k * m.T * 4 + e];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < m.D) y[(int64_t)t * ldy + r + k] = rq_cast<TX>(v[k]);
  }
}

template <typename F>
inline void with_mode(const RqPacked& w, F&& f) {
  switch (rq_mode_of(w)) {
    case RQ_RUNS: f(std::integral_constant<int, RQ_RUNS>{}); break;
    case RQ_SMALL: f(std::integral_constant<int, RQ_SMALL>{}); break;
    default: f(std::integral_constant<int, RQ_ANY>{}); break;
  }
}

}  // namespace

template <typename TX>
void rq_moe_in(const TX* x, int64_t ldx, const RqExperts& gate, int gate_bits, const RqExperts& up, int up_bits,
               const RqMoe& m, hipStream_t s) {
  const dim3 grid((m.I + 15) / 16, rq_units(m.T, m.E, m.K)), block(512);
  auto launch = [&](const RqExperts& of, int bits, int what) {
    rq_with_nbits(bits, [&](auto nb) {
      with_mode(of.w, [&](auto mode) {
        hipLaunchKernelGGL((k_moe_in<TX, decltype(nb)::value, decltype(mode)::value>), grid, block, 0, s, x, ldx, gate, up,
                           what, m);
      });
    });
  };
  if (gate_bits == up_bits && rq_mode_of(gate.w) == rq_mode_of(up.w)) {
    launch(gate, gate_bits, MOE_BOTH);
  } else {
    launch(gate, gate_bits, MOE_GATE);
    launch(up, up_bits, MOE_UP);
  }
}

template <typename TX>
void rq_moe_out(const RqExperts& down, int bits, const RqMoe& m, TX* y, int64_t ldy, hipStream_t s) {
  rq_with_nbits(bits, [&](auto nb) {
    with_mode(down.w, [&](auto mode) {
      constexpr int NB = decltype(nb)::value, MODE = decltype(mode)::value;
      const dim3 grid((m.D + 15) / 16);
      // the copies of the results fit 32 KB of LDS
      if (m.T <= 32)
        hipLaunchKernelGGL((k_moe_out<TX, NB, MODE, 16>), grid, dim3(1024), 16 * m.T * 64, s, down, m, y, ldy);
      else
        hipLaunchKernelGGL((k_moe_out<TX, NB, MODE, 8>), grid, dim3(512), 8 * m.T * 64, s, down, m, y, ldy);
    });
  });
}
