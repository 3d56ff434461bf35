// The two products of a mixture-of-experts layer on the matrix cores (packed_dot.h), for one element type.
#pragma once
#include "pmoe_types.h"

namespace {

enum { MOE_BOTH = 0, MOE_GATE = 1, MOE_UP = 2 };

// Unit u of one token: the u-th of its experts in their order, which every wave chooses for itself (a launch of its
// own for that took 5.6 us, and waits for it before and after).  The first row tile's workgroups leave the units
// for the second product, the first one of them the routing.
struct Lone {
  int expert;
  float weight;
};
__device__ __forceinline__ Lone lone_unit(const RqMoe& m, int unit) {
  const int lane = threadIdx.x & 63;
  RqChoice<MOE_CHOICE> c;
  rq_choose<MOE_CHOICE>(m.logits, m.E, m.K, c);
  float sum = 0.0f;
  float p[MOE_CHOICE];
#pragma unroll
  for (int k = 0; k < MOE_CHOICE; ++k) {
    p[k] = k < c.used ? expf(c.v[k] - c.m) : 0.0f;   // 0 past the last expert
    sum += m.norm && !(c.taken[k] >> lane & 1) ? 0.0f : p[k];
  }
  sum = rq_wave_sum(sum);
  Lone one = {0, 0.0f};
  int before = 0;
#pragma unroll
  for (int k = 0; k < MOE_CHOICE; ++k) {
    const bool taken = c.taken[k] >> lane & 1;
    const uint64_t is = __ballot(taken && before + rq_lanes_before(c.taken[k]) == unit);
    if (is) {
      const int at = __ffsll((unsigned long long)is) - 1;
      one.expert = __builtin_amdgcn_readfirstlane(64 * k + at);
      one.weight = __shfl(p[k], at) / sum;
    }
    before += __popcll(c.taken[k]);
  }
  if (blockIdx.x || threadIdx.x >= 64) return one;
  RqUnit& u = m.units[unit];
  if (lane < 16) u.pairs[lane] = unit;
  if (lane == 0) {
    u.expert = one.expert;
    u.n = 1;
    if (unit == 0) *m.nunits = m.K;
  }
  if (unit == 0 && (m.ids_out || m.weights_out)) {
#pragma unroll
    for (int k = 0; k < MOE_CHOICE; ++k) {
      int place = 0;                                 // chosen experts with larger logits, or equal ones before it
#pragma unroll
      for (int j = 0; j < MOE_CHOICE; ++j)
        for (uint64_t left = c.taken[j]; left; left &= left - 1) {
          const int other = __ffsll((unsigned long long)left) - 1;
          const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)c.key[j], other);
          place += key > c.key[k] || (key == c.key[k] && 64 * j + other < 64 * k + lane) ? 1 : 0;
        }
      if (c.taken[k] >> lane & 1) {
        if (m.ids_out) m.ids_out[place] = 64 * k + lane;
        if (m.weights_out) m.weights_out[place] = p[k] / sum;
      }
    }
  }
  return one;
}

// Grid (row tiles, units): 16 rows, chunks of 128 columns to the waves in turn, joined through LDS in their order.
// BOTH: a wave multiplies the rows of gate and of up by the tokens it has loaded once.  GATE leaves the gate's
// product in fp32, UP takes it from there (weights of different bits or groups).
// 128 registers a lane, two workgroups a CU.  Bound by the weights' bytes: 8 experts of 4096 x 7168 at 5 bits, 32 tokens
// 109 us for 294 MB, 2.7 TB/s, the tokens' loads beside them; 8 of 2048 x 768 at 4 bits, 1 token 12.7 us, 3 of them
// its choice of experts: latency.  Two row tiles a wave, which halve the tokens' loads, need 256 registers: 125 us.
template <typename TX, int NB, int MODE, int NM>
__global__ __launch_bounds__(512, 4) void k_moe_in(const TX* __restrict__ x, int64_t ldx, RqExperts first, RqExperts second,
                                                int what, RqMoe m) {
  __shared__ floatx4 join[NM][8][64];
  extern __shared__ __attribute__((aligned(16))) float scales[];
  const int lane = threadIdx.x & 63, wave = rq_wave(), waves = blockDim.x >> 6;
  const int r0 = blockIdx.x * 16;
  int pair, expert, n;
  float p;
  if (m.logits) {
    const Lone one = lone_unit(m, blockIdx.y);
    pair = blockIdx.y;
    expert = one.expert;
    n = 1;
    p = one.weight;
  } else {
    const RqUnit& u = m.units[blockIdx.y];
    n = u.n;
    if (n == 0) return;
    pair = u.pairs[lane & 15];
    expert = u.expert;
    p = m.weights[pair];
  }
  RqTokens<TX, 1> xs;
  xs.p[0] = x + (int64_t)(pair / m.K) * ldx;
  RqPacked w[NM];
  w[0] = rq_expert(first, expert);
  if constexpr (NM == 2) w[1] = rq_expert(second, expert);
  floatx4 acc[NM][1] = {};
  const bool staged = MODE == RQ_ANY && rq_moe_in_lds(first.w, second.w) > 0;
  if (staged) {
#pragma unroll
    for (int a = 0; a < NM; ++a) rq_stage_scales(w[a], r0, a, NM, threadIdx.x, blockDim.x, scales);
    __syncthreads();
  }
  rq_rows_tokens<NB, MODE, NM, NM>(w, r0, xs, wave, waves, staged ? scales : nullptr, acc);
#pragma unroll
  for (int a = 0; a < NM; ++a) join[a][wave][lane] = acc[a][0];
  __syncthreads();
  if (wave || (lane & 15) >= n) return;
  floatx4 a = join[0][0][lane], b = join[NM - 1][0][lane];
  for (int k = 1; k < waves; ++k) {
    a += join[0][k][lane];
    b += join[NM - 1][k][lane];
  }
  const int r = r0 + 4 * (lane >> 4);
  float* g = m.gate + (int64_t)pair * m.I + r;
  if (what == MOE_GATE) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < m.I) g[k] = a[k];
    return;
  }
  if (what == MOE_UP) {
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = r + k < m.I ? g[k] : 0.0f;
  }
  constexpr int P = MOE_PIECES;
  const int64_t plane = (int64_t)m.T * m.K * m.ldh;
  __hip_bfloat16* row = m.h + (int64_t)pair * m.ldh;
  __hip_bfloat16* h = row + (m.arranged ? rq_arranged(r) : r);                // r is a multiple of 4
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
  if (r0 + 16 >= m.I && m.arranged) {       // the last rows' workgroup fills the last chunk up
    for (int c = m.I + (lane >> 4); c < m.ldh; c += 4)
#pragma unroll
      for (int q = 0; q < P; ++q) row[q * plane + rq_arranged(c)] = __hip_bfloat16(0.0f);
  }
}

// Grid (row tiles, parts): 16 RT rows of down for every unit.  Chunk c of expert e goes to wave (c + e) mod W * parts,
// whatever else is in the batch, and a wave adds every chunk's sums to its own copy of the workgroup's results in
// LDS, in the order of the experts: a token's result depends on how many tokens there are, not on which.
// RUNS: the loads of the next D chunks, of whatever units, are in flight.
// h, in three pieces, is 12 KB a chunk of 16 tokens, ten times a row tile's words: with four row tiles a wave 80 us and
// 4.8 us to join the parts for 8 experts of 7168 x 4096 at 5 bits (147 MB) and 32 tokens.  8 of 768 x 2048 at 4 bits, 1
// token: 12.6 us, latency.
template <typename TX, int NB, int MODE, int RT>
__global__ __launch_bounds__(64 * MOE_OUT_WAVES) void k_moe_out(RqExperts down, RqMoe m, bool staged,
                                                                 TX* __restrict__ y, int64_t ldy) {
  constexpr int P = MOE_PIECES, W = MOE_OUT_WAVES, R4 = 4 * RT;
  extern __shared__ __attribute__((aligned(16))) floatx4 sums[];       // [W][T][R4]: the rows of a token; then the units
  RqUnit* units = reinterpret_cast<RqUnit*>(sums + W * m.T * R4);
  const int lane = threadIdx.x & 63, wave = rq_wave(), i = lane & 15, q = lane >> 4;
  const int r0 = blockIdx.x * 16 * RT, n = __builtin_amdgcn_readfirstlane(*m.nunits);
  for (int k = threadIdx.x; k < m.T * R4 * W; k += 64 * W) sums[k] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = threadIdx.x; k < n * (int)(sizeof(RqUnit) / 4); k += 64 * W)
    reinterpret_cast<int*>(units)[k] = reinterpret_cast<const int*>(m.units)[k];
  __syncthreads();
  floatx4* mine = sums + wave * m.T * R4;
  const int all = W * gridDim.y, self = wave + W * blockIdx.y;         // of the waves that share the rows
  const int nch = (down.w.C + RQ_CHUNK - 1) / RQ_CHUNK;
  auto expert_of = [&](int k) { return __builtin_amdgcn_readfirstlane(units[k].expert); };
  auto begin = [&](int k) { return (self + all - expert_of(k) % all) % all; };       // the wave's first chunk of a unit
  if constexpr (MODE == RQ_RUNS) {
    typedef RqPieces<P, true> X;
    constexpr int D = RT == 1 ? 3 : 2;
    // The wave's chunks in order: unit k, chunk c.
    struct Place {
      int k, c;
    };
    auto next = [&](Place p) {
      p.c += all;
      while (p.k < n && p.c >= nch) {
        ++p.k;
        if (p.k < n) p.c = begin(p.k);
      }
      return p;
    };
    struct Flight {
      RqRunsW<NB, RT> f;
      typename X::raw x[1][4];
      int pair, places, c;                 // places: tokens of the unit, 0 past the last chunk
    };
    Place ahead{0, 0};
    if (n > 0) ahead.c = begin(0) - all;
    ahead = next(ahead);
    const Place first = ahead;
    // Past the end the first chunk is loaded again and nothing is made of it: no load is conditional.
    auto load = [&](Flight& t) {
      const bool is = ahead.k < n;
      const Place p = is ? ahead : first;
      const RqUnit& u = units[p.k];
      t.pair = u.pairs[i];
      t.places = is ? __builtin_amdgcn_readfirstlane(u.n) : 0;
      t.c = p.c;
      X xs;
      xs.p = m.h + (int64_t)t.pair * m.ldh;
      xs.plane = (int64_t)m.T * m.K * m.ldh;
      const RqPacked w[1] = {rq_expert(down, expert_of(p.k))};
      // A lane past the row's last column, where h is 0, loads the last words again.
      const int c = min(p.c * RQ_CHUNK + 32 * q, w[0].C - 32);
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        const uint32_t* row = w[0].q + (int64_t)min(r0 + 16 * a + i, w[0].R - 1) * w[0].ldp;
        __builtin_memcpy(t.f.wd[a], row + (int64_t)(c >> 5) * NB, 4 * NB);
        t.f.sc[a] = rq_load_scales4(w[0], rq_run_group(w[0], p.c * RQ_CHUNK), r0 + 16 * a + 4 * q);
      }
      rq_load_tokens<true>(xs, w[0].C, p.c, t.x);
      ahead = is ? next(ahead) : ahead;
    };
    if (first.k < n) {
      Flight t[D];
#pragma unroll
      for (int u = 0; u < D; ++u) load(t[u]);
      const RqPacked w[1] = {down.w};      // for the groups of rows and columns
      for (;;) {
#pragma unroll
        for (int u = 0; u < D; ++u) {
          if (t[u].places == 0) goto done;
          floatx4 acc[RT][1] = {};
          rq_chunk_runs<X, NB, RT, 1>(w, r0, t[u].c, t[u].f, t[u].x, acc);
          if (i < t[u].places) {
#pragma unroll
            for (int a = 0; a < RT; ++a) mine[t[u].pair / m.K * R4 + 4 * a + q] += acc[a][0];
          }
          load(t[u]);
        }
      }
    done:;
    }
  } else {
    // a wave's own scales, expert by expert
    float* scales = MODE == RQ_ANY && staged ? reinterpret_cast<float*>(units + n) + wave * (down.w.ngroups + 1) * 16 : nullptr;
    for (int k = 0; k < n; ++k) {
      const int pair = units[k].pairs[i];
      RqPieces<P, false> xs;
      xs.p = m.h + (int64_t)pair * m.ldh;
      xs.plane = (int64_t)m.T * m.K * m.ldh;
      const RqPacked w[1] = {rq_expert(down, expert_of(k))};
      floatx4 acc[RT][1] = {};
      if (begin(k) >= nch) continue;
      if (scales) {
        rq_wave_sync();
        rq_stage_scales(w[0], r0, 0, 1, lane, 64, scales);
        rq_wave_sync();
      }
      rq_rows_tokens<NB, MODE, RT, 1>(w, r0, xs, begin(k), all, scales, acc);
      if (i < units[k].n) {
#pragma unroll
        for (int a = 0; a < RT; ++a) mine[pair / m.K * R4 + 4 * a + q] += acc[a][0];
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < m.T * R4; e += 64 * W) {
    const int t = e / R4, r = r0 + 4 * (e % R4);
    floatx4 v = sums[e];
    for (int k = 1; k < W; ++k) v += sums[k * m.T * R4 + e];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (r + k >= m.D) continue;
      if (gridDim.y > 1) m.parts[((int64_t)blockIdx.y * m.T + t) * m.D + r + k] = v[k];
      else y[(int64_t)t * ldy + r + k] = rq_cast<TX>(v[k]);
    }
  }
}
// The sums of the workgroups that share rows, in their order.
template <typename TX>
__global__ __launch_bounds__(256) void k_moe_join(const float* __restrict__ parts, int n, int T, int D, TX* __restrict__ y,
                                                  int64_t ldy) {
  const int r = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (r >= D) return;
  float v = parts[(int64_t)t * D + r];
  for (int k = 1; k < n; ++k) v += parts[((int64_t)k * T + t) * D + r];
  y[(int64_t)t * ldy + r] = rq_cast<TX>(v);
}

template <typename F>
inline void with_mode(int mode, F&& f) {
  switch (mode) {
    case RQ_RUNS: f(std::integral_constant<int, RQ_RUNS>{}); break;
    case RQ_SMALL: f(std::integral_constant<int, RQ_SMALL>{}); break;
    default: f(std::integral_constant<int, RQ_ANY>{}); break;
  }
}

}  // namespace

template <typename TX>
void rq_moe_in(const TX* x, int64_t ldx, const RqExperts& gate, int gate_bits, const RqExperts& up, int up_bits,
               const RqMoe& m, hipStream_t s) {
  const dim3 grid((m.I + 15) / 16, rq_units(m.T, m.E, m.K));
  // Eight waves share the columns, four where there are workgroups enough without (8 experts of 4096 x 7168, 32
  // tokens: 107 us for 111).
  const dim3 block(grid.x * grid.y >= 2048 ? 256 : 512);
  auto launch = [&](const RqExperts& of, int bits, int what, auto both) {
    constexpr int NM = decltype(both)::value ? 2 : 1;
    rq_with_nbits(bits, [&](auto nb) {
      with_mode(rq_mode_of(of.w), [&](auto mode) {
        hipLaunchKernelGGL((k_moe_in<TX, decltype(nb)::value, decltype(mode)::value, NM>), grid, block,
                           decltype(mode)::value == RQ_ANY ? rq_moe_in_lds(of.w, up.w) : 0, s, x, ldx, of, up, what, m);
      });
    });
  };
  if (gate_bits == up_bits && rq_mode_of(gate.w) == rq_mode_of(up.w)) {
    launch(gate, gate_bits, MOE_BOTH, std::true_type{});
  } else {
    launch(gate, gate_bits, MOE_GATE, std::false_type{});
    launch(up, up_bits, MOE_UP, std::false_type{});
  }
}

template <typename TX>
void rq_moe_out(const RqExperts& down, int bits, const RqMoe& m, TX* y, int64_t ldy, hipStream_t s) {
  rq_with_nbits(bits, [&](auto nb) {
    with_mode(rq_moe_out_mode(down.w), [&](auto mode) {
      auto go = [&](auto rt, int parts) {
        constexpr int RT = decltype(rt)::value;
        const int scales = decltype(mode)::value == RQ_ANY ? rq_moe_out_scales(down.w) : 0;
        hipLaunchKernelGGL((k_moe_out<TX, decltype(nb)::value, decltype(mode)::value, RT>),
                           dim3((m.D + 16 * RT - 1) / (16 * RT), parts), dim3(64 * MOE_OUT_WAVES),
                           rq_moe_out_lds(m, RT) + scales, s, down, m, scales > 0, y, ldy);
        if (parts > 1)
          hipLaunchKernelGGL(k_moe_join<TX>, dim3((m.D + 255) / 256, m.T), dim3(256), 0, s, m.parts, parts, m.T, m.D, y, ldy);
      };
      if constexpr (decltype(mode)::value == RQ_RUNS) {
        if (rq_moe_dense(m)) return go(std::integral_constant<int, MOE_OUT_ROWS>{}, rq_moe_parts(m.D));
      }
      go(std::integral_constant<int, 1>{}, 1);
    });
  });
}
