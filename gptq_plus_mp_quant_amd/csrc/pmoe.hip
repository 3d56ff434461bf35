// A mixture-of-experts layer for a few tokens, the experts' linears as packed codes and scales:
//
//   l = x router^T, the K largest of l chosen (equal logits by their index), w = softmax(l) of the chosen
//   (divided by their sum when norm), y = sum_k w_k Wd_k (silu(Wg_k x) * (Wu_k x)).
//
// Four launches, three for one token, five for many: the router's logits; the routing, which sorts the chosen
// (token, expert) pairs into units of up to 16 tokens of one expert (one token's needs no launch); gate, up and
// the activation of every unit; down, summed over a token's experts.  An expert that no token chose is not read,
// one that several chose is read once for 16 of them.
// Router logits, sums, the activation and the sum over experts are fp32 (the activation in three bf16 pieces that
// carry all 24 bits); the one rounding to fewer bits is the result's to x's type.
#include "pmoe_types.h"

namespace {

// A workgroup takes one expert and 8 tokens; its waves take 512 columns in turn, 8 a lane (a router of 128 x 2048, 1 token
// 3 us; of 8 x 4096, 32 tokens 6 us: latency).
constexpr int ROUTER_TOKENS = 8;
template <typename TX>
__global__ __launch_bounds__(256) void k_moe_router(const TX* __restrict__ x, int64_t ldx, int T, int D,
                                                    const TX* __restrict__ router, int64_t ldr, int E,
                                                    float* __restrict__ logits) {
  __shared__ float join[4][ROUTER_TOKENS];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = rq_wave(), t0 = blockIdx.y * ROUTER_TOKENS;
  const TX* r = router + (int64_t)e * ldr;
  const int nt = min(ROUTER_TOKENS, T - t0);
  float s[ROUTER_TOKENS] = {};
  auto add = [&](auto full, int c, int n) {
    constexpr bool FULL = decltype(full)::value;
    const auto w = rq_load_x<FULL>(r + c, n);
#pragma unroll
    for (int t = 0; t < ROUTER_TOKENS; ++t) {
      if (t >= nt) break;
      const auto v = rq_load_x<FULL>(x + (int64_t)(t0 + t) * ldx + c, n);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[t] = __builtin_fmaf((float)v[k], (float)w[k], s[t]);
    }
  };
  const int whole = D / 512 * 512;
#pragma unroll 2
  for (int c = 512 * wave; c < whole; c += 2048) add(std::true_type{}, c + 8 * lane, 8);
  if (whole < D && whole / 512 % 4 == wave) add(std::false_type{}, whole + 8 * lane, D - whole - 8 * lane);
#pragma unroll
  for (int t = 0; t < ROUTER_TOKENS; ++t) {
    if (t >= nt) break;
    const float v = rq_wave_sum(s[t]);
    if (lane == 0) join[wave][t] = v;
  }
  __syncthreads();
  if ((int)threadIdx.x < nt) {
    const int t = threadIdx.x;
    logits[(int64_t)(t0 + t) * E + e] = (join[0][t] + join[1][t]) + (join[2][t] + join[3][t]);
  }
}

// One workgroup.  A wave takes a token: its experts are chosen (rq_choose) and ranked among themselves.  Then a
// wave takes an expert: its pairs in ascending order, cut into units.
// EL: experts a lane holds (its loops are unrolled; 32 tokens to 2 of 8 experts: 8 us, 11 with 16).
template <int EL>
__global__ __launch_bounds__(1024) void k_moe_route(const float* __restrict__ logits, int T, int E, int K, int norm,
                                                    float* __restrict__ weights, int* __restrict__ nunits,
                                                    RqUnit* __restrict__ units, int most, int* __restrict__ ids_out,
                                                    float* __restrict__ weights_out) {
  __shared__ int ids[MOE_TOKENS * MOE_MAX_K];
  __shared__ int first[MOE_MAX_E];                   // the expert's first unit, once they are counted
  __shared__ uint64_t picked[16][MOE_MAX_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int t = wave; t < T; t += 16) {
    RqChoice<EL> c;
    rq_choose<EL>(logits + (int64_t)t * E, E, K, c);
    int at = 0;
#pragma unroll
    for (int u = 0; u < EL; ++u) {
      if (u >= c.used) break;
      if (c.taken[u] >> lane & 1)
        picked[wave][at + rq_lanes_before(c.taken[u])] = ((uint64_t)c.key[u] << 32) | (uint32_t)~(uint32_t)(64 * u + lane);
      at += __popcll(c.taken[u]);
    }
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < EL; ++u) {
      if (u >= c.used) break;
      s += expf(c.v[u] - c.m);                           // 0 past the last expert
    }
    s = rq_wave_sum(s);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint64_t mine = lane < K ? picked[wave][lane] : 0;
    int place = 0;
    for (int j = 0; j < K; ++j) place += picked[wave][j] > mine ? 1 : 0;
    const float p = lane < K ? expf(rq_key_value((uint32_t)(mine >> 32)) - c.m) : 0.0f;
    const float total = norm ? rq_wave_sum(p) : s;
    if (lane < K) {
      const int e = (int)~(uint32_t)mine;
      ids[t * K + place] = e;
      weights[t * K + place] = p / total;
      if (ids_out) ids_out[t * K + place] = e;
      if (weights_out) weights_out[t * K + place] = p / total;
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const int pairs = T * K;
  // Few pairs: one a lane of the first wave, and the lanes of its expert by ten ballots.
  const bool few = pairs <= 64;
  const int own = few && lane < pairs ? ids[lane] : MOE_MAX_E;
  uint64_t same = ~0ull;
  if (few && wave == 0) {
#pragma unroll
    for (int bit = 0; (1 << bit) <= MOE_MAX_E; ++bit) {
      const uint64_t set = __ballot(own >> bit & 1);
      same &= own >> bit & 1 ? set : ~set;
    }
    for (int e = lane; e < E; e += 64) first[e] = 0;
    rq_wave_sync();
    if (lane < pairs) first[own] = (__popcll(same) + 15) / 16;
  }
  for (int e = few ? E : wave; e < E; e += 16) {     // units of every expert
    int n = 0;
    for (int p = 0; p < pairs; p += 64) n += __popcll(__ballot(p + lane < pairs && ids[p + lane] == e));
    if (lane == 0) first[e] = (n + 15) / 16;
  }
  __syncthreads();
  if (wave == 0) {                                   // to the number of units before it
    int before = 0;
    for (int e = 0; e < E; e += 64) {
      const int mine = e + lane < E ? first[e + lane] : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int below = __shfl_up(sum, o);
        sum += lane >= o ? below : 0;
      }
      if (e + lane < E) first[e + lane] = before + sum - mine;
      before += __shfl(sum, 63);
    }
    if (lane == 0) *nunits = before;
    for (int k = before + lane; k < most; k += 64) units[k].n = 0;
  }
  __syncthreads();
  if (few) {
    if (wave || lane >= pairs) return;
    const int n = __popcll(same), before = __popcll(same & ((1ull << lane) - 1));
    RqUnit& u = units[first[own] + before / 16];
    u.pairs[before % 16] = lane;
    if (before % 16 == 0) {
      u.expert = own;
      u.n = min(16, n - before);
    }
    // the expert's last pair fills the places past it with its first
    if (before == n - 1)
      for (int k = before % 16 + 1; k < 16; ++k) u.pairs[k] = __ffsll((unsigned long long)same) - 1;
    return;
  }
  for (int e = wave; e < E; e += 16) {
    int n = 0;
    for (int p = 0; p < pairs; p += 64) {
      const bool is = p + lane < pairs && ids[p + lane] == e;
      const uint64_t mask = __ballot(is);
      const int at = n + rq_lanes_before(mask);
      if (is) units[first[e] + at / 16].pairs[at % 16] = p + lane;
      n += __popcll(mask);
    }
    if (n == 0) continue;
    const int full = (n - 1) / 16;                   // every unit but the last is full
    if (lane <= full) {
      units[first[e] + lane].expert = e;
      units[first[e] + lane].n = lane < full ? 16 : n - 16 * full;
    }
    // the places past the last unit's tokens take the expert's first pair
    int pair0 = -1;
    for (int p = 0; p < pairs && pair0 < 0; p += 64) {
      const uint64_t mask = __ballot(p + lane < pairs && ids[p + lane] == e);
      if (mask) pair0 = p + __ffsll((unsigned long long)mask) - 1;
    }
    if (lane < 16 && lane >= n - 16 * full) units[first[e] + full].pairs[lane] = pair0;
  }
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct Layout {
  int64_t logits, weights, nunits, units, gate, h, parts, total;
};
inline Layout layout(int T, int D, int I, int E, int K) {
  const int64_t n = T < MOE_TOKENS ? T : MOE_TOKENS;
  Layout l;
  l.logits = 0;
  l.weights = l.logits + up256(n * E * 4);
  l.nunits = l.weights + up256(n * K * 4);
  l.units = l.nunits + 256;
  l.gate = l.units + up256((int64_t)rq_units((int)n, E, K) * (int64_t)sizeof(RqUnit));
  l.h = l.gate + up256(n * K * I * 4);
  l.parts = l.h + up256(n * K * (((int64_t)I + 127) / 128 * 128) * 2 * MOE_PIECES);
  l.total = l.parts + up256((int64_t)rq_moe_parts(D) * n * D * 4);
  return l;
}
inline RqExperts experts(const rq_packed_experts* p, int R, int C) {
  return RqExperts{rq_packed(p->qweight, p->ldp, p->scales, p->lds, p->g_idx, R, C, p->ngroups, p->groupsize),
                   p->stride_q, p->stride_scales, C};
}

}  // namespace

extern "C" int64_t rq_packed_moe_workspace_bytes(int T, int D, int I, int E, int K) {
  if (T < 0 || D <= 0 || I <= 0 || E <= 0 || E > MOE_MAX_E || K <= 0 || K > MOE_MAX_K || K > E) return RQ_EINVAL;
  return layout(T, D, I, E, K).total;
}

extern "C" int rq_packed_moe(const void* x, int dtype, int T, int64_t ldx, int D, const void* router, int64_t ldr, int E,
                             int K, int norm, int I, const rq_packed_experts* gate, const rq_packed_experts* up,
                             const rq_packed_experts* down, void* y, int64_t ldy, int* ids_out, float* weights_out,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = rq_packed_moe_workspace_bytes(T, D, I, E, K);
  if (need < 0 || !gate || !up || !down) return RQ_EINVAL;
  const RqExperts g = experts(gate, I, D), u = experts(up, I, D), d = experts(down, D, I);
  if (rq_packed_check(g.w, gate->nbits) != RQ_OK || rq_packed_check(u.w, up->nbits) != RQ_OK ||
      rq_packed_check(d.w, down->nbits) != RQ_OK)
    return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !router || !y || ldx < D || ldr < D || ldy < D || !workspace || workspace_bytes < need) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Layout l = layout(T, D, I, E, K);
  char* ws = (char*)workspace;
  float* logits = (float*)(ws + l.logits);
  float* weights = (float*)(ws + l.weights);
  int* nunits = (int*)(ws + l.nunits);
  RqUnit* units = (RqUnit*)(ws + l.units);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    for (int64_t t0 = 0; t0 < T; t0 += MOE_TOKENS) {
      const int n = (int)(T - t0 < MOE_TOKENS ? T - t0 : MOE_TOKENS);
      const TX* xt = (const TX*)x + t0 * ldx;
      const RqMoe m{n, D, I, E, K, norm, nunits, units, weights, (float*)(ws + l.gate), (__hip_bfloat16*)(ws + l.h),
                    rq_moe_out_mode(d.w) == RQ_RUNS ? (I + 127) / 128 * 128 : I,
                    rq_moe_out_mode(d.w) == RQ_RUNS, (float*)(ws + l.parts),
                    n == 1 && E <= 64 * MOE_CHOICE ? logits : nullptr, ids_out ? ids_out + t0 * K : nullptr,
                    weights_out ? weights_out + t0 * K : nullptr};
      hipLaunchKernelGGL(k_moe_router<TX>, dim3(E, (n + ROUTER_TOKENS - 1) / ROUTER_TOKENS), dim3(256), 0, s, xt,
                         ldx, n, D, (const TX*)router, ldr, E, logits);
      auto route = [&](auto el) {
        hipLaunchKernelGGL(k_moe_route<decltype(el)::value>, dim3(1), dim3(1024), 0, s, logits, n, E, K, norm, weights, nunits,
                           units, rq_units(n, E, K), ids_out ? ids_out + t0 * K : nullptr,
                           weights_out ? weights_out + t0 * K : nullptr);
      };
      if (!m.logits) {                               // else they are chosen where they are needed
        if (E <= 64) route(std::integral_constant<int, 1>{});
        else if (E <= 256) route(std::integral_constant<int, 4>{});
        else route(std::integral_constant<int, MOE_MAX_E / 64>{});
      }
      rq_moe_in<TX>(xt, ldx, g, gate->nbits, u, up->nbits, m, s);
      rq_moe_out<TX>(d, down->nbits, m, (TX*)y + t0 * ldy, ldy, s);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
