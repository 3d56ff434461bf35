// A mixture-of-experts layer for a few tokens, the experts' linears as packed codes and scales:
//
//   l = x router^T, the K largest of l chosen (equal logits by their index), w = softmax(l) of the chosen
//   (divided by their sum when norm), y = sum_k w_k Wd_k (silu(Wg_k x) * (Wu_k x)).
//
// Router logits, products, the activation and the sum over experts are fp32; the one rounding to fewer
// bits is the result's to x's type.
#include "packed_bits.h"

namespace {

constexpr int RW = 4;                 // rows per wave
constexpr int MAX_E = 1024, MAX_K = 64;
constexpr int TOKENS = 64;            // tokens per pass over the experts

// The experts' weights: expert e's entry is w with its pointers moved by e strides.
struct RqExperts {
  RqPacked w;
  int64_t sq, ss, sg;                 // strides of q, scales, g_idx from one expert to the next
};
__device__ __forceinline__ RqPacked expert(const RqExperts& x, int e) {
  RqPacked w = x.w;
  w.q += x.sq * e;
  w.scales += x.ss * e;
  if (w.g_idx) w.g_idx += x.sg * e;
  return w;
}

// acc[i] += sum_c xv[c] * W[r0 + i, c] of the lane's columns
template <int NB, typename TX>
__device__ __forceinline__ void rows_dot(const RqPacked& w, const TX* __restrict__ x, int r0, float (&acc)[RW]) {
  for (int c = (threadIdx.x & 63) * 8; c < w.C; c += 512) {
    const int nc = min(8, w.C - c);
    float xv[8];
    int g[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      xv[k] = k < nc ? rq_load_elem(x + c + k) : 0.0f;
      g[k] = rq_group_of(w, c + (k < nc ? k : 0));
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int r = min(r0 + i, w.R - 1);
      int code[8];
      rq_codes8<NB>(w.q + (int64_t)r * w.ldp, c, nc, code);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        acc[i] = __builtin_fmaf(xv[k], k < nc ? rq_scale_of(w, g[k], r) * (float)code[k] : 0.0f, acc[i]);
    }
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

template <typename TX>
__global__ __launch_bounds__(256) void k_moe_router(const TX* __restrict__ x, int64_t ldx, int D,
                                                    const TX* __restrict__ router, int64_t ldr, int E,
                                                    float* __restrict__ logits) {
  const int e = blockIdx.x * 4 + (threadIdx.x >> 6), t = blockIdx.y;
  if (e >= E) return;
  float s = 0.0f;
  for (int c = threadIdx.x & 63; c < D; c += 64)
    s = __builtin_fmaf(rq_load_elem(x + (int64_t)t * ldx + c), rq_load_elem(router + (int64_t)e * ldr + c), s);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) logits[(int64_t)t * E + e] = s;
}

// One wave per token: an expert's rank is the number of experts before it, so the ranks are a
// permutation whatever the logits hold.
__global__ __launch_bounds__(64) void k_moe_route(const float* __restrict__ logits, int E, int K, int norm,
                                                  int* __restrict__ ids, float* __restrict__ weights,
                                                  int* __restrict__ ids_out, float* __restrict__ weights_out) {
  __shared__ float l[MAX_E];
  __shared__ float chosen[MAX_K];
  const int t = blockIdx.x, lane = threadIdx.x;
  float m = -INFINITY;
  for (int e = lane; e < E; e += 64) {
    const float v = logits[(int64_t)t * E + e];
    l[e] = v;
    m = rq_nan_max(m, v);
  }
  for (int o = 32; o; o >>= 1) m = rq_nan_max(m, __shfl_xor(m, o));
  __syncthreads();
  float s = 0.0f;
  for (int e = lane; e < E; e += 64) {
    const uint32_t mine = rq_order_key(l[e]);
    const float p = expf(l[e] - m);
    s += p;
    int rank = 0;
    for (int j = 0; j < E; ++j) {
      const uint32_t other = rq_order_key(l[j]);
      rank += (other > mine) || (other == mine && j < e);
    }
    if (rank < K) {
      ids[t * K + rank] = e;
      if (ids_out) ids_out[t * K + rank] = e;
      chosen[rank] = p;
    }
  }
  s = wave_sum(s);
  __syncthreads();
  const float p = lane < K ? chosen[lane] : 0.0f;
  const float total = norm ? wave_sum(p) : s;
  if (lane < K) {
    weights[t * K + lane] = p / total;
    if (weights_out) weights_out[t * K + lane] = p / total;
  }
}

// What a gate / up launch leaves: the gate's product, or its activation times the up product.
enum { MOE_GATE = 0, MOE_UP = 1 };

template <typename TX, int NB>
__global__ __launch_bounds__(256) void k_moe_in(const TX* __restrict__ x, int64_t ldx, RqExperts ex, int K,
                                                const int* __restrict__ ids, int mode, float* __restrict__ h) {
  const int pair = blockIdx.y, r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * RW;
  if (r0 >= ex.w.R) return;
  const RqPacked w = expert(ex, ids[pair]);
  float acc[RW] = {};
  rows_dot<NB>(w, x + (int64_t)(pair / K) * ldx, r0, acc);
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const float v = wave_sum(acc[i]);
    if ((threadIdx.x & 63) == 0 && r0 + i < w.R) {
      float* at = h + (int64_t)pair * w.R + r0 + i;
      if (mode == MOE_GATE) *at = v;
      else *at = *at / (1.0f + expf(-*at)) * v;
    }
  }
}

template <typename TX, int NB>
__global__ __launch_bounds__(256) void k_moe_out(const float* __restrict__ h, RqExperts ex, int K,
                                                 const int* __restrict__ ids, const float* __restrict__ weights,
                                                 TX* __restrict__ y, int64_t ldy) {
  const int t = blockIdx.y, r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * RW;
  if (r0 >= ex.w.R) return;
  float acc[RW] = {};
  for (int k = 0; k < K; ++k) {
    const int pair = t * K + k;
    float one[RW] = {};
    rows_dot<NB>(expert(ex, ids[pair]), h + (int64_t)pair * ex.w.C, r0, one);
#pragma unroll
    for (int i = 0; i < RW; ++i) acc[i] = __builtin_fmaf(weights[pair], one[i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const float v = wave_sum(acc[i]);
    if ((threadIdx.x & 63) == 0 && r0 + i < ex.w.R) y[(int64_t)t * ldy + r0 + i] = rq_cast<TX>(v);
  }
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct Layout {
  int64_t logits, ids, weights, h, total;
};
inline Layout layout(int T, int I, int E, int K) {
  const int64_t n = T < TOKENS ? T : TOKENS;
  Layout l;
  l.logits = 0;
  l.ids = l.logits + up256(n * E * 4);
  l.weights = l.ids + up256(n * K * 4);
  l.h = l.weights + up256(n * K * 4);
  l.total = l.h + up256(n * K * I * 4);
  return l;
}
inline RqExperts experts(const rq_packed_experts* p, int R, int C) {
  return RqExperts{RqPacked{p->qweight, p->ldp, p->scales, p->lds, p->g_idx, R, C, p->ngroups, p->groupsize},
                   p->stride_q, p->stride_scales, C};
}

}  // namespace

extern "C" int64_t rq_packed_moe_workspace_bytes(int T, int D, int I, int E, int K) {
  if (T < 0 || D <= 0 || I <= 0 || E <= 0 || E > MAX_E || K <= 0 || K > MAX_K || K > E) return RQ_EINVAL;
  return layout(T, I, E, K).total;
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
  const Layout l = layout(T, I, E, K);
  char* ws = (char*)workspace;
  float* logits = (float*)(ws + l.logits);
  int* ids = (int*)(ws + l.ids);
  float* weights = (float*)(ws + l.weights);
  float* h = (float*)(ws + l.h);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    for (int t0 = 0; t0 < T; t0 += TOKENS) {
      const int n = T - t0 < TOKENS ? T - t0 : TOKENS;
      const TX* xt = (const TX*)x + (int64_t)t0 * ldx;
      const dim3 in((I + 4 * RW - 1) / (4 * RW), n * K), out((D + 4 * RW - 1) / (4 * RW), n);
      hipLaunchKernelGGL(k_moe_router<TX>, dim3((E + 3) / 4, n), dim3(256), 0, s, xt, ldx, D, (const TX*)router, ldr, E,
                         logits);
      hipLaunchKernelGGL(k_moe_route, dim3(n), dim3(64), 0, s, logits, E, K, norm, ids, weights,
                         ids_out ? ids_out + (int64_t)t0 * K : nullptr, weights_out ? weights_out + (int64_t)t0 * K : nullptr);
      rq_with_nbits(gate->nbits, [&](auto nb) {
        hipLaunchKernelGGL((k_moe_in<TX, decltype(nb)::value>), in, dim3(256), 0, s, xt, ldx, g, K, ids, MOE_GATE, h);
      });
      rq_with_nbits(up->nbits, [&](auto nb) {
        hipLaunchKernelGGL((k_moe_in<TX, decltype(nb)::value>), in, dim3(256), 0, s, xt, ldx, u, K, ids, MOE_UP, h);
      });
      rq_with_nbits(down->nbits, [&](auto nb) {
        hipLaunchKernelGGL((k_moe_out<TX, decltype(nb)::value>), out, dim3(256), 0, s, h, d, K, ids, weights,
                           (TX*)y + (int64_t)t0 * ldy, ldy);
      });
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
