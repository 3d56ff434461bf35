// Log probabilities of given tokens, the entropy and the top alternatives of every row of logits, and the
// gradient of the logits.
//
// With m = max z, d_i = z_i - m, s = sum_i exp(d_i):
//   logprob = d_target - log s        H = log s - (sum_i exp(d_i) d_i) / s        p_i = exp(d_i - log s)
//   dz_i = gl (delta_{i,target} - p_i) - gh p_i (log p_i + H)
// Differences from m are formed first, so masks of the type's lowest value cost no precision; a term
// with exp(d_i) = 0 is 0 whatever d_i is (-inf among them).  A row with nothing left (m = -inf) has
// logprob -inf, H = 0 and no gradient.  A NaN or +inf logit makes its row NaN.
// All statistics are fp32.  Equal values are ordered by their index, NaN above everything.
#include "packed_bits.h"

namespace {

constexpr int MAX_TOP = 64;

__device__ __forceinline__ uint64_t top_key(float z, int i) {
  return ((uint64_t)rq_order_key(z) << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)i);
}

template <typename TX>
__global__ __launch_bounds__(256) void k_logprob_rows(const TX* __restrict__ z, int64_t ldz, int V,
                                                      const int64_t* __restrict__ targets, int64_t ignore, int top,
                                                      float* __restrict__ logprob, float* __restrict__ entropy,
                                                      int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
                                                      float* __restrict__ stats) {
  __shared__ float red[3][4];
  __shared__ uint64_t best[4];
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const TX* row = z + n * ldz;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += 256) m = rq_nan_max(m, rq_load_elem(row + i));
  for (int o = 32; o; o >>= 1) m = rq_nan_max(m, __shfl_xor(m, o));
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = rq_nan_max(rq_nan_max(red[0][0], red[0][1]), rq_nan_max(red[0][2], red[0][3]));
  const bool empty = m == -INFINITY;
  float s = 0.0f, a = 0.0f;
  for (int i = threadIdx.x; i < V; i += 256) {
    const float d = rq_load_elem(row + i) - m;
    const float e = expf(d);
    s += e;
    a += e == 0.0f ? 0.0f : e * d;
  }
  for (int o = 32; o; o >>= 1) {
    s += __shfl_xor(s, o);
    a += __shfl_xor(a, o);
  }
  if (lane == 0) {
    red[1][wave] = s;
    red[2][wave] = a;
  }
  __syncthreads();
  s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  a = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const float ls = empty ? 0.0f : logf(s);
  const float H = empty ? 0.0f : ls - a / s;
  if (threadIdx.x == 0) {
    const int64_t t = targets[n];
    float lp = 0.0f;
    if (t != ignore) {
      if (t < 0 || t >= V) lp = __builtin_nanf("");
      else lp = empty ? -INFINITY : (rq_load_elem(row + t) - m) - ls;
    }
    logprob[n] = lp;
    entropy[n] = H;
    stats[3 * n] = m;
    stats[3 * n + 1] = ls;
    stats[3 * n + 2] = H;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t b = 0;
    for (int i = threadIdx.x; i < V; i += 256) {
      const uint64_t key = top_key(rq_load_elem(row + i), i);
      if (key < last && key > b) b = key;
    }
    for (int o = 32; o; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)b, o);
      b = other > b ? other : b;
    }
    __syncthreads();
    if (lane == 0) best[wave] = b;
    __syncthreads();
    for (int q = 0; q < 4; ++q) b = best[q] > b ? best[q] : b;
    last = b;
    if (threadIdx.x == 0) {
      const int i = (int)(0xFFFFFFFFu - (uint32_t)b);
      top_ids[n * top + k] = i;
      top_lp[n * top + k] = empty ? -INFINITY : (rq_key_value((uint32_t)(b >> 32)) - m) - ls;
    }
  }
}

template <typename TX>
__global__ __launch_bounds__(256) void k_logprob_grad(const TX* z, int64_t ldz, int V,
                                                      const int64_t* __restrict__ targets, int64_t ignore,
                                                      const float* __restrict__ stats, const float* __restrict__ gl_,
                                                      const float* __restrict__ gh_, TX* dz, int64_t ldd) {
  const int64_t n = blockIdx.x;
  const int64_t t = targets[n];
  const float m = stats[3 * n], ls = stats[3 * n + 1], H = stats[3 * n + 2];
  const bool empty = m == -INFINITY;
  float gl = t == ignore ? 0.0f : gl_[n];
  if (t != ignore && (t < 0 || t >= V)) gl = __builtin_nanf("");
  const float gh = gh_ ? gh_[n] : 0.0f;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < V; i += 256 * gridDim.y) {
    const float lp = (rq_load_elem(z + n * ldz + i) - m) - ls;
    const float p = expf(lp);
    float g = p == 0.0f ? 0.0f * gl : -p * (gl + gh * (lp + H));
    if (i == t) g += gl;
    dz[n * ldd + i] = rq_cast<TX>(empty ? 0.0f : g);
  }
}

}  // namespace

extern "C" int64_t rq_token_logprobs_workspace_bytes(int64_t N, int V, int top_k) {
  if (N < 0 || V <= 0 || top_k < 0 || top_k > MAX_TOP || top_k > V) return RQ_EINVAL;
  return 0;
}

extern "C" int rq_token_logprobs(const void* logits, int dtype, int64_t N, int64_t ldz, int V, const int64_t* targets,
                                 int64_t ignore_index, int top_k, float* logprob, float* entropy, int64_t* top_ids,
                                 float* top_logprobs, float* stats, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  if (N < 0 || V <= 0 || ldz < V || top_k < 0 || top_k > MAX_TOP || top_k > V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !targets || !logprob || !entropy || !stats || (top_k && (!top_ids || !top_logprobs))) return RQ_EINVAL;
  if (N > INT32_MAX) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    hipLaunchKernelGGL(k_logprob_rows<TX>, dim3((unsigned)N), dim3(256), 0, s, (const TX*)logits, ldz, V, targets,
                       ignore_index, top_k, logprob, entropy, top_ids, top_logprobs, stats);
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int rq_token_logprobs_grad(const void* logits, int dtype, int64_t N, int64_t ldz, int V,
                                      const int64_t* targets, int64_t ignore_index, const float* stats,
                                      const float* grad_logprob, const float* grad_entropy, void* grad_logits,
                                      int64_t ldd, void* stream) {
  if (N < 0 || V <= 0 || ldz < V || ldd < V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !targets || !stats || !grad_logprob || !grad_logits) return RQ_EINVAL;
  if (N > INT32_MAX) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int ny = V > 8192 ? 8 : 1;
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    hipLaunchKernelGGL(k_logprob_grad<TX>, dim3((unsigned)N, ny), dim3(256), 0, s, (const TX*)logits, ldz, V, targets,
                       ignore_index, stats, grad_logprob, grad_entropy, (TX*)grad_logits, ldd);
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
