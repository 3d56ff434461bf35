// The gated half of a feed-forward block with packed weights: what its launches share.  Each element type's kernels
// are a translation unit of their own.
#pragma once
#include "packed_dot.h"
#include "plinear_types.h"

enum { RQ_SILU = 0, RQ_GELU = 1, RQ_GELU_TANH = 2 };

struct RqAct {
  float f, df;
};
// An activation and its derivative.  GELU's tails keep their digits: erfc, and tanh as a logistic function.
__device__ __forceinline__ RqAct rq_act(int kind, float a) {
  if (kind == RQ_SILU) {
    const float s = 1.0f / (1.0f + expf(-a));
    return RqAct{a * s, s * __builtin_fmaf(a, 1.0f - s, 1.0f)};
  }
  if (kind == RQ_GELU) {
    const float s = 0.5f * erfcf(a * -0.70710678118654752f), d = 0.3989422804014327f * expf(-0.5f * a * a);
    return RqAct{a * s, d == 0.0f ? s : __builtin_fmaf(a, d, s)};
  }
  constexpr float K = 1.5957691216057308f, CUBE = 0.044715f;       // 2 sqrt(2 / pi)
  const float s = 1.0f / (1.0f + expf(-K * (a * __builtin_fmaf(CUBE * a, a, 1.0f)))), d = s * (1.0f - s);
  return RqAct{a * s, d == 0.0f ? s : __builtin_fmaf(a * d, K * __builtin_fmaf(3.0f * CUBE * a, a, 1.0f), s)};
}

// h [T, I] = act(x Wg^T) * (x Wu^T); pre (fp32 [T, 2, I], or NULL where both weights go through one launch): the products.
// xa: room for x as RqArranged has it, where rq_gated_arranged says so for one of the weights.
template <typename TX>
void rq_gated_rows(const TX* x, void* xa, int T, int64_t ldx, const RqPacked& gate, int gate_bits, const RqPacked& up, int up_bits,
                   int act, float* pre, TX* h, int64_t ldh, hipStream_t s);
inline bool rq_gated_together(const RqPacked& gate, int gate_bits, const RqPacked& up, int up_bits) {
  return gate_bits == up_bits && rq_whole_mode_of(gate) == rq_whole_mode_of(up);
}
inline bool rq_gated_arranged(int T, const RqPacked& w) { return T > 16 && rq_whole_mode_of(w) == RQ_RUNS; }

// d [2, T, I] = the gradients of the products from grad_h [T, I] and pre [T, 2, I]
template <typename TX>
void rq_gated_pre_grad(const TX* grad_h, int64_t ldg, int T, int I, int act, const float* pre, float* d, hipStream_t s);
// dx [T, C] = the sum of parts [parts, T, C]
template <typename TX>
void rq_gated_join(const float* part, int parts, int T, int C, TX* dx, int64_t ldx, hipStream_t s);
