// The gated half of a feed-forward block with packed weights, and its gradient.
//
//   a = x Wg^T, b = x Wu^T, h = act(a) * b
//   da = dh * b * act'(a), db = dh * act(a), dx = da Wg + db Wu
//
// a, b, da and db are fp32; the one rounding to fewer bits is the result's.
#include "pgated_types.h"

namespace {

constexpr int TOKENS = 1 << 19;             // of one call

struct Weight {
  RqPacked w;
  int nbits;
};
bool weight_of(const rq_packed_weight* p, int R, int C, Weight* out) {
  if (!p) return false;
  *out = Weight{rq_packed(p->qweight, p->ldp, p->scales, p->lds, p->g_idx, R, C, p->ngroups, p->groupsize), p->nbits};
  return rq_packed_check(out->w, p->nbits) == RQ_OK;
}

struct GradSpace {
  int64_t d, part;                          // floats
};
GradSpace grad_space(int T, int I, int C) {
  GradSpace g = {(int64_t)(T < RQ_COL_TOKENS ? T : RQ_COL_TOKENS) * 2 * I, 0};
  for (const int n : {T < RQ_COL_TOKENS ? T : RQ_COL_TOKENS, T % RQ_COL_TOKENS}) {
    const int64_t need = n ? (int64_t)rq_col_split(n, I, C).parts * 2 * n * C : 0;
    g.part = need > g.part ? need : g.part;
  }
  return g;
}

}  // namespace

extern "C" int64_t rq_packed_gated_workspace_bytes(int T, int I, int C, const rq_packed_weight* gate, const rq_packed_weight* up) {
  Weight g, u;
  if (T < 0 || T > TOKENS || I <= 0 || C <= 0 || !weight_of(gate, I, C, &g) || !weight_of(up, I, C, &u)) return RQ_EINVAL;
  return rq_gated_together(g.w, g.nbits, u.w, u.nbits) ? 0 : (int64_t)T * 2 * I * 4;
}

extern "C" int rq_packed_gated(const void* x, int dtype, int T, int64_t ldx, int C, int I, const rq_packed_weight* gate,
                               const rq_packed_weight* up, int activation, float* pre, void* h, int64_t ldh, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  Weight g, u;
  if (T < 0 || T > TOKENS || !weight_of(gate, I, C, &g) || !weight_of(up, I, C, &u)) return RQ_EINVAL;
  if (activation < RQ_SILU || activation > RQ_GELU_TANH) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !h || ldx < C || ldh < I) return RQ_EINVAL;
  if (!pre && !rq_gated_together(g.w, g.nbits, u.w, u.nbits)) {
    if (!workspace || workspace_bytes < (int64_t)T * 2 * I * 4) return RQ_EINVAL;
    pre = (float*)workspace;
  }
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    rq_gated_rows<TX>((const TX*)x, T, ldx, g.w, g.nbits, u.w, u.nbits, activation, pre, (TX*)h, ldh,
                      reinterpret_cast<hipStream_t>(stream));
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int64_t rq_packed_gated_grad_workspace_bytes(int T, int I, int C) {
  if (T < 0 || T > TOKENS || I <= 0 || C <= 0) return RQ_EINVAL;
  const GradSpace g = grad_space(T, I, C);
  return 4 * (g.d + g.part);
}

extern "C" int rq_packed_gated_grad(const void* grad_h, int dtype, int T, int64_t ldg, int I, const float* pre, int activation,
                                    const rq_packed_weight* gate, const rq_packed_weight* up, int C, void* grad_x, int64_t ldx,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  Weight g, u;
  if (T < 0 || T > TOKENS || !weight_of(gate, I, C, &g) || !weight_of(up, I, C, &u)) return RQ_EINVAL;
  if (activation < RQ_SILU || activation > RQ_GELU_TANH) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!grad_h || !pre || !grad_x || ldg < I || ldx < C) return RQ_EINVAL;
  const GradSpace space = grad_space(T, I, C);
  if (!workspace || workspace_bytes < 4 * (space.d + space.part)) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    float *d = (float*)workspace, *part = d + space.d;
    for (int t0 = 0; t0 < T; t0 += RQ_COL_TOKENS) {
      const int n = T - t0 < RQ_COL_TOKENS ? T - t0 : RQ_COL_TOKENS;
      const RqColSplit sp = rq_col_split(n, I, C);
      rq_gated_pre_grad<TX>((const TX*)grad_h + t0 * ldg, ldg, n, I, activation, pre + (int64_t)t0 * 2 * I, d, s);
      rq_cols_parts<float>(d, n, I, g.w, g.nbits, sp, part, s);
      rq_cols_parts<float>(d + (int64_t)n * I, n, I, u.w, u.nbits, sp, part + (int64_t)sp.parts * n * C, s);
      rq_gated_join<TX>(part, 2 * sp.parts, n, C, (TX*)grad_x + t0 * ldx, ldx, s);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
