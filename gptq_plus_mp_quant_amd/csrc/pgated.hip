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

template <typename TX>
int64_t arranged_bytes(TX*, int T, const Weight& g, const Weight& u) {
  return rq_gated_arranged(T, g.w) || rq_gated_arranged(T, u.w) ? rq_arranged_bytes<TX>(T, g.w.C) : 0;
}

struct GradSpace {
  int64_t d, part;                          // floats
};
GradSpace grad_space(int T, int I, int C) {
  // both weights' steps in one launch, or two launches of twice as many parts in all
  const int64_t one = rq_col_parts_floats(T, 2 * rq_col_steps(I), C), two = 2 * rq_col_parts_floats(T, rq_col_steps(I), C);
  return GradSpace{(int64_t)(T < RQ_COL_WIDE ? T : RQ_COL_WIDE) * 2 * I, one > two ? one : two};
}

}  // namespace

extern "C" int64_t rq_packed_gated_workspace_bytes(int T, int I, int C, int dtype, const rq_packed_weight* gate,
                                                   const rq_packed_weight* up) {
  Weight g, u;
  if (T < 0 || T > TOKENS || I <= 0 || C <= 0 || !weight_of(gate, I, C, &g) || !weight_of(up, I, C, &u)) return RQ_EINVAL;
  int64_t bytes = 0;
  if (!rq_with_dtype(dtype, [&](auto* p) { bytes = arranged_bytes(p, T, g, u); })) return RQ_EINVAL;
  return bytes + (rq_gated_together(g.w, g.nbits, u.w, u.nbits) ? 0 : (int64_t)T * 2 * I * 4);
}

extern "C" int rq_packed_gated(const void* x, int dtype, int T, int64_t ldx, int C, int I, const rq_packed_weight* gate,
                               const rq_packed_weight* up, int activation, float* pre, void* h, int64_t ldh, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  Weight g, u;
  if (T < 0 || T > TOKENS || !weight_of(gate, I, C, &g) || !weight_of(up, I, C, &u)) return RQ_EINVAL;
  if (activation < RQ_SILU || activation > RQ_GELU_TANH) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !h || ldx < C || ldh < I) return RQ_EINVAL;
  bool fits = true;
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    const int64_t xa = arranged_bytes(p, T, g, u);
    const bool together = rq_gated_together(g.w, g.nbits, u.w, u.nbits);
    const int64_t need = xa + (pre || together ? 0 : (int64_t)T * 2 * I * 4);
    if (need && (!workspace || workspace_bytes < need)) {
      fits = false;
      return;
    }
    if (!pre && !together) pre = reinterpret_cast<float*>((char*)workspace + xa);
    rq_gated_rows<TX>((const TX*)x, workspace, T, ldx, g.w, g.nbits, u.w, u.nbits, activation, pre, (TX*)h, ldh,
                      reinterpret_cast<hipStream_t>(stream));
  });
  if (!known || !fits) return RQ_EINVAL;
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
    for (int t0 = 0; t0 < T; t0 += RQ_COL_WIDE) {
      const int n = T - t0 < RQ_COL_WIDE ? T - t0 : RQ_COL_WIDE;
      const int64_t plane = (int64_t)n * I;
      rq_gated_pre_grad<TX>((const TX*)grad_h + t0 * ldg, ldg, n, I, activation, pre + (int64_t)t0 * 2 * I, d, s);
      int parts;
      if (rq_cols_together(g.w, g.nbits, u.w, u.nbits)) {
        const RqColSplit sp = rq_col_split_wide(n, 2 * rq_col_steps(I), C);
        rq_cols_parts2(d, n, I, plane, g.w, u.w, g.nbits, sp, part, s);
        parts = sp.parts;
      } else {
        const RqColSplit sp = rq_col_split_wide(n, rq_col_steps(I), C);
        rq_cols_parts<float>(d, n, I, g.w, g.nbits, sp, part, s);
        rq_cols_parts<float>(d + plane, n, I, u.w, u.nbits, sp, part + (int64_t)sp.parts * n * C, s);
        parts = 2 * sp.parts;
      }
      rq_gated_join<TX>(part, parts, n, C, (TX*)grad_x + t0 * ldx, ldx, s);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
