// Products with a packed weight: y = x W^T (+ bias) and its gradient dx = dy W for a few tokens, W read
// as the codes and scales that export_packed stores and never written out.
//
//   y[t, r]  = sum_c x[t, c] * s[g(c), r] * q[r, c] + b[r]
//   dx[t, c] = sum_r dy[t, r] * s[g(c), r] * q[r, c]
//
// Sums are held in fp32; the one rounding to fewer bits is the result's to x's type.
#include "plinear_types.h"

extern "C" int rq_packed_linear(const void* x, int x_dtype, int T, int64_t ldx, int C, const uint32_t* qweight,
                                int64_t ldp, int nbits, int R, const float* scales, int64_t lds, int ngroups,
                                const int32_t* g_idx, int groupsize, const void* bias, void* y, int64_t ldy,
                                void* stream) {
  const RqPacked w = rq_packed(qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize);
  if (T < 0 || rq_packed_check(w, nbits) != RQ_OK) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !y || ldx < C || ldy < R) return RQ_EINVAL;
  const bool known = rq_with_dtype(x_dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    rq_linear_rows<TX>((const TX*)x, T, ldx, w, nbits, (const TX*)bias, (TX*)y, ldy, reinterpret_cast<hipStream_t>(stream));
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int64_t rq_packed_linear_grad_workspace_bytes(int T, int R, int C) {
  if (T < 0 || R <= 0 || C <= 0) return RQ_EINVAL;
  int64_t floats = 0;
  for (const int n : {T < RQ_COL_TOKENS ? T : RQ_COL_TOKENS, T % RQ_COL_TOKENS}) {     // a shorter last launch
    const int64_t need = n ? (int64_t)rq_col_split(n, R, C).parts * n * C : 0;
    floats = need > floats ? need : floats;
  }
  return floats * 4;
}

extern "C" int rq_packed_linear_grad(const void* grad_y, int dtype, int T, int64_t ldg, int C, const uint32_t* qweight,
                                     int64_t ldp, int nbits, int R, const float* scales, int64_t lds, int ngroups,
                                     const int32_t* g_idx, int groupsize, void* grad_x, int64_t ldx, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  const RqPacked w = rq_packed(qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize);
  if (T < 0 || rq_packed_check(w, nbits) != RQ_OK) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!grad_y || !grad_x || ldg < R || ldx < C) return RQ_EINVAL;
  if (!workspace || workspace_bytes < rq_packed_linear_grad_workspace_bytes(T, R, C)) return RQ_EINVAL;
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    rq_linear_cols<TX>((const TX*)grad_y, T, ldg, w, nbits, (float*)workspace, (TX*)grad_x, ldx,
                       reinterpret_cast<hipStream_t>(stream));
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
