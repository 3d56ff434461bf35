// A packed linear with low-rank adapters of several requests, and its gradients.
//
//   y_t  = W x_t + b + s_a B_a (A_a x_t)        a = ids[t], none where that is below 0
//   v_t  = B_a^T dy_t
//   dx_t = W^T dy_t + s_a A_a^T v_t             dA_a = s_a sum_t v_t x_t^T        dB_a = s_a sum_t dy_t (A_a x_t)^T
//
// The low-rank values are fp32 and stay so; sums are fp32, joined in a fixed order; the one rounding to fewer bits is
// the results'.
#include "plora_types.h"

namespace {

constexpr int TOKENS = 1 << 19;             // of one call: grids hold 65535 x 16 tokens and more

bool lora_ok(const void* a, const void* b, int n, int r) { return a && b && n > 0 && n <= 65535 && r > 0 && r <= LORA_MAX_RANK; }
// rank tiles times parts are a grid's third dimension, of both jobs together
bool width_ok(int cols, int r) { return (int64_t)((r + 31) / 32 * 2) * ((cols - 1) / RQ_LORA_COLS + 1) <= 32767; }

struct GradSpace {
  int64_t u, v, part;                       // floats
};
GradSpace grad_space(int T, int R, int C, int r) {
  return GradSpace{rq_low_floats(rq_low(nullptr, T, C, r)), rq_low_floats(rq_low(nullptr, T, R, r)),
                   rq_col_parts_floats(T, rq_col_steps(R), C)};
}

}  // namespace

extern "C" int64_t rq_packed_linear_lora_workspace_bytes(int T, int R, int C, int r, int dtype) {
  if (T < 0 || T > TOKENS || R <= 0 || C <= 0 || r <= 0 || r > LORA_MAX_RANK || !width_ok(C, r)) return RQ_EINVAL;
  int64_t bytes = 4 * rq_low_floats(rq_low(nullptr, T, C, r));
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    if (rq_lora_own(T, R, C, r, sizeof(*p))) bytes = 0;
    else if (T > 16) bytes += rq_arranged_bytes<typename std::remove_pointer<decltype(p)>::type>(T, C);
  });
  return known ? bytes : RQ_EINVAL;
}

extern "C" int rq_packed_linear_lora(const void* x, int dtype, int T, int64_t ldx, int C, const uint32_t* qweight, int64_t ldp,
                                     int nbits, int R, const float* scales, int64_t lds, int ngroups, const int32_t* g_idx,
                                     int groupsize, const void* bias, const void* lora_a, const void* lora_b, int n, int r,
                                     const int64_t* adapter_ids, const float* scaling, float scale, void* y, int64_t ldy,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  const RqPacked w = rq_packed(qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize);
  if (T < 0 || T > TOKENS || rq_packed_check(w, nbits) != RQ_OK || !lora_ok(lora_a, lora_b, n, r) || !width_ok(C, r))
    return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !y || ldx < C || ldy < R) return RQ_EINVAL;
  const int64_t need = rq_packed_linear_lora_workspace_bytes(T, R, C, r, dtype);
  if (need < 0 || (need && (!workspace || workspace_bytes < need))) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    const RqLora<TX> lora{(const TX*)lora_a, (const TX*)lora_b, adapter_ids, scaling, scale, n, r};
    const RqLow low = rq_low(need ? (float*)workspace : nullptr, T, C, r);         // a multiple of 128 bytes
    void* arranged = rq_lora_arranged(T, w) ? (float*)workspace + rq_low_floats(low) : nullptr;
    if (need) rq_lora_down<TX>(rq_down_jobs<TX>(RqDown<TX>{(const TX*)x, ldx, C, 1, low}, nullptr, lora), arranged, nbits, s);
    rq_lora_rows<TX>((const TX*)x, T, ldx, w, nbits, (const TX*)bias, lora, low, arranged, (TX*)y, ldy, s);
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int64_t rq_packed_linear_lora_grad_workspace_bytes(int T, int R, int C, int r) {
  if (T < 0 || T > TOKENS || R <= 0 || C <= 0 || r <= 0 || r > LORA_MAX_RANK || !width_ok(R, r) || !width_ok(C, r)) return RQ_EINVAL;
  const GradSpace g = grad_space(T, R, C, r);
  return 4 * (g.u + g.v + g.part);
}

extern "C" int rq_packed_linear_lora_grad(const void* grad_y, int dtype, int T, int64_t ldg, const void* x, int64_t ldx, int C,
                                          const uint32_t* qweight, int64_t ldp, int nbits, int R, const float* scales,
                                          int64_t lds, int ngroups, const int32_t* g_idx, int groupsize, const void* lora_a,
                                          const void* lora_b, int n, int r, const int64_t* adapter_ids, const float* scaling,
                                          float scale, void* grad_x, int64_t ldgx, void* grad_a, void* grad_b, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  const RqPacked w = rq_packed(qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize);
  if (T < 0 || T > TOKENS || rq_packed_check(w, nbits) != RQ_OK || !lora_ok(lora_a, lora_b, n, r) || !width_ok(C, r) ||
      !width_ok(R, r))
    return RQ_EINVAL;
  if (!grad_a != !grad_b || (T && (!grad_y || !x || ldg < R || ldx < C || (grad_x && ldgx < C)))) return RQ_EINVAL;
  const GradSpace g = grad_space(T, R, C, r);
  if (T && (!workspace || workspace_bytes < 4 * (g.u + g.v + g.part))) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    const RqLora<TX> lora{(const TX*)lora_a, (const TX*)lora_b, adapter_ids, scaling, scale, n, r};
    float* ws = (float*)workspace;
    const RqLow u = rq_low(ws, T, C, r), v = rq_low(ws + g.u, T, R, r);
    float* part = ws + g.u + g.v;
    const TX* dy = (const TX*)grad_y;
    const RqDown<TX> ofx{(const TX*)x, ldx, C, 1, u};
    RqDownJobs<TX> jobs = rq_down_jobs<TX>(RqDown<TX>{dy, ldg, R, 0, v}, grad_a ? &ofx : nullptr, lora);
    if (T && (!grad_x || !rq_jobs_rows(jobs, T < RQ_COL_WIDE ? T : RQ_COL_WIDE, C))) {
      rq_lora_down<TX>(jobs, nullptr, nbits, s);
      jobs.z = 0;
    }
    RqLoraDx<TX> dx{part, 0, 0, 0, nullptr, ldgx};
    for (int t0 = 0; grad_x && t0 < T; t0 += RQ_COL_WIDE) {
      const int k = T - t0 < RQ_COL_WIDE ? T - t0 : RQ_COL_WIDE;
      const RqColSplit sp = rq_col_split_wide(k, rq_col_steps(R), C);
      rq_lora_cols<TX>(dy + t0 * ldg, k, ldg, w, nbits, sp, part, jobs, s);
      jobs.z = 0;
      dx = RqLoraDx<TX>{part, sp.parts, t0, k, (TX*)grad_x + t0 * ldgx, ldgx};
      if (t0 + k < T) rq_lora_grads<TX>(dx, (const TX*)x, ldx, C, dy, ldg, R, T, lora, u, v, nullptr, nullptr, s);
    }
    rq_lora_grads<TX>(dx, (const TX*)x, ldx, C, dy, ldg, R, T, lora, u, v, (TX*)grad_a, (TX*)grad_b, s);
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
