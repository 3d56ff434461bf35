// Products with a packed weight: y = x W^T (+ bias) and its gradient dx = dy W for a few tokens, W read
// as the codes and scales that export_packed stores and never written out.
//
//   y[t, r]  = sum_c x[t, c] * s[g(c), r] * q[r, c] + b[r]
//   dx[t, c] = sum_r dy[t, r] * s[g(c), r] * q[r, c]
//
// Sums are held in fp32; the one rounding to fewer bits is the result's to x's type.
#include "packed_bits.h"

namespace {

// --- y = x W^T, any type, any groups ------------------------------------------------------------
// A wave takes RW rows and TT tokens and runs over the columns, 8 a lane: every weight is
// s * q in fp32, multiplied and added by fmaf; lanes are joined at the end.
constexpr int RW = 4, TT = 8;

template <typename TX, int NB>
__global__ __launch_bounds__(256) void k_packed_rows(const TX* __restrict__ x, int T, int64_t ldx, RqPacked w,
                                                     const TX* __restrict__ bias, TX* __restrict__ y, int64_t ldy) {
  const int lane = threadIdx.x & 63;
  const int r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * RW;
  const int t0 = blockIdx.y * TT;
  if (r0 >= w.R) return;
  float acc[RW][TT];
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[i][t] = 0.0f;
  for (int c = lane * 8; c < w.C; c += 512) {
    const int nc = min(8, w.C - c);
    float xv[TT][8];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        xv[t][k] = (t0 + t < T && k < nc) ? rq_load_elem(x + (int64_t)(t0 + t) * ldx + c + k) : 0.0f;
    int g[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = rq_group_of(w, c + (k < nc ? k : 0));
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int r = min(r0 + i, w.R - 1);
      int code[8];
      rq_codes8<NB>(w.q + (int64_t)r * w.ldp, c, nc, code);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float wv = k < nc ? rq_scale_of(w, g[k], r) * (float)code[k] : 0.0f;
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[i][t] = __builtin_fmaf(xv[t][k], wv, acc[i][t]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RW; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int m = 32; m; m >>= 1) acc[i][t] += __shfl_xor(acc[i][t], m);
      if (lane == 0 && r0 + i < w.R && t0 + t < T) {
        const float b = bias ? rq_load_elem(bias + r0 + i) : 0.0f;
        y[(int64_t)(t0 + t) * ldy + r0 + i] = rq_cast<TX>(acc[i][t] + b);
      }
    }
}

// --- dx = dy W, any type, any groups ------------------------------------------------------------
// A thread takes 8 columns and TT tokens over a range of rows; the ranges' sums are joined, in their
// order, by k_packed_join.
template <typename TX, int NB>
__global__ __launch_bounds__(64) void k_packed_cols(const TX* __restrict__ dy, int T, int64_t ldy, RqPacked w,
                                                    int rows_per, float* __restrict__ part) {
  const int c = (blockIdx.x * 64 + threadIdx.x) * 8;
  const int t0 = blockIdx.z * TT;
  if (c >= w.C) return;
  const int nc = min(8, w.C - c);
  const int ra = blockIdx.y * rows_per, rb = min(w.R, ra + rows_per);
  float acc[8][TT];
  int g[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    g[k] = rq_group_of(w, c + (k < nc ? k : 0));
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[k][t] = 0.0f;
  }
  for (int r = ra; r < rb; ++r) {
    float d[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) d[t] = t0 + t < T ? rq_load_elem(dy + (int64_t)(t0 + t) * ldy + r) : 0.0f;
    int code[8];
    rq_codes8<NB>(w.q + (int64_t)r * w.ldp, c, nc, code);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float wv = rq_scale_of(w, g[k], r) * (float)code[k];
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[k][t] = __builtin_fmaf(d[t], wv, acc[k][t]);
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t)
    if (t0 + t < T)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < nc) part[((int64_t)blockIdx.y * T + t0 + t) * w.C + c + k] = acc[k][t];
}

template <typename TX>
__global__ __launch_bounds__(256) void k_packed_join(const float* __restrict__ part, int nparts, int T, int C,
                                                     TX* __restrict__ dx, int64_t ldx) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  for (int t = blockIdx.y; t < T; t += gridDim.y) {
    float s = 0.0f;
    for (int p = 0; p < nparts; ++p) s += part[((int64_t)p * T + t) * C + c];
    dx[(int64_t)t * ldx + c] = rq_cast<TX>(s);
  }
}

constexpr int TOKENS_PER_LAUNCH = 32768;       // grid.y / grid.z hold at most 65535 blocks

inline int grad_parts(int C, int R) {
  const int cols = (C + 511) / 512;
  int parts = (1024 + cols - 1) / cols;
  parts = parts > (R + 31) / 32 ? (R + 31) / 32 : parts;
  return parts < 1 ? 1 : parts;
}
inline int tokens_per_call(int T) { return T < 64 ? T : 64; }

}  // namespace

extern "C" int rq_packed_linear(const void* x, int x_dtype, int T, int64_t ldx, int C, const uint32_t* qweight,
                                int64_t ldp, int nbits, int R, const float* scales, int64_t lds, int ngroups,
                                const int32_t* g_idx, int groupsize, const void* bias, void* y, int64_t ldy,
                                void* stream) {
  const RqPacked w{qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize};
  if (T < 0 || rq_packed_check(w, nbits) != RQ_OK) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!x || !y || ldx < C || ldy < R) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool known = rq_with_dtype(x_dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    rq_with_nbits(nbits, [&](auto nb) {
      for (int t0 = 0; t0 < T; t0 += TOKENS_PER_LAUNCH) {
        const int n = T - t0 < TOKENS_PER_LAUNCH ? T - t0 : TOKENS_PER_LAUNCH;
        hipLaunchKernelGGL((k_packed_rows<TX, decltype(nb)::value>), dim3((R + 4 * RW - 1) / (4 * RW), (n + TT - 1) / TT),
                           dim3(256), 0, s, (const TX*)x + (int64_t)t0 * ldx, n, ldx, w, (const TX*)bias,
                           (TX*)y + (int64_t)t0 * ldy, ldy);
      }
    });
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int64_t rq_packed_linear_grad_workspace_bytes(int T, int R, int C) {
  if (T < 0 || R <= 0 || C <= 0) return RQ_EINVAL;
  return (int64_t)grad_parts(C, R) * tokens_per_call(T) * C * 4;
}

extern "C" int rq_packed_linear_grad(const void* grad_y, int dtype, int T, int64_t ldg, int C, const uint32_t* qweight,
                                     int64_t ldp, int nbits, int R, const float* scales, int64_t lds, int ngroups,
                                     const int32_t* g_idx, int groupsize, void* grad_x, int64_t ldx, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  const RqPacked w{qweight, ldp, scales, lds, g_idx, R, C, ngroups, groupsize};
  if (T < 0 || rq_packed_check(w, nbits) != RQ_OK) return RQ_EINVAL;
  if (T == 0) return RQ_OK;
  if (!grad_y || !grad_x || ldg < R || ldx < C) return RQ_EINVAL;
  if (!workspace || workspace_bytes < rq_packed_linear_grad_workspace_bytes(T, R, C)) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  float* part = (float*)workspace;
  const int want = grad_parts(C, R);
  const int rows_per = (R + want - 1) / want;
  const int parts = (R + rows_per - 1) / rows_per;
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    rq_with_nbits(nbits, [&](auto nb) {
      for (int t0 = 0; t0 < T; t0 += 64) {
        const int n = T - t0 < 64 ? T - t0 : 64;
        hipLaunchKernelGGL((k_packed_cols<TX, decltype(nb)::value>),
                           dim3((C + 511) / 512, parts, (n + TT - 1) / TT), dim3(64), 0, s,
                           (const TX*)grad_y + (int64_t)t0 * ldg, n, ldg, w, rows_per, part);
        hipLaunchKernelGGL(k_packed_join<TX>, dim3((C + 255) / 256, n), dim3(256), 0, s, part, parts, n, C,
                           (TX*)grad_x + (int64_t)t0 * ldx, ldx);
      }
    });
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
