// Rows of logits: loads and stores of eight at a time.
#pragma once
#include "packed_dot.h"

constexpr float RQ_LOG2E = 1.4426950408889634f;
constexpr int64_t RQ_ROWS_PER_LAUNCH = 1 << 20;

// The 8 logits from column c on that lie before c1; -inf for the others.
template <typename TX>
__device__ __forceinline__ typename RqOperand<TX>::raw rq_load8(const TX* __restrict__ row, int c, int c1) {
  typename RqOperand<TX>::raw v;
  if (c + 8 <= c1) return rq_load_x<true>(row + c, 8);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = -INFINITY;
  if (c < c1) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < c1) __builtin_memcpy((char*)&v + k * sizeof(TX), row + c + k, sizeof(TX));
  }
  return v;
}

template <typename TX>
__device__ __forceinline__ void rq_store8(TX* p, const float (&g)[8]) {
  typename RqOperand<TX>::raw v;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const TX e = rq_cast<TX>(g[k]);
    typename std::remove_reference<decltype(v[0])>::type w;
    __builtin_memcpy(&w, &e, sizeof(TX));
    v[k] = w;
  }
  __builtin_memcpy(p, &v, sizeof(v));
}
