// Distillation from a teacher's top tokens: the divergence of every row and the gradient of the logits.
//
// With the student's q = softmax(z c) over V tokens (c = 1 / temperature) and the teacher's list of K tokens with log
// probabilities t (an id below 0: no entry):
//   RENORMALISE  p_i = softmax(t c) over the list            loss = sum_i p_i (log p_i - log q_i)
//   BUCKET       p_i = exp(t_i), r = 1 - sum p, the rest of the vocabulary one class:
//                loss = sum_i p_i (log p_i - log q_i) + r (log r - log q_rest)
//   mass = sum p + r.   dz_j = g c (q_j mass - p_j) for a listed token, g c w_j F for any other, with w the
//   student's distribution over the others and F = q_rest mass - r (RENORMALISE: w = q, F = mass).
// For q_rest listed tokens are left out of the sum, not subtracted from it, so that a small rest keeps its digits;
// it has a maximum of its own for the same reason.  Terms with p = 0 are 0.  A row without entries, or without a logit
// above -inf, has no gradient.  Differences from a maximum are formed first, in fp32; a lane's sums are fp32.  They are
// joined in 64 bits, as the sums over the list are, a few values a row; the sums that the parts of a cut row hand on are
// rounded to fp32 in between, half a unit beside what the lanes' sums are off by, for half the bytes.
// The rows are bound by the logits' bytes: 2048 x 128256 bf16 95 us, 5.5 TB/s; a few short ones by latency (3 x 32003 fp32, one
// large workgroup each: 10.2 us; cut over several and joined by a second launch 4.9 + 5.6).  The gradient reads and writes them
// once: 1024 x 128256 bf16 114 us, 4.6 TB/s, where a copy reaches 5.1.
#include "logits.h"

namespace {

constexpr int MAX_LIST = 256, MAX_V = 1 << 30;
constexpr int PER_LANE = MAX_LIST / 64;    // entries of a row's list to a lane of its first wave
constexpr int MAX_COLS = 1 << 18;          // columns of a workgroup that keeps a bit for each (32 KB)
constexpr int STATS = 8;
enum { RENORMALISE = 0, BUCKET = 1 };
constexpr double NO_REST = 0x1p-20;        // a remainder up to this beside an empty rest is the list's rounding

struct Teacher {
  const int64_t* ids;       // [N, K]
  const float* t;           // [N, K]
  int K;
  double c;                 // 1 / temperature
  float k, k_low;           // log2(e) / temperature, and what the first rounds off
};

// Maximum and sum of exp((z - m) c); nothing: -inf, 0.
struct Sum {
  float m;
  double s;
};
__device__ __forceinline__ float from(float m) { return m == -INFINITY ? 0.0f : m; }
// exp(d c) for a part's sum: the exponent's rounding, which all of the part would share, is made good.
__device__ __forceinline__ double power(float d, const Teacher& h) {
  const float p = d * h.k, low = __builtin_fmaf(d, h.k, -p) + d * h.k_low;
  const float e = __builtin_amdgcn_exp2f(p);
  return e == 0.0f || p == -INFINITY ? (double)e : (double)e * (1.0 + 0.6931471805599453 * (double)low);
}
__device__ __forceinline__ Sum join(Sum x, Sum y, const Teacher& h) {
  const float m = fmaxf(x.m, y.m), m0 = from(m);
  return Sum{m, x.s * power(x.m - m0, h) + y.s * power(y.m - m0, h)};
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ Sum wave_join(Sum v, const Teacher& h) {
  const float m = wave_max(v.m);
  // 0 times a factor that is 0: a lane without a maximum may still hold a NaN
  return Sum{m, wave_sum(v.s * power(v.m - from(m), h))};
}
// The threads' sums joined in the order of lanes and waves; the first wave's to use.
template <int THREADS>
__device__ __forceinline__ Sum block_join(Sum v, const Teacher& h, Sum* lds) {
  v = wave_join(v, h);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < THREADS / 64; ++w) v = join(v, lds[w], h);
  return v;
}

// Entries of the row's list, of the first wave's lanes: lane l has entries l, l + 64, ...
struct Entry {
  int id;                   // -1: none, V: outside the vocabulary
  float t, z;
};
template <typename TX>
__device__ __forceinline__ void entries_of(const TX* __restrict__ row, int V, int64_t n, const Teacher& h, Entry (&e)[PER_LANE]) {
#pragma unroll
  for (int k = 0; k < PER_LANE; ++k) {
    e[k] = Entry{-1, 0.0f, 0.0f};
    const int at = threadIdx.x + 64 * k;
    if (threadIdx.x < 64 && at < h.K) {
      const int64_t id = h.ids[n * h.K + at];
      e[k].t = h.t[n * h.K + at];
      e[k].id = id < 0 ? -1 : id < V ? (int)id : V;
      if (id >= 0 && id < V) e[k].z = rq_load_elem(row + id);
    }
  }
}

// A row's loss and statistics from the sums over the rest (RENORMALISE: over everything) and over the list, by its first
// wave.
template <int TAIL>
__device__ __forceinline__ void finish_row(int64_t n, int V, const Entry (&e)[PER_LANE], const Teacher& h, Sum rest, Sum list,
                                           float* __restrict__ loss_out, float* __restrict__ stats) {
  float mt = 0.0f;
  if (TAIL == RENORMALISE) {
    mt = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) mt = fmaxf(mt, e[k].id >= 0 ? e[k].t : -INFINITY);
    mt = from(wave_max(mt));
  }
  double at[PER_LANE], x[PER_LANE], total = 0.0;
  bool used = false, outside = false;
#pragma unroll
  for (int k = 0; k < PER_LANE; ++k) {
    at[k] = ((double)e[k].t - mt) * h.c;
    x[k] = e[k].id >= 0 ? exp(at[k]) : 0.0;
    total += x[k];
    used |= e[k].id >= 0;
    outside |= e[k].id == V;
  }
  total = wave_sum(total);
  const double P = TAIL == RENORMALISE ? (total == 0.0 ? 0.0 : total / total) : total;
  const Sum all = TAIL == BUCKET ? join(rest, list, h) : rest;
  const bool empty = all.m == -INFINITY && all.s == 0.0, none = rest.m == -INFINITY && rest.s == 0.0;
  double r = TAIL == BUCKET && !(1.0 - P < 0.0) ? 1.0 - P : 0.0;
  if (none && r <= NO_REST) r = 0.0;
  // four logarithms at once, by four lanes
  const int lane = threadIdx.x & 63;
  const double logs = log(lane == 0 ? all.s : lane == 1 ? rest.s : lane == 2 ? total : r);
  const double m = from(all.m), ls = empty ? 0.0 : __shfl(logs, 0);
  const double lt = TAIL == RENORMALISE && total != 0.0 ? __shfl(logs, 2) : 0.0;
  double loss = 0.0;
#pragma unroll
  for (int k = 0; k < PER_LANE; ++k) {
    const double lq = empty ? -(double)INFINITY : ((double)e[k].z - m) * h.c - ls;
    const double p = TAIL == RENORMALISE && total != 0.0 ? x[k] / total : x[k];
    loss += p == 0.0 ? 0.0 : p * (at[k] - lt - lq);
  }
  loss = wave_sum(loss);
  double mass = P, factor = P, mr = m, lr = ls;
  if (TAIL == BUCKET) {
    mr = from(rest.m);
    lr = none ? 0.0 : __shfl(logs, 1);
    const double lrest = none ? -(double)INFINITY : (mr - m) * h.c + lr - ls;
    if (r != 0.0) loss += r * (__shfl(logs, 3) - lrest);
    mass = P + r;
    factor = exp(lrest) * mass - r;
  }
  if (empty) mass = factor = 0.0;
  if (__any(outside)) loss = mass = factor = __builtin_nan("");
  if (!__any(used)) loss = mass = factor = 0.0;
  if (threadIdx.x == 0) {
    loss_out[n] = (float)loss;
    float* o = stats + n * STATS;
    o[0] = (float)m;
    o[1] = (float)ls;
    o[2] = (float)mr;
    o[3] = (float)lr;
    o[4] = mt;
    o[5] = (float)lt;
    o[6] = (float)mass;
    o[7] = (float)factor;
  }
}

// A workgroup sums columns [c0, c0 + seg_cols) of row blockIdx.x.  SPLIT: c0 = seg_cols blockIdx.y, and k_distill_join
// finishes the row; else that is the row.
template <typename TX, int TAIL, bool SPLIT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_distill_rows(const TX* __restrict__ z, int64_t ldz, int V, int seg_cols, Teacher h,
                                                          float* __restrict__ loss, float* __restrict__ stats,
                                                          float* __restrict__ seg) {
  typedef typename RqOperand<TX>::raw Raw;
  constexpr int U = sizeof(TX) == 2 ? 8 : 4;
  extern __shared__ __attribute__((aligned(16))) uint32_t listed[];     // BUCKET: a bit for every column
  __shared__ Sum lds[THREADS / 64];
  const int64_t n = blockIdx.x;
  const TX* row = z + n * ldz;
  const int c0 = SPLIT ? blockIdx.y * seg_cols : 0, c1 = min(V, c0 + seg_cols);
  Entry e[PER_LANE];
  if (!SPLIT || TAIL == BUCKET) entries_of(row, V, n, h, e);
  uint32_t first = 0;                      // entries that are the first with their id, which lies here
  if (TAIL == BUCKET) {
    for (int w = threadIdx.x; w < (c1 - c0 + 31) / 32; w += THREADS) listed[w] = 0u;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
      if (e[k].id < c0 || e[k].id >= c1) continue;
      const uint32_t bit = 1u << ((e[k].id - c0) & 31);
      if (!(atomicOr(&listed[(e[k].id - c0) >> 5], bit) & bit)) first |= 1u << k;
    }
    __syncthreads();
  }
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(listed);
  float m = -INFINITY, s = 0.0f;
  for (int c = c0 + 8 * (int)threadIdx.x; c < c1; c += 8 * THREADS * U) {
    Raw in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) in[u] = rq_load8<TX>(row, c + 8 * THREADS * u, c1);
    float f[U][8], most = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cu = c + 8 * THREADS * u;
      const uint32_t drop = TAIL == BUCKET && cu < c1 ? bytes[(cu - c0) >> 3] : 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[u][k] = drop >> k & 1 ? -INFINITY : (float)in[u][k];
        most = fmaxf(most, f[u][k]);
      }
    }
    if (most > m) {
      s *= __builtin_amdgcn_exp2f((m - most) * h.k);
      m = most;
    }
    const float m0 = from(m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) s += __builtin_amdgcn_exp2f((f[u][k] - m0) * h.k);
  }
  const Sum rest = block_join<THREADS>(Sum{m, s}, h, lds);
  if (threadIdx.x >= 64) return;
  Sum list = {-INFINITY, 0.0};
  if (TAIL == BUCKET) {
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k)     // a listed NaN or inf makes the row NaN as any other does
      list.m = fmaxf(list.m, first >> k & 1 ? e[k].z : -INFINITY);
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k)
      if (first >> k & 1) list.s += power(e[k].z - from(list.m), h);
    list = wave_join(list, h);
  }
  if (SPLIT) {
    if (threadIdx.x == 0) {
      float* o = seg + (n * gridDim.y + blockIdx.y) * 4;
      o[0] = rest.m;
      o[1] = (float)rest.s;
      o[2] = list.m;
      o[3] = (float)list.s;
    }
  } else {
    finish_row<TAIL>(n, V, e, h, rest, list, loss, stats);
  }
}

template <typename TX, int TAIL>
__global__ __launch_bounds__(64) void k_distill_join(const TX* __restrict__ z, int64_t ldz, int V, Teacher h,
                                                     const float* __restrict__ seg, int segs, float* __restrict__ loss,
                                                     float* __restrict__ stats) {
  const int64_t n = blockIdx.x;
  Entry e[PER_LANE];
  entries_of(z + n * ldz, V, n, h, e);
  Sum rest = {-INFINITY, 0.0}, list = {-INFINITY, 0.0};
  for (int p = threadIdx.x; p < segs; p += 64) {
    const floatx4 o = *reinterpret_cast<const floatx4*>(seg + (n * segs + p) * 4);
    rest = join(rest, Sum{o[0], o[1]}, h);
    if (TAIL == BUCKET) list = join(list, Sum{o[2], o[3]}, h);
  }
  rest = wave_join(rest, h);
  if (TAIL == BUCKET) list = wave_join(list, h);
  finish_row<TAIL>(n, V, e, h, rest, list, loss, stats);
}

// The gradient: every column as if it were outside the list, then the listed ones of the workgroup's columns over
// them.  z and dz may be the same memory: a thread reads what it writes first, and listed logits before anything is written.
constexpr int THREADS = MAX_LIST, GRAD_COLS = 8 * THREADS * 4;

template <typename TX>
__global__ __launch_bounds__(THREADS) void k_distill_grad(const TX* z, int64_t ldz, int V, Teacher h,
                                                          const float* __restrict__ stats, const float* __restrict__ gl,
                                                          TX* dz, int64_t ldd) {
  typedef typename RqOperand<TX>::raw Raw;
  __shared__ int ids[MAX_LIST];
  __shared__ float ps[MAX_LIST];
  const int64_t n = blockIdx.x;
  const TX* row = z + n * ldz;
  TX* out = dz + n * ldd;
  const float* st = stats + n * STATS;
  const float m = st[0], ls = st[1], mr = st[2], lr = st[3], mt = st[4], lt = st[5], mass = st[6], factor = st[7];
  const bool none = mass == 0.0f;                  // nothing to learn from this row
  const float g = none ? 0.0f : gl[n] * (float)h.c;
  const float ls2 = lr * RQ_LOG2E, scale = g * factor;
  auto gradient = [&](float v) { return none ? 0.0f : __builtin_amdgcn_exp2f((v - mr) * h.k - ls2) * scale; };
  int id = -1;
  float zi = 0.0f;
  for (int c0 = blockIdx.y * GRAD_COLS; c0 < V; c0 += GRAD_COLS * gridDim.y) {
    const int at0 = c0 + 8 * (int)threadIdx.x;
    Raw r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at0 + 8 * THREADS * u + 8 <= V) r[u] = rq_load_x<true>(row + at0 + 8 * THREADS * u, 8);
    if (c0 == (int)blockIdx.y * GRAD_COLS && (int)threadIdx.x < h.K) {        // the list, while they are on their way
      const int64_t i = h.ids[n * h.K + threadIdx.x];
      id = i < 0 || i >= V ? -1 : (int)i;
      if (id >= 0) zi = rq_load_elem(row + id);
      ids[threadIdx.x] = id;
      ps[threadIdx.x] = expf((h.t[n * h.K + threadIdx.x] - mt) * (float)h.c - lt);
    }
    if (z == dz) __syncthreads();                  // listed logits are read before they are written over
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = at0 + 8 * THREADS * u;
      if (at + 8 <= V) {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = gradient((float)r[u][k]);
        rq_store8<TX>(out + at, o);
      } else {
        for (int i = at; i < V; ++i) out[i] = rq_cast<TX>(gradient(rq_load_elem(row + i)));
      }
    }
  }
  __syncthreads();
  if (id < 0 || id / GRAD_COLS % (int)gridDim.y != (int)blockIdx.y) return;
  float p = 0.0f;                                  // of all entries with this id
  for (int j = 0; j < h.K; ++j) p += ids[j] == id ? ps[j] : 0.0f;
  out[id] = rq_cast<TX>(none ? 0.0f : g * (__builtin_amdgcn_exp2f((zi - m) * h.k - ls * RQ_LOG2E) * mass - p));
}

// How a row is cut: into one workgroup where the rows alone fill the GPU, and where a large one reads it in the
// time that a second launch takes; fewer and longer rows over more.
constexpr int LARGE = 1024, ALONE = 1 << 16;
struct Cut {
  int segs, cols;
  bool large;
};
inline Cut cut_of(int64_t N, int V) {
  if (N < 512 && V <= ALONE) return Cut{1, (V + 31) / 32 * 32, V > 8 * THREADS};
  const int64_t fill = N >= 512 ? 1 : (1024 + N - 1) / N, most = ((int64_t)V + 4095) / 4096, least = ((int64_t)V + MAX_COLS - 1) / MAX_COLS;
  int64_t segs = fill < most ? fill : most;
  segs = segs > least ? segs : least;
  const int cols = (int)(((V + segs - 1) / segs + 31) / 32 * 32);
  return Cut{(V + cols - 1) / cols, cols, false};
}

inline bool bad_sizes(int64_t N, int V, int K, double temperature, int tail) {
  return N < 0 || V <= 0 || V > MAX_V || K <= 0 || K > MAX_LIST || !(temperature >= 1e-6 && temperature <= 1e6) ||
         (tail != RENORMALISE && (tail != BUCKET || temperature != 1.0));
}
inline Teacher teacher(const int64_t* ids, const float* t, int K, double temperature) {
  const double k = 1.4426950408889634 / temperature;
  return Teacher{ids, t, K, 1.0 / temperature, (float)k, (float)(k - (float)k)};
}
template <typename F>
inline bool with_tail(int dtype, int tail, F&& f) {
  return rq_with_dtype(dtype, [&](auto* p) {
    if (tail == BUCKET) f(p, std::integral_constant<int, BUCKET>{});
    else f(p, std::integral_constant<int, RENORMALISE>{});
  });
}

}  // namespace

extern "C" int64_t rq_distill_loss_workspace_bytes(int64_t N, int V) {
  if (N < 0 || V <= 0 || V > MAX_V) return RQ_EINVAL;
  if (N == 0) return 0;
  const Cut cut = cut_of(N, V);
  return cut.segs > 1 ? N * cut.segs * 16 : 0;
}

extern "C" int rq_distill_loss(const void* logits, int dtype, int64_t N, int64_t ldz, int V, const int64_t* teacher_ids,
                               const float* teacher_logprobs, int K, double temperature, int tail, float* loss,
                               float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
  if (bad_sizes(N, V, K, temperature, tail) || ldz < V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !teacher_ids || !teacher_logprobs || !loss || !stats) return RQ_EINVAL;
  const int64_t need = rq_distill_loss_workspace_bytes(N, V);
  if (need && (!workspace || workspace_bytes < need)) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Cut cut = cut_of(N, V);
  const bool known = with_tail(dtype, tail, [&](auto* ptr, auto of) {
    typedef typename std::remove_pointer<decltype(ptr)>::type TX;
    constexpr int TAIL = decltype(of)::value;
    const size_t lds = TAIL == BUCKET ? (size_t)cut.cols / 8 : 0;
    for (int64_t n = 0; n < N; n += RQ_ROWS_PER_LAUNCH) {
      const unsigned rows = (unsigned)(N - n < RQ_ROWS_PER_LAUNCH ? N - n : RQ_ROWS_PER_LAUNCH);
      const Teacher h = teacher(teacher_ids + n * K, teacher_logprobs + n * K, K, temperature);
      const TX* z = (const TX*)logits + n * ldz;
      float* seg = (float*)workspace + n * cut.segs * 4;
      auto rows_of = [&](auto split, auto threads) {
        hipLaunchKernelGGL((k_distill_rows<TX, TAIL, decltype(split)::value, decltype(threads)::value>), dim3(rows, cut.segs),
                           dim3(decltype(threads)::value), lds, s, z, ldz, V, cut.cols, h, loss + n, stats + n * STATS, seg);
      };
      if (cut.segs > 1) {
        rows_of(std::true_type{}, std::integral_constant<int, 256>{});
        hipLaunchKernelGGL((k_distill_join<TX, TAIL>), dim3(rows), dim3(64), 0, s, z, ldz, V, h, seg, cut.segs, loss + n,
                           stats + n * STATS);
      } else if (cut.large) {
        rows_of(std::false_type{}, std::integral_constant<int, LARGE>{});
      } else {
        rows_of(std::false_type{}, std::integral_constant<int, 256>{});
      }
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int rq_distill_loss_grad(const void* logits, int dtype, int64_t N, int64_t ldz, int V, const int64_t* teacher_ids,
                                    const float* teacher_logprobs, int K, double temperature, int tail, const float* stats,
                                    const float* grad_loss, void* grad_logits, int64_t ldd, void* stream) {
  if (bad_sizes(N, V, K, temperature, tail) || ldz < V || ldd < V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !teacher_ids || !teacher_logprobs || !stats || !grad_loss || !grad_logits) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int rounds = (V + GRAD_COLS - 1) / GRAD_COLS, ny = rounds < 64 ? rounds : 64;
  const bool known = rq_with_dtype(dtype, [&](auto* ptr) {
    typedef typename std::remove_pointer<decltype(ptr)>::type TX;
    for (int64_t n = 0; n < N; n += RQ_ROWS_PER_LAUNCH) {
      const unsigned rows = (unsigned)(N - n < RQ_ROWS_PER_LAUNCH ? N - n : RQ_ROWS_PER_LAUNCH);
      hipLaunchKernelGGL(k_distill_grad<TX>, dim3(rows, ny), dim3(THREADS), 0, s, (const TX*)logits + n * ldz,
                         ldz, V, teacher(teacher_ids + n * K, teacher_logprobs + n * K, K, temperature), stats + n * STATS,
                         grad_loss + n, (TX*)grad_logits + n * ldd, ldd);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
