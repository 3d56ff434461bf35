// Log probabilities of given tokens, the entropy and the top alternatives of every row of logits, and the
// gradient of the logits.
//
// With m = max z, d_i = z_i - m, s = sum_i exp(d_i):
//   logprob = d_target - log s        H = log s - (sum_i exp(d_i) d_i) / s        p_i = exp(d_i - log s)
//   dz_i = gl (delta_{i,target} - p_i) - gh p_i (log p_i + H)
// Differences from m are formed first, so masks of the type's lowest value cost no precision; a term
// with exp(d_i) = 0 is 0 whatever d_i is (-inf among them).  A row with nothing but -inf (m = -inf, s = 0) has
// logprob -inf, H = 0 and no gradient.  A NaN or +inf logit makes its row NaN.
// All statistics are fp32.  Equal values are ordered by their index, NaN above everything.
//
// Forward, one pass over the logits.  A wave runs over a segment of a row, 8 logits a lane and load.  Each
// lane keeps its own running maximum m, sum s and sum a of exp(d) d in units of log 2 (when m grows by D:
// s f and f (a - D s), f = exp(-D)).  The maximum passes NaNs over; they reach the sums.
// The alternatives cost the pass nothing but the maxima: the top_k-th largest of the lanes' maxima is a bar
// that at least top_k logits reach and, the lanes being many more than top_k, few others.  Each lane also
// leaves a maximum for every block of its loads, and the few blocks that reach the bar are read again (from
// the caches) for the logits that do.  2048 rows of 128256 bf16 with 5 alternatives take 129 us, 525 MB read: 4.1 TB/s,
// where a copy of that size reaches 5.0 (read and written).
// A row's segments are joined by one wave: in the workgroup that has the whole row, or by k_logprob_join
// where a row is cut over many workgroups.
#include "logits.h"

namespace {

constexpr int MAX_TOP = 64, MAX_V = 1 << 30;
constexpr int LIST = 320;                  // candidates a wave holds
constexpr float LN2 = 0.6931471805599453f;
constexpr float LOW = -200.0f;             // 2^LOW is 0 in fp32: stands for any lower exponent where it is a factor
__device__ __forceinline__ uint64_t top_key(float z, int i) {
  return ((uint64_t)rq_order_key(z) << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// LDS of one wave is written and read by that wave alone: its accesses are issued in order, so only the
// compiler has to be kept from moving them.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// How many of the first n lanes hold a larger key.
__device__ __forceinline__ int lane_rank(uint64_t key, int n) {
  int place = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) place += lane_value(key, j) > key ? 1 : 0;
  return place;
}

// A value that at least k <= 64 of the lanes' reach, the k-th largest or what is left of it when no more do.
__device__ __forceinline__ uint32_t kth_largest(uint32_t mine, int k) {
  uint32_t least = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t tried = least | (1u << bit);
    const int reach = __popcll(__ballot(mine >= tried));
    if (reach >= k) least = tried;
    if (reach == k) break;
  }
  return least;
}

struct Stat {
  float m, s, a;
};
// Two parts of a row as one.  An empty part has m = -inf, s = a = 0.
__device__ __forceinline__ Stat join(Stat x, Stat y) {
  const float m = fmaxf(x.m, y.m);
  if (m == -INFINITY) return Stat{m, x.s + y.s, x.a + y.a};
  const float dx = (x.m - m) * RQ_LOG2E, dy = (y.m - m) * RQ_LOG2E;            // <= 0, -inf for an empty part
  const float fx = __builtin_amdgcn_exp2f(dx), fy = __builtin_amdgcn_exp2f(dy);
  Stat r;
  r.m = m;
  r.s = fx * x.s + fy * y.s;
  r.a = fx * (x.a + fmaxf(dx, LOW) * x.s) + fy * (y.a + fmaxf(dy, LOW) * y.s);
  return r;
}
__device__ __forceinline__ Stat wave_join(Stat v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = join(v, Stat{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.a, o)});
  return v;
}

// The k <= 64 largest of n <= LIST distinct keys of a wave's list, in order, to its front; the places
// past n get 0.  Over 64 keys are first cut to k: the k-th largest is found bit by bit from the number of
// keys that reach a value.  ids: every key's index is below it (the bits above are ones in every key).
__device__ __forceinline__ void keep_top(uint64_t* list, int n, int k, int ids) {
  const int lane = threadIdx.x & 63;
  if (n > 64) {
    uint64_t mine[LIST / 64];
#pragma unroll
    for (int u = 0; u < LIST / 64; ++u) mine[u] = lane + 64 * u < n ? list[lane + 64 * u] : 0;
    const int used = (n + 63) / 64;
    const int low = 32 - __builtin_clz(ids);
    uint64_t least = (uint64_t)(uint32_t)~((1u << low) - 1u);
    for (int bit = 63; bit >= 0; --bit) {
      if (bit < 32 && bit >= low) continue;
      const uint64_t tried = least | (1ull << bit);
      int reach = 0;
#pragma unroll
      for (int u = 0; u < LIST / 64; ++u)
        if (u < used) reach += __popcll(__ballot(mine[u] >= tried));
      if (reach >= k) least = tried;
      if (reach == k) break;
    }
    wave_fence();
    int at = 0;
#pragma unroll
    for (int u = 0; u < LIST / 64; ++u) {
      if (u < used) {
        const bool stays = mine[u] >= least;
        const uint64_t mask = __ballot(stays);
        if (stays) list[at + lanes_before(mask)] = mine[u];
        at += __popcll(mask);
      }
    }
    wave_fence();
    n = k;
  }
  const uint64_t mine = lane < n ? list[lane] : 0;
  const int place = lane_rank(mine, n);
  wave_fence();
  if (lane < n && place < k) list[place] = mine;
  if (lane >= n && lane < k) list[lane] = 0;
  wave_fence();
}

// Joins the parts of one row (their statistics, and their k best each) and writes its results; one wave.
// list: LIST keys of LDS.
template <typename TX, typename Parts>
__device__ __forceinline__ void finish_row(const TX* __restrict__ row, int V, int64_t n, int nparts, const Parts& parts,
                                           uint64_t* list, int64_t target, int64_t ignore, int top,
                                           float* __restrict__ logprob, float* __restrict__ entropy,
                                           int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
                                           float* __restrict__ stats) {
  const int lane = threadIdx.x & 63;
  Stat v = {-INFINITY, 0.0f, 0.0f};
  for (int p = lane; p < nparts; p += 64) v = join(v, parts.stat(p));
  v = wave_join(v);
  const bool empty = v.m == -INFINITY && v.s == 0.0f;      // the maximum passes NaNs over, the sum does not
  const float ls = empty ? 0.0f : logf(v.s);
  const float H = empty ? 0.0f : ls - LN2 * (v.a / v.s);
  if (lane == 0) {
    float lp = 0.0f;
    if (target != ignore) {
      if (target < 0 || target >= V) lp = __builtin_nanf("");
      else lp = empty ? -INFINITY : (rq_load_elem(row + target) - v.m) - ls;
    }
    logprob[n] = lp;
    entropy[n] = H;
    stats[3 * n] = v.m;
    stats[3 * n + 1] = ls;
    stats[3 * n + 2] = H;
  }
  if (!top) return;
  // A value is among the top only if it reaches the top-th largest of the parts' best values.
  uint64_t floor_key = 0;
  if (nparts > 8) {
    uint64_t best = 0;
    for (int p = lane; p < nparts; p += 64) {
      const uint64_t o = parts.key(p, 0);
      best = o > best ? o : best;
    }
    const uint32_t least = kth_largest((uint32_t)(best >> 32), top);
    floor_key = (uint64_t)least << 32;
    // Where more of them are equal the exact key is found, or every part's list would pass.
    if (__popcll(__ballot((uint32_t)(best >> 32) >= least)) > top) {
      const uint64_t is = __ballot(lane_rank(best, 64) == top - 1 && best != 0);
      if (is) floor_key = lane_value(best, __ffsll((unsigned long long)is) - 1);
    }
  }
  int count = 0;
  for (int p0 = 0; p0 < nparts; p0 += 64) {
    constexpr int AHEAD = 4;
    uint64_t next[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) next[u] = p0 + lane < nparts && u < top ? parts.key(p0 + lane, u) : 0;
    for (int k = 0; k < top; ++k) {
      const uint64_t key = next[0];
#pragma unroll
      for (int u = 0; u + 1 < AHEAD; ++u) next[u] = next[u + 1];
      next[AHEAD - 1] = p0 + lane < nparts && k + AHEAD < top ? parts.key(p0 + lane, k + AHEAD) : 0;
      const bool take = key != 0 && key >= floor_key;
      const uint64_t mask = __ballot(take);
      if (!mask) break;                              // the parts' lists are in order
      if (take) list[count + lanes_before(mask)] = key;
      count += __popcll(mask);
      wave_fence();
      if (count > LIST - 64) {
        keep_top(list, count, top, V);
        count = top;
        const uint64_t last = list[top - 1];
        floor_key = last > floor_key ? last : floor_key;
      }
    }
  }
  keep_top(list, count, top, V);
  if (lane < top) {
    const uint64_t key = list[lane];
    const int i = (int)(0xFFFFFFFFu - (uint32_t)key);
    top_ids[n * top + lane] = i;
    top_lp[n * top + lane] = empty ? -INFINITY : (rq_key_value((uint32_t)(key >> 32)) - v.m) - ls;
  }
}

// The next float above v (inf for inf and NaN).
__device__ __forceinline__ float above(float v) {
  if (!(v < INFINITY)) return INFINITY;
  const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
  return __uint_as_float((b & 0x80000000u) ? b - 1 : b + 1);
}

// A wave's segment [c0, c1) of a row, in rounds of U loads of 512 columns, blocks of `rounds` rounds each.
template <typename TX>
struct Scan {
  static constexpr int U = sizeof(TX) == 2 ? 8 : 4, ROUND = 512 * U;
  const TX* row;
  int c0, c1, rounds;
};
constexpr int W = 4, BLOCKS = 8;           // waves of a workgroup; blocks at most for which a wave leaves maxima

// The lane's statistics of the segment; most: its maxima of the blocks, 64 floats a block.
template <typename TX>
__device__ __forceinline__ Stat scan_segment(const Scan<TX>& sc, float* most) {
  typedef typename RqOperand<TX>::raw Raw;
  constexpr int U = Scan<TX>::U;
  const int lane = threadIdx.x & 63, c1 = sc.c1;
  Raw in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) in[u] = rq_load8<TX>(sc.row, sc.c0 + 512 * u + 8 * lane, c1);
  Stat v = {-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < 8; ++k) v.m = fmaxf(v.m, (float)in[u][k]);
  // Exponents are f log2e - shift with shift = fl(m log2e), one fma: the sums are off by the factor
  // 2^(m log2e - shift), which is taken out at the end.  It is within 2^(+-1/16) up to |shift| = WIDE; beyond (wide: masks
  // of a large negative number in everything so far, the type's lowest value among them, or +inf) exponents are
  // (f - m) log2e.
  constexpr float WIDE = 0x1p20f;
  auto is_wide = [](float at) { return __builtin_fabsf(at) > WIDE; };
  float shift = v.m == -INFINITY ? 0.0f : v.m * RQ_LOG2E;
  float block = -INFINITY;
  int round = 0;
  for (int c = sc.c0; c < c1; c += 512 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cu = c + 512 * u;
      if (cu >= c1) break;
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = (float)in[u][k];
      in[u] = rq_load8<TX>(sc.row, cu + 512 * U + 8 * lane, c1);
      float big = f[0];
#pragma unroll
      for (int k = 1; k < 8; ++k) big = fmaxf(big, f[k]);
      block = fmaxf(block, big);
      if (big > v.m) {                     // the maximum grows
        const float grown = big * RQ_LOG2E;
        // far: from what the sums' exponents were taken from to what they are taken from now.  One of them is wide only
        // if -shift or grown is (a lane without a maximum so far has shift 0 and sums of 0).
        float far = shift - grown;
        if (__any(__builtin_fmaxf(-shift, grown) > WIDE)) {
          if (is_wide(shift)) far = is_wide(grown) ? (v.m - big) * RQ_LOG2E : __builtin_fmaf(v.m, RQ_LOG2E, -grown);
          else if (is_wide(grown)) far = __builtin_fmaf(-big, RQ_LOG2E, shift);
        }
        const float D = __builtin_amdgcn_fmed3f(far, LOW, 1.0f);
        const float scale = v.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(D);
        v.a = scale * (v.a + D * v.s);
        v.s *= scale;
        v.m = big;
        shift = grown;
      }
      auto add = [&](float x) {
        const float e = __builtin_amdgcn_exp2f(x);
        v.s += e;
        v.a = __builtin_fmaf(e, __builtin_amdgcn_fmed3f(x, LOW, 1.0f), v.a);
      };
      if (__any(is_wide(shift))) {
#pragma unroll
        for (int k = 0; k < 8; ++k) add(is_wide(shift) ? (f[k] - v.m) * RQ_LOG2E : __builtin_fmaf(f[k], RQ_LOG2E, -shift));
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) add(__builtin_fmaf(f[k], RQ_LOG2E, -shift));
      }
    }
    if (++round % sc.rounds == 0 || c + 512 * U >= c1) {
      most[(round - 1) / sc.rounds * 64 + lane] = block;
      block = -INFINITY;
    }
  }
  const float off = v.m == -INFINITY || is_wide(shift) ? 0.0f : __builtin_fmaf(v.m, RQ_LOG2E, -shift);
  const float back = __builtin_amdgcn_exp2f(-off);
  v.a = back * (v.a - off * v.s);
  v.s *= back;
  return v;
}

// A float that at least k <= 64 of the workgroup's logits reach: the k-th largest of 64 maxima, each over one
// lane of every wave (order keys).  About 64 ln(64 / (64 - k)) logits reach it: 5 for k = 5, 24 for 20, 300
// for 64.  (The k-th largest of all lanes' maxima lets fewer pass, and took 5 us
// longer to find.)
__device__ __forceinline__ float bar_of(const uint32_t* keys, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t mine = keys[lane];
#pragma unroll
  for (int u = 1; u < W; ++u) mine = max(mine, keys[64 * u + lane]);
  const uint32_t least = kth_largest(mine, k);
  return rq_key_value(min(max(least, 0x007FFFFFu), 0xFF800000u));       // from -inf to inf, which NaNs reach too
}

// The segment's logits that reach the bar, the top of them in order to the front of list (0 where there are
// fewer).  nan: the lane may hold a NaN or inf, which its maxima do not show.
template <typename TX>
__device__ __forceinline__ void collect(const Scan<TX>& sc, const float* most, bool nan, float bar, int top, uint64_t* list) {
  typedef typename RqOperand<TX>::raw Raw;
  constexpr int U = Scan<TX>::U;
  const int lane = threadIdx.x & 63, c1 = sc.c1, width = Scan<TX>::ROUND * sc.rounds;
  int count = 0;
  bool strict = false;       // the bar has been moved up by a bit: values equal to what it was come too late
  for (int c = sc.c0, b = 0; c < c1; c += width, ++b) {
    if (!__any(!(most[b * 64 + lane] < bar) || nan)) continue;
    const int end = (int)min((int64_t)c1, (int64_t)c + width);
    for (int cr = c; cr < end; cr += 512 * U) {
      Raw in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = rq_load8<TX>(sc.row, cr + 512 * u + 8 * lane, c1);
      uint32_t passed = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        bool any = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) any = any || !((float)in[u][k] < bar);
        if (__any(any && cr + 512 * u + 8 * lane < c1)) passed |= 1u << u;
      }
      for (; passed; passed &= passed - 1) {
        const int u0 = __ffs(passed) - 1, at = cr + 512 * u0 + 8 * lane;
        Raw x = in[0];
#pragma unroll
        for (int u = 1; u < U; ++u)
          if (u == u0) x = in[u];
        float f[8];
        uint32_t takes = 0, equals = 0;              // of the lane's eight
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          f[k] = (float)x[k];
          takes |= at + k < c1 && !(f[k] < bar) ? 1u << k : 0u;
          equals |= f[k] == bar ? 1u << k : 0u;
        }
        equals &= takes;
        if (__any(equals != 0)) {
          // Of the values equal to the bar the first top suffice (a lane's eight lie before the next lane's).
          int before = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) before += lanes_before(__ballot(equals >> k & 1));
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (equals >> k & 1)
              if (before++ >= top) takes &= ~(1u << k);
        }
        // One of each lane at a time: mostly one is all.
        while (__any(takes != 0)) {
          if (count > LIST - 64) {
            keep_top(list, count, top, c1);
            count = top;
            const float last = rq_key_value((uint32_t)(list[top - 1] >> 32));
            if (last > bar) {
              bar = last;
              strict = false;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (f[k] < bar) takes &= ~(1u << k);
            }
          }
          const bool take = takes != 0;
          const int k0 = __ffs(takes) - 1;
          float v = f[0];
#pragma unroll
          for (int k = 1; k < 8; ++k) v = k == k0 ? f[k] : v;
          const uint64_t mask = __ballot(take);
          if (take) list[count + lanes_before(mask)] = top_key(v, at + k0);
          count += __popcll(mask);
          takes &= takes - 1;                        // 0 stays 0
          wave_fence();
        }
        // top values that reach the bar are held: equal ones of later loads come after them
        if (count >= top && !strict) {
          bar = above(bar);
          strict = true;
        }
      }
    }
  }
  keep_top(list, count, top, c1);
}

struct LdsParts {
  const Stat* st;
  const uint64_t* lists;
  __device__ Stat stat(int p) const { return st[p]; }
  __device__ uint64_t key(int p, int k) const { return lists[p * LIST + k]; }
};
struct MemParts {
  const float* st;
  const uint64_t* keys;
  int top;
  __device__ Stat stat(int p) const { return Stat{st[3 * p], st[3 * p + 1], st[3 * p + 2]}; }
  __device__ uint64_t key(int p, int k) const { return keys[(int64_t)p * top + k]; }
};

// W waves to a workgroup, a segment of row blockIdx.x each.  SPLIT: segment W blockIdx.y + wave, its results go
// to the workspace; else the W segments are the row and the first wave finishes it.
template <typename TX, bool SPLIT>
__global__ __launch_bounds__(64 * W, sizeof(TX) == 2 ? 5 : 4) void k_logprob_rows(
    const TX* __restrict__ z, int64_t ldz, int V, int segs, int seg_cols, const int64_t* __restrict__ targets,
    int64_t ignore, int top, float* __restrict__ logprob, float* __restrict__ entropy, int64_t* __restrict__ top_ids,
    float* __restrict__ top_lp, float* __restrict__ stats, float* __restrict__ seg_stats, uint64_t* __restrict__ seg_keys) {
  __shared__ uint64_t lists[(SPLIT ? W : W + 1) * LIST];
  __shared__ float most[W * BLOCKS * 64];
  __shared__ uint32_t maxima[W * 64];
  __shared__ Stat st[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = blockIdx.x;
  const int seg = SPLIT ? blockIdx.y * W + wave : wave;
  const int c0 = (int)min((int64_t)V, (int64_t)seg * seg_cols);
  const int per = (seg_cols + Scan<TX>::ROUND - 1) / Scan<TX>::ROUND;
  const Scan<TX> sc{z + n * ldz, c0, min(V, c0 + seg_cols), (per + BLOCKS - 1) / BLOCKS};
  uint64_t* list = lists + wave * LIST;
  const Stat mine = scan_segment<TX>(sc, most + wave * BLOCKS * 64);
  const Stat v = wave_join(mine);
  if (!SPLIT && lane == 0) st[wave] = v;
  if (top) {
    const bool nan = mine.s != mine.s;
    maxima[threadIdx.x] = nan ? 0xFFFFFFFFu : rq_order_key(mine.m);
    __syncthreads();
    collect<TX>(sc, most + wave * BLOCKS * 64, nan, bar_of(maxima, top), top, list);
  }
  if constexpr (SPLIT) {
    if (lane == 0) {
      float* o = seg_stats + (n * segs + seg) * 3;
      o[0] = v.m;
      o[1] = v.s;
      o[2] = v.a;
    }
    if (lane < top) seg_keys[(n * segs + seg) * top + lane] = list[lane];
  } else {
    __syncthreads();
    if (wave == 0)
      finish_row<TX>(sc.row, V, n, W, LdsParts{st, lists}, lists + W * LIST, targets[n], ignore, top, logprob, entropy,
                     top_ids, top_lp, stats);
  }
}

template <typename TX>
__global__ __launch_bounds__(64) void k_logprob_join(const TX* __restrict__ z, int64_t ldz, int V, int segs,
                                                     const int64_t* __restrict__ targets, int64_t ignore, int top,
                                                     float* __restrict__ logprob, float* __restrict__ entropy,
                                                     int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
                                                     float* __restrict__ stats, const float* __restrict__ seg_stats,
                                                     const uint64_t* __restrict__ seg_keys) {
  __shared__ uint64_t list[LIST];
  const int64_t n = blockIdx.x;
  finish_row<TX>(z + n * ldz, V, n, segs, MemParts{seg_stats + n * segs * 3, seg_keys + n * segs * top, top}, list, targets[n],
                 ignore, top, logprob, entropy, top_ids, top_lp, stats);
}

// How a row is cut: into one workgroup's 4 segments where the rows alone fill the GPU or are short; fewer rows
// over more workgroups, down to 2048 columns a wave, and a second launch joins them (one row of 128256 bf16,
// 20 alternatives: 11.5 + 6.6 us, a chain of latencies; one workgroup of 16 waves took 30).
struct Split {
  int segs, cols;
};
inline Split split_of(int64_t N, int V) {
  const int64_t fill = N >= 512 ? W : (2048 + N - 1) / N, most = (V + 2047) / 2048;
  const int64_t segs = ((fill < most ? fill : most) + W - 1) / W * W;
  return Split{(int)segs, (int)(((V + segs - 1) / segs + 7) / 8 * 8)};
}

// --- the gradient ---------------------------------------------------------------------------
// A workgroup takes rounds of 8192 columns of a row, 4 x 8 a thread: read once, written once.  z and dz may
// be the same memory (a thread reads what it writes first).  1024 rows of 128256 bf16: 108 us for 525 MB,
// 4.9 TB/s, a copy's rate; 12 rows of 32003 fp32 4.8 us, a launch.
constexpr int GRAD_COLS = 8192;

template <typename TX>
__global__ __launch_bounds__(256) void k_logprob_grad(const TX* z, int64_t ldz, int V,
                                                      const int64_t* __restrict__ targets, int64_t ignore,
                                                      const float* __restrict__ stats, const float* __restrict__ gl_,
                                                      const float* __restrict__ gh_, TX* dz, int64_t ldd) {
  typedef typename RqOperand<TX>::raw Raw;
  const int64_t n = blockIdx.x;
  const int64_t t = targets[n];
  const float m = stats[3 * n], ls = stats[3 * n + 1], H = stats[3 * n + 2];
  const bool empty = m == -INFINITY && ls == 0.0f;
  float gl = t == ignore ? 0.0f : gl_[n];
  if (t != ignore && (t < 0 || t >= V)) gl = __builtin_nanf("");
  const float gh = gh_ ? gh_[n] : 0.0f;
  const float c = gl + gh * H;
  const TX* row = z + n * ldz;
  TX* out = dz + n * ldd;
  // -p (gl + gh (log p + H)); 0 where p is 0
  auto gradient = [&](float v, int i) {
    const float lp = (v - m) - ls;
    const float p = __builtin_amdgcn_exp2f(lp * RQ_LOG2E);
    float g = -p * __builtin_fmaf(gh, fmaxf(lp, LOW), c);
    if (i == t) g += gl;
    return empty ? 0.0f : g;
  };
  for (int c0 = blockIdx.y * GRAD_COLS; c0 < V; c0 += GRAD_COLS * gridDim.y) {
    const int at0 = c0 + 8 * (int)threadIdx.x;
    Raw r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at0 + 2048 * u + 8 <= V) r[u] = rq_load_x<true>(row + at0 + 2048 * u, 8);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = at0 + 2048 * u;
      if (at + 8 <= V) {
        float g[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = gradient((float)r[u][k], at + k);
        rq_store8<TX>(out + at, g);
      } else {
        for (int i = at; i < V; ++i) out[i] = rq_cast<TX>(gradient(rq_load_elem(row + i), i));
      }
    }
  }
}

}  // namespace

extern "C" int64_t rq_token_logprobs_workspace_bytes(int64_t N, int V, int top_k) {
  if (N < 0 || V <= 0 || V > MAX_V || top_k < 0 || top_k > MAX_TOP || top_k > V) return RQ_EINVAL;
  if (N == 0) return 0;
  const Split sp = split_of(N, V);
  return sp.segs > W ? N * sp.segs * (top_k * 8 + 12) : 0;
}

extern "C" int rq_token_logprobs(const void* logits, int dtype, int64_t N, int64_t ldz, int V, const int64_t* targets,
                                 int64_t ignore_index, int top_k, float* logprob, float* entropy, int64_t* top_ids,
                                 float* top_logprobs, float* stats, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  const int64_t need = rq_token_logprobs_workspace_bytes(N, V, top_k);
  if (need < 0 || ldz < V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !targets || !logprob || !entropy || !stats || (top_k && (!top_ids || !top_logprobs))) return RQ_EINVAL;
  if (need && (!workspace || workspace_bytes < need)) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Split sp = split_of(N, V);
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    if (sp.segs > W) {                               // N < 512
      uint64_t* keys = (uint64_t*)workspace;
      float* st = (float*)(keys + N * sp.segs * top_k);
      hipLaunchKernelGGL((k_logprob_rows<TX, true>), dim3((unsigned)N, sp.segs / W), dim3(64 * W), 0, s, (const TX*)logits,
                         ldz, V, sp.segs, sp.cols, targets, ignore_index, top_k, logprob, entropy, top_ids, top_logprobs,
                         stats, st, keys);
      hipLaunchKernelGGL(k_logprob_join<TX>, dim3((unsigned)N), dim3(64), 0, s, (const TX*)logits, ldz, V, sp.segs, targets,
                         ignore_index, top_k, logprob, entropy, top_ids, top_logprobs, stats, st, keys);
      return;
    }
    for (int64_t n = 0; n < N; n += RQ_ROWS_PER_LAUNCH) {
      const int64_t rows = N - n < RQ_ROWS_PER_LAUNCH ? N - n : RQ_ROWS_PER_LAUNCH;
      hipLaunchKernelGGL((k_logprob_rows<TX, false>), dim3((unsigned)rows), dim3(64 * W), 0, s, (const TX*)logits + n * ldz,
                         ldz, V, sp.segs, sp.cols, targets + n, ignore_index, top_k, logprob + n, entropy + n,
                         top_ids + n * top_k, top_logprobs + n * top_k, stats + 3 * n, nullptr, nullptr);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}

extern "C" int rq_token_logprobs_grad(const void* logits, int dtype, int64_t N, int64_t ldz, int V,
                                      const int64_t* targets, int64_t ignore_index, const float* stats,
                                      const float* grad_logprob, const float* grad_entropy, void* grad_logits,
                                      int64_t ldd, void* stream) {
  if (N < 0 || V <= 0 || V > MAX_V || ldz < V || ldd < V) return RQ_EINVAL;
  if (N == 0) return RQ_OK;
  if (!logits || !targets || !stats || !grad_logprob || !grad_logits) return RQ_EINVAL;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int rounds = (V + GRAD_COLS - 1) / GRAD_COLS, ny = rounds < 64 ? rounds : 64;
  const bool known = rq_with_dtype(dtype, [&](auto* p) {
    typedef typename std::remove_pointer<decltype(p)>::type TX;
    for (int64_t n = 0; n < N; n += RQ_ROWS_PER_LAUNCH) {
      const int64_t rows = N - n < RQ_ROWS_PER_LAUNCH ? N - n : RQ_ROWS_PER_LAUNCH;
      hipLaunchKernelGGL(k_logprob_grad<TX>, dim3((unsigned)rows, ny), dim3(256), 0, s, (const TX*)logits + n * ldz, ldz, V,
                         targets + n, ignore_index, stats + 3 * n, grad_logprob + n, grad_entropy ? grad_entropy + n : nullptr,
                         (TX*)grad_logits + n * ldd, ldd);
    }
  });
  if (!known) return RQ_EINVAL;
  RQ_CHECK_LAUNCH();
  return RQ_OK;
}
