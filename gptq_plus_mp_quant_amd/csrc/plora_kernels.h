// The products with low-rank adapters, for one element type.
//
// Bound, for few tokens, by the packed weight's bytes and by latency: what the adapters add is a few operations and a
// launch.  Hence their products ride in the packed weight's launches, and what precedes them is one short launch (or
// none).  Measured, 4-bit bf16: 48 tokens of 16 adapters of rank 32, 14336 x 4096, 5.8 + 28.2 us; one token, 4096 x 4096, rank 16,
// 13.5 us; gradients of 128 tokens, 4096 x 14336, rank 64, 65.8 + 19.8 us, 7 tokens of 1026 x 1365 along an order 11.0 + 6.5.
//
// A tile is 16 tokens, as with the packed weight, and goes once over every adapter that one of them has: the matrix
// cores' columns are tokens, so what another adapter makes of a token is dropped, not added as 0 (an adapter that holds an
// inf or NaN spoils its own tokens only).
#pragma once
#include "plora_down.h"
#include "plinear_rows.h"

namespace {

constexpr int ARRANGED_CHUNKS = 16, DOWN_WAVES = 16;
// Both jobs, and behind them chunks of the first's x to be arranged.
template <typename TX>
__global__ __launch_bounds__(64 * DOWN_WAVES) void k_lora_down(RqDownJobs<TX> jobs, RqArrange arrange) {
  __shared__ floatx4 join[DOWN_WAVES * 64];
  if ((int)blockIdx.z >= jobs.z) {
    const RqDown<TX>& d = jobs.first;
    const int ch = (blockIdx.z - jobs.z) * ARRANGED_CHUNKS, chunks = (d.cols + RQ_CHUNK - 1) / RQ_CHUNK;
    if (blockIdx.y == 0)
      rq_arrange<TX>(d.x, d.low.T, d.ldx, d.cols, blockIdx.x, ch, min(ch + ARRANGED_CHUNKS, chunks), arrange.paired, threadIdx.x,
                     blockDim.x, arrange.out);
    return;
  }
  rq_lora_down_job<TX, DOWN_WAVES>(jobs, blockIdx.x, blockIdx.y, blockIdx.z, join);
}

// Eight ranks of a token, its parts joined in their order.
__device__ __forceinline__ floatx8 low8(const RqLow& low, int64_t t, int rank) {
  floatx8 v = rq_load_as<floatx8>(low.u + low.at(0, t) + rank);
#pragma unroll 2
  for (int p = 1; p < low.parts; ++p) v += rq_load_as<floatx8>(low.u + low.at(p, t) + rank);
  return v;
}

// The adapter's side of s B u as bf16 pieces, exactly: bf16 as it is, fp16's 11 bits in two, fp32 in three.
template <typename TX> struct LoraPieces;
template <> struct LoraPieces<__hip_bfloat16> { static constexpr int n = 1; };
template <> struct LoraPieces<__half> { static constexpr int n = 2; };
template <> struct LoraPieces<float> { static constexpr int n = 3; };
__device__ __forceinline__ bf16x8 without_inf(bf16x8 v) {
  bf16x8 o;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float f = (float)v[k];
    o[k] = __builtin_fabsf(f) == INFINITY ? (__bf16)0.0f : v[k];
  }
  return o;
}

// s B u to the sums of a row tile: 32 ranks of an adapter at a time, dealt to the waves by adapter and rank alone, so that
// a token's bits do not depend on its companions.  u goes in as three bf16 pieces (24 bits), B in as many as hold it; products of
// pieces i and j with i + j > 2, at most 2^-22 of a term, are left out.  An inf's product with a piece of 0 would be a
// NaN that the formula does not have: past a number's first piece the other side's infs are 0.  Of the 28.2 us
// above they take 10 (18.0 with no adapter for any token); as fp32 matrix instructions they took nearly twice as long.
template <typename TX>
struct RqLowRank {
  static constexpr bool arranged = true, whole = true;
  static constexpr int staged_groups = RQ_STAGED_GROUPS - 16;      // u lies behind the scales, in 64 KB
  RqLora<TX> lora;
  RqLow low;
  const void* arranged_x;
  bool own;                 // no launch made u: each workgroup makes it for itself, in LDS from float own_at on
  int own_at;
  size_t own_lds(size_t lds) {
    own_at = (int)(lds / 4);
    return own ? lds + (size_t)low.T * low.ranks * 4 : lds;
  }
  // u of at most 16 tokens: the waves take steps of 32 columns in turn, eight in flight, and are joined in their order.
  __device__ __forceinline__ void prepare(const TX* __restrict__ x, int T, int64_t ldx, int C, int wave, int waves, float* lds) const {
    typedef typename RqOperand<TX>::raw Raw;
    if (!own) return;
    floatx4* join = reinterpret_cast<floatx4*>(lds);
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int mine = i < T ? lora.of(i) : -1;
    for (uint64_t pending = __ballot(lane < 16 && mine >= 0 && mine < lora.n); pending;) {
      const int lead = __ffsll((unsigned long long)pending) - 1, a = __builtin_amdgcn_readlane(mine, lead);
      pending &= ~__ballot(mine == a);
      const TX* xs = x + (int64_t)(mine == a ? i : lead) * ldx;
      for (int rank = 0; rank < low.ranks; rank += 16) {
        const TX* as = lora.a + ((int64_t)a * lora.r + min(rank + i, lora.r - 1)) * C;
        floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        int c = 32 * wave;
        if (rank < lora.r) {
          for (; c + 32 * (7 * waves + 1) <= C; c += 32 * 8 * waves) {
            Raw xv[8], av[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              xv[k] = rq_load_x<true>(xs + c + 32 * k * waves + 8 * q, 8);
              av[k] = rq_load_x<true>(as + c + 32 * k * waves + 8 * q, 8);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) acc = rq_mfma32(av[k], xv[k], acc);
          }
          for (; c + 32 <= C; c += 32 * waves)
            acc = rq_mfma32(rq_load_x<true>(as + c + 8 * q, 8), rq_load_x<true>(xs + c + 8 * q, 8), acc);
          if (c < C) {
            const int n = C - c - 8 * q;             // the lane's columns (may be none)
            acc = rq_mfma32(rq_load_x<false>(as + c + 8 * q, n), rq_load_x<false>(xs + c + 8 * q, n), acc);
          }
        }
        join[wave * 64 + lane] = acc;
        __syncthreads();
        if (wave == 0) {
          for (int w = 1; w < waves; ++w) acc += join[w * 64 + lane];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (rank + 4 * q + k >= lora.r) acc[k] = 0.0f;
          if (mine == a) *reinterpret_cast<floatx4*>(lds + own_at + i * low.ranks + rank + 4 * q) = acc;
        }
        __syncthreads();
      }
    }
  }
  template <int RT, int NT>
  __device__ __forceinline__ void add(int r0, int R, int t0, int T, int wave, int waves, const float* lds,
                                      floatx4 (&acc)[RT][NT]) const {
    constexpr int PW = LoraPieces<TX>::n;
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int mine = lane < 16 * NT && t0 + lane < T ? lora.of(t0 + lane) : -1;
    int whose[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) whose[b] = __shfl(mine, 16 * b + i);
    for (uint64_t pending = __ballot(mine >= 0 && mine < lora.n); pending;) {
      const int a = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)pending) - 1);
      const uint64_t who = __ballot(mine == a);
      pending &= ~who;
      int turn = wave - a % waves;                   // the first of its rank tiles that this wave takes
      turn = turn < 0 ? turn + waves : turn;
      if (32 * turn >= lora.r) continue;
      const float s = lora.scale_of(a);
      for (int k0 = 32 * turn; k0 < lora.r; k0 += 32 * waves) {
        const int k = k0 + 8 * q;
        bf16x8 w[RT][PW], first[RT];
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          const TX* p = lora.b + ((int64_t)a * R + min(rq_tile_row<true>(r0 + 16 * m, R) + i, R - 1)) * lora.r + k;
          const typename RqOperand<TX>::raw e = k + 8 <= lora.r ? rq_load_x<true>(p, 8) : rq_load_x<false>(p, lora.r - k);
          if constexpr (PW == 1) {
            w[m][0] = e;
          } else {
            floatx8 f;
            rq_floats(e, f);
            rq_operand<PW>(f, w[m]);
          }
          first[m] = without_inf(w[m][0]);
        }
#pragma unroll
        for (int b = 0; b < NT; ++b) {
          if (!(who >> (16 * b) & 0xFFFF)) continue;
          bf16x8 u[3];
          const int t = min(t0 + 16 * b + i, T - 1);
          floatx8 f;
          if (NT == 1 && own) f = rq_load_as<floatx8>(lds + own_at + t * low.ranks + k);
          else f = low8(low, t, k);
          rq_operand<3>(f, u);
          bf16x8 lead = u[0];
          if constexpr (PW > 1) lead = without_inf(lead);
#pragma unroll
          for (int m = 0; m < RT; ++m) {
            floatx4 part = rq_mfma(w[m][0], u[0], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
            part = rq_mfma(first[m], u[1], part);
            part = rq_mfma(first[m], u[2], part);
            if constexpr (PW > 1) {
              part = rq_mfma(w[m][1], lead, part);
              part = rq_mfma(w[m][1], u[1], part);
            }
            if constexpr (PW > 2) part = rq_mfma(w[m][2], lead, part);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[m][b][j] = whose[b] == a ? __builtin_fmaf(s, part[j], acc[m][b][j]) : acc[m][b][j];
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NT; ++b)
      if (whose[b] == lora.n) {
#pragma unroll
        for (int m = 0; m < RT; ++m) acc[m][b] = floatx4{1.0f, 1.0f, 1.0f, 1.0f} * __builtin_nanf("");
      }
  }
};

// --- the gradients, once the parts of dy W are there --------------------------------------------
// One launch: workgroups for da and db and, behind them, for dx.  Bound by the latency of loads that lie in other XCDs'
// caches: four parts' and a wave's eight rows are in flight at once.
constexpr int WINDOW = 512;

// dx of 16 tokens and 64 columns a workgroup: its waves deal the parts among them, and the adapters' ranks, 32 at a time, by
// adapter and rank alone; joined through LDS in their order.  Lane 16 q + j has columns 4j..4j+3 of ranks 8q..8q+7,
// product n takes the n-th of each, so that D's column j is column 4j + n.
constexpr int DX_COLS = 64, GRAD_WAVES = 4;
template <typename TX>
__device__ __forceinline__ void lora_dx(int block, const float* __restrict__ part, int parts, int64_t t0, int T, int C,
                                        const RqLora<TX>& lora, const RqLow& v, TX* __restrict__ dx, int64_t ldx, floatx4* lds) {
  const int lane = threadIdx.x & 63, wave = rq_wave(), j = lane & 15, q = lane >> 4;
  const int ctiles = (C + DX_COLS - 1) / DX_COLS, c = block % ctiles * DX_COLS + 4 * j, tw = block / ctiles * 16;
  const int nc = C - c;                            // <= 0: none
  const int mine = tw + j < T ? lora.of(t0 + tw + j) : -1;
  int own[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) own[k] = __shfl(mine, 4 * q + k);
  floatx4 o[4];                                    // of token 4q + k
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (int m = wave; m < parts; m += GRAD_WAVES)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] += rq_load4(part + ((int64_t)m * T + min(tw + 4 * q + k, T - 1)) * C + c, nc);
  for (uint64_t pending = __ballot(lane < 16 && mine >= 0 && mine < lora.n); pending;) {
    const int a = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)pending) - 1);
    pending &= ~__ballot(mine == a);
    const int first = 32 * ((wave - a + 2) & (GRAD_WAVES - 1));
    if (first >= lora.r) continue;
    const float s = lora.scale_of(a);
    floatx4 low[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) low[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = first; k0 < lora.r; k0 += 32 * GRAD_WAVES) {
      const floatx8 vt = low8(v, t0 + min(tw + j, T - 1), k0 + 8 * q);
      floatx4 row[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) row[k] = rq_load4(lora.a + ((int64_t)a * lora.r + min(k0 + 8 * q + k, lora.r - 1)) * C + c, nc);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool is = k0 + 8 * q + k < lora.r;
#pragma unroll
        for (int n = 0; n < 4; ++n) low[n] = rq_mfma4(vt[k], is ? row[k][n] : 0.0f, low[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k][n] = own[k] == a ? __builtin_fmaf(s, low[n][k], o[k][n]) : o[k][n];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) lds[(wave * 4 + k) * 64 + lane] = o[k];
  __syncthreads();
  // wave w: token 4q + w
  const bool none = __shfl(mine, 4 * q + wave) >= lora.n;
  const int t = tw + 4 * q + wave;
  if (t >= T) return;
  floatx4 r = lds[wave * 64 + lane];
#pragma unroll
  for (int w = 1; w < GRAD_WAVES; ++w) r += lds[(w * 4 + wave) * 64 + lane];
  TX* out = dx + (int64_t)t * ldx + c;
  TX e[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) e[n] = rq_cast<TX>(none ? __builtin_nanf("") : r[n]);
  if (nc >= 4) {
    __builtin_memcpy(out, e, sizeof(e));
  } else {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n < nc) out[n] = e[n];
  }
}

// da and db.  Blocks (tiles of 128 columns of x, then of dy; rank tiles; adapters from a0 on): the tokens of the adapter, four to a
// matrix instruction, sixteen in flight, to the waves in turn.  Lane 16 q + i holds columns 8i..8i+7 of token q, and product n takes
// the n-th of each, so that D's column i is column 8i + n.
template <typename TX>
__device__ __forceinline__ void lora_outer(int block, int a0, const TX* __restrict__ x, int64_t ldx, int C, const TX* __restrict__ dy,
                                           int64_t ldy, int R, int T, const RqLora<TX>& lora, const RqLow& u, const RqLow& v,
                                           TX* __restrict__ da, TX* __restrict__ db, floatx4* lds) {
  typedef typename RqOperand<TX>::raw Raw;
  __shared__ int list[WINDOW];
  __shared__ int count;
  const int lane = threadIdx.x & 63, wave = rq_wave(), i = lane & 15, q = lane >> 4;
  const int ctiles = (C + 127) / 128, tiles = ctiles + (R + 127) / 128, rtiles = (lora.r + 15) / 16;
  const int tile = block % tiles, a = a0 + block / tiles / rtiles, rank = block / tiles % rtiles * 16;
  const bool of_a = tile < ctiles;                   // da: v with x; db: u with dy
  const int width = of_a ? C : R, col = (of_a ? tile : tile - ctiles) * 128 + 8 * i;
  const TX* src = of_a ? x : dy;
  const int64_t ld = of_a ? ldx : ldy;
  const RqLow low = of_a ? v : u;
  floatx4 acc[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) acc[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  bool any = false;                                // tokens with this adapter
  for (int64_t w0 = 0; w0 < T; w0 += WINDOW) {
    if (wave == 0) {
      int n = 0;
      for (int k = 0; k < WINDOW && w0 + k < T; k += 64) {
        const bool is = w0 + k + lane < T && lora.of(w0 + k + lane) == a;
        const uint64_t mask = __ballot(is);
        if (is) list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = k + lane;
        n += __popcll(mask);
      }
      if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    any |= n > 0;
    for (int g = 16 * wave; g < n; g += 16 * GRAD_WAVES) {
      float m[4];
      Raw r[4];
      int64_t t[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        t[h] = w0 + list[g + 4 * h + q < n ? g + 4 * h + q : 0];
        m[h] = 0.0f;
        r[h] = col + 8 <= width ? rq_load_x<true>(src + t[h] * ld + col, 8) : rq_load_x<false>(src + t[h] * ld + col, width - col);
      }
      for (int p0 = 0; p0 < low.parts; p0 += 4) {      // four parts' loads at once, the last again past it
        float e[4][4];
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int h = 0; h < 4; ++h) e[p][h] = low.u[low.at(min(p0 + p, low.parts - 1), t[h]) + rank + i];
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int h = 0; h < 4; ++h) m[h] += p0 + p < low.parts ? e[p][h] : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (g + 4 * h >= n) break;
        const bool is = g + 4 * h + q < n;
        floatx8 f;
        rq_floats(r[h], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = rq_mfma4(is ? m[h] : 0.0f, is ? f[k] : 0.0f, acc[k]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) lds[(wave * 8 + n) * 64 + lane] = acc[n];
  __syncthreads();
  const float s = any ? lora.scale_of(a) : 0.0f;   // 0, whatever the scaling of an adapter that nobody has
  if (of_a) {
    // wave w: rank 4q + w, eight columns
    const int k = rank + 4 * q + wave;
    if (k >= lora.r) return;
    TX* out = da + ((int64_t)a * lora.r + k) * C + col;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float o = 0.0f;
      for (int w = 0; w < GRAD_WAVES; ++w) o += lds[(w * 8 + n) * 64 + lane][wave];
      if (col + n < C) out[n] = rq_cast<TX>(s * o);
    }
  } else {
    // wave w: rows 2w and 2w + 1 of the lane's eight, four ranks
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = 2 * wave + h, row = col + n;
      floatx4 o = lds[n * 64 + lane];
      for (int w = 1; w < GRAD_WAVES; ++w) o += lds[(w * 8 + n) * 64 + lane];
      if (row >= R) continue;
      TX* out = db + ((int64_t)a * R + row) * lora.r + rank + 4 * q;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (rank + 4 * q + k < lora.r) out[k] = rq_cast<TX>(s * o[k]);
    }
  }
}

template <typename TX>
__global__ __launch_bounds__(64 * GRAD_WAVES, 4) void k_lora_grads(RqLoraDx<TX> g, int outer, int a0, const TX* x, int64_t ldx, int C,
                                                                 const TX* dy, int64_t ldy, int R, int T, RqLora<TX> lora, RqLow u,
                                                                 RqLow v, TX* da, TX* db) {
  __shared__ floatx4 lds[GRAD_WAVES * 8 * 64];
  if ((int)blockIdx.x >= outer) lora_dx<TX>(blockIdx.x - outer, g.part, g.parts, g.t0, g.T, C, lora, v, g.dx, g.ldx, lds);
  else lora_outer<TX>(blockIdx.x, a0, x, ldx, C, dy, ldy, R, T, lora, u, v, da, db, lds);
}

}  // namespace

template <typename TX>
void rq_lora_down(const RqDownJobs<TX>& jobs, void* arranged, int nbits, hipStream_t s) {
  const int chunks = (jobs.first.cols + RQ_CHUNK - 1) / RQ_CHUNK, more = arranged ? (chunks + ARRANGED_CHUNKS - 1) / ARRANGED_CHUNKS : 0;
  hipLaunchKernelGGL(k_lora_down<TX>, dim3(jobs.tiles, jobs.adapters, jobs.z + more), dim3(64 * DOWN_WAVES), 0, s, jobs,
                     RqArrange{arranged, rq_pairs<TX>(nbits)});
}

template <typename TX>
void rq_lora_rows(const TX* x, int T, int64_t ldx, const RqPacked& w, int nbits, const TX* bias, const RqLora<TX>& lora,
                  const RqLow& low, const void* arranged, TX* y, int64_t ldy, hipStream_t s) {
  rq_with_nbits(nbits, [&](auto nb) {
    linear_rows<TX, decltype(nb)::value>(x, T, ldx, w, bias, y, ldy, RqLowRank<TX>{lora, low, arranged, low.u == nullptr, 0}, s);
  });
}

template <typename TX>
void rq_lora_grads(const RqLoraDx<TX>& g, const TX* x, int64_t ldx, int C, const TX* dy, int64_t ldy, int R, int T,
                   const RqLora<TX>& lora, const RqLow& u, const RqLow& v, TX* da, TX* db, hipStream_t s) {
  // A launch holds fewer than 2^32 threads along a dimension: adapters past that go into further launches.  One adapter's
  // workgroups, at most 2^20 (by width_ok), and dx's, at most 2^23 of 256 tokens, always fit.
  constexpr int64_t MOST = ((1ll << 32) - 1) / (64 * GRAD_WAVES);
  int64_t ndx = g.dx ? (int64_t)((C + DX_COLS - 1) / DX_COLS) * ((g.T + 15) / 16) : 0;
  const int64_t each = da ? (int64_t)((C + 127) / 128 + (R + 127) / 128) * ((lora.r + 15) / 16) : 0;
  const int n = da ? lora.n : 0;
  for (int a0 = 0; ndx || a0 < n; ndx = 0) {
    const int64_t fit = each ? (MOST - ndx) / each : 0;
    const int adapters = (int)(fit < n - a0 ? fit : n - a0);
    hipLaunchKernelGGL(k_lora_grads<TX>, dim3((unsigned)(ndx + adapters * each)), dim3(64 * GRAD_WAVES), 0, s, g, (int)(adapters * each),
                       a0, x, ldx, C, dy, ldy, R, T, lora, u, v, da, db);
    a0 += adapters;
  }
}
