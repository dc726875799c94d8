// fmxq_logprobs.hip -- log probabilities of given tokens through a quantized vocabulary head, the
// entropy and the likeliest tokens, and their gradient.
//
// With l = h . deq(W)^T / T over the tokens and p = softmax(l):
//   lse = log sum exp(l),  logp_j = l_j - lse,  H = -sum_v p_v log p_v
//   dl_v = sum_j a_j [id_j = v] - p_v (A + c (log p_v + H)),  A = sum_j a_j,  dh = (1 / T) sum_v dl_v W_v
// for upstream gradients a_j of logp_j and c of H.
//
// Scores: the product's epilogue leaves a few numbers of every tile of a row (HeadTile), relative to
// the tile's largest logit and without it.  A row is then joined relative to its largest logit:
// with `others` the sum of the other tokens' exponentials, -log p of the likeliest token is
// log1p(others) and H = log1p(others) + sum_v p_v (top - l_v): sums of positive terms, which keep
// their precision in rows that are sure.
// The likeliest tokens: the n largest logits lie in the n tiles whose largest are highest, but for what
// fp32 sums are off by, so of the exponentials, which the product leaves in bf16, a row reads the tiles
// that come within that of the n-th.  What comes within that and bf16's rounding of it is a
// candidate, whose logit is summed again in 64 bits: that decides the order, and equal ones go to
// the lowest token.
// Gradient: the logits' product again, whose epilogue writes dl (without the given tokens) in bf16,
// and dl . deq(W); the given tokens' share enters at the end in fp32, as 1 - p from log p.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_grad_tile.hpp"
#include "fmxq_head_row.hpp"
#include "fmxq_internal.hpp"

namespace fmxq {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 64;
// Candidates: within this of the n-th logit (units of log 2), beside what fp32 sums are off by: two
// roundings to bf16 are 0.0057.
constexpr float kNear = 0.0225f;
// Exponentials below 2^-kLost are taken as lost.
constexpr float kLost = 120.f, kLostBelow = 0x1p-120f;

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The logit of token v for row m in units of log 2, summed in 64 bits (its products are exact
// there); NaN counts as the lowest.  With SIZE also the sum of the products' magnitudes, and whether
// the row has a value other than 0.
template <bool SIZE>
__device__ __forceinline__ double logit64(const HeadScore& a, int64_t m, int v, float* size, bool* some) {
  constexpr int B = 4;  // chunks of 512 columns that are requested together
  const uint16_t* h = a.h + m * a.K;
  const int K = (int)a.K;
  double t = 0.;
  float mag = 0.f;
  uint32_t any = 0;
  for (int c0 = 8 * (threadIdx.x & 63); c0 < K; c0 += 512 * B) {
    Packed8 p[B];
    u32x4 x[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int c = c0 + 512 * i < K ? c0 + 512 * i : c0;
      p[i] = load8(a, v, c);
      x[i] = *reinterpret_cast<const u32x4*>(h + c);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (c0 + 512 * i >= K) break;
      float wv[8];
      deq8(p[i], a.bits, wv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t = __builtin_fma((double)wv[2 * j], (double)bf16_lo(x[i][j]), t);
        t = __builtin_fma((double)wv[2 * j + 1], (double)bf16_hi(x[i][j]), t);
        if constexpr (SIZE) {
          mag += fabsf(wv[2 * j] * bf16_lo(x[i][j])) + fabsf(wv[2 * j + 1] * bf16_hi(x[i][j]));
          any |= x[i][j] & 0x7fff7fffu;
        }
      }
    }
  }
  const double scale = 1.4426950408889634 / (double)a.temperature;
  t = wave_sum64(t) * scale;
  if constexpr (SIZE) {
    *size = wave_sum(mag) * (float)scale;
    *some = __any(any != 0);
  }
  return t == t ? t : -__builtin_huge_val();
}
__device__ __forceinline__ double logit64(const HeadScore& a, int64_t m, int v) {
  return logit64<false>(a, m, v, nullptr, nullptr);
}

// Floats in their order as whole numbers.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// The rank-th largest of n keys (1 <= rank <= n), and how many of those equal to it are among the
// rank largest: a byte a pass.  lds: 258 words.
template <int T, class Key>
__device__ __forceinline__ uint32_t select_key(uint32_t n, uint32_t rank, Key key, uint32_t* lds,
                                               uint32_t* equal) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += T) lds[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += T) {
      const uint32_t k = key(i);
      if (shift == 24 || (k ^ prefix) >> (shift + 8) == 0) atomicAdd(&lds[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 64) {
      const int b = 255 - 4 * lane;  // the lane's bins b, b - 1, b - 2, b - 3
      const uint32_t c[4] = {lds[b], lds[b - 1], lds[b - 2], lds[b - 3]};
      const uint32_t sum = c[0] + c[1] + c[2] + c[3];
      uint32_t at = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = (uint32_t)__shfl_up((int)at, o, 64);
        if (lane >= o) at += u;
      }
      at -= sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (at < rank && rank <= at + c[i]) {
          lds[256] = (uint32_t)(b - i);
          lds[257] = rank - at;
        }
        at += c[i];
      }
    }
    __syncthreads();
    prefix |= lds[256] << shift;
    rank = lds[257];
    __syncthreads();
  }
  *equal = rank;
  return prefix;
}

// A candidate, and whether it comes before another.
struct Best {
  double l;
  int id;
};
__device__ __forceinline__ bool before(double l, int id, double l2, int id2) {
  return l > l2 || (l == l2 && id < id2);
}

// (Blocks for few rows take more of LDS; of the others several share it: with 4096 and 2048 there too, 2048
// rows of 1002 tiles took 212 us in place of 159.)
template <int T>
struct ScoreShared {
  static constexpr uint32_t kKeptTiles = T > 256 ? 4096 : 1280;
  static constexpr int kCandidates = T > 256 ? 2048 : 1024;
  uint32_t sel[258], keys[kKeptTiles];
  uint64_t red[T / 64];
  float sum[2][T / 64];
  uint32_t tiles[T + 128];
  double lead;
  float size;
  uint32_t zeros, ntiles, ncand, nbest;
  double bl[2][kMaxTop], cl[kCandidates];
  int bi[2][kMaxTop], ci[kCandidates];
};

// The candidates so far join the best n, which end in set `to`.
template <int T>
__device__ __forceinline__ void join_candidates(const HeadScore& a, int64_t m, int n, int from, int to,
                                                ScoreShared<T>& s) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const int nc = (int)s.ncand, nb = (int)s.nbest;
  for (int i = wave; i < nc; i += T / 64) {
    const double l = logit64(a, m, s.ci[i]);
    if ((tid & 63) == 0) s.cl[i] = l;
  }
  __syncthreads();
  for (int i = tid; i < nb + nc; i += T) {
    const double l = i < nb ? s.bl[from][i] : s.cl[i - nb];
    const int id = i < nb ? s.bi[from][i] : s.ci[i - nb];
    int rank = 0;
    for (int j = 0; j < nb; ++j) rank += before(s.bl[from][j], s.bi[from][j], l, id);
    for (int j = 0; j < nc; ++j) rank += before(s.cl[j], s.ci[j], l, id);
    if (rank < n) {
      s.bl[to][rank] = l;
      s.bi[to][rank] = id;
    }
  }
  __syncthreads();
  if (tid == 0) {
    s.nbest = nb + nc < n ? nb + nc : n;
    s.ncand = 0;
  }
  __syncthreads();
}

// A block joins the tiles of a row.
template <int T>
__global__ __launch_bounds__(T) void head_score_kernel(HeadScore a, const HeadTile* __restrict__ score,
                                                       int64_t stat_tiles, int tw,
                                                       const uint16_t* __restrict__ e, int64_t lde) {
  constexpr int W = T / 64;
  __shared__ ScoreShared<T> s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.x;
  const uint32_t nt = (uint32_t)((a.V + tw - 1) / tw);
  const HeadTile* st = score + m * stat_tiles;
  // The largest logit and the first tile that has it.
  // (The order of the tiles' tops stays in LDS where it has room.)
  uint64_t lead = 0;
  const bool kept = nt <= s.kKeptTiles;
#pragma unroll 4
  for (uint32_t t = tid; t < nt; t += T) {
    const uint32_t o = order_key(st[t].top);
    if (kept) s.keys[t] = o;
    const uint64_t k = (uint64_t)o << 32 | (0xffffffffu - t);
    lead = k > lead ? k : lead;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t k = __shfl_xor(lead, o, 64);
    lead = k > lead ? k : lead;
  }
  if (lane == 0) s.red[wave] = lead;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) lead = s.red[i] > lead ? s.red[i] : lead;
  const uint32_t lt = 0xffffffffu - (uint32_t)lead;
  const float top = key_value((uint32_t)(lead >> 32));
  const int first = (int)((int64_t)lt * tw + st[lt].first);  // (past the vocabulary in a row that is not finite)
  float others = 0.f, low = 0.f;
#pragma unroll 4
  for (uint32_t t = tid; t < nt; t += T) {
    const HeadTile h = st[t];
    const float d = top - h.top, f = __builtin_amdgcn_exp2f(-d);
    const float sum = t == lt ? h.sum : (1.f + h.sum) * f;
    others += sum;
    low += h.low * f;
    low = __builtin_fmaf(d, sum, low);
  }
  others = wave_sum(others);
  low = wave_sum(low);
  if (lane == 0) {
    s.sum[0][wave] = others;
    s.sum[1][wave] = low;
  }
  __syncthreads();
  others = low = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    others += s.sum[0][i];
    low += s.sum[1][i];
  }
  const bool bad = !(fabsf(top) < INFINITY) || !(others < INFINITY) || !(low < INFINITY);
  const float nan = __builtin_nanf("");
  const float lz = bad ? nan : log1pf(others);
  if (tid == 0) {
    a.lse[m] = bad ? nan : __builtin_fmaf(top, kLn2, lz);
    a.entropy[m] = bad ? nan : lz + kLn2 * (low / (1.f + others));
  }
  const int n = a.top, k = a.k;
  if (n + k == 0) return;
  // The given tokens' logits, and that of the likeliest, in 64 bits.
  for (int j = wave; j <= k; j += W) {
    const int id = j < k ? a.ids[m * k + j] : first;
    if (j < k && id >= a.V && lane == 0) atomicOr(a.flag, 1u);
    if (bad || id < 0 || id >= a.V) continue;
    const int v = __builtin_amdgcn_readfirstlane(id);
    if (j < k) {
      const double l = v == first ? 0. : logit64(a, m, v);
      if (lane == 0) s.cl[j] = l;
    } else {
      float size;
      bool some;
      const double l = logit64<true>(a, m, v, &size, &some);
      if (lane == 0) {
        s.lead = l;
        s.size = size;
        s.zeros = !some;
      }
    }
  }
  if (tid == 0) s.ntiles = s.ncand = s.nbest = 0;
  __syncthreads();
  // log p of a token from its logit, relative to the likeliest one's, which is what the others leave: their
  // sum relative to that one's 64-bit logit too, so that what its fp32 sum is off by is in neither.
  const float d = bad ? nan : (float)((double)top - s.lead);
  const float left = bad             ? nan
                     : others == 0.f ? 0.f
                     : d < 64.f      ? log1pf(others * __builtin_amdgcn_exp2f(d))
                                     : __builtin_fmaf(d, kLn2, logf(others));
  auto logp = [&](int id, double l) {
    return bad ? nan : id == first ? -left : (float)((l - s.lead) * 0.6931471805599453 - (double)left);
  };
  if (tid < k) {
    const int id = a.ids[m * k + tid];
    a.logp[m * k + tid] = id >= 0 && id < a.V ? logp(id, s.cl[tid]) : 0.f;
  }
  if (n == 0) return;
  int32_t* ids = a.top_ids + m * n;
  float* lps = a.top_logp + m * n;
  if (bad || s.zeros || (top == 0.f && others == (float)(a.V - 1) && low == 0.f)) {
    // No order, or a row of zeros, or a head of zeros for the row (all of its logits 0 in fp32): all
    // alike.  (The search would sum every token again: 100 ms for one row of 128256 x 4096.)
    for (int i = tid; i < n; i += T) {
      ids[i] = bad ? -1 : i;
      lps[i] = -left;
    }
    return;
  }
  auto tile_key = [&](uint32_t t) { return kept ? s.keys[t] : order_key(st[t].top); };
  const int sh = __builtin_ctz(tw);
  const uint16_t* er = e + m * lde;
  // Column c of a tile: its token and its logit to bf16's precision, or where its exponential leaves
  // the type's range, `lost` below the tile's largest (which it is at least).
  auto column = [&](uint32_t t, uint32_t c, int* id, float lost) {
    const int64_t v = (int64_t)t * tw + c;
    *id = (int)v;
    if (v >= a.V) return -INFINITY;
    const float x = bf16_bits_to_f32(er[v]);
    return st[t].top - (x < kLostBelow ? lost : -__builtin_amdgcn_logf(x));
  };
  // The n-th logit: a bound below it that n columns reach, the n-th highest tile's largest, or of few
  // tiles the n-th column's.
  uint32_t equal;
  float nth;
  if (nt >= (uint32_t)n) {
    nth = key_value(select_key<T>(nt, n, tile_key, s.sel, &equal));
  } else {
    nth = key_value(select_key<T>(nt * (uint32_t)tw, n, [&](uint32_t i) {
            int id;
            return order_key(column(i >> sh, i & (tw - 1), &id, INFINITY));
          }, s.sel, &equal));
  }
  // Two fp32 logits that differ by more than this are in their exact order: twice what a sum of K
  // products is off by, for tokens whose products are up to twice as large as the likeliest one's.
  const float off = 4.f * (float)(a.K + 16) * 0x1p-24f * fmaxf(s.size, fabsf(nth));
  const float tile_least = nt >= (uint32_t)n ? nth - off : -INFINITY, least = nth - (kNear + off);
  int set = 0;
  for (uint32_t t0 = 0; t0 < nt;) {
    // Tiles that may hold one, as many as the list does, and their columns.
    for (; t0 < nt; t0 += T) {
      const bool full = s.ntiles > 128;
      __syncthreads();
      if (full) break;
      const uint32_t t = t0 + tid;
      if (t < nt && key_value(tile_key(t)) >= tile_least) s.tiles[atomicAdd(&s.ntiles, 1u)] = t;
      __syncthreads();
    }
    const uint32_t cols = s.ntiles * (uint32_t)tw;
    for (uint32_t i0 = 0; i0 < cols; i0 += T) {
      int id;
      const uint32_t i = i0 + tid;
      if (i < cols && column(s.tiles[i >> sh], i & (tw - 1), &id, kLost) >= least && id < a.V)
        s.ci[atomicAdd(&s.ncand, 1u)] = id;
      __syncthreads();
      const bool full = s.ncand > s.kCandidates - T;
      __syncthreads();
      if (full) {
        join_candidates<T>(a, m, n, set, set ^ 1, s);
        set ^= 1;
      }
    }
    __syncthreads();
    if (tid == 0) s.ntiles = 0;
    __syncthreads();
  }
  join_candidates<T>(a, m, n, set, set ^ 1, s);
  set ^= 1;
  for (int i = tid; i < n; i += T) {
    const bool on = i < (int)s.nbest;
    ids[i] = on ? s.bi[set][i] : -1;
    lps[i] = on ? logp(s.bi[set][i], s.bl[set][i]) : nan;
  }
}

// ---- gradient -----------------------------------------------------------------------

// A row's upstream gradients, lane j's entry among them.
struct GradRow {
  int v;       // the lane's token, or -1
  float a, A;  // of the lane's entry, of all
  float c;
  bool empty;  // nothing flows back
};
__device__ __forceinline__ GradRow grad_row(const HeadScoreGrad& a, int64_t m, bool report) {
  const int lane = threadIdx.x & 63;
  GradRow r{-1, 0.f, 0.f, 0.f, false};
  if (lane < a.k) {
    const int id = a.ids[m * a.k + lane];
    if (id >= 0 && id < a.V) {
      r.v = id;
      r.a = a.grad_logp[m * a.k + lane];
    } else if (report && id >= a.V) {
      atomicOr(a.flag, 1u);
    }
  }
  r.A = a.k > 1 ? wave_sum(r.a) : __shfl(r.a, 0, 64);
  r.c = a.grad_entropy ? a.grad_entropy[m] : 0.f;
  r.empty = r.c == 0.f && !__any(r.a != 0.f);
  return r;
}

// A wave a row: what the epilogue of the logits needs (store_coef).
__global__ __launch_bounds__(256) void score_rows_kernel(HeadScoreGrad a, f32x4* __restrict__ rows) {
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.M) return;
  const GradRow r = grad_row(a, m, true);
  if ((threadIdx.x & 63) == 0)
    rows[m] = f32x4{a.lse[m] * kLog2e, r.c == 0.f ? r.A : __builtin_fmaf(r.c, a.entropy[m], r.A), r.c * kLn2,
                    0.f};
}

// dh: the sum of the slices and the given tokens' share, 8 columns a thread.  With WS = 4 the waves
// of a block share the slices and the entries of 512 columns (many slices, or entries).
template <int WS>
__global__ __launch_bounds__(256) void score_dh_kernel(HeadScoreGrad a, const float* __restrict__ slices,
                                                       int splits) {
  __shared__ float coef[64];
  __shared__ int tokens[64], empty;
  __shared__ f32x4 part[WS > 1 ? 2 * 256 : 1];
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c0 = (int64_t)blockIdx.y * (WS > 1 ? 512 : 2048);
  const int64_t c = c0 + 8 * (WS > 1 ? lane : (int)threadIdx.x);
  if (wave == 0) {
    const GradRow r = grad_row(a, m, false);
    // The gradients of the row's entries of the lane's token and of its others, and whether an
    // earlier lane has the token.
    float mine = 0.f, rest = 0.f;
    bool again = false;
    for (int j = 0; j < a.k; ++j) {
      const int v = __builtin_amdgcn_readlane(r.v, j);
      const float g = __shfl(r.a, j, 64);
      if (v == r.v) {
        mine += g;
        again |= j < lane;
      } else {
        rest += g;
      }
    }
    float d = 0.f;
    const bool on = r.v >= 0 && !again;
    if (on) {
      const float lp = a.logp[m * a.k + lane], p = expf(lp);
      d = mine * -expm1f(lp) - p * rest;
      if (r.c != 0.f && p != 0.f) d -= p * (r.c * (lp + a.entropy[m]));
    }
    coef[lane] = d;
    tokens[lane] = on ? r.v : -1;
    if (lane == 0) empty = r.empty;
  }
  f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  if (c < a.K) {
#pragma unroll 8
    for (int s = WS > 1 ? wave : 0; s < splits; s += WS) {
      const f32x4* p = reinterpret_cast<const f32x4*>(slices + ((int64_t)s * a.M + m) * a.K + c);
      v[0] += p[0];
      v[1] += p[1];
    }
  }
  __syncthreads();
  if (c < a.K) {
    constexpr int B = 4;  // entries that are requested together
    for (int i0 = WS > 1 ? wave : 0; i0 < a.k; i0 += B * WS) {
      Packed8 p[B];
      int id[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        id[i] = i0 + i * WS < a.k ? tokens[i0 + i * WS] : -1;
        p[i] = load8(a, id[i] < 0 ? 0 : id[i], (int)c);
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (__builtin_amdgcn_readfirstlane(id[i]) < 0) continue;
        const float co = coef[i0 + i * WS];
        float wv[8];
        deq8(p[i], a.bits, wv);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = __builtin_fmaf(co, wv[j], v[j >> 2][j & 3]);
      }
    }
  }
  const float scale = 1.f / a.temperature;
  if constexpr (WS > 1) {
    part[2 * threadIdx.x] = v[0];
    part[2 * threadIdx.x + 1] = v[1];
    __syncthreads();
    const float* p = reinterpret_cast<const float*>(part) + 2 * threadIdx.x;
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      lo += p[512 * w];
      hi += p[512 * w + 1];
    }
    const int64_t n = c0 + 2 * threadIdx.x;
    if (n < a.K)
      *reinterpret_cast<uint32_t*>(a.dh + m * a.K + n) = empty ? 0u : pack_bf16x2(lo * scale, hi * scale);
  } else if (c < a.K) {
    v[0] *= scale;
    v[1] *= scale;
    u32x4 o = {pack_bf16x2(v[0][0], v[0][1]), pack_bf16x2(v[0][2], v[0][3]),
               pack_bf16x2(v[1][0], v[1][1]), pack_bf16x2(v[1][2], v[1][3])};
    if (empty) o = u32x4{0u, 0u, 0u, 0u};
    *reinterpret_cast<u32x4*>(a.dh + m * a.K + c) = o;
  }
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Rows are scored in chunks whose tiles and exponentials take about this much.
constexpr int64_t kScoreBytes = (int64_t)1 << 30;

constexpr int64_t kFewRows = 512;
struct ScorePlan {
  HeadPlan p;
  bool thin;
  int stat_width;
  int64_t stat_tiles, lde;
  size_t e, panel, xp, bytes;  // the tiles' numbers begin the workspace
};
int64_t score_rows(int64_t M, int64_t V, int top) {
  const int64_t row = up(V, kGradTileCols) * (top ? 2 : 0) + up(V, kGradTileCols) / kThinStatWidth * 16;
  return std::min(M, std::max<int64_t>(kScoreBytes / row / 256 * 256, 256));
}
ScorePlan score_plan(int64_t M, int64_t V, int64_t K, int k, int top, int cus) {
  ScorePlan s{};
  s.p = head_plan(M, V, K, std::max(k, 1), false, cus);
  s.lde = up(V, kGradTileCols);
  s.thin = thin_supported(M, V, K);
  s.stat_width = s.thin ? kThinStatWidth : s.p.stat_width;
  s.stat_tiles = s.lde / s.stat_width;
  size_t at = (size_t)up(M * s.stat_tiles * (int64_t)sizeof(HeadTile), 256);
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
  };
  s.e = take(top ? M * s.lde * 2 : 0);
  s.panel = take(s.p.panel && !s.p.skinny ? s.p.piece * K * 2 : 0);
  s.xp = take(s.p.skinny ? skinny_pack_bytes(M, K) : 0);
  s.bytes = at;
  return s;
}

// The product of the logits of tokens v0 .. v0 + n, but for its epilogue.
template <class Args>
GradGemm logits_gemm(const Args& a, int64_t v0, int64_t n) {
  GradGemm g;
  g.a = a.h;
  g.lda = g.a_cols = a.K;
  g.M = a.M;
  g.N = n;
  g.C = a.K;
  g.c_split = up(a.K, 64);
  g.w = a.w + v0 * (a.K * a.bits / 32);
  g.scales = a.scales + v0 * (a.K / a.group_size);
  g.biases = a.biases + v0 * (a.K / a.group_size);
  g.group_size = a.group_size;
  g.bits = a.bits;
  g.logit_scale = kLog2e / a.temperature;
  return g;
}
hipError_t launch_logits(GradGemm& g, const HeadPlan& p, uint16_t* panel, void* xp, bool keep,
                         hipStream_t stream) {
  if (p.skinny && skinny_pack_bytes(g.M, g.C)) g.xp = xp;
  if (p.panel && (keep || !p.skinny)) {
    if (hipError_t r = launch_dequantize(g.w, g.scales, g.biases, panel, g.N, g.C, g.group_size, g.bits, stream))
      return r;
    g.panel = panel;
    g.ldp = g.C;
  }
  return p.skinny  ? launch_skinny_gemm(g, false, stream)
         : p.panel ? launch_panel_gemm(g, false, stream)
                   : launch_grad_gemm(g, false, p.bm, stream);
}

}  // namespace

size_t head_score_bytes(int64_t M, int64_t V, int64_t K, int k, int top, int cus) {
  const int64_t rows = score_rows(M, V, top);
  size_t most = score_plan(rows, V, K, k, top, cus).bytes;
  if (M % rows) most = std::max(most, score_plan(M % rows, V, K, k, top, cus).bytes);
  return most;
}

hipError_t launch_head_score(const HeadScore& all, int cus, void* ws, hipStream_t stream) {
  char* base = static_cast<char*>(ws);
  const int64_t rows = score_rows(all.M, all.V, all.top);
  for (int64_t r0 = 0; r0 < all.M; r0 += rows) {
    HeadScore a = all;
    a.M = std::min(rows, all.M - r0);
    a.h += r0 * a.K;
    if (a.k) {
      a.ids += r0 * a.k;
      a.logp += r0 * a.k;
    }
    a.entropy += r0;
    a.lse += r0;
    if (a.top) {
      a.top_ids += r0 * a.top;
      a.top_logp += r0 * a.top;
    }
    const ScorePlan s = score_plan(a.M, a.V, a.K, a.k, a.top, cus);
    HeadTile* score = reinterpret_cast<HeadTile*>(base);
    uint16_t* e = a.top ? reinterpret_cast<uint16_t*>(base + s.e) : nullptr;
    for (int64_t v0 = 0; v0 < a.V; v0 += s.p.piece) {
      GradGemm g = logits_gemm(a, v0, std::min(a.V - v0, s.p.piece));
      g.epi = kEpiScores;
      g.score = score + v0 / s.stat_width;
      g.stat_tiles = s.stat_tiles;
      g.e = e ? e + v0 : nullptr;
      g.lde = s.lde;
      if (hipError_t r = s.thin ? launch_thin_gemm(g, stream)
                                : launch_logits(g, s.p, reinterpret_cast<uint16_t*>(base + s.panel), base + s.xp,
                                                false, stream))
        return r;
    }
    // Few rows: more threads each, where the latency of one row is what counts.
    const unsigned n = (unsigned)a.M;
    if (a.M <= kFewRows)
      head_score_kernel<1024><<<n, 1024, 0, stream>>>(a, score, s.stat_tiles, s.stat_width, e, s.lde);
    else
      head_score_kernel<256><<<n, 256, 0, stream>>>(a, score, s.stat_tiles, s.stat_width, e, s.lde);
    if (hipError_t r = hipGetLastError()) return r;
  }
  return hipSuccess;
}

size_t head_score_grad_bytes(int64_t M, int64_t V, int64_t K, int k, int cus) {
  return head_plan(M, V, K, k, true, cus).bytes + (size_t)up(M * 16, 256);
}

hipError_t launch_head_score_grad(const HeadScoreGrad& a, int cus, void* ws, hipStream_t stream) {
  const HeadPlan p = head_plan(a.M, a.V, a.K, a.k, true, cus);
  char* base = static_cast<char*>(ws);
  uint16_t* e = reinterpret_cast<uint16_t*>(base + p.e);
  float* slices = reinterpret_cast<float*>(base + p.slices);
  f32x4* rows = reinterpret_cast<f32x4*>(base + p.bytes);
  score_rows_kernel<<<(unsigned)((a.M + 3) / 4), 256, 0, stream>>>(a, rows);
  if (hipError_t r = hipGetLastError()) return r;
  for (int i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(a.V - v0, p.piece);
    GradGemm g = logits_gemm(a, v0, n);
    g.epi = kEpiCoef;
    g.rows = reinterpret_cast<const float*>(rows);
    g.e = e;
    g.lde = up(n, kGradTileCols);
    g.wanted = a.ids;
    g.wanted_k = a.k;
    g.wanted_none = -1;
    g.first_token = v0;
    if (hipError_t r = launch_logits(g, p, reinterpret_cast<uint16_t*>(base + p.panel_at), base + p.xp, true, stream))
      return r;
    GradGemm d = g;
    d.epi = kEpiStats;
    d.a = e;
    d.lda = g.lde;
    d.a_cols = up(n, p.stat_width);  // columns that the tiles have written
    d.N = a.K;
    d.C = n;
    d.splits = p.splits;
    d.c_split = p.c_split;
    d.out = slices;
    d.add = i > 0;
    if (hipError_t r = p.panel         ? launch_panel_gemm(d, true, stream)
                       : p.grad_skinny ? launch_skinny_gemm(d, true, stream)
                                       : launch_grad_gemm(d, true, p.grad_bm, stream))
      return r;
  }
  if (p.splits >= 8 || a.k >= 8) {
    const dim3 grid((unsigned)a.M, (unsigned)((a.K + 511) / 512));
    score_dh_kernel<4><<<grid, 256, 0, stream>>>(a, slices, p.splits);
  } else {
    const dim3 grid((unsigned)a.M, (unsigned)((a.K + 2047) / 2048));
    score_dh_kernel<1><<<grid, 256, 0, stream>>>(a, slices, p.splits);
  }
  return hipGetLastError();
}

}  // namespace fmxq
