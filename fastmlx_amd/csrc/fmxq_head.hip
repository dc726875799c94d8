// fmxq_head.hip -- losses over a quantized vocabulary head: cross entropy and the divergence
// from a teacher's top logits, with the gradient of the hidden states.
//
// With l = h . deq(W)^T / T (T = 1 for cross entropy), p = softmax(l) and q the wanted
// distribution, which has at most k entries a row (one for cross entropy):
//   lse  = log sum_v exp(l_v)
//   loss = T^2 sum_j q_j (log q_j - l_j + lse)
//   dh   = g T (sum_v p_v W_v - sum_j q_j W_j)
// The vocabulary is walked in pieces.  A piece's product leaves e = 2^(l - m) in bf16 with m
// the largest l of the row in a tile, rounded to a multiple of 64, and the tile's sum; the join
// brings the tiles of a row to one m (a power of two: no second rounding; with m the largest l
// itself nearly all tiles needed it, which took 50 us of a piece of 2048 rows by 32064 tokens
// where the join now takes 17), and e . deq(W) is added to fp32 sums that are scaled by the
// change of m.  The wanted entries are left out of e and of the sums.  Their exponentials and their
// share p_j - q_j enter at the end in fp32: where one of them takes nearly everything, the loss and
// the gradient are what the other tokens leave, which no sum over all of them holds.
//
// e and the weights' panel pass through memory because a piece of either (256 MB at most) stays
// in the last-level cache; recomputing the logits for the gradient would cost a third product.
// Bound: the two products.  2048 rows, 128256 x 4096: 3.97 to 4.16 ms, of them the products 3.65 to
// 3.9, the panels 0.24 and the kernels here 0.07 ms.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_grad_tile.hpp"
#include "fmxq_head_row.hpp"
#include "fmxq_internal.hpp"

namespace fmxq {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// The token of entry j of row m, or -1: absent, or out of range (which raises the flag).
__device__ __forceinline__ int64_t token_of(const HeadLoss& a, int64_t m, int j, bool report) {
  const int32_t id = a.ids[m * a.k + j];
  if (a.teacher ? id < 0 : id == a.ignore) return -1;
  if (id < 0 || id >= a.V) {
    if (report) atomicOr(a.flag, 1u);
    return -1;
  }
  return id;
}

// The logit of token v for row m in units of log 2, fp32 sums over the wave.
__device__ __forceinline__ float logit_of(const HeadLoss& a, int64_t m, int64_t v, float scale) {
  constexpr int B = 4;  // chunks of 512 columns that are requested together
  const uint16_t* h = a.h + m * a.K;
  const int K = (int)a.K;
  float t = 0.f;
  for (int c0 = 8 * (threadIdx.x & 63); c0 < K; c0 += 512 * B) {
    Packed8 p[B];
    u32x4 x[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int c = c0 + 512 * i < K ? c0 + 512 * i : c0;
      p[i] = load8(a, (int)v, c);
      x[i] = *reinterpret_cast<const u32x4*>(h + c);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (c0 + 512 * i >= K) break;
      float wv[8];
      deq8(p[i], a.bits, wv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t = __builtin_fmaf(wv[2 * j], bf16_lo(x[i][j]), t);
        t = __builtin_fmaf(wv[2 * j + 1], bf16_hi(x[i][j]), t);
      }
    }
  }
  return wave_sum(t) * scale;
}

// d - 1 + exp(-d) for |d| < 1/2, where it nears d^2 / 2: its series, cut off below 1e-7 of it.
__device__ __forceinline__ float excess(float d) {
  float s = 1.f / 40320;
  s = __builtin_fmaf(s, d, -1.f / 5040);
  s = __builtin_fmaf(s, d, 1.f / 720);
  s = __builtin_fmaf(s, d, -1.f / 120);
  s = __builtin_fmaf(s, d, 1.f / 24);
  s = __builtin_fmaf(s, d, -1.f / 6);
  s = __builtin_fmaf(s, d, 0.5f);
  return s * (d * d);
}

// log(1 + a / b) for 0 <= a <= b, relative to itself: 2 atanh(a / (2 b + a)), whose series over at most
// 1/3 is cut off below 1e-8 of it.
__device__ __forceinline__ float log1p_ratio(float a, float b) {
  const float t = a / (2.f * b + a), u = t * t;
  float s = 1.f / 15;
  s = __builtin_fmaf(s, u, 1.f / 13);
  s = __builtin_fmaf(s, u, 1.f / 11);
  s = __builtin_fmaf(s, u, 1.f / 9);
  s = __builtin_fmaf(s, u, 1.f / 7);
  s = __builtin_fmaf(s, u, 1.f / 5);
  s = __builtin_fmaf(s, u, 1.f / 3);
  s = __builtin_fmaf(s, u, 1.f);
  return 2.f * t * s;
}

// A row's tokens, lane j's entry among them, from the row's final (m, sum over the tokens that are
// not wanted) and the entry's logit l2: exponentials relative to 2^top.
//
// Nothing in it is the difference of near equals, which a row that is sure of what it wants would
// make of log q - log p and of p - q (a loss of 1e-6 came out as one of -3e-6): 1 - p of the likeliest
// entry is what the others leave, and its -log p is log1p of their ratio; q alike.
struct HeadRow {
  int v;                // the lane's token, or -1
  bool first, twice;    // an id that a row names twice is one token
  bool led, t_led;      // the likeliest entry, of the row's and of the teacher's
  bool empty;           // no wanted entry: loss and gradient are 0
  float l, e, p;
  float top, rest, rest_scale;  // rest: the tokens that are not wanted
  float others, z;              // all tokens but the likeliest entry; all
  float t, t_others, q;  // the teacher's logit less the row's largest, in units of log 2
                         // (cross entropy: a teacher with one entry)
};
// An entry's logit, and whether the row names its token in an earlier entry or in another one.
struct Entry {
  float l2;
  uint32_t again, twice;
};
__device__ __forceinline__ HeadRow read_row(const HeadLoss& a, int64_t m, float2 st, Entry en) {
  const int lane = threadIdx.x & 63;
  HeadRow r;
  r.v = -1;
  r.t = -INFINITY;
  if (lane < a.k) {
    if (!a.teacher) r.t = 0.f;
    else if (a.teacher_bf16) r.t = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.teacher)[m * a.k + lane]);
    else r.t = reinterpret_cast<const float*>(a.teacher)[m * a.k + lane];
    r.v = (int)token_of(a, m, lane, false);
  }
  r.first = r.v >= 0 && !en.again;
  r.twice = r.v >= 0 && en.twice;
  r.l = r.v >= 0 ? en.l2 : -INFINITY;
  if (r.v < 0) r.t = -INFINITY;
  float most = r.l, t_top = r.t;
  if (a.k > 1) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      most = fmaxf(most, __shfl_xor(most, o, 64));
      t_top = fmaxf(t_top, __shfl_xor(t_top, o, 64));
    }
  } else {
    most = __shfl(most, 0, 64);
    t_top = __shfl(t_top, 0, 64);
  }
  r.empty = t_top == -INFINITY && !__any(r.t != r.t);
  const uint64_t t_at = __ballot(r.t == t_top);
  r.t_led = t_at && lane == __builtin_ctzll(t_at);
  // The difference first: a logit of the type's lowest value times log2 e would be -infinity.
  r.t = (r.t - t_top) * (kLog2e / a.temperature);
  r.top = fmaxf(st.x, most);
  r.rest_scale = __builtin_amdgcn_exp2f(st.x - r.top);
  r.rest = st.y * r.rest_scale;
  r.e = __builtin_amdgcn_exp2f(r.l - r.top);
  const float w = r.empty ? 0.f : __builtin_amdgcn_exp2f(r.t);
  const uint64_t at = __ballot(r.first && r.l == most);
  const int lead = at ? __builtin_ctzll(at) : -1, v_lead = __shfl(r.v, lead & 63, 64);
  r.led = at && r.v == v_lead;
  float others = r.first && lane != lead ? r.e : 0.f;
  r.t_others = r.t_led ? 0.f : w;
  if (a.k > 1) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      others += __shfl_xor(others, o, 64);
      r.t_others += __shfl_xor(r.t_others, o, 64);
    }
  } else {
    others = __shfl(others, 0, 64);
    r.t_others = __shfl(r.t_others, 0, 64);
  }
  r.others = r.rest + others;
  r.z = r.others + (at ? __builtin_amdgcn_exp2f(most - r.top) : 0.f);
  r.p = r.e / r.z;
  r.q = w / (1.f + r.t_others);
  return r;
}

// lse and the loss.  With d_j = log q_j - log p_j and p_rest the share of the tokens that are not
// wanted,
//   sum_j q_j d_j = sum_j q_j (d_j - 1 + exp(-d_j)) + p_rest,
// because the q_j add up to 1 and the p_j = q_j exp(-d_j) to 1 - p_rest.  No term is negative.
// (Of an id named twice the terms are not, and its p counts once.)
__device__ __forceinline__ void store_loss(const HeadLoss& a, int64_t m, const HeadRow& r) {
  const float log2_z = __builtin_amdgcn_logf(r.z);
  const float neg_log_p = r.led && r.others < r.e ? log1p_ratio(r.others, r.e)
                                                  : (r.top - r.l + log2_z) * kLn2;
  float neg_log_q = 0.f;
  if (a.k > 1)
    neg_log_q = r.t_led && r.t_others < 1.f ? log1p_ratio(r.t_others, 1.f)
                                            : (__builtin_amdgcn_logf(1.f + r.t_others) - r.t) * kLn2;
  const float d = neg_log_p - neg_log_q, p_once = r.first ? r.p : 0.f;
  // Entries of no weight (q = 0) add their p; NaN stays.
  float term = !r.twice && fabsf(d) < 0.5f ? r.q * excess(d) : r.q * (d - 1.f) + p_once;
  if (r.q == 0.f) term = p_once;
  if (r.v < 0) term = 0.f;
  term = a.k > 1 ? wave_sum(term) : term;
  if ((threadIdx.x & 63) != 0) return;
  a.lse[m] = (r.top + log2_z) * kLn2;
  // One factor T at a time: T T alone leaves fp32's range where the loss need not.
  a.loss[m] = r.empty ? 0.f : (term + r.rest / r.z) * a.temperature * a.temperature;
}

// The lane's coefficient of W_id, and the factor of the sums over e.
__device__ __forceinline__ float row_coef(const HeadLoss& a, int64_t m, const HeadRow& r,
                                          float* factor) {
  float q = r.q, not_q = r.t_led ? r.t_others / (1.f + r.t_others) : 1.f - r.q;
  if (__any(r.twice)) {
    float all = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const float qj = __shfl(q, j, 64);
      if (__builtin_amdgcn_readlane(r.v, j) == r.v) all += qj;
    }
    if (r.twice) {
      q = all;
      not_q = 1.f - q;
    }
  }
  const float g = (a.grad_loss ? a.grad_loss[m] : 1.f) * a.temperature;
  *factor = g * r.rest_scale / r.z;
  if (!r.first) return 0.f;
  return g * (q > 0.5f ? not_q - (r.led ? r.others / r.z : 1.f - r.p) : r.p - q);
}

// Block (row, chunk): the row's running (m, sum) after this piece, and the chunk's e brought to it.
// in / out are the states before and after; chunk 0 writes out and the factor of the earlier
// pieces' sums and, after the last piece, finishes the row where no gradient follows.  After the
// last piece the blocks of a row share its wanted entries (sel).
// A chunk is a multiple of 64 tiles: a wave looks at 64 tiles' exponents at once and, where
// none differs from the row's, as in most rows, leaves their e alone.
__global__ __launch_bounds__(256) void head_join_kernel(HeadLoss a, const float2* __restrict__ stats,
                                                        int64_t stat_tiles, int tw,
                                                        const float2* in, float2* out,
                                                        float* factor, uint16_t* e, int64_t lde,
                                                        int tiles, int chunk, bool last, float scale,
                                                        Entry* sel) {
  __shared__ float red[4], red2[4];
  __shared__ Entry entries[64];
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float2* st = stats + m * stat_tiles;
  const float2 old = in ? in[m] : make_float2(-INFINITY, 0.f);
  float top = old.x;
  for (int64_t t = tid; t < tiles; t += 256) top = fmaxf(top, st[t].x);
  top = wave_max(top);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float2 now = make_float2(0.f, 0.f);
  if (blockIdx.y == 0) {
    float sum = 0.f;
    for (int64_t t = tid; t < tiles; t += 256)
      sum = __builtin_fmaf(st[t].y, __builtin_amdgcn_exp2f(st[t].x - top), sum);
    sum = wave_sum(sum);
    if (lane == 0) red2[wave] = sum;
    __syncthreads();
    if (wave == 0) {
      // The first piece starts from nothing: its factor is never used on anything but zeros.
      const float f = in ? __builtin_amdgcn_exp2f(old.x - top) : 0.f;
      now = make_float2(top,
                        (in ? old.y * f : 0.f) + (red2[0] + red2[1]) + (red2[2] + red2[3]));
      if (lane == 0) {
        out[m] = now;
        if (factor) factor[m] = f;
      }
    }
  }
  if (last)
    for (int j = 4 * blockIdx.y + wave; j < a.k; j += 4 * gridDim.y) {
      const int64_t v = token_of(a, m, j, lane == 0);
      uint64_t same = 1;
      if (a.k > 1) same = __ballot(lane < a.k && a.ids[m * a.k + lane] == (int32_t)v);
      const Entry en = {v >= 0 ? logit_of(a, m, v, scale) : 0.f, (same & ((1ull << j) - 1)) != 0,
                        (same & (same - 1)) != 0};
      if (lane == 0) (e ? sel + m * a.k : entries)[j] = en;
    }
  if (last && !e) {
    __syncthreads();
    if (wave == 0) store_loss(a, m, read_row(a, m, now, lane < a.k ? entries[lane] : Entry{}));
  }
  if (!e) return;
  uint16_t* row = e + m * lde;
  const int ta = (int)blockIdx.y * chunk, tb = ta + chunk < tiles ? ta + chunk : tiles;
  for (int t0 = ta + 64 * wave; t0 < tb; t0 += 256) {
    const float f = t0 + lane < tb ? __builtin_amdgcn_exp2f(st[t0 + lane].x - top) : 1.f;
    if (!__any(f != 1.f)) continue;
    for (int c = 8 * lane; c < 64 * tw; c += 512) {
      const float ft = __shfl(f, c >> __builtin_ctz(tw), 64);
      if (ft == 1.f) continue;
      uint16_t* at = row + (int64_t)t0 * tw + c;
      u32x4 v = *reinterpret_cast<u32x4*>(at);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = pack_bf16x2(bf16_lo(v[j]) * ft, bf16_hi(v[j]) * ft);
      *reinterpret_cast<u32x4*>(at) = v;
    }
  }
}

// A row's loss and gradient: the slices' sum times the row's factor, plus the wanted entries'
// share, 8 columns a thread.  With WS = 4 the waves of a block share the slices and the
// entries of 512 columns (many slices, or entries), else each takes columns of its own.
template <int WS>
__global__ __launch_bounds__(256) void head_dh_kernel(HeadLoss a, const float* __restrict__ slices,
                                                      int splits, const float2* __restrict__ state,
                                                      const Entry* __restrict__ sel) {
  __shared__ float coef[64], factor;
  __shared__ int any;
  __shared__ f32x4 part[WS > 1 ? 2 * 256 : 1];
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c0 = (int64_t)blockIdx.y * (WS > 1 ? 512 : 2048);
  const int64_t c = c0 + 8 * (WS > 1 ? lane : (int)threadIdx.x);
  if (wave == 0) {
    const HeadRow r = read_row(a, m, state[m], lane < a.k ? sel[m * a.k + lane] : Entry{});
    if (blockIdx.y == 0) store_loss(a, m, r);
    float f;
    coef[lane] = row_coef(a, m, r, &f);
    if (lane == 0) {
      factor = f;
      any = !r.empty;
    }
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
  v[0] *= factor;
  v[1] *= factor;
  if (c < a.K) {
    constexpr int B = 4;  // entries that are requested together
    for (int i0 = WS > 1 ? wave : 0; i0 < a.k; i0 += B * WS) {
      Packed8 p[B];
      int id[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        id[i] = i0 + i * WS < a.k ? (int)token_of(a, m, i0 + i * WS, false) : -1;
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
      *reinterpret_cast<uint32_t*>(a.dh + m * a.K + n) = any ? pack_bf16x2(lo, hi) : 0u;
  } else if (c < a.K) {
    u32x4 o = {pack_bf16x2(v[0][0], v[0][1]), pack_bf16x2(v[0][2], v[0][3]),
               pack_bf16x2(v[1][0], v[1][1]), pack_bf16x2(v[1][2], v[1][3])};
    if (!any) o = u32x4{0u, 0u, 0u, 0u};
    *reinterpret_cast<u32x4*>(a.dh + m * a.K + c) = o;
  }
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace

// Most bytes of a piece's e, and of its panel of dequantized weights.
constexpr int64_t kHeadPieceBytes = 256 << 20;
constexpr int64_t kHeadPanelBytes = 256 << 20;
// Rows from which the weights are dequantized to a panel beforehand: for two products, where
// five tiles of 256 rows take as long either way (128256 x 4096: 2.75 ms) and eight 4.0 against
// 4.4 ms; for the logits alone, where the panel's 0.24 ms are won back later (1025 rows 1.34
// against 1.50 ms, 1700 rows 1.89 against 2.07, 2048 rows 2.13 against 2.09).
constexpr int64_t kHeadPanelRows = 1025, kScorePanelRows = 1793;

// Few tokens for many rows: the tiles of the logits leave most of the chip idle and each walks
// the whole width, about 2 us a 64-deep step; the kernel for few rows has a block for every
// 32 tokens of every 64 rows and takes about 1.1 ns a block's step.  (500 rows over 1200
// tokens, 4096 wide: 130 against 30 us.)
bool few_tokens(int64_t M, int64_t V, int bm, int cus) {
  const int64_t tiles = (M + bm - 1) / bm * ((V + kLogitCols - 1) / kLogitCols);
  const int64_t waves = (tiles + cus - 1) / cus;
  const int64_t chunks = (M + kSkinnyRows - 1) / kSkinnyRows;
  return chunks <= 65535 && chunks * ((V + 31) / 32) * 11 < waves * 20000;
}

HeadPlan head_plan(int64_t M, int64_t V, int64_t K, int k, bool grad, int cus) {
  HeadPlan p{};
  p.panel = M >= (grad ? kHeadPanelRows : kScorePanelRows) && panel_gemm_supported(K);
  p.bm = p.panel ? kPanelRows : std::max(grad_gemm_rows(M), 128);
  p.grad_bm = p.panel ? kPanelRows : grad_gemm_rows(M);
  int64_t piece = grad ? std::max<int64_t>(kHeadPieceBytes / 2 / M, 2048) : V;
  if (p.panel) piece = std::min(piece, std::max<int64_t>(kHeadPanelBytes / 2 / K, 2048));
  // What the launches take: blocks of 256 tokens by bm rows, or 32 by 64, and e's rows as an operand.
  piece = std::min(piece, (kMaxBlocks - 1) / ((M + p.bm - 1) / p.bm) * kLogitCols);
  piece = std::min(piece, kMaxBlocks * 32 - kGradTileCols);
  if (grad) piece = std::min(piece, kMaxLda / kGradTileCols * kGradTileCols);
  p.pieces = (int)((V + piece - 1) / piece);
  piece = up((V + p.pieces - 1) / p.pieces, kGradTileCols);
  p.pieces = (int)((V + piece - 1) / piece);
  p.piece = piece;
  p.grad_skinny = M <= kGradSkinnyRows && skinny_gemm_supported(piece, piece, K);
  p.skinny = skinny_gemm_supported(K, 32, K) && (M <= kSkinnyRows || few_tokens(M, piece, p.bm, cus));
  p.stat_width = p.skinny ? kSkinnyStatWidth : p.panel ? kPanelStatWidth : kGradStatWidth;
  // Without a gradient the tiles of all pieces are joined at once.
  p.stat_tiles = (grad ? piece : up(V, kGradTileCols)) / p.stat_width;
  // Parts of the gradient product's contraction: enough blocks for the chip, each walking
  // 256 tokens at least.
  const int64_t cols = p.grad_skinny ? kSkinnyCols : p.grad_bm > 128 ? kGradTileCols : kGradCols;
  const int64_t tiles = (p.grad_skinny ? 1 : (M + p.grad_bm - 1) / p.grad_bm) * ((K + cols - 1) / cols);
  const int64_t want = (p.grad_bm > 128 ? cus : 2 * cus) / tiles;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, piece / 256));
  p.c_split = up((piece + p.splits - 1) / p.splits, 64);
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
  };
  p.stats = take(M * p.stat_tiles * 8);
  p.state = take(2 * M * 8);
  p.sel = take(M * k * (int64_t)sizeof(Entry));
  p.factor = take(M * 4);
  if (grad) {
    p.e = take(M * piece * 2);
    p.slices = take((int64_t)p.splits * M * K * 4);
  }
  if (p.panel) p.panel_at = take(piece * K * 2);
  if (p.skinny) p.xp = take(skinny_pack_bytes(M, K));
  p.bytes = at;
  return p;
}

hipError_t launch_head_loss(const HeadLoss& a, const HeadPlan& p, void* ws, hipStream_t stream) {
  char* base = static_cast<char*>(ws);
  float2* stats = reinterpret_cast<float2*>(base + p.stats);
  float2* state = reinterpret_cast<float2*>(base + p.state);
  Entry* sel = reinterpret_cast<Entry*>(base + p.sel);
  float* factor = reinterpret_cast<float*>(base + p.factor);
  uint16_t* e = a.dh ? reinterpret_cast<uint16_t*>(base + p.e) : nullptr;
  float* slices = a.dh ? reinterpret_cast<float*>(base + p.slices) : nullptr;
  const float scale = kLog2e / a.temperature;
  uint16_t* panel = p.panel ? reinterpret_cast<uint16_t*>(base + p.panel_at) : nullptr;
  // (in, out): the running state before and after the pieces joined so far.
  auto join = [&](int i, int64_t v0, int64_t n, int64_t lde) {
    // About 4096 blocks: each reads all statistics of its row, so more of them cost (1000 rows of
    // 128256 tokens, 64 entries: 148 us with 16 blocks a row, 110 with 4), and fewer leave
    // compute units idle.
    const int64_t tiles = (n + p.stat_width - 1) / p.stat_width;
    const int64_t most = std::max((tiles + 63) / 64, v0 + n == a.V ? (a.k + 3) / 4 : (int64_t)1);
    const int64_t by = e ? std::max<int64_t>(1, std::min(most, 4096 / a.M)) : 1;
    const int64_t chunk = up((tiles + by - 1) / by, 64);
    head_join_kernel<<<dim3((unsigned)a.M, (unsigned)by), 256, 0, stream>>>(
        a, stats, p.stat_tiles, p.stat_width, i ? state + (i & 1) * a.M : nullptr,
        state + ((i + 1) & 1) * a.M, factor, e, lde, (int)tiles, (int)chunk, v0 + n == a.V, scale, sel);
    return hipGetLastError();
  };
  for (int i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = std::min(a.V - v0, p.piece);
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
    g.stats = stats + (e ? 0 : v0 / p.stat_width);
    g.stat_tiles = p.stat_tiles;
    g.e = e;
    g.lde = up(n, kGradTileCols);
    g.logit_scale = scale;
    g.wanted = a.ids;
    g.wanted_k = a.k;
    g.wanted_none = a.teacher ? -1 : a.ignore;
    g.first_token = v0;
    if (p.skinny && skinny_pack_bytes(a.M, a.K)) g.xp = base + p.xp;
    if (p.panel && (e || !p.skinny)) {
      if (hipError_t r = launch_dequantize(g.w, g.scales, g.biases, panel, n, a.K, a.group_size, a.bits,
                                           stream))
        return r;
      g.panel = panel;
      g.ldp = a.K;
    }
    if (hipError_t r = p.skinny  ? launch_skinny_gemm(g, false, stream)
                       : p.panel ? launch_panel_gemm(g, false, stream)
                                 : launch_grad_gemm(g, false, p.bm, stream))
      return r;
    if (!e) continue;
    if (hipError_t r = join(i, v0, n, g.lde)) return r;
    GradGemm d = g;
    d.a = e;
    d.lda = g.lde;
    d.a_cols = up(n, p.stat_width);  // columns that the tiles have written
    d.N = a.K;
    d.C = n;
    d.splits = p.splits;
    d.c_split = p.c_split;
    d.out = slices;
    d.add = i > 0;
    d.factor = factor;
    if (hipError_t r = p.panel         ? launch_panel_gemm(d, true, stream)
                       : p.grad_skinny ? launch_skinny_gemm(d, true, stream)
                                       : launch_grad_gemm(d, true, p.grad_bm, stream))
      return r;
  }
  if (!e)
    if (hipError_t r = join(0, 0, a.V, 0)) return r;
  if (!a.dh) return hipSuccess;
  const float2* end = state + (p.pieces & 1) * a.M;
  if (p.splits >= 8 || a.k >= 8) {
    const dim3 grid((unsigned)a.M, (unsigned)((a.K + 511) / 512));
    head_dh_kernel<4><<<grid, 256, 0, stream>>>(a, slices, p.splits, end, sel);
  } else {
    const dim3 grid((unsigned)a.M, (unsigned)((a.K + 2047) / 2048));
    head_dh_kernel<1><<<grid, 256, 0, stream>>>(a, slices, p.splits, end, sel);
  }
  return hipGetLastError();
}

}  // namespace fmxq
