// fmxq_grad_tile.hpp -- what the products of fmxq_grad_gemm.hip and fmxq_grad_panel.hip
// share: the LDS layout of a 64-deep stage, buffer resources, and the epilogues.
//
// The weights are the first operand of v_mfma_f32_32x32x16_bf16, so a lane holds 16 columns
// of one output row (8 g + 4 h + 0..3 for g = 0..3, h its half of the wave): what a softmax
// wants of a row is reduced in registers, and stores take 4 neighbouring columns.
#pragma once
#include "fmxq_common.hpp"
#include "fmxq_grad.hpp"
#include "fmxq_lora_tile.hpp"

namespace fmxq {

typedef __attribute__((address_space(3))) void lds_t;

// 16-byte chunk c of row r sits at chunk position c ^ swz(r) of the row's 128 LDS bytes: 8
// consecutive rows at one chunk hit 8 distinct positions.
__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// s_waitcnt with vmcnt = vm and lgkmcnt = lgkm (expcnt left alone).
__device__ __forceinline__ constexpr int wait_enc(int vm, int lgkm) {
  return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8);
}

// A buffer of `bytes` at p, both the same in every lane.  They pass through readfirstlane
// because the compiler may hold a uniform value in vector registers, and then loops over the
// lanes' resources at every load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int64_t bytes) {
  const int64_t b = bytes < 0 ? 0 : bytes < 0x7fffffff ? bytes : 0x7fffffff;
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane((int)b), 0x00020000);
}

// dequantize's value: bf16(bf16(q s) + b), two at a time (low half first).  The empty asm hides
// where the pair comes from: the compiler takes a pack whose halves are used apart for two
// conversions.
__device__ __forceinline__ uint32_t deq_pair(float q0, float q1, float s0, float s1, float b0,
                                             float b1) {
  uint32_t m = pack_bf16x2(q0 * s0, q1 * s1);
  asm("" : "+v"(m));
  return pack_bf16x2(bf16_lo(m) + b0, bf16_hi(m) + b1);
}

// The other half of the wave's value.
__device__ __forceinline__ uint32_t other_half(uint32_t u) {
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return (threadIdx.x & 32) ? p[0] : p[1];
}
__device__ __forceinline__ float other_half(float v) {
  return __uint_as_float(other_half(__float_as_uint(v)));
}

// Rows mw .. of 32 MI (below mend), columns nw .. of 32 NJ: input gradients.
template <int MI, int NJ>
__device__ __forceinline__ void store_grad(const GradGemm& g, const f32x16 (&acc)[MI][NJ],
                                           int64_t mw, int64_t mend, int64_t nw, int64_t split) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    if (m >= mend) continue;
    if (g.y) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t n = nw + 32 * j + 8 * q + 4 * h;
          if (n < g.N)
            *reinterpret_cast<u32x2*>(g.y + m * g.ldy + n) =
                u32x2{pack_bf16x2(acc[i][j][4 * q], acc[i][j][4 * q + 1]),
                      pack_bf16x2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
        }
    } else {
      float* o = g.out + (split * g.M + m) * g.N;
      const float f = g.factor ? g.factor[m] : 1.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t n = nw + 32 * j + 8 * q + 4 * h;
          if (n >= g.N) continue;
          f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                     acc[i][j][4 * q + 3]};
          if (g.add) {
            const f32x4 old = *reinterpret_cast<const f32x4*>(o + n);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(old[e], f, v[e]);
          }
          *reinterpret_cast<f32x4*>(o + n) = v;
        }
    }
  }
}

// The column of an id that a row wants, counted from n0; ids of no token land behind the last.
__device__ __forceinline__ uint32_t wanted_column(const GradGemm& g, int32_t id, int64_t n0) {
  return id == g.wanted_none ? ~0u : (uint32_t)id - (uint32_t)(g.first_token + n0);
}

// out[i][j]: a bit for each of the 32 columns from nw + 32 j on that the lane's row of group i (from
// mw on) of the tile of BM x BN at (m0, n0) wants.  One id a row: the block has read them to `one`.
// Of more, all T threads of the block read the tile's rows' ids here, and their bits meet in
// `lds` (BM * BN / 8 bytes that no wave uses any more).
template <int BM, int BN, int T, int MI, int NJ>
__device__ __forceinline__ void find_wanted(const GradGemm& g, int64_t m0, int64_t rows, int64_t n0,
                                            int64_t mw, int64_t nw, const int32_t* one,
                                            uint32_t* lds, uint32_t (&out)[MI][NJ]) {
  const int r32 = threadIdx.x & 31;
  if (g.wanted_k == 1) {
    asm volatile("" ::: "memory");  // written before the steps' barriers
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const uint32_t c = wanted_column(g, one[mw - m0 + 32 * i + r32], nw);
#pragma unroll
      for (int j = 0; j < NJ; ++j) out[i][j] = c >> 5 == (uint32_t)j ? 1u << (c & 31) : 0u;
    }
    return;
  }
  const uint32_t k = (uint32_t)g.wanted_k, n = (uint32_t)rows * k;
  const uint32_t per_k = 0xffffffffu / k + 1;  // i / k as the high half of a product (i < 2^14)
  constexpr int B = 32;  // ids that are requested together
  int32_t id[B];
  auto load = [&](uint32_t i0) {
#pragma unroll
    for (int j = 0; j < B; ++j) id[j] = g.wanted[m0 * k + (i0 + j * T < n ? i0 + j * T : 0)];
  };
  load(threadIdx.x);
  __syncthreads();
  for (int i = threadIdx.x; i < BM * BN / 32; i += T) lds[i] = 0;
  __syncthreads();
  for (uint32_t i0 = threadIdx.x; i0 < n; i0 += B * T) {
    if (i0 >= B * T) load(i0);
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const uint32_t i = i0 + j * T, c = wanted_column(g, id[j], n0);
      if (c < BN && i < n) atomicOr(&lds[__umulhi(i, per_k) * (BN / 32) + (c >> 5)], 1u << (c & 31));
    }
  }
  __syncthreads();
  const uint32_t* mine = lds + (mw - m0 + r32) * (BN / 32) + (nw - n0) / 32;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) out[i][j] = mine[i * 32 * (BN / 32) + j];
}

// The softmax statistics of a tile of 32 NJ columns, and e.  They are relative to the nearest
// multiple of kStatStep (units of log 2) to the row's largest logit in the tile: bf16 and fp32
// keep their precision at any exponent, so tiles of a row whose logits reach about as far share
// one and need no rescaling, and where they differ 2^-kStatStep is still a normal number.
//
// The row's wanted tokens are left out, and enter the row's sums with its loss: where one of them
// takes nearly everything, what the others leave is the loss, and could not be had from a sum
// that holds both (out: find_wanted's bits).  A tile without other tokens has the sum 0 of kNoStat.
constexpr float kStatStep = 64.f;
constexpr float kNoStat = -3.4028234663852886e38f;  // below every tile's; differences stay numbers

template <int MI, int NJ>
__device__ __forceinline__ void store_stats(const GradGemm& g, f32x16 (&acc)[MI][NJ],
                                            const uint32_t (&out)[MI][NJ], int64_t mw, int64_t mend,
                                            int64_t nw) {
  // The scaled logits are rounded once and the same values everywhere: an unrounded product
  // passes the largest one by half a unit, which among logits of 1e10 is no power of two.
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  if (nw >= g.N) {  // no token here: zeros where a product reads whole tiles
    if (g.e)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t m = mw + 32 * i + r32, n = nw + 32 * j + 8 * q + 4 * h;
            if (m < mend && n < g.lde) *reinterpret_cast<u32x2*>(g.e + m * g.lde + n) = u32x2{0u, 0u};
          }
    return;
  }
  const bool full = nw + 32 * NJ <= g.N;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    uint32_t some = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) some |= out[i][j];
    if (__any(some != 0))
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (!__any(out[i][j] != 0)) continue;
        const uint32_t mine = out[i][j] >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((mine >> (8 * (r >> 2) + (r & 3))) & 1u) acc[i][j][r] = -INFINITY;
      }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[i][j][r] *= g.logit_scale;
        if (full || nw + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3) < g.N) top = fmaxf(top, acc[i][j][r]);
      }
    top = fmaxf(top, other_half(top));
    const float mx = top == -INFINITY ? kNoStat : kStatStep * rintf(top * (1.f / kStatStep));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = nw + 32 * j + 8 * q + 4 * h;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = __builtin_amdgcn_exp2f(acc[i][j][4 * q + e] - mx);
          if (!full && n + e >= g.N) v[e] = 0.f;
          sum += v[e];
        }
        if (g.e && m < mend)
          *reinterpret_cast<u32x2*>(g.e + m * g.lde + n) =
              u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    sum += other_half(sum);
    if (h == 0 && m < mend) g.stats[m * g.stat_tiles + nw / (32 * NJ)] = make_float2(mx, sum);
  }
}

// What log probabilities need of a tile of 32 NJ columns (HeadTile), in units of log 2: its largest
// logit m and the first column that has it, and of the other columns the sums of 2^(l - m) and of
// 2^(l - m) (m - l).  That column takes no part in the sums, so that where one token takes nearly
// everything, what the others leave is not the difference of near equals.  A logit of minus infinity (0
// times infinity in the second sum), as any other that is not finite, leaves NaN.  With e, also
// bf16(2^(l - m)), zeros from column N to the tile's end.
template <int MI, int NJ>
__device__ __forceinline__ void store_scores(const GradGemm& g, f32x16 (&acc)[MI][NJ], int64_t mw,
                                             int64_t mend, int64_t nw) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  if (nw >= g.N) return;
  const int left = g.N - nw < 32 * NJ ? (int)(g.N - nw) : 32 * NJ;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[i][j][r] *= g.logit_scale;
        if (32 * j + 8 * (r >> 2) + 4 * h + (r & 3) < left) top = fmaxf(top, acc[i][j][r]);
      }
    top = fmaxf(top, other_half(top));
    uint32_t first = 32 * NJ;
#pragma unroll
    for (int j = NJ - 1; j >= 0; --j)
#pragma unroll
      for (int r = 15; r >= 0; --r) {
        const uint32_t c = 32 * j + 8 * (r >> 2) + 4 * h + (r & 3);
        if (acc[i][j][r] == top && (int)c < left) first = c;
      }
    const uint32_t theirs = other_half(first);
    first = first < theirs ? first : theirs;
    float sum = 0.f, low = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * j + 8 * q + 4 * h;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = top - acc[i][j][4 * q + e];
          v[e] = c + e < left ? __builtin_amdgcn_exp2f(-d) : 0.f;
          const float w = (uint32_t)(c + e) == first || c + e >= left ? 0.f : v[e];
          sum += w;
          low = __builtin_fmaf(w, c + e < left ? d : 0.f, low);
        }
        if (g.e && m < mend)
          *reinterpret_cast<u32x2*>(g.e + m * g.lde + nw + c) =
              u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    sum += other_half(sum);
    low += other_half(low);
    if (h == 0 && m < mend)
      g.score[m * g.stat_tiles + nw / (32 * NJ)] = HeadTile{top, sum, low, first};
  }
}

// The gradient of log probabilities and entropy for the logits of a tile:
//   d = -p (a + c (log p + entropy)),  p = 2^(l - lse),
// as bf16 in e, zeros for the row's wanted tokens (whose share enters later, in fp32) and from column N to
// the tile's end.  bf16, which the product behind takes: an entry is off by 2^-8 of itself at most, as in the
// losses' gradients, before the result's own rounding.  (1000 rows, 128256 x 4096: dh is 0.00184 off in the 2-norm,
// of which its own rounding alone is 0.00166; 37 rows 0.00169.  What is left in a second bf16 value would be
// as many rows again for that product: 1.08 and 1.96 ms of a step of 3.3.)
template <int MI, int NJ>
__device__ __forceinline__ void store_coef(const GradGemm& g, const f32x16 (&acc)[MI][NJ],
                                           const uint32_t (&out)[MI][NJ], int64_t mw, int64_t mend,
                                           int64_t nw) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int64_t ln = g.N - nw;
  const int left = ln < 0 ? 0 : ln < 32 * NJ ? (int)ln : 32 * NJ;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    const f32x4 row = reinterpret_cast<const f32x4*>(g.rows)[m < mend ? m : mend - 1];
    const float lse = row[0], a = row[1], c2 = row[2];  // c in units of log 2, c entropy in a
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t mine = out[i][j] >> (4 * h);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * j + 8 * q + 4 * h;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lp = __builtin_fmaf(acc[i][j][4 * q + e], g.logit_scale, -lse);
          const float p = __builtin_amdgcn_exp2f(lp);
          v[e] = -p * __builtin_fmaf(c2, lp, a);
          if (p == 0.f || c + e >= left || ((mine >> (8 * q + e)) & 1u)) v[e] = 0.f;
        }
        if (m < mend && nw + c < g.lde)
          *reinterpret_cast<u32x2*>(g.e + m * g.lde + nw + c) =
              u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    }
  }
}

// The product itself: rows of y, of any width, or a part's fp32 slice (N a multiple of 4).
template <int MI, int NJ>
__device__ __forceinline__ void store_out(const GradGemm& g, f32x16 (&acc)[MI][NJ], int64_t mw,
                                          int64_t mend, int64_t nw, int64_t split) {
  if (g.lora.u && split == 0)
    add_lora<MI, NJ>(g.lora, [&](int i, int j) -> f32x16& { return acc[i][j]; }, mw, mend, nw, g.N);
  if (!g.y || ((g.N | g.ldy) & 3) == 0) {
    store_grad<MI, NJ>(g, acc, mw, mend, nw, split);
    return;
  }
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    if (m >= mend) continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t n = nw + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3);
        if (n < g.N) g.y[m * g.ldy + n] = (uint16_t)f32_to_bf16_rne(acc[i][j][r]);
      }
  }
}

// Whether an epilogue leaves out the row's wanted tokens.
constexpr bool epi_wants(int epi) { return epi == kEpiStats || epi == kEpiCoef; }

// A tile's epilogue of logits.
template <int EPI, int MI, int NJ>
__device__ __forceinline__ void store_logits(const GradGemm& g, f32x16 (&acc)[MI][NJ],
                                             const uint32_t (&out)[MI][NJ], int64_t mw, int64_t mend,
                                             int64_t nw, int64_t split) {
  if constexpr (EPI == kEpiStats) store_stats<MI, NJ>(g, acc, out, mw, mend, nw);
  else if constexpr (EPI == kEpiScores) store_scores<MI, NJ>(g, acc, mw, mend, nw);
  else if constexpr (EPI == kEpiOut) store_out<MI, NJ>(g, acc, mw, mend, nw, split);
  else store_coef<MI, NJ>(g, acc, out, mw, mend, nw);
}

}  // namespace fmxq
