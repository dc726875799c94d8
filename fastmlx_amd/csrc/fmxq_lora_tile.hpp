// fmxq_lora_tile.hpp -- an adapter's part in the epilogue of a product.
#pragma once
#include "fmxq_common.hpp"
#include "fmxq_grad.hpp"

namespace fmxq {

// A row's adapter, or -1.
__device__ __forceinline__ int adapter_of(const LoraAdd& l, int64_t m) {
  const int e = l.ids[m];
  return e >= 0 && e < l.E ? e : -1;
}

// The adapters' part of a tile of N columns in all: rows mw .. of 32 MI (below mend), columns nw .. of 32
// NJ, in accumulators at(i, j) of products whose first operand were the weights.  Rows of 32 that share
// an adapter add it to the sums; others take the adapters in turn, each apart, so that one's infinities
// reach its own rows only.  (All groups of a wave at once would hide more of the loads, but the branches
// around so many accumulators spill them.)
template <int MI, int NJ, class At>
__device__ __forceinline__ void add_lora(const LoraAdd& l, At&& at, int64_t mw, int64_t mend, int64_t nw,
                                         int64_t N) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int chunks = l.r / 8, steps = (chunks + 1) / 2;
  if (nw >= N) return;
  int64_t n[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) n[j] = (nw + 32 * j + r32 < N ? nw + 32 * j + r32 : N - 1) * l.r;
  int e[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    e[i] = adapter_of(l, m < mend ? m : mend - 1);
    if (m >= mend) e[i] = -1;
  }
  const u32x4 zero = {0u, 0u, 0u, 0u};
  auto load = [&](const uint16_t* p, int c) {
    return __builtin_bit_cast(bf16x8, c < chunks ? *reinterpret_cast<const u32x4*>(p + 8 * c) : zero);
  };
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = mw + 32 * i + r32;
    const bool in = m < mend;
    uint64_t some = __ballot(e[i] >= 0);
    if (!some) continue;
    const uint16_t* u = l.u + (in ? m : mend - 1) * l.parts * l.r;
    const int first = __builtin_amdgcn_readlane(e[i], __builtin_ctzll(some));
    if (__ballot(!in || e[i] == first) == ~0ull) {
      const uint16_t* v = l.v + (int64_t)first * l.n * l.r;
      for (int s = 0; s < steps; s += 2) {
        bf16x8 u0[2], u1[2], b[2][NJ];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          u0[k] = load(u, 2 * (s + k) + h);
          u1[k] = load(u + l.r, 2 * (s + k) + h);
#pragma unroll
          for (int j = 0; j < NJ; ++j) b[k][j] = load(v + n[j], 2 * (s + k) + h);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            at(i, j) = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[k][j], u0[k], at(i, j), 0, 0, 0);
            at(i, j) = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[k][j], u1[k], at(i, j), 0, 0, 0);
          }
      }
      continue;
    }
    while (some) {
      const int cur = __builtin_amdgcn_readlane(e[i], __builtin_ctzll(some));
      const uint16_t* v = l.v + (int64_t)cur * l.n * l.r;
      const bool mine = e[i] == cur;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        f32x16 t;
#pragma unroll
        for (int x = 0; x < 16; ++x) t[x] = 0.f;
        for (int s = 0; s < steps; ++s) {
          const bf16x8 u0 = load(u, 2 * s + h), u1 = load(u + l.r, 2 * s + h);
          const bf16x8 b = load(v + n[j], 2 * s + h);
          t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, u0, t, 0, 0, 0);
          t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, u1, t, 0, 0, 0);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) at(i, j)[x] += mine ? t[x] : 0.f;
      }
      if (mine) e[i] = -1;
      some = __ballot(e[i] >= 0);
    }
  }
}

// The same for one row and four neighbouring columns from n on (all of them in the adapter's rows of
// v), added to v4.
__device__ __forceinline__ void add_lora4(const LoraAdd& l, int e, int64_t m, int64_t n, f32x4& v4) {
  const uint16_t* u = l.u + m * l.parts * l.r;
  const uint16_t* b = l.v + ((int64_t)e * l.n + n) * l.r;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int j = 0; j < l.r; j += 8) {
    const u32x4 u0 = *reinterpret_cast<const u32x4*>(u + j), u1 = *reinterpret_cast<const u32x4*>(u + l.r + j);
    u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const u32x4*>(b + i * l.r + j);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float lo = bf16_lo(u0[k]) + bf16_lo(u1[k]), hi = bf16_hi(u0[k]) + bf16_hi(u1[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = __builtin_fmaf(bf16_lo(w[i][k]), lo, s[i]);
        s[i] = __builtin_fmaf(bf16_hi(w[i][k]), hi, s[i]);
      }
    }
  }
  v4 += s;
}

// ... and for one row and column.
__device__ __forceinline__ float lora_value(const LoraAdd& l, int e, int64_t m, int64_t n) {
  const uint16_t* u = l.u + m * l.parts * l.r;
  const uint16_t* b = l.v + ((int64_t)e * l.n + n) * l.r;
  float s = 0.f;
#pragma unroll 4
  for (int j = 0; j < l.r; j += 8) {
    const u32x4 u0 = *reinterpret_cast<const u32x4*>(u + j), u1 = *reinterpret_cast<const u32x4*>(u + l.r + j);
    const u32x4 w = *reinterpret_cast<const u32x4*>(b + j);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s = __builtin_fmaf(bf16_lo(w[k]), bf16_lo(u0[k]) + bf16_lo(u1[k]), s);
      s = __builtin_fmaf(bf16_hi(w[k]), bf16_hi(u0[k]) + bf16_hi(u1[k]), s);
    }
  }
  return s;
}

}  // namespace fmxq
