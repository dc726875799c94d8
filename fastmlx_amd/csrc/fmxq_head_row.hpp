// fmxq_head_row.hpp -- single rows of a quantized head, as the losses (fmxq_head.hip) and the log
// probabilities (fmxq_logprobs.hip) read them.
#pragma once
#include "fmxq_common.hpp"
#include "fmxq_grad_tile.hpp"

namespace fmxq {

// 8 packed values of row `row`, which is the same in every lane, from column c on.
struct Packed8 {
  u32x2 w;
  uint16_t s, b;
};
template <class Args>
__device__ __forceinline__ Packed8 load8(const Args& a, int row, int c) {
  const int64_t r = __builtin_amdgcn_readfirstlane(row);
  const int gs = __builtin_ctz(a.group_size);
  const int64_t g0 = r * (a.K >> gs);
  Packed8 p;
  if (a.bits == 4) p.w = u32x2{(a.w + r * (a.K >> 3))[(uint32_t)c >> 3], 0u};
  else p.w = *reinterpret_cast<const u32x2*>(a.w + r * (a.K >> 2) + ((uint32_t)c >> 2));
  p.s = (a.scales + g0)[(uint32_t)c >> gs];
  p.b = (a.biases + g0)[(uint32_t)c >> gs];
  return p;
}

// Their dequantized values (fmxq_dequantize's bits).
__device__ __forceinline__ void deq8(const Packed8& p, int bits, float* v) {
  const float s = bf16_bits_to_f32(p.s), b = bf16_bits_to_f32(p.b);
  // Bytes: the even and the odd values.
  uint32_t lo = p.w[0] & 0x0F0F0F0Fu, hi = (p.w[0] >> 4) & 0x0F0F0F0Fu;
  if (bits == 8) {
    lo = __builtin_amdgcn_perm(p.w[1], p.w[0], 0x06040200u);
    hi = __builtin_amdgcn_perm(p.w[1], p.w[0], 0x07050301u);
  }
  asm("" : "+v"(lo), "+v"(hi));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t t = deq_pair((float)((lo >> (8 * j)) & 0xffu), (float)((hi >> (8 * j)) & 0xffu), s,
                                s, b, b);
    v[2 * j] = bf16_lo(t);
    v[2 * j + 1] = bf16_hi(t);
  }
}

}  // namespace fmxq
