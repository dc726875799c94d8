// fmxq_thin.hip -- products x . deq(W)^T of up to 16 rows with fmxq_dequantize's bits: outputs with an
// adapter's part, or logits with what log probabilities need of them.
//
// A block takes 16 weight rows and its 8 waves steps of 256 values in turn: lane r16 of quarter q4 holds
// values 64 q4 .. + 64 of row r16, so a wave's loads of a step are whole 128-byte lines (4 bits; 256
// bytes at 8), and any two lanes of a quarter share x's addresses.  16x16x32 MFMAs take the lane's chunks of
// 8 values in order, weights first: a lane ends with outputs 4 q4 .. + 4 of row r16 of x.
//
// Bound: the dequantization's VALU instructions (5 a weight: two roundings; 6.4e12 weights a second
// on the whole chip), and for small matrices the launch, the loads' latency and the sum over waves.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_grad_tile.hpp"
#include "fmxq_mfma_frag.hpp"

namespace fmxq {
namespace {

constexpr int kStep = 256;  // values of a wave's step
constexpr uint32_t kOut = 0x7ffffff0u;  // an offset past every buffer: loads give zero

template <int BITS, int GS, int EPI>
__global__ __launch_bounds__(512, 8) void thin_kernel(GradGemm g) {
  constexpr int NW = BITS / 2;             // 16-byte loads of a lane's weights in a step
  constexpr int NG = GS < 64 ? 64 / GS : 1;  // groups of a lane's 64 values
  __shared__ f32x4 part[8][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int K = (int)g.C, steps = (K + kStep - 1) / kStep;
  const int64_t wpr = (int64_t)K * BITS / 32, gpr = K / GS;
  const int64_t rows = g.N - n0 < 16 ? g.N - n0 : 16;
  const __amdgpu_buffer_rsrc_t wr = rsrc(g.w + n0 * wpr, rows * wpr * 4);
  const __amdgpu_buffer_rsrc_t sr = rsrc(g.scales + n0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t br = rsrc(g.biases + n0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t xr = rsrc(g.a, g.M * g.lda * 2);
  const uint32_t wo = (uint32_t)(r16 * wpr * 4), so = (uint32_t)(r16 * gpr * 2);
  // Rows past M read the last one's values and are not stored.
  const uint32_t xo = (uint32_t)((r16 < g.M ? r16 : g.M - 1) * g.lda * 2);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  struct Weights {
    u32x4 w[NW];
    uint16_t s[NG], b[NG];
  };
  // Values past the row are those of scale and bias 0.
  auto load = [&](int step, Weights& p) {
    const int k = kStep * step + 64 * q4;
    const uint32_t o = step < steps && k < K ? wo + (uint32_t)(k * BITS / 8) : kOut;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      p.w[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, (int)o, 16 * i, 0));
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const uint32_t so_i = step < steps && k + GS * i < K ? so + (uint32_t)((k + GS * i) / GS * 2) : kOut;
      p.s[i] = __builtin_amdgcn_raw_buffer_load_b16(sr, (int)so_i, 0, 0);
      p.b[i] = __builtin_amdgcn_raw_buffer_load_b16(br, (int)so_i, 0, 0);
    }
  };
  Weights w;
  load(wave, w);
  for (int step = wave; step < steps; step += 8) {
    const int k = kStep * step + 64 * q4;
    Weights next;
    load(step + 8, next);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x4 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int kc = k + 32 * half + 8 * c;
        x[c] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(xr, (int)(kc < K ? xo + (uint32_t)(kc * 2) : kOut), 0, 0));
      }
      const int gi = NG > 1 ? half * NG / 2 : 0;
      const bool in = k + 32 * half < K;  // (the second half of a row's last 64 may be past it)
      const float s = in ? bf16_bits_to_f32(w.s[gi]) : 0.f, b = in ? bf16_bits_to_f32(w.b[gi]) : 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        bf16x8 f;
        if constexpr (BITS == 4) f = deq_exact4(w.w[half][c], s, s * 0.0625f, b);
        else f = deq_exact8(w.w[2 * half + c / 2][2 * (c & 1)], w.w[2 * half + c / 2][2 * (c & 1) + 1], s, b);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, x[c]), acc, 0, 0, 0);
      }
    }
    w = next;
  }
  part[wave][lane] = acc;
  __syncthreads();
  if constexpr (EPI == kEpiOut) {
    // Thread: one output of one row.
    if (tid >= 256) return;
    const int m = tid >> 4, i = tid & 15;
    if (m >= g.M || n0 + i >= g.N) return;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += part[k][16 * (i >> 2) + m][i & 3];
    const int e = g.lora.u ? adapter_of(g.lora, m) : -1;
    if (e >= 0) v += lora_value(g.lora, e, m, n0 + i);
    g.y[m * g.ldy + n0 + i] = (uint16_t)f32_to_bf16_rne(v);
  } else {
    // One wave: lane (row of x, 4 tokens); as store_scores.
#pragma clang fp contract(off)
    if (wave) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) v += part[k][lane];
    const int left = (int)rows;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] *= g.logit_scale;
      if (4 * q4 + i < left) top = fmaxf(top, v[i]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int first = 16;
#pragma unroll
    for (int i = 3; i >= 0; --i)
      if (v[i] == top && 4 * q4 + i < left) first = 4 * q4 + i;
    int o = __shfl_xor(first, 16, 64);
    first = first < o ? first : o;
    o = __shfl_xor(first, 32, 64);
    first = first < o ? first : o;
    float sum = 0.f, low = 0.f, ex[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 4 * q4 + i;
      const float d = top - v[i];
      ex[i] = c < left ? __builtin_amdgcn_exp2f(-d) : 0.f;
      const float t = c == first || c >= left ? 0.f : ex[i];
      sum += t;
      low = __builtin_fmaf(t, c < left ? d : 0.f, low);
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    low += __shfl_xor(low, 16, 64);
    low += __shfl_xor(low, 32, 64);
    if (r16 >= g.M) return;
    if (g.e)
      *reinterpret_cast<u32x2*>(g.e + r16 * g.lde + n0 + 4 * q4) =
          u32x2{pack_bf16x2(ex[0], ex[1]), pack_bf16x2(ex[2], ex[3])};
    if (q4 == 0) g.score[r16 * g.stat_tiles + blockIdx.x] = HeadTile{top, sum, low, (uint32_t)first};
  }
}

template <int BITS, int GS>
hipError_t launch_thin(const GradGemm& g, hipStream_t stream) {
  const int64_t blocks = (g.N + 15) / 16;
  if (blocks >= kMaxBlocks) return hipErrorInvalidConfiguration;
  if (g.epi == kEpiOut) thin_kernel<BITS, GS, kEpiOut><<<(unsigned)blocks, 512, 0, stream>>>(g);
  else thin_kernel<BITS, GS, kEpiScores><<<(unsigned)blocks, 512, 0, stream>>>(g);
  return hipGetLastError();
}

}  // namespace

// Byte offsets of 16 rows are 32 bits: x, 8-bit weights.
static bool row_ok(int64_t K) { return 16 * K * 2 < 0x7ffffff0LL; }
bool thin_supported(int64_t M, int64_t N, int64_t K) {
  if (M > kThinRows || !row_ok(K) || (N + 15) / 16 >= kMaxBlocks) return false;
  return M <= 4 || N <= ((int64_t)1 << 29) / M / std::max<int64_t>(K, 1);
}

hipError_t launch_thin_gemm(const GradGemm& g, hipStream_t stream) {
  if (!g.a || !g.w || !logits_operands(g) || (g.epi != kEpiOut && g.epi != kEpiScores) || (g.epi == kEpiOut && !g.y) ||
      g.M > kThinRows || !row_ok(g.lda) || !row_ok(g.C) || g.lda % 8 || g.splits != 1)
    return hipErrorInvalidValue;
  if (g.M < 1 || g.N < 1) return hipSuccess;
  if (g.bits == 4)
    return g.group_size == 32   ? launch_thin<4, 32>(g, stream)
           : g.group_size == 64 ? launch_thin<4, 64>(g, stream)
                                : launch_thin<4, 128>(g, stream);
  return g.group_size == 32   ? launch_thin<8, 32>(g, stream)
         : g.group_size == 64 ? launch_thin<8, 64>(g, stream)
                              : launch_thin<8, 128>(g, stream);
}

}  // namespace fmxq
