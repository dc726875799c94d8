// fmxq_grad_skinny.hip -- the products of fmxq_grad_gemm.hip for up to 64 rows, where the
// packed weights are the work: every weight is read and dequantized once, in the registers
// of the wave that multiplies it, with no stage in LDS and no barrier before the last sum.
//
// Logits: a block takes 32 tokens and its 8 waves every eighth 64-deep step of the hidden
// width; a lane holds 32 values of one token's row.
// Input gradients: a block takes 256 outputs and its waves share the contraction in steps of
// 16 weight rows; lane r32 of half h holds the word of outputs 8 r32 .. + 8 in rows 8 h ..
// + 8, and matrix column r32 of tile j is output 8 r32 + j, so that a word's values go to
// eight tiles and never have to cross lanes.  With two row tiles (more than 32 rows) a wave
// takes four of the eight.
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr uint32_t kOut = 0x7ffffff0u;  // an offset past every buffer: loads give zero

template <int BITS, int MT>
__global__ __launch_bounds__(512, 2) void logits_skinny_kernel(GradGemm g) {
  constexpr int NW = BITS / 4;  // 16-byte weight loads per lane and step
  __shared__ __attribute__((aligned(16))) float part[8 * MT * 1024];
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const int K = (int)g.C;
  const int64_t wpr = (int64_t)K * BITS / 32, gpr = K / g.group_size;
  const int gs = __builtin_ctz(g.group_size);
  const int64_t rows = g.N - n0 < 32 ? g.N - n0 : 32;
  const __amdgpu_buffer_rsrc_t wr = rsrc(g.w + n0 * wpr, rows * wpr * 4);
  const __amdgpu_buffer_rsrc_t sr = rsrc(g.scales + n0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t br = rsrc(g.biases + n0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t ar = rsrc(g.a, g.M * g.lda * 2);
  // Rows of x past M lie past its buffer.
  uint32_t ao[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) ao[i] = (uint32_t)((r32 + 32 * i) * g.lda * 2);
  const int wo = r32 * (int)wpr * 4;

  struct Step {
    u32x4 w[NW], x[MT][4];
    uint16_t s, b;
  };
  // A half past the row's end (and a step past the last) takes the row's last values against
  // zeros of x.
  auto load = [&](int step, Step& p) {
    const int k = 64 * step + 32 * h, kw = k < K ? k : K - 32;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      p.w[i] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, wo + kw * BITS / 8, 16 * i, 0));
    const int so = (r32 * (int)gpr + (kw >> gs)) * 2;
    p.s = __builtin_amdgcn_raw_buffer_load_b16(sr, so, 0, 0);
    p.b = __builtin_amdgcn_raw_buffer_load_b16(br, so, 0, 0);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint32_t o = k < K ? ao[m] + 2 * k : kOut;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p.x[m][i] =
            __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ar, (int)o, 16 * i, 0));
    }
  };
  f32x16 acc[MT][1];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[m][0][r] = 0.f;
  auto use = [&](const Step& p) {
    const float s = bf16_bits_to_f32(p.s), b = bf16_bits_to_f32(p.b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 o;
      if constexpr (BITS == 4) {
        uint32_t e = p.w[0][i] & 0x0F0F0F0Fu, d = (p.w[0][i] >> 4) & 0x0F0F0F0Fu;
        asm("" : "+v"(e), "+v"(d));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = deq_pair((float)((e >> (8 * j)) & 0xffu), (float)((d >> (8 * j)) & 0xffu), s, s, b, b);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t v = p.w[i >> 1][2 * (i & 1) + (j >> 1)] >> (16 * (j & 1));
          o[j] = deq_pair((float)(v & 0xffu), (float)((v >> 8) & 0xffu), s, s, b, b);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[m][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, o),
                                                            __builtin_bit_cast(bf16x8, p.x[m][i]),
                                                            acc[m][0], 0, 0, 0);
    }
  };
  const int steps = (K + 63) / 64;
  Step p0, p1;
  load(wave, p0);
  for (int k = wave; k < steps; k += 16) {
    load(k + 8, p1);
    use(p0);
    load(k + 16, p0);
    use(p1);
  }
  // The waves' sums, in the order of the waves; wave m finishes row tile m.
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(part + (((wave * MT + m) * 4 + q) * 64 + lane) * 4) =
          f32x4{acc[m][0][4 * q], acc[m][0][4 * q + 1], acc[m][0][4 * q + 2], acc[m][0][4 * q + 3]};
  __syncthreads();
  if (wave >= MT) return;
  f32x16 sum[1][1];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(part + (((w * MT + wave) * 4 + q) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += u[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[0][0][4 * q + e] = v[e];
  }
  store_stats<1, 1>(g, sum, 32 * wave, g.M, n0);
}

template <int BITS, int MT, bool G32>
__global__ __launch_bounds__(512, 2) void grad_skinny_kernel(GradGemm g) {
  constexpr int JN = 8 / MT, NP = 8 / MT;  // tiles of a wave, waves along the contraction
  constexpr int NG = G32 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float part[2][8 * 1024];
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave % MT, np = wave / MT;
  const int64_t tn = (g.N + kGradTileCols - 1) / kGradTileCols;
  const int64_t split = blockIdx.x / tn, n0 = blockIdx.x % tn * kGradTileCols;
  const int64_t c0 = split * g.c_split;
  const int64_t c1 = c0 + g.c_split < g.C ? c0 + g.c_split : g.C;
  const int64_t wpr = g.N * BITS / 32, gpr = g.N / g.group_size;
  const int64_t rows = c1 > c0 ? c1 - c0 : 0;
  const __amdgpu_buffer_rsrc_t wr = rsrc(g.w + c0 * wpr, rows * wpr * 4);
  const __amdgpu_buffer_rsrc_t sr = rsrc(g.scales + c0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t br = rsrc(g.biases + c0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t ar = rsrc(g.a, g.M * g.lda * 2);
  // Columns past the weight's last are clamped into its rows; they are not stored.
  const int64_t unit = n0 / 8 + r32 < g.N / 8 ? n0 / 8 + r32 : g.N / 8 - 1;
  constexpr bool kPair = BITS == 8 && MT == 1;  // both words of a unit
  const uint32_t wo = (uint32_t)(8 * h * wpr * 4 + unit * BITS + (BITS == 8 && MT == 2 ? 4 * half : 0));
  // Scales: lane i of an octet (whose 64 columns share a group; 32 of them in groups of 32)
  // loads row i's and the others take it from there.
  const int srow = 8 * h + (G32 ? r32 & 3 : r32 & 7);
  const uint32_t so = (uint32_t)((srow * gpr + unit * 8 / g.group_size) * 2);
  uint32_t ao[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) ao[m] = (uint32_t)((r32 + 32 * m) * g.lda * 2);
  const uint32_t acols = (uint32_t)g.a_cols;

  struct Step {
    uint32_t w[kPair ? 16 : 8];
    u32x4 a[MT];
    uint16_t s[NG], b[NG];
  };
  // Rows past the part lie past its buffers.
  auto load = [&](int step, Step& p) {
    const uint32_t r = 16 * (uint32_t)step, o = wo + r * (uint32_t)(wpr * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int oi = (int)(o + (uint32_t)(i * wpr * 4));
      if constexpr (kPair) {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(wr, oi, 0, 0));
        p.w[2 * i] = v[0];
        p.w[2 * i + 1] = v[1];
      } else {
        p.w[i] = __builtin_amdgcn_raw_buffer_load_b32(wr, oi, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int oi = (int)(so + (r + 4 * i) * (uint32_t)(gpr * 2));
      p.s[i] = __builtin_amdgcn_raw_buffer_load_b16(sr, oi, 0, 0);
      p.b[i] = __builtin_amdgcn_raw_buffer_load_b16(br, oi, 0, 0);
    }
    const uint32_t col = (uint32_t)c0 + r + 8 * h;
#pragma unroll
    for (int m = 0; m < MT; ++m)
      p.a[m] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             ar, (int)(col < acols ? ao[m] + 2 * col : kOut), 0, 0));
  };
  f32x16 acc[JN][MT];
#pragma unroll
  for (int j = 0; j < JN; ++j)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][m][r] = 0.f;
  auto use = [&](const Step& p) {
    uint32_t sb[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) sb[i] = (uint32_t)p.s[i] | ((uint32_t)p.b[i] << 16);
    uint32_t rs[8];
    auto from = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      // Lane (octet, or half octet, of this one) | i.
      constexpr int pattern = G32 ? (0x1c | ((i & 3) << 5)) : (0x18 | (i << 5));
      rs[i] = (uint32_t)__builtin_amdgcn_ds_swizzle((int)sb[G32 ? i >> 2 : 0], pattern);
    };
    from(std::integral_constant<int, 0>{});
    from(std::integral_constant<int, 1>{});
    from(std::integral_constant<int, 2>{});
    from(std::integral_constant<int, 3>{});
    from(std::integral_constant<int, 4>{});
    from(std::integral_constant<int, 5>{});
    from(std::integral_constant<int, 6>{});
    from(std::integral_constant<int, 7>{});
    uint32_t lo[8], hi[8];  // the rows' values of even and odd columns (4 bits), or bytes
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (BITS == 4) {
        const uint32_t v = MT == 2 && half ? p.w[i] >> 16 : p.w[i];
        lo[i] = v & 0x0F0F0F0Fu;
        hi[i] = (v >> 4) & 0x0F0F0F0Fu;
      } else if constexpr (kPair) {
        lo[i] = p.w[2 * i];
        hi[i] = p.w[2 * i + 1];
      } else {
        lo[i] = p.w[i];
        hi[i] = 0;
      }
      asm("" : "+v"(lo[i]), "+v"(hi[i]));
    }
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      auto value = [&](int i) {
        if constexpr (BITS == 4) return (float)(((j & 1 ? hi[i] : lo[i]) >> (8 * (j >> 1))) & 0xffu);
        else return (float)(((j < 4 ? lo[i] : hi[i]) >> (8 * (j & 3))) & 0xffu);
      };
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = deq_pair(value(2 * i), value(2 * i + 1), bf16_lo(rs[2 * i]), bf16_lo(rs[2 * i + 1]),
                        bf16_hi(rs[2 * i]), bf16_hi(rs[2 * i + 1]));
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[j][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, o),
                                                            __builtin_bit_cast(bf16x8, p.a[m]),
                                                            acc[j][m], 0, 0, 0);
    }
  };
  const int steps = (int)((rows + 15) / 16);
  Step p0, p1;
  load(np, p0);
  for (int k = np; k < steps; k += 2 * NP) {
    load(k + NP, p1);
    use(p0);
    load(k + 2 * NP, p0);
    use(p1);
  }
  // Tile by tile the waves' sums meet in LDS; a thread adds the NP of 2 MT registers of one
  // lane and keeps them, and ends up with JN neighbouring outputs of each.
  constexpr int TR = 2 * MT, PL = 16 / TR;  // registers of a thread, threads of a lane
  const int th = tid / (512 / MT), in = tid % (512 / MT), ln = in / PL, r0 = in % PL * TR;
  float out[JN][MT][TR];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int j = t / MT, m = t % MT;
    float* buf = part[t & 1];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(buf + ((wave * 4 + q) * 64 + lane) * 4) = f32x4{
          acc[j][m][4 * q], acc[j][m][4 * q + 1], acc[j][m][4 * q + 2], acc[j][m][4 * q + 3]};
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TR; ++r) out[j][m][r] = 0.f;
#pragma unroll
    for (int w = 0; w < NP; ++w) {
      const float* v = buf + (((w * MT + th) * 4 + r0 / 4) * 64 + ln) * 4 + r0 % 4;
#pragma unroll
      for (int r = 0; r < TR; ++r) out[j][m][r] += v[r];
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = (ln & 31) + 32 * m;
    if (row >= g.M) continue;
    const float f = g.factor ? g.factor[row] : 0.f;
#pragma unroll
    for (int r = 0; r < TR; ++r) {
      const int reg = r0 + r;
      const int64_t n = n0 + 8 * (8 * (reg >> 2) + 4 * (ln >> 5) + (reg & 3)) + JN * th;
      if (n >= g.N) continue;
      if (g.y) {
#pragma unroll
        for (int j = 0; j < JN; j += 4)
          *reinterpret_cast<u32x2*>(g.y + row * g.ldy + n + j) =
              u32x2{pack_bf16x2(out[j][m][r], out[j + 1][m][r]),
                    pack_bf16x2(out[j + 2][m][r], out[j + 3][m][r])};
      } else {
        float* o = g.out + (split * g.M + row) * g.N + n;
#pragma unroll
        for (int j = 0; j < JN; j += 4) {
          f32x4 v = {out[j][m][r], out[j + 1][m][r], out[j + 2][m][r], out[j + 3][m][r]};
          if (g.factor) {
            const f32x4 old = *reinterpret_cast<const f32x4*>(o + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(old[e], f, v[e]);
          }
          *reinterpret_cast<f32x4*>(o + j) = v;
        }
      }
    }
  }
}

template <int BITS, int MT>
hipError_t launch(const GradGemm& g, bool nn, hipStream_t stream) {
  if (!nn) {
    const int64_t blocks = (g.N + 31) / 32;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    logits_skinny_kernel<BITS, MT><<<(unsigned)blocks, 512, 0, stream>>>(g);
  } else {
    const int64_t blocks = (g.N + kGradTileCols - 1) / kGradTileCols * g.splits;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (g.group_size == 32) grad_skinny_kernel<BITS, MT, true><<<(unsigned)blocks, 512, 0, stream>>>(g);
    else grad_skinny_kernel<BITS, MT, false><<<(unsigned)blocks, 512, 0, stream>>>(g);
  }
  return hipGetLastError();
}

}  // namespace

// Byte offsets of a call's rows are 32 bits: 64 rows of x, 32 weight rows of the logits, a
// part's weight rows of the gradient and the steps that are requested past its end.
bool skinny_gemm_supported(int64_t M, int64_t lda, int64_t weight_rows, int64_t weight_cols) {
  return M <= kSkinnyRows && 64 * lda * 2 < 0x7ffffff0LL &&
         (weight_rows + 1024) * weight_cols < 0x7fff0000LL;
}

hipError_t launch_skinny_gemm(const GradGemm& g, bool nn, hipStream_t stream) {
  if (!skinny_gemm_supported(g.M, g.lda, nn ? g.c_split : 32, nn ? g.N : g.C) || g.tiles || g.lda % 8 ||
      g.a_cols % 8 || g.c_split % 16)
    return hipErrorInvalidValue;
  if (g.M < 1 || g.N < 1 || g.splits < 1) return hipSuccess;
  if (g.bits == 4) return g.M <= 32 ? launch<4, 1>(g, nn, stream) : launch<4, 2>(g, nn, stream);
  return g.M <= 32 ? launch<8, 1>(g, nn, stream) : launch<8, 2>(g, nn, stream);
}

}  // namespace fmxq
