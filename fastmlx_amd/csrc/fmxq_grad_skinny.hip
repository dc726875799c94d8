// fmxq_grad_skinny.hip -- the products of fmxq_grad_gemm.hip for few rows, where the
// packed weights are the work: every weight is read and dequantized once, in the registers
// of the wave that multiplies it, with no stage in LDS and no barrier before the last sum.
//
// Logits: a block takes 32 tokens and up to 64 rows (more rows in chunks of 64 where the tokens
// are few), each of its 8 waves an eighth of the hidden width in 64-deep steps; a lane holds 32
// values of one token's row.
// Input gradients (48 rows at most): a block takes 128 outputs and its waves every eighth step
// of 32 weight rows; lane r16 of quarter q4 holds the word of outputs 8 r16 .. + 8 in rows
// 8 q4 .. + 8, and column r16 of v_mfma_f32_16x16x32_bf16's tile j is output 8 r16 + j, so that
// a word's values go to eight tiles and never have to cross lanes.
//
// Bound: waiting for loads.  A wave requests a step's weights, scales and x and uses them at once;
// the other waves hide a part of it.  31 to 45% of the wave cycles wait, and the dequantization's
// VALU instructions (6 a weight, with the roundings that make it exact) fill 34 to 50% of the
// SIMDs' cycles, the MFMAs 3 to 8%.  Below about 20 us also the launch and the sum over the waves.
// Measured: logits of one row, 32000 x 2048, 4 bits: 19 us; of 16 rows, 32000 x 2560 in
// groups of 32: 29 us; of 37 rows, 50257 x 1024, 8 bits: 27 us; gradients of the last two
// 28 and 32 us; of 13 rows, 4096 x 4096: 9 us; logits of one row, 128256 x 4096: 131 us.
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr uint32_t kOut = 0x7ffffff0u;  // an offset past every buffer: loads give zero

// x in the order in which the logits' waves read it: 16 bytes a lane, the four chunks of a
// 64-deep step of a 32-row tile one after the other, zeros past M and K.
__global__ __launch_bounds__(256) void pack_x_kernel(const uint16_t* __restrict__ a, int64_t lda,
                                                     int64_t M, int64_t K, u32x4* __restrict__ xp,
                                                     int mt, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  a += (int64_t)blockIdx.y * kSkinnyRows * lda;
  M -= (int64_t)blockIdx.y * kSkinnyRows;
  xp += blockIdx.y * n;
  const int lane = (int)i & 63, c = (int)(i >> 6) & 3;
  const int64_t t = i >> 8;  // step mt + row tile
  const int64_t m = t % mt * 32 + (lane & 31), k = t / mt * 64 + 32 * (lane >> 5) + 8 * c;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (m < M && k < K) v = *reinterpret_cast<const u32x4*>(a + m * lda + k);
  xp[i] = v;
}

template <int BITS, int MT, bool PACKED, int EPI>
__global__ __launch_bounds__(512, MT == 1 ? 8 : 4) void logits_skinny_kernel(GradGemm g) {
  constexpr int NW = BITS / 4;  // 16-byte weight loads per lane and step
  __shared__ __attribute__((aligned(16))) float part[8 * MT * 1024];
  __shared__ uint32_t want[16 * 32];
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const int64_t m0 = (int64_t)blockIdx.y * kSkinnyRows;
  const int64_t M = g.M - m0 < kSkinnyRows ? g.M - m0 : kSkinnyRows;
  const int K = (int)g.C;
  const int gs = __builtin_ctz(g.group_size);
  const int64_t wpr = (int64_t)K * BITS / 32, gpr = K >> gs;
  const int64_t rows = g.N - n0 < 32 ? g.N - n0 : 32;
  const __amdgpu_buffer_rsrc_t wr = rsrc(g.w + n0 * wpr, rows * wpr * 4);
  const __amdgpu_buffer_rsrc_t sr = rsrc(g.scales + n0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t br = rsrc(g.biases + n0 * gpr, rows * gpr * 2);
  const int steps = (K + 63) / 64;
  const __amdgpu_buffer_rsrc_t ar =
      PACKED ? rsrc(static_cast<const uint8_t*>(g.xp) + blockIdx.y * ((int64_t)steps * MT * 4096),
                    (int64_t)steps * MT * 4096)
             : rsrc(g.a + m0 * g.lda, M * g.lda * 2);
  // Rows past M read the last one's values and are not stored: lanes at one address cost the
  // data path one access, lanes past a buffer one each.  (With the scales' loads below, one
  // row, 4096 wide, 128256 tokens: 162 before, 131 us; 16 rows 218 and 175.)
  uint32_t ao[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    ao[i] = PACKED ? (uint32_t)(i * 4096 + lane * 16)
                   : (uint32_t)((r32 + 32 * i < M ? r32 + 32 * i : M - 1) * g.lda * 2);
  const int wo = r32 * (int)wpr * 4;
  f32x16 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[m][r] = 0.f;
  // A wave's steps are consecutive, so that one load fetches the scales of four groups of a
  // row, at an even one (a 2-byte load of 32 rows costs the data path as many accesses).
  const int st0 = steps * wave / 8, st1 = steps * (wave + 1) / 8;
  const bool wide = !(gpr & 1) && gpr >= 4 &&
                    !((reinterpret_cast<uintptr_t>(g.scales) | reinterpret_cast<uintptr_t>(g.biases)) & 3);
  const int sw = r32 * (int)gpr * 2;
  int first = -4;  // the group whose scales are sv's first
  u32x2 sv = {0u, 0u}, bv = {0u, 0u};
  // Loads are hidden by the other waves: up to eight on a SIMD.
  for (int step = st0; step < st1; ++step) {
    // A half past the row's end takes the row's last values against zeros of x.
    const int k = 64 * step + 32 * h, kw = k < K ? k : K - 32;
    if (wide) {
      const int gu = (64 * step) >> gs;
      if (gu >= first + 4 || first < 0) {
        first = (gu & ~1) < (int)gpr - 4 ? gu & ~1 : (int)gpr - 4;
        sv = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(sr, sw, 2 * first, 0));
        bv = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(br, sw, 2 * first, 0));
      }
    } else {
      first = kw >> gs;
      sv[0] = __builtin_amdgcn_raw_buffer_load_b16(sr, sw + 2 * first, 0, 0);
      bv[0] = __builtin_amdgcn_raw_buffer_load_b16(br, sw + 2 * first, 0, 0);
    }
    u32x4 w[NW], x[MT][4];
#pragma unroll
    for (int i = 0; i < NW; ++i)
      w[i] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, wo + kw * BITS / 8, 16 * i, 0));
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint32_t o = PACKED ? ao[m] + (uint32_t)step * (MT * 4096) : k < K ? ao[m] + 2 * k : kOut;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[m][i] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(ar, (int)o, (PACKED ? 1024 : 16) * i, 0));
    }
    const int at = (kw >> gs) - first;  // 0 .. 3
    const float s = __uint_as_float(((at & 2 ? sv[1] : sv[0]) << (at & 1 ? 0 : 16)) & 0xffff0000u);
    const float b = __uint_as_float(((at & 2 ? bv[1] : bv[0]) << (at & 1 ? 0 : 16)) & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 o;
      if constexpr (BITS == 4) {
        uint32_t e = w[0][i] & 0x0F0F0F0Fu, d = (w[0][i] >> 4) & 0x0F0F0F0Fu;
        asm("" : "+v"(e), "+v"(d));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = deq_pair((float)((e >> (8 * j)) & 0xffu), (float)((d >> (8 * j)) & 0xffu), s, s, b, b);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t v = w[i >> 1][2 * (i & 1) + (j >> 1)] >> (16 * (j & 1));
          o[j] = deq_pair((float)(v & 0xffu), (float)((v >> 8) & 0xffu), s, s, b, b);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, o),
                                                         __builtin_bit_cast(bf16x8, x[m][i]), acc[m],
                                                         0, 0, 0);
    }
  }
  // The columns that the rows want: wave m, m + MT, ... share the ids of row tile m, two lanes a wave.
  constexpr int SH = 16 / MT;
  const int row = 32 * (wave % MT) + r32, share = 2 * (wave / MT) + h;
  uint32_t some = 0;
  if (epi_wants(EPI) && row < M)
    for (int j = share; j < g.wanted_k; j += SH) {
      const uint32_t c = wanted_column(g, g.wanted[(m0 + row) * g.wanted_k + j], n0);
      if (c < 32) some |= 1u << c;
    }
  if (epi_wants(EPI)) want[share * (MT * 32) + row] = some;
  // The waves' sums, in the order of the waves; wave m finishes row tile m.
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(part + (((wave * MT + m) * 4 + q) * 64 + lane) * 4) =
          f32x4{acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
  __syncthreads();
  if constexpr (EPI == kEpiOut) {
    // All waves: thread t takes 4 columns of a row, the adapter's part value by value (rows of a decode
    // batch have adapters of their own, which tiles would take in turn: 48 rows of 32 adapters of rank 16
    // 33.8 us that way, 31.2 this way).  It reads B again for every row: 64 rows, 14336 x 4096, rank 16, 64 and
    // 128 with what comes before 30, 39 and 52 us of one adapter, 32, 63 and 111 of 32.
    if (tid >= MT * 256) return;
    const int mt = tid >> 8, q = (tid >> 6) & 3;
    const int64_t m = m0 + 32 * mt + r32, n = n0 + 8 * q + 4 * h;
    if (m >= g.M || n >= g.N) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w)
      v += *reinterpret_cast<const f32x4*>(part + (((w * MT + mt) * 4 + q) * 64 + lane) * 4);
    const int e = g.lora.u ? adapter_of(g.lora, m) : -1;
    uint16_t* y = g.y + m * g.ldy + n;
    if (((g.N | g.ldy) & 3) == 0) {
      if (e >= 0) add_lora4(g.lora, e, m, n, v);
      *reinterpret_cast<u32x2*>(y) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      return;
    }
    for (int i = 0; i < 4 && n + i < g.N; ++i) {
      const float s = v[i] + (e >= 0 ? lora_value(g.lora, e, m, n + i) : 0.f);
      y[i] = (uint16_t)f32_to_bf16_rne(s);
    }
    return;
  }
  if (wave >= MT) return;
  uint32_t out[1][1] = {{0u}};
  if (epi_wants(EPI))
    for (int i = 0; i < SH && i < g.wanted_k; ++i) out[0][0] |= want[i * (MT * 32) + row];
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
  store_logits<EPI>(g, sum, out, m0 + 32 * wave, g.M, n0, 0);
}

template <int BITS, int MT, bool G32, bool LORA>
__global__ __launch_bounds__(512, MT == 1 ? 4 : 2) void grad_skinny_kernel(GradGemm g) {
  constexpr int NG = G32 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float part[8 * 2048];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tn = (int)((g.N + kSkinnyCols - 1) / kSkinnyCols);
  const int split = (int)(blockIdx.x / tn);
  const int64_t n0 = (int64_t)(blockIdx.x % tn) * kSkinnyCols;
  const int64_t c0 = split * g.c_split;
  const int64_t c1 = c0 + g.c_split < g.C ? c0 + g.c_split : g.C;
  const int gs = __builtin_ctz(g.group_size);
  const int64_t wpr = g.N * BITS / 32, gpr = g.N >> gs;
  const int64_t rows = c1 > c0 ? c1 - c0 : 0;
  const __amdgpu_buffer_rsrc_t wr = rsrc(g.w + c0 * wpr, rows * wpr * 4);
  const __amdgpu_buffer_rsrc_t sr = rsrc(g.scales + c0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t br = rsrc(g.biases + c0 * gpr, rows * gpr * 2);
  const __amdgpu_buffer_rsrc_t ar = rsrc(g.a, g.M * g.lda * 2);
  // Columns past the weight's last are clamped into its rows; they are not stored.
  const int unit = (int)(n0 / 8 + r16 < g.N / 8 ? n0 / 8 + r16 : g.N / 8 - 1);
  const uint32_t wo = (uint32_t)(8 * q4 * wpr * 4 + unit * BITS);
  // Scales: lane i of an octet (whose 64 columns share a group; 32 of them in groups of 32)
  // loads row i's and the others take it from there.
  const int srow = 8 * q4 + (G32 ? r16 & 3 : r16 & 7);
  const uint32_t so = (uint32_t)((srow * gpr + (unit * 8 >> gs)) * 2);
  uint32_t ao[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) ao[m] = (uint32_t)((r16 + 16 * m) * g.lda * 2);
  const uint32_t acols = (uint32_t)g.a_cols;

  struct Step {
    uint32_t w[BITS == 8 ? 16 : 8];
    u32x4 a[MT];
    uint16_t s[NG], b[NG];
  };
  // Rows past the part lie past its buffers.
  auto load = [&](int step, Step& p) {
    const uint32_t r = 32 * (uint32_t)step, o = wo + r * (uint32_t)(wpr * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int oi = (int)(o + (uint32_t)(i * wpr * 4));
      if constexpr (BITS == 8) {
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
    const uint32_t col = (uint32_t)c0 + r + 8 * q4;
#pragma unroll
    for (int m = 0; m < MT; ++m)
      p.a[m] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             ar, (int)(col < acols ? ao[m] + 2 * col : kOut), 0, 0));
  };
  f32x4 acc[8][MT];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[j][m] = f32x4{0.f, 0.f, 0.f, 0.f};
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
    uint32_t lo[8], hi[8];  // the rows' values of even and odd columns, or bytes
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (BITS == 4) {
        lo[i] = p.w[i] & 0x0F0F0F0Fu;
        hi[i] = (p.w[i] >> 4) & 0x0F0F0F0Fu;
      } else {
        lo[i] = p.w[2 * i];
        hi[i] = p.w[2 * i + 1];
      }
      asm("" : "+v"(lo[i]), "+v"(hi[i]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
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
        acc[j][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o),
                                                            __builtin_bit_cast(bf16x8, p.a[m]),
                                                            acc[j][m], 0, 0, 0);
    }
  };
  const int steps = (int)((rows + 31) / 32);
  Step p0;
  if constexpr (MT == 1) {
    // Four waves on a SIMD hide each other's loads.
    for (int k = wave; k < steps; k += 8) {
      load(k, p0);
      use(p0);
    }
  } else {
    Step p1;
    load(wave, p0);
    for (int k = wave; k < steps; k += 16) {
      load(k + 8, p1);
      use(p0);
      load(k + 16, p0);
      use(p1);
    }
  }
  // Row tile by row tile the waves' sums meet in LDS and are added in the order of the waves.
  // Register r of a lane and tile j is row r16, output 8 (4 q4 + r) + j of the block's: a
  // lane's 16-byte unit 2 r + (j / 4) at position unit ^ (lane & 7).
  const int ln = tid >> 3, un = tid & 7;  // the unit that this thread adds up
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int jh = 0; jh < 2; ++jh)
        *reinterpret_cast<f32x4*>(part + ((wave * 64 + lane) * 8 + ((2 * r + jh) ^ (lane & 7))) * 4) =
            f32x4{acc[4 * jh][m][r], acc[4 * jh + 1][m][r], acc[4 * jh + 2][m][r], acc[4 * jh + 3][m][r]};
    __syncthreads();
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(part + ((w * 64 + ln) * 8 + (un ^ (ln & 7))) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += u[e];
    }
    const int64_t row = (ln & 15) + 16 * m;
    const int64_t n = n0 + 8 * (4 * (ln >> 4) + (un >> 1)) + 4 * (un & 1);
    if (row >= g.M || n >= g.N) continue;
    if constexpr (LORA) {
      const int e = split == 0 ? adapter_of(g.lora, row) : -1;
      if (e >= 0) add_lora4(g.lora, e, row, n, v);
    }
    if (g.y) {
      *reinterpret_cast<u32x2*>(g.y + row * g.ldy + n) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    } else {
      float* o = g.out + (split * g.M + row) * g.N + n;
      if (g.add) {
        const f32x4 old = *reinterpret_cast<const f32x4*>(o);
        const float f = g.factor ? g.factor[row] : 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(old[e], f, v[e]);
      }
      *reinterpret_cast<f32x4*>(o) = v;
    }
  }
}

template <int BITS, int MT, int EPI>
hipError_t launch_logits(const GradGemm& g, hipStream_t stream) {
  const int64_t blocks = (g.N + 31) / 32, chunks = (g.M + kSkinnyRows - 1) / kSkinnyRows;
  if (blocks >= kMaxBlocks || chunks > 65535) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks, (unsigned)chunks);
  if (!g.xp) {
    logits_skinny_kernel<BITS, MT, false, EPI><<<grid, 512, 0, stream>>>(g);
    return hipGetLastError();
  }
  const int64_t n = (g.C + 63) / 64 * MT * 256;
  pack_x_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)chunks), 256, 0, stream>>>(
      g.a, g.lda, g.M, g.C, reinterpret_cast<u32x4*>(g.xp), MT, n);
  if (hipError_t e = hipGetLastError()) return e;
  logits_skinny_kernel<BITS, MT, true, EPI><<<grid, 512, 0, stream>>>(g);
  return hipGetLastError();
}

template <int EPI>
hipError_t launch_logits_of(const GradGemm& g, hipStream_t stream) {
  if (g.bits == 4)
    return g.M <= 32 ? launch_logits<4, 1, EPI>(g, stream) : launch_logits<4, 2, EPI>(g, stream);
  return g.M <= 32 ? launch_logits<8, 1, EPI>(g, stream) : launch_logits<8, 2, EPI>(g, stream);
}

template <int BITS, int MT>
hipError_t launch_grad(const GradGemm& g, hipStream_t stream) {
  const int64_t blocks = (g.N + kSkinnyCols - 1) / kSkinnyCols * g.splits;
  if (blocks >= kMaxBlocks) return hipErrorInvalidConfiguration;
  const unsigned n = (unsigned)blocks;
  if (g.lora.u) {
    if (g.group_size == 32) grad_skinny_kernel<BITS, MT, true, true><<<n, 512, 0, stream>>>(g);
    else grad_skinny_kernel<BITS, MT, false, true><<<n, 512, 0, stream>>>(g);
  } else {
    if (g.group_size == 32) grad_skinny_kernel<BITS, MT, true, false><<<n, 512, 0, stream>>>(g);
    else grad_skinny_kernel<BITS, MT, false, false><<<n, 512, 0, stream>>>(g);
  }
  return hipGetLastError();
}

}  // namespace

// Byte offsets of a block's rows are 32 bits: 64 rows of x, 32 weight rows of the logits, a
// part's weight rows of the gradient and the steps that are requested past its end.
bool skinny_gemm_supported(int64_t lda, int64_t weight_rows, int64_t weight_cols) {
  return 64 * lda * 2 < 0x7ffffff0LL && (weight_rows + 1024) * weight_cols < 0x7fff0000LL;
}

hipError_t launch_skinny_gemm(const GradGemm& g, bool nn, hipStream_t stream) {
  if (!g.a || !g.w || (nn ? !g.out && !g.y : !logits_operands(g)) ||
      (nn && g.M > kGradSkinnyRows) ||
      !skinny_gemm_supported(g.lda, nn ? g.c_split : 32, nn ? g.N : g.C) || g.offsets || g.lda % 8 ||
      g.a_cols % 8 || g.c_split % 16)
    return hipErrorInvalidValue;
  if (g.M < 1 || g.N < 1 || g.splits < 1) return hipSuccess;
  if (nn) {
    const int mt = (int)(g.M + 15) / 16;
    if (g.bits == 4)
      return mt == 1   ? launch_grad<4, 1>(g, stream)
             : mt == 2 ? launch_grad<4, 2>(g, stream)
                       : launch_grad<4, 3>(g, stream);
    return mt == 1   ? launch_grad<8, 1>(g, stream)
           : mt == 2 ? launch_grad<8, 2>(g, stream)
                     : launch_grad<8, 3>(g, stream);
  }
  return g.epi == kEpiStats    ? launch_logits_of<kEpiStats>(g, stream)
         : g.epi == kEpiScores ? launch_logits_of<kEpiScores>(g, stream)
         : g.epi == kEpiCoef   ? launch_logits_of<kEpiCoef>(g, stream)
                               : launch_logits_of<kEpiOut>(g, stream);
}

}  // namespace fmxq
