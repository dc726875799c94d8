// fmxq_grad_panel.hip -- the products of fmxq_grad_gemm.hip for many rows: the weights are
// dequantized to a bf16 panel once, and both operands of the product go to LDS without
// passing through registers.
//
// Tile: 256 rows by 256 columns, 64 deep steps in two LDS stages, 4 waves of 128 x 128 (one
// per SIMD, 256 accumulators each).  A step's fragments of 16 contraction values are read
// while the MFMAs of the 16 before run; the barrier sits before the last quarter's MFMAs,
// when every wave has read the stage, so the next stage's first fragments and the DMA that
// refills this one are under way while they run.
#include <algorithm>
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr int kS = 64;  // contraction values per step
constexpr int kN = kGradTileCols;

template <bool NN>
__global__ __launch_bounds__(256, 1) void panel_gemm_kernel(GradGemm g) {
  constexpr int BM = kPanelRows, MI = 4, NJ = 4;
  constexpr int XI = BM / 32, YI = kN / 32;  // DMA instructions per wave and step
  __shared__ __attribute__((aligned(1024))) uint8_t as0[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t as1[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs0[kN * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs1[kN * 128];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;

  // Row tiles fastest; every eighth block runs on one XCD, and those take neighbouring tiles.
  const int64_t tn = (g.N + kN - 1) / kN, tm = (g.M + BM - 1) / BM;
  const int64_t total = (int64_t)gridDim.x;
  int64_t b = blockIdx.x;
  if ((total & 7) == 0) b = (b & 7) * (total >> 3) + (b >> 3);
  const int64_t split = b / (tm * tn);
  b -= split * tm * tn;
  const int64_t m0 = b % tm * BM, n0 = b / tm * kN;
  const int64_t rows = g.M - m0 < BM ? g.M - m0 : BM, cols = g.N - n0 < kN ? g.N - n0 : kN;
  const int64_t c0 = split * g.c_split;
  const int64_t c1 = c0 + g.c_split < g.C ? c0 + g.c_split : g.C;
  const int nk = c1 > c0 ? (int)((c1 - c0 + kS - 1) / kS) : 0;
  auto as = [&](int st) -> uint8_t* { return st == 0 ? as0 : as1; };
  auto bs = [&](int st) -> uint8_t* { return st == 0 ? bs0 : bs1; };

  const __amdgpu_buffer_rsrc_t ares = rsrc(g.a + m0 * g.lda, rows * g.lda * 2);
  const __amdgpu_buffer_rsrc_t bres = rsrc(g.panel + n0 * g.ldp, cols * g.ldp * 2);
  // Instruction i of a wave fills rows 8 (8 wave + i) .. + 8 of a stage; lane L lands at row
  // L / 8, chunk position L % 8.
  const int chunk8 = ((lane & 7) ^ swz(lane >> 3)) * 8;  // rows 8 i differ in swz's last bit
  uint32_t ao[XI], bo[YI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = 8 * (XI * wave + i) + (lane >> 3);
    ao[i] = row < rows ? (uint32_t)(row * g.lda * 2) : 0x7ffffff0u;
  }
#pragma unroll
  for (int i = 0; i < YI; ++i) {
    const int row = 8 * (YI * wave + i) + (lane >> 3);
    bo[i] = row < cols ? (uint32_t)(row * g.ldp * 2) : 0x7ffffff0u;
  }
  auto issue = [&](int k, int st) {
    const int64_t kc = c0 + (int64_t)k * kS;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t col = kc + (chunk8 ^ (8 * p));
      const uint32_t va = k < nk && col < g.a_cols ? (uint32_t)(col * 2) : 0x7ffffff0u;
      const uint32_t vb = k < nk && col < g.C ? (uint32_t)(col * 2) : 0x7ffffff0u;
#pragma unroll
      for (int i = p; i < XI; i += 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lds_t*)(as(st) + 8 * (XI * wave + i) * 128),
                                                 16, (int)__builtin_elementwise_add_sat(ao[i], va), 0, 0, 0);
#pragma unroll
      for (int i = p; i < YI; i += 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(bres, (lds_t*)(bs(st) + 8 * (YI * wave + i) * 128),
                                                 16, (int)__builtin_elementwise_add_sat(bo[i], vb), 0, 0, 0);
    }
  };

  uint32_t fo[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) fo[s] = r32 * 128 + (((2 * s + h) ^ swz(r32)) << 4);

  f32x16 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  bf16x8 a0[MI], a1[MI], b0[NJ], b1[NJ];
  auto read = [&](bf16x8 (&af)[MI], bf16x8 (&bf)[NJ], int st, int s) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      bf[j] = *reinterpret_cast<const bf16x8*>(bs(st) + (wn * NJ + j) * 4096 + fo[s]);
#pragma unroll
    for (int i = 0; i < MI; ++i)
      af[i] = *reinterpret_cast<const bf16x8*>(as(st) + (wm * MI + i) * 4096 + fo[s]);
  };
  auto mfmas = [&](const bf16x8 (&af)[MI], const bf16x8 (&bf)[NJ]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
  };
  // One fragment read under each of the first MFMAs of a quarter.
  auto pace = [&]() {
#pragma unroll
    for (int t = 0; t < MI * NJ; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                     // MFMA
      if (t < MI + NJ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // DS read
    }
  };
  auto step = [&](int k, auto stc) {
    constexpr int st = decltype(stc)::value;
    read(a1, b1, st, 1);
    mfmas(a0, b0);
    pace();
    read(a0, b0, st, 2);
    mfmas(a1, b1);
    pace();
    read(a1, b1, st, 3);
    mfmas(a0, b0);
    pace();
    // The next stage has landed and this one is read.
    __builtin_amdgcn_s_waitcnt(wait_enc(0, 0));
    __builtin_amdgcn_s_barrier();
    issue(k + 2, st);
    read(a0, b0, st ^ 1, 0);
    mfmas(a1, b1);
#pragma unroll
    for (int t = 0; t < MI * NJ; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (t < MI + NJ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // VMEM (the DMA)
    }
  };
  if (nk > 0) {
    issue(0, 0);
    __builtin_amdgcn_sched_barrier(0);  // the wait counts on this order
    issue(1, 1);
    __builtin_amdgcn_s_waitcnt(wait_enc(XI + YI, 15));
    __builtin_amdgcn_s_barrier();
    read(a0, b0, 0, 0);
    // Two steps a turn, the last one on zeros where nk is odd.
    for (int k = 0; k < nk; k += 2) {
      step(k, std::integral_constant<int, 0>{});
      step(k + 1, std::integral_constant<int, 1>{});
    }
    __builtin_amdgcn_s_waitcnt(wait_enc(0, 0));
  }
  const int64_t mw = m0 + wm * MI * 32, nw = n0 + wn * NJ * 32;
  if constexpr (NN) store_grad<MI, NJ>(g, acc, mw, m0 + rows, nw, split);
  else store_stats<MI, NJ>(g, acc, mw, m0 + rows, nw);
}

// A thread takes 8 rows of 8 columns: the roundings pack any two values, so the block comes
// out transposed at no cost.  Lanes 8 c .. 8 c + 7 hold 64 rows of one 8-column unit and
// store 128 contiguous bytes of a panel row.
template <int BITS>
__global__ __launch_bounds__(256) void dequant_transposed_kernel(
    const uint32_t* __restrict__ w, const uint16_t* __restrict__ scales,
    const uint16_t* __restrict__ biases, uint16_t* __restrict__ panel, int64_t n, int64_t K,
    int64_t ld, int group_size) {
  constexpr int WPU = BITS / 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t units = K / 8, gpr = K / group_size;
  const int64_t r0 = (int64_t)blockIdx.y * 64 + 8 * (lane & 7);
  const int64_t u = ((int64_t)blockIdx.x * 4 + wave) * 8 + (lane >> 3);
  if (u >= units || r0 >= ld) return;
  float q[8][8], s[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + i;
    uint32_t x[2] = {0u, 0u};
    s[i] = b[i] = 0.f;
    if (r < n) {
      x[0] = w[(r * units + u) * WPU];
      if (WPU == 2) x[1] = w[(r * units + u) * WPU + 1];
      const int64_t grp = r * gpr + u * 8 / group_size;
      s[i] = bf16_bits_to_f32(scales[grp]);
      b[i] = bf16_bits_to_f32(biases[grp]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      q[i][j] = BITS == 4 ? (float)((x[0] >> (4 * j)) & 15u)
                          : (float)((x[j >> 2] >> (8 * (j & 3))) & 255u);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = pack_bf16x2(q[2 * i][j] * s[2 * i], q[2 * i + 1][j] * s[2 * i + 1]);
      o[i] = pack_bf16x2(bf16_lo(m) + b[2 * i], bf16_hi(m) + b[2 * i + 1]);
    }
    *reinterpret_cast<u32x4*>(panel + (u * 8 + j) * ld + r0) = o;
  }
}

}  // namespace

hipError_t launch_panel_gemm(const GradGemm& g, bool nn, hipStream_t stream) {
  if (!g.a || !g.panel || (nn ? !g.out && !g.y : !g.stats) || kPanelRows * g.lda * 2 >= 0x7ffffff0LL || kN * g.ldp * 2 >= 0x7ffffff0LL || g.c_split % kS ||
      g.lda % 8 || g.a_cols % 8 || g.ldp % 8 || g.offsets)
    return hipErrorInvalidValue;
  const int64_t blocks = (g.M + kPanelRows - 1) / kPanelRows * ((g.N + kN - 1) / kN) * g.splits;
  if (blocks < 1) return hipSuccess;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  if (nn) panel_gemm_kernel<true><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else panel_gemm_kernel<false><<<(unsigned)blocks, 256, 0, stream>>>(g);
  return hipGetLastError();
}

hipError_t launch_dequant_transposed(const uint32_t* w, const uint16_t* scales,
                                     const uint16_t* biases, uint16_t* panel, int64_t n, int64_t K,
                                     int64_t ld, int group_size, int bits, hipStream_t stream) {
  const int64_t by = (ld + 63) / 64;
  if (ld % 8 || by > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((K / 8 + 31) / 32), (unsigned)by);
  if (bits == 4)
    dequant_transposed_kernel<4><<<grid, 256, 0, stream>>>(w, scales, biases, panel, n, K, ld, group_size);
  else
    dequant_transposed_kernel<8><<<grid, 256, 0, stream>>>(w, scales, biases, panel, n, K, ld, group_size);
  return hipGetLastError();
}

}  // namespace fmxq
