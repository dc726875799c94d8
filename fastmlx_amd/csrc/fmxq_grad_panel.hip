// fmxq_grad_panel.hip -- the products of fmxq_grad_gemm.hip for many rows: the weights are
// dequantized to a bf16 panel once, and both operands of the product go to LDS without
// passing through registers.
//
// One panel [tokens, width] serves both products.  The logits' contraction runs along its
// rows: a stage holds 256 rows of 64 values.  The gradient's runs across them: a stage holds
// 64 rows of 256 columns, and ds_read_b64_tr_b16 turns it on the way to the registers (16 lanes
// give 4 rows of 16 columns and get 4 rows' values of one column each).
//
// Tile: 256 rows by 256 columns, 64 deep steps in two LDS stages, 4 waves of 128 x 128 (one
// per SIMD, 256 accumulators each).  A step's fragments of 16 contraction values are read
// while the MFMAs of the 16 before run; the barrier sits before the last quarter's MFMAs,
// when every wave has read the stage, so the next stage's first fragments and the DMA that
// refills this one are under way while they run.
//
// Bound: MFMAs at the clock that the power limit leaves.  Measured for 2048 rows, 32064 x 4096:
// the gradient 440 to 455 us, 1.18 to 1.22 PFLOP/s; the logits with their statistics 488 us,
// 1.10 PFLOP/s (the epilogue's exponentials; a large library product ran at 1.20 there).
#include <algorithm>
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr int kS = 64;  // contraction values per step
constexpr int kN = kGradTileCols;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <bool NN, int EPI = kEpiStats>
__global__ __launch_bounds__(256, 1) void panel_gemm_kernel(GradGemm g) {
  constexpr int BM = kPanelRows, MI = 4, NJ = 4;
  constexpr int XI = BM / 32, YI = kN / 32;  // DMA instructions per wave and step
  __shared__ __attribute__((aligned(1024))) uint8_t as0[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t as1[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs0[kN * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs1[kN * 128];
  __shared__ int32_t one[NN ? 1 : BM];  // the rows' wanted tokens, where they have one
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
  // Instruction i of a wave fills rows 8 (8 wave + i) .. + 8 of a stage; lane L lands at row
  // L / 8, chunk position L % 8.
  const int chunk8 = ((lane & 7) ^ swz(lane >> 3)) * 8;  // rows 8 i differ in swz's last bit
  uint32_t ao[XI], bo[YI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = 8 * (XI * wave + i) + (lane >> 3);
    ao[i] = row < rows ? (uint32_t)(row * g.lda * 2) : 0x7ffffff0u;
  }
  // nn: instruction i fills rows 2 (8 wave + i) .. + 2 of 512 bytes; the row's 64-byte blocks
  // sit at block ^ turn(row), so that the 8 rows of a turning read meet 8 different ones.
  auto turn = [](int row) { return (row & 3) | ((row >> 3) & 1) << 2; };
  const __amdgpu_buffer_rsrc_t bres = rsrc(g.panel + n0 * g.ldp, cols * g.ldp * 2);  // nt
#pragma unroll
  for (int i = 0; i < YI; ++i) {
    if constexpr (NN) {
      const int row = 2 * (YI * wave + i) + (lane >> 5), at = lane & 31;
      const int unit = ((at >> 2) ^ turn(row)) * 4 + (at & 3);
      bo[i] = (uint32_t)(row * g.ldp * 2 + (n0 + 8 * unit) * 2);
    } else {
      const int row = 8 * (YI * wave + i) + (lane >> 3);
      bo[i] = row < cols ? (uint32_t)(row * g.ldp * 2) : 0x7ffffff0u;
    }
  }
  auto issue = [&](int k, int st) {
    const int64_t kc = c0 + (int64_t)k * kS;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t col = kc + (chunk8 ^ (8 * p));
      const uint32_t va = k < nk && col < g.a_cols ? (uint32_t)(col * 2) : 0x7ffffff0u;
#pragma unroll
      for (int i = p; i < XI; i += 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lds_t*)(as(st) + 8 * (XI * wave + i) * 128),
                                                 16, (int)__builtin_elementwise_add_sat(ao[i], va), 0, 0, 0);
      if constexpr (!NN) {
        const uint32_t vb = k < nk && col < g.C ? (uint32_t)(col * 2) : 0x7ffffff0u;
#pragma unroll
        for (int i = p; i < YI; i += 2)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(bres, (lds_t*)(bs(st) + 8 * (YI * wave + i) * 128),
                                                   16, (int)__builtin_elementwise_add_sat(bo[i], vb), 0, 0, 0);
      }
    }
    if constexpr (NN) {
      // Rows past the part lie past the buffer; columns past N belong to the next row and to
      // outputs that are not stored.
      const int64_t left = k < nk ? (c1 - kc < kS ? c1 - kc : kS) : 0;
      const __amdgpu_buffer_rsrc_t br = rsrc(g.panel + kc * g.ldp, left * g.ldp * 2);
#pragma unroll
      for (int i = 0; i < YI; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(br, (lds_t*)(bs(st) + 2 * (YI * wave + i) * 512), 16,
                                                 (int)bo[i], 0, 0, 0);
    }
  };

  uint32_t fo[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) fo[s] = r32 * 128 + (((2 * s + h) ^ swz(r32)) << 4);
  // nn: the lane's 8 bytes of row 8 h + lane % 16 / 4, block 4 wn (block j: flipped by j).
  const int trow = 8 * h + ((lane & 15) >> 2);
  const uint32_t to = (uint32_t)(trow * 512 + (((4 * wn) ^ turn(trow)) << 6) + ((lane >> 4) & 1) * 32 +
                                 (lane & 3) * 8);

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
    for (int j = 0; j < NJ; ++j) {
      if constexpr (NN) {
        uint8_t* p = bs(st) + (to ^ (uint32_t)(j << 6)) + s * 8192;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 2048));
        bf[j] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        bf[j] = *reinterpret_cast<const bf16x8*>(bs(st) + (wn * NJ + j) * 4096 + fo[s]);
      }
    }
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
  // The next quarter's fragment reads (two a turned fragment) under the first MFMAs of this.
  constexpr int RD = MI + (NN ? 2 : 1) * NJ;
  auto pace = [&]() {
#pragma unroll
    for (int t = 0; t < MI * NJ; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                     // MFMA
      if (t < RD) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);         // DS read
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
      if (t < RD) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // VMEM (the DMA)
    }
  };
  int32_t id = -1;
  if (!NN && epi_wants(EPI) && g.wanted_k == 1 && tid < rows) id = g.wanted[m0 + tid];
  if (nk > 0) {
    issue(0, 0);
    __builtin_amdgcn_sched_barrier(0);  // the wait counts on this order
    issue(1, 1);
    __builtin_amdgcn_s_waitcnt(wait_enc(XI + YI, 15));
    if (!NN) one[tid] = id;
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
  if constexpr (NN && EPI == kEpiOut) store_out<MI, NJ>(g, acc, mw, m0 + rows, nw, split);
  else if constexpr (NN) store_grad<MI, NJ>(g, acc, mw, m0 + rows, nw, split);
  else {
    uint32_t out[MI][NJ];
    if constexpr (epi_wants(EPI))
      find_wanted<BM, kN, 256>(g, m0, rows, n0, mw, nw, one, reinterpret_cast<uint32_t*>(as0),
                               out);
    store_logits<EPI>(g, acc, out, mw, m0 + rows, nw, split);
  }
}

}  // namespace

hipError_t launch_panel_gemm(const GradGemm& g, bool nn, hipStream_t stream) {
  if (!g.a || !g.panel || (nn ? !g.out && !g.y : !logits_operands(g)) || g.lda > kMaxLda ||
      !panel_gemm_supported(g.ldp) || g.c_split % kS ||
      g.lda % 8 || g.a_cols % 8 || g.ldp % 8 || g.offsets)
    return hipErrorInvalidValue;
  const int64_t blocks = (g.M + kPanelRows - 1) / kPanelRows * ((g.N + kN - 1) / kN) * g.splits;
  if (blocks < 1) return hipSuccess;
  if (blocks >= kMaxBlocks) return hipErrorInvalidConfiguration;
  if (nn && g.lora.u) panel_gemm_kernel<true, kEpiOut><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else if (nn) panel_gemm_kernel<true><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else if (g.epi == kEpiOut) panel_gemm_kernel<false, kEpiOut><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else if (g.epi == kEpiStats) panel_gemm_kernel<false, kEpiStats><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else if (g.epi == kEpiScores) panel_gemm_kernel<false, kEpiScores><<<(unsigned)blocks, 256, 0, stream>>>(g);
  else panel_gemm_kernel<false, kEpiCoef><<<(unsigned)blocks, 256, 0, stream>>>(g);
  return hipGetLastError();
}

}  // namespace fmxq
