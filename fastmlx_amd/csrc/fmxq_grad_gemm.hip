// fmxq_grad_gemm.hip -- MFMA products with dequantized weights for training: the logits of
// a quantized head with the statistics of their softmax (nt), and the input gradient
// dx = dy . deq(W) of a quantized product (nn), of one matrix or of expert runs.
//
// Tile: BM rows by 256 columns, 64 deep contraction steps, 4 waves.  A goes global -> LDS
// with buffer_load ... lds; the packed weights go global -> registers two steps ahead, are
// dequantized there to fmxq_dequantize's bits and written to LDS.  Both stages hold rows of
// 64 contraction values (128 bytes), so one fragment read serves both forms: where the
// weights are packed along the outputs (nn), a thread takes 8 rows of one word column, and
// the transposition costs nothing: the roundings pack any two values.
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr int kS = 64;   // contraction values per step
constexpr int kN = kGradTileCols;

template <int BM>
struct GradCfg {
  static constexpr int WM = BM >= 128 ? 2 : 1;   // waves along the rows
  static constexpr int WN = 4 / WM;              // and along the columns
  static constexpr int MI = BM / WM / 32;        // 32-row groups of a wave
  static constexpr int NJ = kN / WN / 32;        // 32-column groups
};

// Value j (0..7) of 8 packed values as a float; the masks let each be one byte conversion.
template <int BITS>
struct Q8;
template <>
struct Q8<4> {
  uint32_t e, o;
  __device__ __forceinline__ explicit Q8(const uint32_t* w) {
    e = w[0] & 0x0F0F0F0Fu;
    o = (w[0] >> 4) & 0x0F0F0F0Fu;
    asm("" : "+v"(e), "+v"(o));
  }
  __device__ __forceinline__ float at(int j) const {
    return (float)((((j & 1) ? o : e) >> (8 * (j >> 1))) & 0xffu);
  }
};
template <>
struct Q8<8> {
  uint32_t w0, w1;
  __device__ __forceinline__ explicit Q8(const uint32_t* w) : w0(w[0]), w1(w[1]) {}
  __device__ __forceinline__ float at(int j) const {
    return (float)(((j < 4 ? w0 : w1) >> (8 * (j & 3))) & 0xffu);
  }
};

template <int BM, int BITS, bool G32, bool NN>
__global__ __launch_bounds__(256, 1) void grad_gemm_kernel(GradGemm g) {
  using C = GradCfg<BM>;
  constexpr int WN = C::WN, MI = C::MI, NJ = C::NJ;
  constexpr int WPU = BITS / 4;              // words of 8 values
  constexpr int XI = BM / 32;                // A DMA instructions per wave and step
  constexpr int NSB = G32 ? 4 : 2;           // scale and bias loads per thread and step
  constexpr int NLD = (NN ? 8 : 2 * WPU) + NSB;  // loads per thread and step
  __shared__ __attribute__((aligned(1024))) uint8_t as0[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t as1[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs0[kN * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs1[kN * 128];
  __shared__ __attribute__((aligned(16))) uint32_t sbx[NN ? 4 * 64 * (G32 ? 2 : 1) : 4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  // Tile of this block: row tiles fastest, so that the blocks of one XCD (every eighth)
  // share weight columns.
  const int64_t tn = (g.N + kN - 1) / kN;
  const int64_t tm = g.tiles ? g.max_tiles : (g.M + BM - 1) / BM;
  const int64_t total = (int64_t)gridDim.x;
  int64_t b = blockIdx.x;
  if ((total & 7) == 0) b = (b & 7) * (total >> 3) + (b >> 3);
  const int64_t split = b / (tm * tn);
  b -= split * tm * tn;
  const int64_t mt = b % tm, nt = b / tm;
  int64_t m0 = mt * BM, rows = g.M - m0 < BM ? g.M - m0 : BM;
  const int64_t n0 = nt * kN;
  const uint32_t* w = g.w;
  const uint16_t *scales = g.scales, *biases = g.biases;
  const int64_t wk = NN ? g.N : g.C;             // values of a weight row
  const int64_t wpr = wk * BITS / 32, gpr = wk / g.group_size;
  if (NN && g.tiles) {
    if (mt >= (int64_t)*g.ntile) return;
    m0 = g.tiles[3 * mt];
    rows = g.tiles[3 * mt + 1];
    const int64_t e = g.tiles[3 * mt + 2];
    w += e * g.C * wpr;
    scales += e * g.C * gpr;
    biases += e * g.C * gpr;
  }
  const int64_t c0 = split * g.c_split;
  const int64_t c1 = c0 + g.c_split < g.C ? c0 + g.c_split : g.C;
  const int nk = c1 > c0 ? (int)((c1 - c0 + kS - 1) / kS) : 0;

  auto as = [&](int st) -> uint8_t* { return st == 0 ? as0 : as1; };
  auto bs = [&](int st) -> uint8_t* { return st == 0 ? bs0 : bs1; };

  // ---- A: wave w, instruction i fills rows 8 (XI w + i) .. + 8 of the stage.
  const __amdgpu_buffer_rsrc_t ares = rsrc(g.a + m0 * g.lda, rows * g.lda * 2);
  uint32_t ao[XI], ac[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = 8 * (XI * wave + i) + (lane >> 3);
    ac[i] = ((lane & 7) ^ swz(row)) * 8;
    ao[i] = row < rows ? (uint32_t)(row * g.lda * 2) : 0xffffffffu;
  }
  auto issue_a = [&](int k, int st) {
    const int64_t kc = c0 + (int64_t)k * kS;
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t off = (ao[i] != 0xffffffffu && kc + ac[i] < g.a_cols && k < nk)
                               ? ao[i] + (uint32_t)(kc + ac[i]) * 2
                               : 0x7ffffff0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lds_t*)(as(st) + 8 * (XI * wave + i) * 128),
                                               16, (int)off, 0, 0, 0);
    }
  };

  // ---- B: packed words and scales of a step in registers.
  struct Packed {
    uint32_t w[8 * WPU];
    uint16_t s[NSB / 2], b[NSB / 2];
  };
  Packed pk[2];
  const int q = lane & 7, c = lane >> 3;  // nn: rows 8 q .. + 8, word column c of the wave's 8
  auto issue_b = [&](int k, Packed& p) {
    const int64_t kc = c0 + (int64_t)k * kS;
    if constexpr (NN) {
      const int64_t left = k < nk ? (c1 - kc < kS ? c1 - kc : kS) : 0;
      const int64_t col = n0 + 64 * wave;
      // Columns past the weight's last are clamped into its rows; they are not stored.
      const int64_t wcol = col / 8 + c < wk / 8 ? col / 8 + c : wk / 8 - 1;
      const __amdgpu_buffer_rsrc_t wr = rsrc(w + kc * wpr, left * wpr * 4);
      const uint32_t o = (uint32_t)((8 * q) * wpr * 4 + wcol * WPU * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int oi = (int)(o + (uint32_t)(i * wpr * 4));
        if constexpr (WPU == 1) {
          p.w[i] = __builtin_amdgcn_raw_buffer_load_b32(wr, oi, 0, 0);
        } else {
          const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(wr, oi, 0, 0));
          p.w[2 * i] = v[0];
          p.w[2 * i + 1] = v[1];
        }
      }
      const __amdgpu_buffer_rsrc_t sr = rsrc(scales + kc * gpr, left * gpr * 2);
      const __amdgpu_buffer_rsrc_t br = rsrc(biases + kc * gpr, left * gpr * 2);
#pragma unroll
      for (int i = 0; i < NSB / 2; ++i) {
        int64_t grp = (col + 32 * i) / g.group_size;
        if (grp > gpr - 1) grp = gpr - 1;
        const int so = (int)((lane * gpr + grp) * 2);
        p.s[i] = __builtin_amdgcn_raw_buffer_load_b16(sr, so, 0, 0);
        p.b[i] = __builtin_amdgcn_raw_buffer_load_b16(br, so, 0, 0);
      }
    } else {
      const int64_t nrows = g.N - n0 < kN ? g.N - n0 : kN;
      const __amdgpu_buffer_rsrc_t wr = rsrc(w + n0 * wpr, nrows * wpr * 4);
      const uint32_t o = (uint32_t)(tid * wpr * 4 + kc / 8 * WPU * 4);
#pragma unroll
      for (int i = 0; i < 2 * WPU; ++i) {
        const u32x4 v =
            __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, (int)o + 16 * i, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) p.w[4 * i + j] = v[j];
      }
      const __amdgpu_buffer_rsrc_t sr = rsrc(scales + n0 * gpr, nrows * gpr * 2);
      const __amdgpu_buffer_rsrc_t br = rsrc(biases + n0 * gpr, nrows * gpr * 2);
#pragma unroll
      for (int i = 0; i < NSB / 2; ++i) {
        // A step past the row's end takes the row's last group: finite weights against
        // zeros of A.
        int64_t grp = (kc + 32 * i) / g.group_size;
        if (grp > gpr - 1) grp = gpr - 1;
        const int so = (int)((tid * gpr + grp) * 2);
        p.s[i] = __builtin_amdgcn_raw_buffer_load_b16(sr, so, 0, 0);
        p.b[i] = __builtin_amdgcn_raw_buffer_load_b16(br, so, 0, 0);
      }
    }
  };
  // nn: the scales and biases of the wave's 64 rows, one pair a word, through LDS.
  uint32_t sb8[8];
  auto share_sb = [&](const Packed& p) {
    if constexpr (NN) {
#pragma unroll
      for (int i = 0; i < NSB / 2; ++i)
        sbx[(wave * (NSB / 2) + i) * 64 + lane] = (uint32_t)p.s[i] | ((uint32_t)p.b[i] << 16);
      const int half = G32 ? c >> 2 : 0;
      const u32x4* v = reinterpret_cast<const u32x4*>(sbx + (wave * (NSB / 2) + half) * 64 + 8 * q);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sb8[4 * i + j] = v[i][j];
    }
  };
  // Quarter t of the step's weights: two 16-byte chunks of the stage.
  auto dequant = [&](const Packed& p, int st, int t) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = 2 * t + u;
      u32x4 o;
      int row, chunk;
      if constexpr (NN) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Q8<BITS> q0(p.w + 2 * i * WPU), q1(p.w + (2 * i + 1) * WPU);
          o[i] = deq_pair(q0.at(j), q1.at(j), bf16_lo(sb8[2 * i]), bf16_lo(sb8[2 * i + 1]),
                          bf16_hi(sb8[2 * i]), bf16_hi(sb8[2 * i + 1]));
        }
        row = 64 * wave + 8 * c + j;
        chunk = q;
      } else {
        const float s = bf16_bits_to_f32(p.s[G32 ? j >> 2 : 0]);
        const float bb = bf16_bits_to_f32(p.b[G32 ? j >> 2 : 0]);
        const Q8<BITS> qq(p.w + j * WPU);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = deq_pair(qq.at(2 * i), qq.at(2 * i + 1), s, s, bb, bb);
        row = tid;
        chunk = j;
      }
      *reinterpret_cast<u32x4*>(bs(st) + row * 128 + ((chunk ^ swz(row)) << 4)) = o;
    }
  };

  f32x16 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // Fragment of sub-step s: row r32 of a 32-row group, chunk 2 s + h.
  uint32_t fo[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) fo[s] = r32 * 128 + (((2 * s + h) ^ swz(r32)) << 4);

  // Step k, staged in st: the next step's A and the packed weights of the one after are
  // requested, then the MFMAs run with the next step's dequantization between them.
  auto step = [&](int k, auto stc) {
    constexpr int st = decltype(stc)::value;
    issue_a(k + 1, st ^ 1);
    __builtin_amdgcn_sched_barrier(0);
    issue_b(k + 2, pk[st]);
    __builtin_amdgcn_sched_barrier(0);
    share_sb(pk[st ^ 1]);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 af[MI], bf[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i)
        af[i] = *reinterpret_cast<const bf16x8*>(as(st) + (wm * MI + i) * 4096 + fo[s]);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        bf[j] = *reinterpret_cast<const bf16x8*>(bs(st) + (wn * NJ + j) * 4096 + fo[s]);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
      dequant(pk[st ^ 1], st ^ 1, s);
    }
    // The next step's A has landed (only the packed loads of the step after it are
    // younger) and its weights are written.
    __builtin_amdgcn_s_waitcnt(wait_enc(NLD, 0));
    __builtin_amdgcn_s_barrier();
  };
  if (nk > 0) {
    issue_a(0, 0);
    issue_b(0, pk[0]);
    issue_b(1, pk[1]);
    share_sb(pk[0]);
#pragma unroll
    for (int s = 0; s < 4; ++s) dequant(pk[0], 0, s);
    __builtin_amdgcn_s_waitcnt(wait_enc(0, 0));
    __builtin_amdgcn_s_barrier();
    int k = 0;
    for (; k + 1 < nk; k += 2) {
      step(k, std::integral_constant<int, 0>{});
      step(k + 1, std::integral_constant<int, 1>{});
    }
    if (k < nk) step(k, std::integral_constant<int, 0>{});
    __builtin_amdgcn_s_waitcnt(wait_enc(0, 0));
  }

  const int64_t mw = m0 + wm * MI * 32, nw = n0 + wn * NJ * 32;
  if constexpr (NN) store_grad<MI, NJ>(g, acc, mw, m0 + rows, nw, split);
  else store_stats<MI, NJ>(g, acc, mw, m0 + rows, nw);
}

template <int BM, bool NN>
hipError_t launch_bm(const GradGemm& g, hipStream_t stream) {
  const int64_t tn = (g.N + kN - 1) / kN, tm = g.tiles ? g.max_tiles : (g.M + BM - 1) / BM;
  const int64_t blocks = tm * tn * g.splits;
  if (blocks < 1) return hipSuccess;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(256);
  if (g.bits == 4) {
    if (g.group_size == 32) grad_gemm_kernel<BM, 4, true, NN><<<grid, block, 0, stream>>>(g);
    else grad_gemm_kernel<BM, 4, false, NN><<<grid, block, 0, stream>>>(g);
  } else {
    if (g.group_size == 32) grad_gemm_kernel<BM, 8, true, NN><<<grid, block, 0, stream>>>(g);
    else grad_gemm_kernel<BM, 8, false, NN><<<grid, block, 0, stream>>>(g);
  }
  return hipGetLastError();
}

}  // namespace

int grad_gemm_rows(int64_t M) { return M <= 32 ? 32 : M <= 64 ? 64 : 128; }

int grad_gemm_stat_width(int64_t M) { return grad_gemm_rows(M) >= 128 ? 128 : 64; }

hipError_t launch_grad_gemm(const GradGemm& g, bool nn, int bm, hipStream_t stream) {
  // Offsets into one tile's rows and into 64 or 256 weight rows are 32 bits.
  if (128 * g.lda * 2 >= 0x7ffffff0LL || 256 * (nn ? g.N : g.C) >= 0x7ffffff0LL || g.c_split % kS ||
      g.lda % 8 || g.a_cols % 8)
    return hipErrorInvalidValue;
  switch (bm) {
    case 32: return nn ? launch_bm<32, true>(g, stream) : launch_bm<32, false>(g, stream);
    case 64: return nn ? launch_bm<64, true>(g, stream) : launch_bm<64, false>(g, stream);
    case 128: return nn ? launch_bm<128, true>(g, stream) : launch_bm<128, false>(g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace fmxq

// ---- around the products --------------------------------------------------------

namespace fmxq {
namespace {

__global__ __launch_bounds__(256) void sum_slices_kernel(const float* __restrict__ slices,
                                                         int splits, uint16_t* __restrict__ y,
                                                         int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; 4 * i < n;
       i += (int64_t)gridDim.x * 256) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(slices + s * n + 4 * i);
    *reinterpret_cast<u32x2*>(y + 4 * i) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  }
}

__global__ __launch_bounds__(256) void pad_rows_kernel(const uint16_t* __restrict__ src,
                                                       uint16_t* __restrict__ dst, int64_t M,
                                                       int64_t N, int64_t ld) {
  const int64_t units = ld / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * units;
       i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / units, c = (i - m * units) * 8;
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = c + 2 * j < N ? src[m * N + c + 2 * j] : 0u;
      const uint32_t hi = c + 2 * j + 1 < N ? src[m * N + c + 2 * j + 1] : 0u;
      v[j] = lo | (hi << 16);
    }
    *reinterpret_cast<u32x4*>(dst + m * ld + c) = u32x4{v[0], v[1], v[2], v[3]};
  }
}

// One block: the offsets are checked, then each thread cuts a range of experts' runs.
__global__ __launch_bounds__(1024) void run_tiles_kernel(const int32_t* __restrict__ offsets,
                                                         int64_t E, int64_t S, int bm,
                                                         uint32_t* __restrict__ tiles,
                                                         uint32_t* __restrict__ ntile,
                                                         uint32_t* flag) {
  __shared__ uint32_t wsum[16], bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int64_t e = tid; e <= E; e += 1024) {
    const int64_t o = offsets[e];
    if (o < 0 || o > S || (e > 0 && o < offsets[e - 1])) bad = 1;
  }
  __syncthreads();
  if (bad) {
    if (tid == 0) {
      *ntile = 0;
      atomicOr(flag, 1u);
    }
    return;
  }
  const int64_t per = (E + 1023) / 1024;
  const int64_t e0 = tid * per < E ? tid * per : E, e1 = e0 + per < E ? e0 + per : E;
  uint32_t n = 0;
  for (int64_t e = e0; e < e1; ++e) n += (uint32_t)((offsets[e + 1] - offsets[e] + bm - 1) / bm);
  uint32_t inc = n;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_up((int)inc, o, 64);
    if (lane >= o) inc += t;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  uint32_t at = inc - n;
  for (int i = 0; i < wave; ++i) at += wsum[i];
  if (tid == 1023) *ntile = at + n;
  for (int64_t e = e0; e < e1; ++e)
    for (int64_t r = offsets[e]; r < offsets[e + 1]; r += bm, ++at) {
      const int64_t left = offsets[e + 1] - r;
      tiles[3 * at] = (uint32_t)r;
      tiles[3 * at + 1] = (uint32_t)(left < bm ? left : bm);
      tiles[3 * at + 2] = (uint32_t)e;
    }
}

// Rows before the first run and behind the last (all of them where the offsets are bad, which
// run_tiles_kernel shows by listing no tile).
__global__ __launch_bounds__(256) void zero_uncovered_kernel(const int32_t* __restrict__ offsets,
                                                             int64_t E, int64_t S,
                                                             const uint32_t* __restrict__ ntile,
                                                             uint16_t* __restrict__ dx, int64_t N) {
  const bool none = *ntile == 0;
  const int64_t lo = none ? S : offsets[0], hi = none ? S : offsets[E];
  const int64_t units = N / 8, n = (lo + S - hi) * units;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    int64_t r = i / units;
    const int64_t c = i - r * units;
    if (r >= lo) r += hi - lo;
    *reinterpret_cast<u32x4*>(dx + r * N + 8 * c) = u32x4{0u, 0u, 0u, 0u};
  }
}

unsigned blocks_for(int64_t items, int64_t per, int64_t most) {
  const int64_t b = (items + per - 1) / per;
  return (unsigned)(b < 1 ? 1 : b < most ? b : most);
}

}  // namespace

hipError_t launch_sum_slices(const float* slices, int splits, uint16_t* y, int64_t M, int64_t N,
                             hipStream_t stream) {
  sum_slices_kernel<<<blocks_for(M * N / 4, 256, 4096), 256, 0, stream>>>(slices, splits, y, M * N);
  return hipGetLastError();
}

hipError_t launch_pad_rows(const uint16_t* src, uint16_t* dst, int64_t M, int64_t N, int64_t ld,
                           hipStream_t stream) {
  pad_rows_kernel<<<blocks_for(M * ld / 8, 256, 8192), 256, 0, stream>>>(src, dst, M, N, ld);
  return hipGetLastError();
}

hipError_t launch_run_tiles(const int32_t* offsets, int64_t E, int64_t S, int bm, uint32_t* tiles,
                            uint32_t* ntile, uint16_t* dx, int64_t N, uint32_t* flag,
                            hipStream_t stream) {
  run_tiles_kernel<<<1, 1024, 0, stream>>>(offsets, E, S, bm, tiles, ntile, flag);
  if (hipError_t e = hipGetLastError()) return e;
  zero_uncovered_kernel<<<256, 256, 0, stream>>>(offsets, E, S, ntile, dx, N);
  return hipGetLastError();
}

}  // namespace fmxq
