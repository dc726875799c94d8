// fmxq_grad_gemm.hip -- MFMA products with dequantized weights for training: the logits of
// a quantized head with the statistics of their softmax (nt), and the input gradient
// dx = dy . deq(W) of a quantized product (nn), of one matrix or of expert runs.
//
// Tile: BM rows by BN columns, 64 deep contraction steps in two LDS stages, a wave for every 32
// columns; two waves on a SIMD: of one block for the logits (BN = 256), of two for the
// gradients (BN = 128), whose contraction is often short and whose first loads and last stores
// then run under the other block's steps.  A goes global -> LDS with
// buffer_load ... lds; the packed weights go global -> registers some steps ahead, are
// dequantized there to fmxq_dequantize's bits and written to LDS.  Both stages hold rows of
// 64 contraction values (128 bytes), so one fragment read serves both forms: where the
// weights are packed along the outputs (nn), a thread takes 4 rows of 8 columns, and
// the transposition costs nothing: the roundings pack any two values.
//
// The barrier of a step sits before its last quarter's MFMAs, when every wave has read the
// stage: the next fragments, the DMA that refills this stage and the first share of its
// weights' dequantization run under them.
//
// Bound: MFMAs and dequantization in turn (a weight is dequantized once for every BM rows).  In the
// 256-row tiles the two waves of a SIMD hardly overlap them: 45% of the cycles are MFMAs and 50%
// VALU, 509 rows over 151936 x 2048.  Short contractions and expert runs of few rows are bound by
// the latency of the weights instead.
// Measured: logits of 509 rows, 151936 x 2048, 4 bits: 329 to 357 us, 0.89 to 0.96 PFLOP/s; gradients
// of 1000 rows, 128256 x 4096: 1.13 to 1.2 ms, 0.88 to 0.93 PFLOP/s; of 256 / 512 / 1024 rows, 14336 x
// 4096: 0.56 / 0.75 / 0.88 PFLOP/s; of 8192 rows in 64 expert runs, 512 x 2048, 8 bits: 67 us, 0.26
// PFLOP/s and 1.7 TB/s.
#include <type_traits>

#include "fmxq_grad_tile.hpp"

namespace fmxq {
namespace {

constexpr int kS = 64;   // contraction values per step

// Chunk c of row r at position c ^ swz8(r): distinct for 8 consecutive rows (fragment reads),
// and for 8 rows 8 apart (the transposing writes).
__device__ __forceinline__ int swz8(int r) { return (r ^ (r >> 3)) & 7; }

template <int BM, int BN>
struct GradCfg {
  static constexpr int W = BN / 32;              // waves
  static constexpr int WM = BM >= 64 ? 2 : 1;    // ... along the rows
  static constexpr int WN = W / WM;              // and along the columns
  static constexpr int MI = BM / WM / 32;        // 32-row groups of a wave
  static constexpr int NJ = BN / WN / 32;        // 32-column groups
  static constexpr int CB = BN / 64;             // 64-column blocks
};

// Tile mt of BM-row tiles over the expert runs [offsets[e], offsets[e + 1]): its first row,
// rows and expert, or rows = 0 behind the last tile.  Then *spare is the number of tiles
// behind the last one up to and with this one, of *spares in all, and rows *lo .. *hi are
// what the runs cover (nothing where the offsets decrease or leave 0 .. S).  All threads of
// the block take part, each in a range of experts; lds: T / 64 + 4 words.
template <int T>
__device__ __forceinline__ int64_t run_tile(const GradGemm& g, int64_t mt, int BM, int64_t* m0,
                                            int64_t* expert, int64_t* spare, int64_t* spares,
                                            int64_t* lo, int64_t* hi, int* lds) {
  uint32_t* wsum = reinterpret_cast<uint32_t*>(lds);
  int *found = lds + T / 64, &bad = lds[T / 64 + 3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* off = g.offsets;
  const int E = (int)g.experts, S = (int)g.M;
  const int per = (E + T - 1) / T, e0 = tid * per < E ? tid * per : E, e1 = e0 + per < E ? e0 + per : E;
  if (tid == 0) {
    bad = 0;
    found[1] = 0;
  }
  __syncthreads();
  uint32_t n = 0;
  bool ok = true;
  for (int e = e0; e < e1; ++e) {
    const int a = off[e], b = off[e + 1];
    ok = ok && a >= 0 && b >= a && b <= S;
    n += (uint32_t)((b - a + BM - 1) / BM);
  }
  if (!ok) bad = 1;
  uint32_t inc = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_up((int)inc, o, 64);
    if (lane >= o) inc += t;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  uint32_t at = inc - n, all = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    if (i < wave) at += wsum[i];
    all += wsum[i];
  }
  const int wrong = bad;
  if (wrong) all = 0;
  else if (mt >= at && mt < at + n) {
    for (int e = e0; e < e1; ++e) {
      const int a = off[e], b = off[e + 1], k = (b - a + BM - 1) / BM;
      if (mt < at + k) {
        const int r = a + (int)(mt - at) * BM;
        found[0] = r;
        found[1] = b - r < BM ? b - r : BM;
        found[2] = e;
        break;
      }
      at += k;
    }
  }
  __syncthreads();
  // Uniform for the compiler too: buffer resources made of them stay in scalar registers.
  *m0 = __builtin_amdgcn_readfirstlane(found[0]);
  *expert = __builtin_amdgcn_readfirstlane(found[2]);
  all = __builtin_amdgcn_readfirstlane(all);
  *spare = mt - all;
  *spares = g.max_tiles - all;
  *lo = all ? off[0] : S;
  *hi = all ? off[E] : S;
  const int rows = __builtin_amdgcn_readfirstlane(found[1]);
  if (wrong && blockIdx.x == 0 && tid == 0) atomicOr(g.flag, 1u);
  __syncthreads();  // lds may be overwritten
  return rows;
}

// Value j of 8 packed values as a float: a byte conversion each, after the masks.
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

template <int BM, int BN, int BITS, bool G32, bool NN>
__global__ __launch_bounds__(BN * 2, NN && BM < 64 ? 3 : 2) void grad_gemm_kernel(GradGemm g) {
  using C = GradCfg<BM, BN>;
  constexpr int W = C::W, WN = C::WN, MI = C::MI, NJ = C::NJ, CB = C::CB;
  constexpr int XI = BM / (8 * W);           // A DMA instructions per wave and step
  static_assert(XI * 8 * W == BM, "the waves' DMA instructions fill the rows");
  constexpr int WPU = BITS / 4;              // words of 8 values
  constexpr int NLD = (NN ? 4 : WPU) + 2;    // loads per thread and step
  // Stages of A, and steps whose packed weights are in registers or on their way.  Three for
  // the gradients, whose short steps (half the columns) end before memory answers.
  constexpr int AS = BN == 128 ? 3 : 2;
  // Each stage an LDS object of its own, so that the compiler can tell a DMA's target from
  // the reads of another stage.
  __shared__ __attribute__((aligned(1024))) uint8_t as0[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t as1[BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t as2[AS > 2 ? BM * 128 : 16];
  __shared__ __attribute__((aligned(1024))) uint8_t bs0[BN * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t bs1[BN * 128];
  __shared__ int32_t one[NN ? 1 : BM];  // the rows' wanted tokens, where they have one

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  // Tile of this block; every eighth block runs on one XCD.  One matrix: row tiles fastest in
  // contiguous shares, so that the blocks of an XCD share weight columns.  Expert runs: an
  // XCD takes every eighth row tile with all its columns, so that its rows are read once
  // (8192 rows of 64 experts of 512 x 2048, 8 bits: 300 MB past L2 the other way).
  const uint32_t tn = (uint32_t)((g.N + BN - 1) / BN);
  const uint32_t tm = (uint32_t)(g.offsets ? g.max_tiles : (g.M + BM - 1) / BM);
  const uint32_t total = gridDim.x;
  uint32_t b = blockIdx.x, split = 0;
  int64_t mt, nt;
  if (NN && g.offsets) {
    mt = (b & 7) + 8 * ((b >> 3) / tn);
    nt = (b >> 3) % tn;
  } else {
    if ((total & 7) == 0) b = (b & 7) * (total >> 3) + (b >> 3);
    split = b / (tm * tn);
    b -= split * (tm * tn);
    mt = b % tm;
    nt = b / tm;
  }
  int64_t m0 = mt * BM, rows = g.M - m0 < BM ? g.M - m0 : BM;
  const int64_t n0 = nt * BN;
  const uint32_t* w = g.w;
  const uint16_t *scales = g.scales, *biases = g.biases;
  const int gs = __builtin_ctz(g.group_size);
  const int64_t wk = NN ? g.N : g.C;             // values of a weight row
  const int64_t wpr = wk * BITS / 32, gpr = wk >> gs;
  if (NN && g.offsets) {
    int64_t e, spare, spares, lo, hi;
    rows = run_tile<C::W * 64>(g, mt, BM, &m0, &e, &spare, &spares, &lo, &hi,
                                 reinterpret_cast<int*>(as0));
    if (rows == 0) {
      // The tiles behind the last one zero the rows of no expert.
      const int64_t units = (g.N - n0 < BN ? g.N - n0 : BN) / 8;
      for (int64_t i = tid + spare * (C::W * 64); i < (lo + g.M - hi) * units;
           i += spares * (C::W * 64)) {
        int64_t r = i / units;
        const int64_t c = i - r * units;
        if (r >= lo) r += hi - lo;
        *reinterpret_cast<u32x4*>(g.y + r * g.ldy + n0 + 8 * c) = u32x4{0u, 0u, 0u, 0u};
      }
      return;
    }
    w += e * g.C * wpr;
    scales += e * g.C * gpr;
    biases += e * g.C * gpr;
  }
  const int64_t c0 = split * g.c_split;
  const int64_t c1 = c0 + g.c_split < g.C ? c0 + g.c_split : g.C;
  const int nk = c1 > c0 ? (int)((c1 - c0 + kS - 1) / kS) : 0;

  auto as = [&](int st) -> uint8_t* { return st == 0 ? as0 : st == 1 ? as1 : as2; };
  auto bs = [&](int st) -> uint8_t* { return st == 0 ? bs0 : bs1; };

  // ---- A: instruction i of a wave fills rows 8 (XI wave + i) .. + 8 of the stage.
  // (Rows past the tile's lie past its buffer.)
  const __amdgpu_buffer_rsrc_t ares = rsrc(g.a + m0 * g.lda, rows * g.lda * 2);
  const int arow = 8 * XI * wave + (lane >> 3);
  const uint32_t ao = (uint32_t)(arow * g.lda * 2), a8 = (uint32_t)(8 * g.lda * 2);
  const uint32_t ac = ((lane & 7) ^ swz8(arow)) * 8;  // the row 8 i further flips i into it
  const uint32_t acols = (uint32_t)g.a_cols;
  auto issue_a = [&](int k, int st) {
    const uint32_t kc = (uint32_t)c0 + (uint32_t)k * kS, end = k < nk ? acols : 0u;
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t col = kc + (ac ^ (8 * ((XI * wave + i) ^ (XI * wave))));
      const uint32_t off = col < end ? ao + i * a8 + col * 2 : 0x7ffffff0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lds_t*)(as(st) + 8 * (XI * wave + i) * 128),
                                               16, (int)off, 0, 0, 0);
    }
  };

  // ---- B: packed words and scales of a step in registers.
  struct Packed {
    uint32_t w[4 * WPU];
    uint16_t s, b;
  };
  Packed pk[AS];
  // nn: wave (column block, half); lane: rows 8 q + 4 half .. + 4, unit c of 8 columns.
  const int cb = wave % CB, half = wave / CB, q = lane >> 3, c = lane & 7;
  // nt: row (token) tid / 2, its contraction half tid % 2: a load then meets 32 rows' lines, of
  // which two lanes take their share (half as long in the data path as 64 rows).
  const int trow = tid >> 1, kh = tid & 1;
  uint32_t wo, so;
  if constexpr (NN) {
    // Columns past the weight's last are clamped into its rows; they are not stored.
    const int64_t u = n0 / 8 + 8 * cb + c;
    const int unit = (int)(u < wk / 8 ? u : wk / 8 - 1);
    wo = (uint32_t)((8 * q + 4 * half) * wpr * 4 + unit * BITS);
    // Lane c of an octet (whose 64 columns share a group; 32 of them in groups of 32) loads a
    // row's scale and the others take it from there.  A load of 64 rows costs the data path 64
    // lines whatever it takes of them, so none is repeated within a wave: an octet's upper
    // half loads the biases where the lower half's scales serve it too.
    so = (uint32_t)(((8 * q + 4 * half + (c & 3)) * gpr + (unit * 8 >> gs)) * 2);
  } else {
    wo = (uint32_t)(trow * wpr * 4);
    so = (uint32_t)(trow * gpr * 2);
  }
  const int64_t nrows = g.N - n0 < BN ? g.N - n0 : BN;
  auto issue_b = [&](int k, Packed& p) {
    const int64_t kc = c0 + (int64_t)k * kS;
    if constexpr (NN) {
      const int64_t left = k < nk ? (c1 - kc < kS ? c1 - kc : kS) : 0;
      const __amdgpu_buffer_rsrc_t wr = rsrc(w + kc * wpr, left * wpr * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int o = (int)(wo + (uint32_t)(i * wpr * 4));
        if constexpr (BITS == 8) {
          const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(wr, o, 0, 0));
          p.w[2 * i] = v[0];
          p.w[2 * i + 1] = v[1];
        } else {
          p.w[i] = __builtin_amdgcn_raw_buffer_load_b32(wr, o, 0, 0);
        }
      }
      // (Lanes that load nothing here have offsets past the buffer.)
      const __amdgpu_buffer_rsrc_t sr = rsrc(scales + kc * gpr, left * gpr * 2);
      const __amdgpu_buffer_rsrc_t br = rsrc(biases + kc * gpr, left * gpr * 2);
      p.s = __builtin_amdgcn_raw_buffer_load_b16(sr, (int)(G32 || c < 4 ? so : 0x7ffffff0u), 0, 0);
      p.b = __builtin_amdgcn_raw_buffer_load_b16(br, (int)(G32 || c >= 4 ? so : 0x7ffffff0u), 0, 0);
    } else {
      // A half step past the row's end takes the row's last values against zeros of A.
      const int kq = (int)(kc + 32 * kh < wk ? kc + 32 * kh : wk - 32);
      const __amdgpu_buffer_rsrc_t wr = rsrc(w + n0 * wpr, nrows * wpr * 4);
#pragma unroll
      for (int i = 0; i < WPU; ++i) {
        const u32x4 v = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, (int)(wo + kq * BITS / 8), 16 * i, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) p.w[4 * i + j] = v[j];
      }
      const __amdgpu_buffer_rsrc_t sr = rsrc(scales + n0 * gpr, nrows * gpr * 2);
      const __amdgpu_buffer_rsrc_t br = rsrc(biases + n0 * gpr, nrows * gpr * 2);
      const int o = (int)(so + 2 * (kq >> gs));
      p.s = __builtin_amdgcn_raw_buffer_load_b16(sr, o, 0, 0);
      p.b = __builtin_amdgcn_raw_buffer_load_b16(br, o, 0, 0);
    }
  };
  // nn: the scales and biases of the lane's four rows.
  float rsc[4], rbi[4];
  auto share = [&](const Packed& p) {
    if constexpr (NN) {
      const int sb = (int)((uint32_t)p.s | ((uint32_t)p.b << 16));
      auto from = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (G32) {  // lane i of the half octet holds both
          const uint32_t v = (uint32_t)__builtin_amdgcn_ds_swizzle(sb, 0x1c | (i << 5));
          rsc[i] = bf16_lo(v);
          rbi[i] = bf16_hi(v);
        } else {
          rsc[i] = bf16_lo((uint32_t)__builtin_amdgcn_ds_swizzle(sb, 0x18 | (i << 5)));
          rbi[i] = bf16_hi((uint32_t)__builtin_amdgcn_ds_swizzle(sb, 0x18 | ((4 + i) << 5)));
        }
      };
      from(std::integral_constant<int, 0>{});
      from(std::integral_constant<int, 1>{});
      from(std::integral_constant<int, 2>{});
      from(std::integral_constant<int, 3>{});
    }
  };
  // Quarter t of the thread's weights: 16 bytes of the stage.
  auto dequant = [&](const Packed& p, int st, int t) {
    if constexpr (NN) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = 2 * t + u, row = 64 * cb + 8 * c + j;
        u32x2 o;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Q8<BITS> a(p.w + 2 * i * WPU), z(p.w + (2 * i + 1) * WPU);
          o[i] = deq_pair(a.at(j), z.at(j), rsc[2 * i], rsc[2 * i + 1], rbi[2 * i], rbi[2 * i + 1]);
        }
        *reinterpret_cast<u32x2*>(bs(st) + row * 128 + ((q ^ swz8(row)) << 4) + 8 * half) = o;
      }
    } else {
      const float s = bf16_bits_to_f32(p.s), bb = bf16_bits_to_f32(p.b);
      const Q8<BITS> v(p.w + t * WPU);
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = deq_pair(v.at(2 * i), v.at(2 * i + 1), s, s, bb, bb);
      *reinterpret_cast<u32x4*>(bs(st) + trow * 128 + (((4 * kh + t) ^ swz8(trow)) << 4)) = o;
    }
  };

  f32x16 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // Fragment of sub-step s in a 32-row group: row r32, chunk 2 s + h.  The chunk's position is
  // an exclusive or with the swizzle, which the sub-step and the group's parity enter as
  // constants: one register an operand (kept from the compiler, which would hold them all).
  uint32_t fa = (uint32_t)((wm * MI * 32 + r32) * 128 + ((h ^ swz8(wm * MI * 32 + r32)) << 4));
  uint32_t fb = (uint32_t)((wn * NJ * 32 + r32) * 128 + ((h ^ swz8(wn * NJ * 32 + r32)) << 4));
  auto frag = [&](const uint8_t* stage, uint32_t f, int i, int s) {
    return *reinterpret_cast<const bf16x8*>(stage + (f ^ (uint32_t)(64 * (i & 1) ^ 32 * s)) + i * 4096);
  };
  bf16x8 a0[MI], a1[MI], b0[NJ], b1[NJ];
  auto read = [&](bf16x8 (&af)[MI], bf16x8 (&bf)[NJ], int sa, int sb, int s) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) bf[j] = frag(bs(sb), fb, j, s);
#pragma unroll
    for (int i = 0; i < MI; ++i) af[i] = frag(as(sa), fa, i, s);
  };
  auto mfmas = [&](const bf16x8 (&af)[MI], const bf16x8 (&bf)[NJ]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
  };
  // The dequantization's work in even shares under `quarters` quarters of a step's MFMAs.
  // (The logits' larger tile has no registers left for it.)
  auto pace = [&](int quarters) {
    if constexpr (BN == 256) return;
#pragma unroll
    for (int t = 0; t < quarters * MI * NJ; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                 // MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                 // DS read
      __builtin_amdgcn_sched_group_barrier(0x002, 56 / (MI * NJ), 0);    // VALU
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);                 // DS write
    }
  };
  // Step k (st = k modulo the stages' common period), its A in stage k % AS, its weights in
  // stage k % 2; the weights of step k + 1 go to the other stage, their first chunk during the
  // step before.
  auto step = [&](int k, auto stc) {
    constexpr int st = decltype(stc)::value, a = st % AS, a1s = (st + 1) % AS, a2s = (st + 2) % AS;
    constexpr int b = st % 2;
    asm volatile("" : "+v"(fa), "+v"(fb));
    read(a1, b1, a, b, 1);
    mfmas(a0, b0);
    dequant(pk[a1s], b ^ 1, 1);
    read(a0, b0, a, b, 2);
    mfmas(a1, b1);
    dequant(pk[a1s], b ^ 1, 2);
    read(a1, b1, a, b, 3);
    mfmas(a0, b0);
    dequant(pk[a1s], b ^ 1, 3);
    pace(3);
    // Step k + 1's A has landed (younger are the weights of AS - 1 steps and the A of AS - 2),
    // its weights are written, and this stage is read.
    __builtin_amdgcn_s_waitcnt(wait_enc(NLD + (AS - 2) * (XI + NLD), 0));
    __builtin_amdgcn_s_barrier();
    issue_a(k + AS, a);
    __builtin_amdgcn_sched_barrier(0);
    issue_b(k + 1 + AS, pk[a1s]);
    __builtin_amdgcn_sched_barrier(0);
    read(a0, b0, a1s, b ^ 1, 0);
    share(pk[a2s]);
    mfmas(a1, b1);
    dequant(pk[a2s], b, 0);
    pace(1);
  };
  int32_t id = -1;
  if (!NN && g.wanted_k == 1 && tid < rows) id = g.wanted[m0 + tid];
  if (nk > 0) {
#pragma unroll
    for (int i = 0; i < AS; ++i) {  // the waits count on this order
      issue_b(i, pk[i]);
      __builtin_amdgcn_sched_barrier(0);
      issue_a(i, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    share(pk[0]);
#pragma unroll
    for (int t = 0; t < 4; ++t) dequant(pk[0], 0, t);
    if (!NN && tid < BM) one[tid] = id;  // the loads behind it have landed
    __builtin_amdgcn_s_waitcnt(wait_enc((AS - 1) * (XI + NLD), 0));
    __builtin_amdgcn_s_barrier();
    issue_b(AS, pk[0]);
    __builtin_amdgcn_sched_barrier(0);
    read(a0, b0, 0, 0, 0);
    share(pk[1]);
    dequant(pk[1], 1, 0);
    if constexpr (AS == 2) {
      // Two steps a turn, the last one on zeros where nk is odd.
      for (int k = 0; k < nk; k += 2) {
        step(k, std::integral_constant<int, 0>{});
        step(k + 1, std::integral_constant<int, 1>{});
      }
    } else {
      for (int k = 0;; k += 6) {
        step(k, std::integral_constant<int, 0>{});
        if (k + 1 >= nk) break;
        step(k + 1, std::integral_constant<int, 1>{});
        if (k + 2 >= nk) break;
        step(k + 2, std::integral_constant<int, 2>{});
        if (k + 3 >= nk) break;
        step(k + 3, std::integral_constant<int, 3>{});
        if (k + 4 >= nk) break;
        step(k + 4, std::integral_constant<int, 4>{});
        if (k + 5 >= nk) break;
        step(k + 5, std::integral_constant<int, 5>{});
        if (k + 6 >= nk) break;
      }
    }
    __builtin_amdgcn_s_waitcnt(wait_enc(0, 0));
  }
  const int64_t mw = m0 + wm * MI * 32, nw = n0 + wn * NJ * 32;
  if constexpr (NN) store_grad<MI, NJ>(g, acc, mw, m0 + rows, nw, split);
  else {
    uint32_t out[MI][NJ];
    find_wanted<BM, BN, W * 64>(g, m0, rows, n0, mw, nw, one, reinterpret_cast<uint32_t*>(as0),
                                      out);
    store_stats<MI, NJ>(g, acc, out, mw, m0 + rows, nw);
  }
}

template <int BM, bool NN>
hipError_t launch_bm(const GradGemm& g, hipStream_t stream) {
  constexpr int BN = NN && BM < 256 ? kGradCols : kLogitCols;
  const int64_t tn = (g.N + BN - 1) / BN, tm = g.offsets ? g.max_tiles : (g.M + BM - 1) / BM;
  const int64_t blocks = tm * tn * g.splits;
  if (blocks < 1) return hipSuccess;
  if (blocks >= kMaxBlocks) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks), block(BN * 2);
  const bool g32 = NN && g.group_size == 32;
  if (g.bits == 4) {
    if (g32) grad_gemm_kernel<BM, BN, 4, NN, NN><<<grid, block, 0, stream>>>(g);
    else grad_gemm_kernel<BM, BN, 4, false, NN><<<grid, block, 0, stream>>>(g);
  } else {
    if (g32) grad_gemm_kernel<BM, BN, 8, NN, NN><<<grid, block, 0, stream>>>(g);
    else grad_gemm_kernel<BM, BN, 8, false, NN><<<grid, block, 0, stream>>>(g);
  }
  return hipGetLastError();
}

}  // namespace

// The lowest tile that holds the rows: a higher one multiplies zeros, a lower one dequantizes
// twice.  128 rows through 14336 x 4096 take 41 us in 128-row tiles, 129 in 256-row ones 46; 64
// expert runs of 128 rows, 512 x 2048, 47 us in 128-row tiles and 62 in 256-row ones, of 129 rows
// 87 and 64; runs of 128 in the mean with Zipf-like lengths 69 and 81, of 256 and more the higher
// tile takes 0.74 to 0.87 of the time.
int grad_gemm_rows(int64_t M) { return M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256; }

hipError_t launch_grad_gemm(const GradGemm& g, bool nn, int bm, hipStream_t stream) {
  // Offsets into one tile's rows and into 64 or 256 weight rows are 32 bits.
  if (!g.a || !g.w || (nn ? !g.out && !g.y : !g.stats || !g.wanted) || g.lda > kMaxLda ||
      256 * (nn ? g.N : g.C) >= 0x7ffffff0LL || g.c_split % kS || g.lda % 8 || g.a_cols % 8 ||
      (g.offsets && (!nn || !g.y || !g.flag || g.splits != 1)))
    return hipErrorInvalidValue;
  switch (bm) {
    case 32: return nn ? launch_bm<32, true>(g, stream) : hipErrorInvalidValue;
    case 64: return nn ? launch_bm<64, true>(g, stream) : hipErrorInvalidValue;
    case 128: return nn ? launch_bm<128, true>(g, stream) : launch_bm<128, false>(g, stream);
    case 256: return nn ? launch_bm<256, true>(g, stream) : launch_bm<256, false>(g, stream);
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

}  // namespace fmxq
