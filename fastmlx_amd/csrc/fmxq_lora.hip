// fmxq_lora.hip -- low-rank adapters of many requests beside a quantized product, and their
// gradients:
//   y  = x deq(W)^T + s_e (x A_e^T) B_e^T       for rows of adapter e
//   dx = dy deq(W) + dt A_e,  dt = s_e dy B_e
//   dA_e = sum dt^T x,  dB_e = s_e sum dy^T t   over e's rows, t = x A_e^T
// t and dt are fp32, as the sums of parts of the contraction.  As an operand of a matrix product
// each is a few bf16 values that add up to it: two (off by 2^-17 of it, where the result's own
// rounding to bf16 is 2^-8) for y and dx, three (all 24 bits) for the fp32 gradients, so that no
// step rounds to bf16 but the result's.
//
// The products with W take the adapter's part in their epilogue (add_lora): y and dx are written once,
// from fp32 sums.  Here are the narrow products around them.  Their rows are ordered by adapter
// beforehand; a tile that holds several is walked once for each and keeps the rows that are the
// adapter's own, so that one adapter's infinities reach no other row.  Few rows are taken one at a
// time instead.
// Of v_mfma_f32_16x16x32_bf16 the second operand gives a lane its row, so a lane holds 4
// neighbouring values of the first operand's index.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_internal.hpp"
#include "fmxq_train.hpp"

namespace fmxq {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTile = 32;  // rows of a shrink's tile: two MFMA tiles

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two jobs of one launch.
template <class Job>
struct Pair {
  Job job[2];
};

// Position p's row, and its adapter or -1.
struct RowOf {
  int64_t m;
  int e;
};
__device__ __forceinline__ RowOf row_of(const LoraRows& l, int64_t p) {
  RowOf r{0, -1};
  if (p >= l.M) return r;
  r.m = l.order ? l.order[p] : p;
  const int e = l.adapters[r.m];
  r.e = e >= 0 && e < l.E ? e : -1;
  return r;
}
// The next adapter of the wave's two rows a lane: one that no earlier turn took, or -1.
__device__ __forceinline__ int next_adapter(int e0, int e1) {
  const uint64_t b0 = __ballot(e0 >= 0), b1 = __ballot(e1 >= 0);
  if (b0) return __builtin_amdgcn_readlane(e0, __builtin_ctzll(b0));
  if (b1) return __builtin_amdgcn_readlane(e1, __builtin_ctzll(b1));
  return -1;
}

// ---- order ------------------------------------------------------------------------

// A stable counting sort of up to kSortRows rows by adapter in one block (rows without one last): its
// 16 waves take consecutive rows.  (2048 rows of 8 adapters: the two launches of the sort for any number
// 10.5 us.)
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kSortBuckets = 512;
__global__ __launch_bounds__(kSortThreads) void lora_sort_kernel(const int32_t* __restrict__ adapters, int M, int E,
                                                                 int bits, uint32_t* __restrict__ order,
                                                                 uint32_t* __restrict__ offsets) {
  __shared__ uint32_t cur[kSortWaves][kSortBuckets], sums[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kSortWaves * kSortBuckets; i += kSortThreads) cur[i / kSortBuckets][i % kSortBuckets] = 0;
  __syncthreads();
  const int per = (M + kSortThreads - 1) / kSortThreads * 64;
  const int r0 = wave * per < M ? wave * per : M, r1 = r0 + per < M ? r0 + per : M;
  auto bucket = [&](int m) {
    const int e = adapters[m];
    return e >= 0 && e < E ? e : E;
  };
  for (int m = r0 + lane; m < r1; m += 64) atomicAdd(&cur[wave][bucket(m)], 1u);
  __syncthreads();
  // Bucket tid's rows, those of the buckets before it, and each wave's first position in it.
  uint32_t n = 0;
  if (tid <= E)
    for (int w = 0; w < kSortWaves; ++w) n += cur[w][tid];
  uint32_t at = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)at, o, 64);
    if (lane >= o) at += u;
  }
  if (lane == 63) sums[wave] = at;
  __syncthreads();
  at -= n;
  for (int w = 0; w < wave; ++w) at += sums[w];
  if (tid <= E) {
    offsets[tid] = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = cur[w][tid];
      cur[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int m = r0 + lane; m - lane < r1; m += 64) {
    const bool on = m < r1;
    const uint32_t b = on ? (uint32_t)bucket(m) : 0u;
    uint64_t same = __ballot(on);
    for (int i = 0; i < bits; ++i) {
      const uint64_t set = __ballot((b >> i) & 1u);
      same &= (b >> i) & 1u ? set : ~set;
    }
    const uint64_t before = same & ((1ull << lane) - 1);
    if (on) order[cur[wave][b] + (uint32_t)__popcll(before)] = (uint32_t)m;
    // The wave's own LDS accesses, in order.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (on && before == 0) cur[wave][b] += (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// ---- t = P . V_e^T ----------------------------------------------------------------

// Block: 32 positions and a part of the contraction, whose 32-deep steps its 8 waves take in turn, the
// next ones' loads under way.
template <int RT>
__global__ __launch_bounds__(512) void lora_shrink_kernel(LoraRows l, Pair<LoraShrink> jobs) {
  constexpr int R = RT < 4 ? 2 * RT : 8;  // the sums that meet in LDS at once
  __shared__ __attribute__((aligned(16))) f32x4 part[8][R][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool second = (int)blockIdx.y >= jobs.job[0].splits;
  const LoraShrink& a = jobs.job[second];
  const int split = (int)blockIdx.y - (second ? jobs.job[0].splits : 0);
  const int64_t p0 = (int64_t)blockIdx.x * kTile;
  // (Positions past the last take its row's values and no part.)
  const int64_t q0 = p0 + r16 < l.M ? p0 + r16 : l.M - 1, q1 = p0 + 16 + r16 < l.M ? p0 + 16 + r16 : l.M - 1;
  const int64_t m0 = l.order ? l.order[q0] : q0, m1 = l.order ? l.order[q1] : q1;
  int e0 = l.adapters[m0], e1 = l.adapters[m1];
  if (wave == 0 && blockIdx.y == 0 && (e0 >= l.E || e1 >= l.E)) atomicOr(l.flag, 1u);
  if (e0 >= l.E || p0 + r16 >= l.M) e0 = -1;
  if (e1 >= l.E || p0 + 16 + r16 >= l.M) e1 = -1;
  const int steps = (int)((a.C + 31) / 32);
  const int s0 = (int)((int64_t)steps * split / a.splits);
  const int s1 = (int)((int64_t)steps * (split + 1) / a.splits);
  const uint16_t *x0 = a.p + m0 * a.ldp, *x1 = a.p + m1 * a.ldp;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int cur; (cur = next_adapter(e0, e1)) >= 0;) {
    const uint16_t* vr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int j = 16 * i + r16;
      vr[i] = a.v + ((int64_t)cur * l.r + (j < l.r ? j : 0)) * a.ldv;
    }
    f32x4 acc[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Steps that are loaded together: more only where one alone leaves a wave waiting between its products
    // (2048 rows of 4096 and 14336 values, us with 1 and 2: rank 32 20, 25; rank 64 64.6, 63.4).
    constexpr int U = RT == 4 ? 2 : 1;
    struct Steps {
      u32x4 x[U][2], b[U][RT];
    };
    auto load = [&](int s, Steps& v) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t c = 32 * (int64_t)(s + k) + 8 * q4;
        const bool in = s + k < s1 && c < a.C;
        v.x[k][0] = in ? *reinterpret_cast<const u32x4*>(x0 + c) : zero;
        v.x[k][1] = in ? *reinterpret_cast<const u32x4*>(x1 + c) : zero;
#pragma unroll
        for (int i = 0; i < RT; ++i) v.b[k][i] = in ? *reinterpret_cast<const u32x4*>(vr[i] + c) : zero;
      }
    };
    auto multiply = [&](const Steps& v) {
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          acc[0][i] = mfma(v.b[k][i], v.x[k][0], acc[0][i]);
          acc[1][i] = mfma(v.b[k][i], v.x[k][1], acc[1][i]);
        }
    };
    Steps v0, v1;
    const int s = s0 + U * wave;
    load(s, v0);
    for (int k = s; k < s1; k += 16 * U) {
      load(k + 8 * U, v1);
      multiply(v0);
      load(k + 16 * U, v0);
      multiply(v1);
    }
    // The waves' sums, in their order.
#pragma unroll
    for (int i0 = 0; i0 < RT; i0 += R / 2) {
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        part[wave][2 * i][lane] = acc[0][i0 + i];
        part[wave][2 * i + 1][lane] = acc[1][i0 + i];
      }
      __syncthreads();
      if (wave < R) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += part[k][wave][lane];
        const int j = 16 * (i0 + (wave >> 1)) + 4 * q4, half = wave & 1;
        if ((half ? e1 : e0) == cur && j < l.r)
          *reinterpret_cast<f32x4*>(a.t + ((int64_t)split * l.M + p0 + 16 * half + r16) * l.r + j) = sum;
      }
      __syncthreads();
    }
    if (e0 == cur) e0 = -1;
    if (e1 == cur) e1 = -1;
  }
}

// Words that a product behind this launch wants zero.
__device__ __forceinline__ void clear(const Zeros& z) {
  if (blockIdx.y) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < z.n; i += (int64_t)gridDim.x * 256) z.p[i] = 0u;
}

// A value as the bf16 values that add up to it.  A finite value's parts are finite, also where it is
// beyond bf16's largest; an infinity is all in the first part, as infinity less infinity would make
// NaN of it.
__device__ __forceinline__ float to_part(float v) {
  constexpr float kMost = 0x1.fep127f;
  return fabsf(v) < INFINITY ? __builtin_amdgcn_fmed3f(v, -kMost, kMost) : v;
}
__device__ __forceinline__ float left_of(float v, float part) { return fabsf(v) < INFINITY ? v - part : 0.f; }

template <int PARTS>
__device__ __forceinline__ void store_parts(uint16_t* u, int r, float v) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    const uint32_t h = f32_to_bf16_rne(to_part(v));
    u[k * r] = (uint16_t)h;
    v = left_of(v, bf16_bits_to_f32(h));
  }
}

// A thread for 8 values of a row: the sum of the shrink's parts, scaled, in bf16 parts.
__global__ __launch_bounds__(256) void lora_parts_kernel(LoraRows l, Pair<LoraShrink> jobs, int parts,
                                                         const float* __restrict__ scales, Zeros z) {
  clear(z);
  const LoraShrink& a = jobs.job[blockIdx.y];
  const int chunks = l.r / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, p = i / chunks;
  const int j = (int)(i - p * chunks) * 8;
  if (p >= l.M) return;
  const RowOf w = row_of(l, p);
  if (w.e < 0) return;
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) {
    const f32x4* t = reinterpret_cast<const f32x4*>(a.t + ((int64_t)k * l.M + p) * l.r + j);
    lo += t[0];
    hi += t[1];
  }
  const float s = scales[w.e];
  lo *= s;
  hi *= s;
  uint16_t* u = a.u + w.m * parts * l.r + j;
  for (int k = 0; k < parts; ++k) {
    u32x4 o;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      o[x] = pack_bf16x2(to_part(lo[2 * x]), to_part(lo[2 * x + 1]));
      o[2 + x] = pack_bf16x2(to_part(hi[2 * x]), to_part(hi[2 * x + 1]));
    }
    *reinterpret_cast<u32x4*>(u + k * l.r) = o;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      lo[2 * x] = left_of(lo[2 * x], bf16_lo(o[x]));
      lo[2 * x + 1] = left_of(lo[2 * x + 1], bf16_hi(o[x]));
      hi[2 * x] = left_of(hi[2 * x], bf16_lo(o[2 + x]));
      hi[2 * x + 1] = left_of(hi[2 * x + 1], bf16_hi(o[2 + x]));
    }
  }
}

// A wave for every value.
__global__ __launch_bounds__(256) void lora_shrink_rows_kernel(LoraRows l, LoraShrink a,
                                                               const float* __restrict__ scales, Zeros z) {
  clear(z);
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, j = 4 * blockIdx.y + (threadIdx.x >> 6);
  const int e = l.adapters[m];
  if (e < 0 || e >= l.E) {
    if (e >= l.E && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(l.flag, 1u);
    return;
  }
  const uint16_t *x = a.p + m * a.ldp, *w = a.v + ((int64_t)e * l.r + j) * a.ldv;
  float s = 0.f;
  constexpr int U = 8;
  for (int64_t c0 = 8 * lane; c0 < a.C; c0 += 512 * U) {
    u32x4 p[U], v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t c = c0 + 512 * k;
      p[k] = v[k] = u32x4{0u, 0u, 0u, 0u};
      if (c < a.C) {
        p[k] = *reinterpret_cast<const u32x4*>(x + c);
        v[k] = *reinterpret_cast<const u32x4*>(w + c);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = __builtin_fmaf(bf16_lo(p[k][i]), bf16_lo(v[k][i]), s);
        s = __builtin_fmaf(bf16_hi(p[k][i]), bf16_hi(v[k][i]), s);
      }
  }
  s = wave_sum(s) * scales[e];
  if (lane == 0) store_parts<2>(a.u + m * 2 * l.r + j, l.r, s);
}

// ---- g_e = sum P^T u -----------------------------------------------------------------

// Byte offset of a row of P's tile in LDS: 16 columns of the 16 rows that the quarters of a wave read at
// once (rows 8 q .. + 4) fall into all banks twice, the least that 512 bytes take.
__device__ __forceinline__ int tile_row(int row) { return row * 288 + (row >> 3) * 128; }
constexpr int kOuterRows = 64;      // of a step
constexpr int kOuterStretch = 256;  // whose rows are found together
constexpr int kTileBytes = kOuterRows * 288 + kOuterRows / 8 * 128;

// A lane's 8 values of one column in rows 8 q4 .. + 8: p is the address of 8 bytes of row 8 q4 +
// r16 / 4, and p4 that of the row 4 further on.
__device__ __forceinline__ u32x4 turned(const uint8_t* p, const uint8_t* p4) {
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p4);
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Adapter e's positions in parts of `chunk`; the parts of one that has several go to slots of `part`.
struct Run {
  int64_t lo, hi;
};
__device__ __forceinline__ Run run_of(const LoraRows& l, int64_t e) {
  return l.offsets ? Run{l.offsets[e], l.offsets[e + 1]} : Run{0, l.M};
}
// (A run of more than a chunk has at most 2 (len / chunk) parts, so runs' slots are apart.)
__device__ __forceinline__ int64_t slot_of(const Run& r, int64_t chunk) { return r.lo / chunk * 2; }

// The launch's blocks: `blocks` of job 0, then job 1's.
struct OuterGrid {
  int64_t chunk[2];
  uint32_t tiles[2], blocks;
};

// Block: 128 columns of P and all of the rank, over a part of adapter e's rows in steps of 64.  A step's
// rows are loaded while the one before is multiplied; which rows they are is found beforehand, so that
// no load waits for another.
template <int RT>
__global__ __launch_bounds__(256) void lora_outer_kernel(LoraRows l, Pair<LoraOuter> jobs, OuterGrid grid) {
  constexpr int UP = RT * 32 + 32;                 // bytes of a row of u in LDS
  constexpr int UC = RT * 2;                       // its 16-byte chunks
  constexpr int TU = kOuterRows * UC * kLoraParts, NU = (TU + 255) / 256;  // ... of a step, and a thread's
  __shared__ __attribute__((aligned(16))) uint8_t ps[kTileBytes];
  __shared__ __attribute__((aligned(16))) uint8_t us[kLoraParts][kOuterRows * UP];
  __shared__ int row_of_pos[kOuterStretch + kOuterRows];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool second = blockIdx.x >= grid.blocks;
  const LoraOuter& o = jobs.job[second];
  const int64_t chunk = grid.chunk[second];
  const uint32_t b = blockIdx.x - (second ? grid.blocks : 0), tiles = grid.tiles[second];
  const int64_t c0 = (int64_t)(b % tiles) * 128, pt = b / tiles, e = blockIdx.y;
  const Run run = run_of(l, e);
  const int64_t begin = run.lo + pt * chunk;
  if (begin >= run.hi && pt > 0) return;
  const int64_t end = begin + chunk < run.hi ? begin + chunk : run.hi;
  const bool alone = run.hi - run.lo <= chunk;
  float* out = alone ? o.g + e * o.C * l.r : o.part + (slot_of(run, chunk) + pt) * o.C * l.r;
  f32x4 acc[2][RT];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u32x4 zero = {0u, 0u, 0u, 0u};
  // Rows of a stretch of kOuterStretch positions, or -1.  (Without an order the one adapter's rows are
  // those that name it.)
  auto find_rows = [&](int64_t p0) {
    for (int i = tid; i < kOuterStretch; i += 256) {
      const int64_t pos = p0 + i;
      int m = -1;
      if (pos < end) {
        if (l.order) m = (int)l.order[pos];
        else if (l.adapters[pos] == 0) m = (int)pos;
      }
      row_of_pos[i] = m;
    }
  };
  struct Step {
    u32x4 p[4], u[NU];
  };
  auto load = [&](int at, Step& v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t m = row_of_pos[at + (tid >> 4) + 16 * k], c = c0 + 8 * (tid & 15);
      v.p[k] = m >= 0 && c < o.C ? *reinterpret_cast<const u32x4*>(o.p + m * o.ldp + c) : zero;
    }
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const int i = tid + 256 * k, row = i / (UC * kLoraParts), c = i % (UC * kLoraParts);
      const int part = c / UC, j = c % UC * 8;
      const int64_t m = i < TU ? row_of_pos[at + row] : -1;
      v.u[k] = m >= 0 && j < l.r ? *reinterpret_cast<const u32x4*>(o.u + (m * kLoraParts + part) * l.r + j) : zero;
    }
  };
  auto multiply = [&](const Step& v) {
    __syncthreads();  // the step before has been read
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<u32x4*>(ps + tile_row((tid >> 4) + 16 * k) + 16 * (tid & 15)) = v.p[k];
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const int i = tid + 256 * k, row = i / (UC * kLoraParts), c = i % (UC * kLoraParts);
      if (i < TU) *reinterpret_cast<u32x4*>(us[c / UC] + row * UP + c % UC * 16) = v.u[k];
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kOuterRows / 32; ++kk) {
      const int tr = 32 * kk + 8 * q4 + (r16 >> 2), at = 8 * (r16 & 3);
      u32x4 pf[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = 2 * (32 * wave + 16 * k) + at;
        pf[k] = turned(ps + tile_row(tr) + col, ps + tile_row(tr + 4) + col);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int x = 0; x < kLoraParts; ++x) {
          const uint8_t* q = us[x] + tr * UP + 32 * i + at;
          const u32x4 uf = turned(q, q + 4 * UP);
          acc[0][i] = mfma(uf, pf[0], acc[0][i]);
          acc[1][i] = mfma(uf, pf[1], acc[1][i]);
        }
    }
  };
  for (int64_t p0 = begin; p0 < end; p0 += kOuterStretch) {
    __syncthreads();  // the stretch before is done with its rows
    find_rows(p0);
    __syncthreads();
    const int n = end - p0 < kOuterStretch ? (int)(end - p0) : kOuterStretch;
    Step a, b;
    load(0, a);
    for (int at = 0; at < n; at += 2 * kOuterRows) {
      load(at + kOuterRows, b);
      multiply(a);
      if (at + kOuterRows >= n) break;
      if (at + 2 * kOuterRows < n) load(at + 2 * kOuterRows, a);
      multiply(b);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t c = c0 + 32 * wave + 16 * k + r16;
      const int j = 16 * i + 4 * q4;
      if (c >= o.C || j >= l.r) continue;
      if (o.rows_r) {
#pragma unroll
        for (int x = 0; x < 4; ++x) out[(j + x) * o.C + c] = acc[k][i][x];
      } else {
        *reinterpret_cast<f32x4*>(out + c * l.r + j) = acc[k][i];
      }
    }
}

// The sums of parts, of the adapters that have several.
__global__ __launch_bounds__(256) void lora_outer_sum_kernel(LoraRows l, Pair<LoraOuter> jobs, OuterGrid grid) {
  const int64_t e = blockIdx.y;
  const Run run = run_of(l, e);
  const LoraOuter& o = jobs.job[blockIdx.z];
  const int64_t chunk = grid.chunk[blockIdx.z], size = o.C * l.r;
  if (run.hi - run.lo <= chunk) return;
  const int64_t parts = (run.hi - run.lo + chunk - 1) / chunk;
  const float* from = o.part + slot_of(run, chunk) * size;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 1024) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int64_t k = 0; k < parts; ++k) s += *reinterpret_cast<const f32x4*>(from + k * size + i);
    *reinterpret_cast<f32x4*>(o.g + e * size + i) = s;
  }
}

// ---- turned matrices -------------------------------------------------------------------

__global__ __launch_bounds__(256) void lora_turn_kernel(LoraRows l, Pair<LoraTurn> jobs, uint32_t blocks) {
  __shared__ uint16_t s[32][33];
  const int64_t e = blockIdx.y;
  if (l.offsets && l.offsets[e] == l.offsets[e + 1]) return;
  const bool second = blockIdx.x >= blocks;
  const LoraTurn& t = jobs.job[second];
  const uint32_t b = blockIdx.x - (second ? blocks : 0), tc = (uint32_t)((t.C + 31) / 32);
  const int64_t r0 = (int64_t)(b / tc) * 32, c0 = (int64_t)(b % tc) * 32;
  const int x = threadIdx.x & 31, yy = threadIdx.x >> 5;
#pragma unroll
  for (int i = yy; i < 32; i += 8)
    s[i][x] = r0 + i < t.R && c0 + x < t.C ? t.in[(e * t.R + r0 + i) * t.C + c0 + x] : 0;
  __syncthreads();
#pragma unroll
  for (int i = yy; i < 32; i += 8)
    if (c0 + i < t.C && r0 + x < t.ldo) t.out[(e * t.C + c0 + i) * t.ldo + r0 + x] = s[x][i];
}

bool rank_ok(int r) { return r >= 8 && r <= kLoraMaxRank && r % 8 == 0; }
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up(int64_t v, int64_t to) { return div_up(v, to) * to; }

template <class Job>
Pair<Job> pair_of(const Job* j, int n) {
  return Pair<Job>{{j[0], j[n - 1]}};
}

// Rows of a part: whole runs where the columns alone fill the chip (four blocks a compute unit),
// else as many parts as do, of 256 rows at least.
int64_t outer_chunk(int64_t M, int64_t C) {
  const int64_t tiles = std::max<int64_t>(div_up(C, 128), 1), parts = std::max<int64_t>(1024 / tiles, 1);
  return std::max<int64_t>(up(div_up(M, parts), kOuterRows), 256);
}
int64_t outer_parts(int64_t M, int64_t C) { return std::max<int64_t>(div_up(M, outer_chunk(M, C)), 1); }

}  // namespace

bool lora_sort_supported(int64_t M, int64_t E) { return M <= 16 * kSortThreads && E < kSortBuckets; }
hipError_t launch_lora_sort(const int32_t* adapters, int64_t M, int64_t E, uint32_t* order, uint32_t* offsets,
                            hipStream_t stream) {
  if (M < 1 || !lora_sort_supported(M, E)) return hipErrorInvalidValue;
  int bits = 1;
  while (E >= ((int64_t)1 << bits)) ++bits;
  lora_sort_kernel<<<1, kSortThreads, 0, stream>>>(adapters, (int)M, (int)E, bits, order, offsets);
  return hipGetLastError();
}

// Parts that leave each of a block's 8 waves 4 steps, while the blocks are no more than two for each of
// 256 compute units.
int lora_splits(int64_t M, int64_t C) {
  const int64_t tiles = std::max<int64_t>(div_up(M, kTile), 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, C / (32 * 8 * 4), 16}));
}

hipError_t launch_lora_shrink(const LoraRows& l, const LoraShrink* s, int n, hipStream_t stream) {
  if (!rank_ok(l.r) || n < 1 || n > 2) return hipErrorInvalidValue;
  int64_t splits = 0;
  for (int i = 0; i < n; ++i) {
    if (s[i].ldp % 8 || s[i].ldv % 8 || s[i].C % 8 || s[i].splits < 1) return hipErrorInvalidValue;
    splits += s[i].splits;
  }
  if (l.M < 1) return hipSuccess;
  const dim3 grid((unsigned)div_up(l.M, kTile), (unsigned)splits);
  const Pair<LoraShrink> jobs = pair_of(s, n);
  if (l.r <= 16) lora_shrink_kernel<1><<<grid, 512, 0, stream>>>(l, jobs);
  else if (l.r <= 32) lora_shrink_kernel<2><<<grid, 512, 0, stream>>>(l, jobs);
  else if (l.r <= 64) lora_shrink_kernel<4><<<grid, 512, 0, stream>>>(l, jobs);
  else lora_shrink_kernel<8><<<grid, 512, 0, stream>>>(l, jobs);
  return hipGetLastError();
}

hipError_t launch_lora_parts(const LoraRows& l, const LoraShrink* s, int n, int parts, const float* scales,
                             const Zeros& z, hipStream_t stream) {
  if (!rank_ok(l.r) || n < 1 || n > 2) return hipErrorInvalidValue;
  if (l.M < 1) return hipSuccess;
  const dim3 grid((unsigned)div_up(l.M * (l.r / 8), 256), (unsigned)n);
  lora_parts_kernel<<<grid, 256, 0, stream>>>(l, pair_of(s, n), parts, scales, z);
  return hipGetLastError();
}

hipError_t launch_lora_shrink_rows(const LoraRows& l, const LoraShrink& s, const float* scales,
                                   const Zeros& z, hipStream_t stream) {
  if (!rank_ok(l.r) || s.ldp % 8 || s.ldv % 8 || s.C % 8 || l.order) return hipErrorInvalidValue;
  if (l.M < 1) return hipSuccess;
  lora_shrink_rows_kernel<<<dim3((unsigned)l.M, (unsigned)(l.r / 4)), 256, 0, stream>>>(l, s, scales, z);
  return hipGetLastError();
}

int64_t lora_outer_floats(int64_t M, int64_t C, int r) {
  const int64_t chunk = outer_chunk(M, C);
  return M > chunk ? 2 * (M / chunk + 1) * C * r : 0;
}
int64_t lora_outer_blocks(int64_t M, int64_t C, int64_t E) {
  return div_up(C, 128) * outer_parts(M, C) * E;
}

hipError_t launch_lora_outer(const LoraRows& l, const LoraOuter* o, int n, hipStream_t stream) {
  if (!rank_ok(l.r) || n < 1 || n > 2 || l.E < 1 || (!l.offsets && l.E != 1)) return hipErrorInvalidValue;
  OuterGrid g{};
  int64_t blocks = 0, size = 0;
  bool sums = false;
  for (int i = 0; i < n; ++i) {
    if (o[i].ldp % 8 || o[i].C < 1) return hipErrorInvalidValue;
    g.chunk[i] = outer_chunk(l.M, o[i].C);
    g.tiles[i] = (uint32_t)div_up(o[i].C, 128);
    blocks += g.tiles[i] * outer_parts(l.M, o[i].C);
    if (i == 0) g.blocks = (uint32_t)blocks;
    sums = sums || l.M > g.chunk[i];
    size = std::max(size, o[i].C * l.r);
  }
  if (blocks * l.E >= kLoraMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)l.E);
  const Pair<LoraOuter> jobs = pair_of(o, n);
  if (l.r <= 16) lora_outer_kernel<1><<<grid, 256, 0, stream>>>(l, jobs, g);
  else if (l.r <= 32) lora_outer_kernel<2><<<grid, 256, 0, stream>>>(l, jobs, g);
  else if (l.r <= 64) lora_outer_kernel<4><<<grid, 256, 0, stream>>>(l, jobs, g);
  else lora_outer_kernel<8><<<grid, 256, 0, stream>>>(l, jobs, g);
  if (hipError_t e = hipGetLastError()) return e;
  if (!sums) return hipSuccess;
  const dim3 sum((unsigned)std::min<int64_t>(div_up(size, 1024), 1024), (unsigned)l.E, (unsigned)n);
  lora_outer_sum_kernel<<<sum, 256, 0, stream>>>(l, jobs, g);
  return hipGetLastError();
}

int64_t lora_turn_blocks(int64_t C, int64_t ldo, int64_t E) { return div_up(C, 32) * div_up(ldo, 32) * E; }

hipError_t launch_lora_turn(const LoraRows& l, const LoraTurn* t, int n, hipStream_t stream) {
  if (n < 1 || n > 2 || l.E < 1) return hipErrorInvalidValue;
  int64_t blocks = 0, first = 0;
  for (int i = 0; i < n; ++i) {
    if (t[i].R < 1 || t[i].C < 1) return hipErrorInvalidValue;
    blocks += lora_turn_blocks(t[i].C, t[i].ldo, 1);
    if (i == 0) first = blocks;
  }
  if (blocks * l.E >= kLoraMaxBlocks) return hipErrorInvalidValue;
  lora_turn_kernel<<<dim3((unsigned)blocks, (unsigned)l.E), 256, 0, stream>>>(l, pair_of(t, n), (uint32_t)first);
  return hipGetLastError();
}

// ---- the product with an adapter's part --------------------------------------------------

namespace {
// Rows from which the weights are dequantized to a panel beforehand, and most bytes of one.
constexpr int64_t kOutPanelRows = 1793;
constexpr int64_t kOutPanelBytes = 512 << 20;
constexpr int kOutCus = 256;  // compute units that plans are made for
}  // namespace

// Times of the three kernels that take more than 64 rows, in us.  Chunks of 64 rows on the kernel for
// few rows: 0.8 ns a 64-deep step of a block of 32 outputs (65 to 128 rows, 4096 x 4096: 18 us, 256 rows
// 33; 512 rows, 1024 x 4096: 29).  The wide product: 1 PFLOP/s, 20 us of ends, and 0.8 us for each part of a cut
// tile, which its last block adds up (128 rows 4096 x 4096 33 us, 14336 x 4096 42, 4096 x 14336 56; 256
// rows, 14336 x 4096: 62; 512 rows, 1024 x 4096: 40).
static double few_rows_us(int64_t M, int64_t N, int64_t K) {
  return 4. + 0.8e-3 * (double)(div_up(M, kSkinnyRows) * div_up(N, 32) * div_up(K, 64));
}
static double wide_us(int64_t M, int64_t N, int64_t K, const WidePlan& w) {
  const double parts = w.sk_len > 0 ? (double)w.nk / w.sk_len : 0.;
  return 20. + 2e-9 * (double)(up(M, w.bm) * N) * (double)K + 0.8 * parts;
}

OutPlan out_plan(int64_t M, int64_t N, int64_t K) {
  constexpr int cus = kOutCus;
  OutPlan p{};
  // The largest format's limits, so that a plan goes by the sizes alone.
  alignas(16) static uint16_t any;  // an aligned address
  const QmmArgs q{&any, reinterpret_cast<const uint32_t*>(&any), &any, &any, nullptr, &any, M, N, K, K, N, 32, 8};
  p.thin = thin_supported(M, N, K);
  const bool chunks = skinny_gemm_supported(K, 32, K) && div_up(M, kSkinnyRows) <= 65535;
  p.skinny = !p.thin && chunks && M <= kSkinnyRows;
  if (!p.thin && !p.skinny && qmm_wide_supported(q)) {
    p.wide = !chunks || wide_us(M, N, K, qmm_wide_plan(M, N, K, cus)) < few_rows_us(M, N, K);
    p.skinny = !p.wide;
  }
  // What the wide product does not take: widths that are no multiple of 256, outputs of 8.
  const bool rest = !p.thin && !p.skinny && !p.wide;
  p.panel = rest && M >= kOutPanelRows && panel_gemm_supported(K);
  p.bm = p.panel ? kPanelRows : std::max(grad_gemm_rows(M), 128);
  if (rest && chunks && few_tokens(M, N, p.bm, cus)) {
    p.skinny = true;
    p.panel = false;
  }
  p.piece = N;
  if (p.panel)
    p.piece = std::min<int64_t>(N, std::max<int64_t>(kOutPanelBytes / 2 / K / kLogitCols * kLogitCols, kLogitCols));
  // Parts of the contraction where the tiles leave compute units idle, of 256 values at least.
  p.splits = 1;
  const int64_t tiles = div_up(M, p.bm) * div_up(N, kLogitCols);
  if (rest && !p.skinny && N % 4 == 0 && p.piece == N)
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(cus / std::max<int64_t>(tiles, 1), K / 256));
  p.c_split = up(div_up(K, p.splits), 64);
  p.splits = (int)std::max<int64_t>(1, div_up(K, p.c_split));
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
  };
  if (p.wide) {
    const WidePlan w = qmm_wide_plan(M, N, K, cus);
    p.slices = take(w.ws_floats * 4);
    p.counters = w.sk_len > 0 ? w.tiles : 0;
    p.count_at = take(p.counters * 4);
  } else {
    p.slices = take(p.splits > 1 ? p.splits * M * N * 4 : 0);
  }
  p.panel_at = take(p.panel ? p.piece * K * 2 : 0);
  p.xp = take(p.skinny ? skinny_pack_bytes(M, K) : 0);
  p.bytes = at;
  return p;
}

hipError_t launch_out(const uint16_t* x, const uint32_t* w, const uint16_t* scales, const uint16_t* biases,
                      const LoraAdd& lora, uint16_t* y, int64_t M, int64_t N, int64_t K, int group_size,
                      int bits, const OutPlan& p, void* ws, uint32_t* flag, hipStream_t stream) {
  char* base = static_cast<char*>(ws);
  if (p.wide) {
    QmmArgs q{x, w, scales, biases, nullptr, y, M, N, K, K, N, group_size, bits};
    q.ws = reinterpret_cast<float*>(base + p.slices);
    q.tile_count = reinterpret_cast<uint32_t*>(base + p.count_at);
    return launch_qmm_wide(q, qmm_wide_plan(M, N, K, kOutCus), flag, stream, &lora);
  }
  uint16_t* panel = reinterpret_cast<uint16_t*>(base + p.panel_at);
  float* slices = reinterpret_cast<float*>(base + p.slices);
  for (int64_t n0 = 0; n0 < N; n0 += p.piece) {
    GradGemm g;
    g.epi = kEpiOut;
    g.a = x;
    g.lda = g.a_cols = K;
    g.M = M;
    g.N = std::min(p.piece, N - n0);
    g.C = K;
    g.c_split = p.c_split;
    g.splits = p.splits;
    g.w = w + n0 * (K * bits / 32);
    g.scales = scales + n0 * (K / group_size);
    g.biases = biases + n0 * (K / group_size);
    g.group_size = group_size;
    g.bits = bits;
    g.lora = lora;
    g.lora.v = lora.v + n0 * lora.r;
    if (p.splits > 1) {
      g.out = slices;
    } else {
      g.y = y + n0;
      g.ldy = N;
    }
    if (p.skinny && skinny_pack_bytes(M, K)) g.xp = base + p.xp;
    if (p.panel) {
      if (hipError_t r = launch_dequantize(g.w, g.scales, g.biases, panel, g.N, K, group_size, bits, stream))
        return r;
      g.panel = panel;
      g.ldp = K;
    }
    if (hipError_t r = p.thin    ? launch_thin_gemm(g, stream)
                       : p.skinny ? launch_skinny_gemm(g, false, stream)
                       : p.panel  ? launch_panel_gemm(g, false, stream)
                                  : launch_grad_gemm(g, false, p.bm, stream))
      return r;
  }
  return p.splits > 1 ? launch_sum_slices(slices, p.splits, y, M, N, stream) : hipSuccess;
}

}  // namespace fmxq
