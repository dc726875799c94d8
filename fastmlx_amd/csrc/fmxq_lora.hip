// fmxq_lora.hip -- low-rank adapters of many requests beside a quantized product, and their
// gradients:
//   y  += s_e (x A_e^T) B_e^T                   for rows of adapter e
//   dx += dt A_e,  dt = s_e dy B_e
//   dA_e = sum dt^T x,  dB_e = s_e sum dy^T t   over e's rows, t = x A_e^T
// t and dt are fp32, as the sums of parts of the contraction; as an operand of a matrix product
// each is two bf16 values whose sum keeps 16 bits of it, so that no step rounds to bf16 but the
// result's.
//
// Rows in tiles (16x16x32 MFMAs) are ordered by adapter beforehand; a tile that holds several is
// walked once for each and keeps the rows that are the adapter's own, so that one adapter's
// infinities reach no other row.  Few rows are taken one at a time instead.
// The second operand of an MFMA gives a lane its row, so a lane holds 4 neighbouring values of
// the first operand's index.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_train.hpp"

namespace fmxq {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTile = 32;  // rows of a tile: two MFMA tiles

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

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

// 8 fp32 values as two rows of bf16 whose sum is the value to 16 bits.
__device__ __forceinline__ void split8(const float* v, u32x4* hi, u32x4* lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    (*hi)[i] = h;
    (*lo)[i] = pack_bf16x2(v[2 * i] - bf16_lo(h), v[2 * i + 1] - bf16_hi(h));
  }
}

// ---- t = P . V_e^T ----------------------------------------------------------------

// Block: 32 positions and a part of the contraction, whose 32-deep steps its 8 waves take in turn.
template <int RT>
__global__ __launch_bounds__(512) void lora_shrink_kernel(LoraRows l, const uint16_t* __restrict__ p,
                                                          int64_t ldp, const uint16_t* __restrict__ v,
                                                          int64_t ldv, int64_t C, float* __restrict__ t) {
  __shared__ __attribute__((aligned(16))) f32x4 part[8][2][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t p0 = (int64_t)blockIdx.x * kTile;
  const RowOf w0 = row_of(l, p0 + r16), w1 = row_of(l, p0 + 16 + r16);
  if (wave == 0 && blockIdx.y == 0 && q4 == 0) {
    const bool bad = (p0 + r16 < l.M && l.adapters[w0.m] >= l.E) ||
                     (p0 + 16 + r16 < l.M && l.adapters[w1.m] >= l.E);
    if (bad) atomicOr(l.flag, 1u);
  }
  const int steps = (int)((C + 31) / 32);
  const int s0 = (int)((int64_t)steps * blockIdx.y / gridDim.y);
  const int s1 = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y);
  const uint16_t *x0 = p + w0.m * ldp, *x1 = p + w1.m * ldp;
  int e0 = w0.e, e1 = w1.e;
  for (int cur; (cur = next_adapter(e0, e1)) >= 0;) {
    const uint16_t* vr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int j = 16 * i + r16;
      vr[i] = v + ((int64_t)cur * l.r + (j < l.r ? j : 0)) * ldv;
    }
    f32x4 acc[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = s0 + wave; s < s1; s += 8) {
      const int64_t c = 32 * (int64_t)s + 8 * q4;
      const bool in = c < C;
      const u32x4 zero = {0u, 0u, 0u, 0u};
      const u32x4 a0 = in ? *reinterpret_cast<const u32x4*>(x0 + c) : zero;
      const u32x4 a1 = in ? *reinterpret_cast<const u32x4*>(x1 + c) : zero;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const u32x4 b = in ? *reinterpret_cast<const u32x4*>(vr[i] + c) : zero;
        acc[0][i] = mfma(b, a0, acc[0][i]);
        acc[1][i] = mfma(b, a1, acc[1][i]);
      }
    }
    // The waves' sums, in their order.
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      part[wave][0][lane] = acc[0][i];
      part[wave][1][lane] = acc[1][i];
      __syncthreads();
      if (wave < 2) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += part[k][wave][lane];
        const int j = 16 * i + 4 * q4;
        if ((wave ? e1 : e0) == cur && j < l.r)
          *reinterpret_cast<f32x4*>(t + ((int64_t)blockIdx.y * l.M + p0 + 16 * wave + r16) * l.r + j) = sum;
      }
      __syncthreads();
    }
    if (e0 == cur) e0 = -1;
    if (e1 == cur) e1 = -1;
  }
}

// A wave for every value of t.
__global__ __launch_bounds__(256) void lora_shrink_rows_kernel(LoraRows l, const uint16_t* __restrict__ p,
                                                               int64_t ldp, const uint16_t* __restrict__ v,
                                                               int64_t ldv, int64_t C, float* __restrict__ t) {
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, j = 4 * blockIdx.y + (threadIdx.x >> 6);
  const int e = l.adapters[m];
  if (e < 0 || e >= l.E) {
    if (e >= l.E && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(l.flag, 1u);
    return;
  }
  const uint16_t *x = p + m * ldp, *w = v + ((int64_t)e * l.r + j) * ldv;
  float s = 0.f;
#pragma unroll 4
  for (int64_t c = 8 * lane; c < C; c += 512) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(x + c), b = *reinterpret_cast<const u32x4*>(w + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = __builtin_fmaf(bf16_lo(a[i]), bf16_lo(b[i]), s);
      s = __builtin_fmaf(bf16_hi(a[i]), bf16_hi(b[i]), s);
    }
  }
  s = wave_sum(s);
  if (lane == 0) t[m * l.r + j] = s;
}

// ---- y += s t . V_e^T --------------------------------------------------------------

// 8 values of t at position p from j on, all parts, times s.
__device__ __forceinline__ void load_t8(const LoraRows& l, const float* t, int splits, int64_t p, int j,
                                        float s, float* v) {
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
  for (int k = 0; k < splits; ++k) {
    const f32x4* q = reinterpret_cast<const f32x4*>(t + ((int64_t)k * l.M + p) * l.r + j);
    a += q[0];
    b += q[1];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i] * s;
    v[4 + i] = b[i] * s;
  }
}

// Block: 32 positions by 512 columns, 128 a wave.  MFMA tile j takes the columns 32 (i % 4) + 8 (i / 4) +
// j of the wave's, so that a lane's 8 tiles are 8 neighbouring columns.  KS: 32-deep steps of the
// rank; 0: up to 16, where one step takes both halves of t.
template <int KS>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraRows l, const float* __restrict__ t,
                                                          int splits, const float* __restrict__ scales,
                                                          const uint16_t* __restrict__ v,
                                                          uint16_t* __restrict__ y, int64_t N, bool wide) {
  constexpr int NF = KS ? KS : 1;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tn = (uint32_t)((N + 511) / 512);
  const int64_t p0 = (int64_t)(blockIdx.x / tn) * kTile, n0 = (int64_t)(blockIdx.x % tn) * 512 + 128 * wave;
  if (n0 >= N) return;
  const RowOf w[2] = {row_of(l, p0 + r16), row_of(l, p0 + 16 + r16)};
  int e0 = w[0].e, e1 = w[1].e;
  const int chunks = l.r / 8;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int cur; (cur = next_adapter(e0, e1)) >= 0;) {
    const bool mine[2] = {e0 == cur, e1 == cur};
    const float s = scales[cur];
    u32x4 hi[2][NF], lo[2][NF];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < NF; ++k) {
        hi[m][k] = lo[m][k] = zero;
        const int c = KS ? 4 * k + q4 : q4 % chunks;
        if (mine[m] && c < chunks) {
          float f[8];
          load_t8(l, t, splits, p0 + 16 * m + r16, 8 * c, s, f);
          split8(f, &hi[m][k], &lo[m][k]);
        }
        if constexpr (KS == 0)  // the first `chunks` quarters hi, the next ones lo
          hi[m][k] = q4 < chunks ? hi[m][k] : q4 < 2 * chunks ? lo[m][k] : zero;
      }
    f32x4 acc[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      acc[j][0] = acc[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int64_t n = n0 + 32 * (r16 & 3) + 8 * (r16 >> 2) + j;
      const uint16_t* vr = v + ((int64_t)cur * N + (n < N ? n : N - 1)) * l.r;
#pragma unroll
      for (int k = 0; k < NF; ++k) {
        const int c = KS ? 4 * k + q4 : q4 % chunks;
        const u32x4 b = c < chunks && (KS || q4 < 2 * chunks) ? *reinterpret_cast<const u32x4*>(vr + 8 * c) : zero;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          acc[j][m] = mfma(b, hi[m][k], acc[j][m]);
          if constexpr (KS > 0) acc[j][m] = mfma(b, lo[m][k], acc[j][m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (!mine[m]) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + 32 * q + 8 * q4;
        uint16_t* o = y + w[m].m * N + n;
        if (wide) {
          if (n >= N) continue;
          u32x4 d = *reinterpret_cast<const u32x4*>(o);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            d[i] = pack_bf16x2(bf16_lo(d[i]) + acc[2 * i][m][q], bf16_hi(d[i]) + acc[2 * i + 1][m][q]);
          *reinterpret_cast<u32x4*>(o) = d;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < N) o[j] = (uint16_t)f32_to_bf16_rne(bf16_bits_to_f32(o[j]) + acc[j][m][q]);
        }
      }
    }
    if (e0 == cur) e0 = -1;
    if (e1 == cur) e1 = -1;
  }
}

// A thread for every value of y.
__global__ __launch_bounds__(256) void lora_expand_rows_kernel(LoraRows l, const float* __restrict__ t,
                                                               const float* __restrict__ scales,
                                                               const uint16_t* __restrict__ v,
                                                               uint16_t* __restrict__ y, int64_t N) {
  const int64_t m = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int e = l.adapters[m];
  if (e < 0 || e >= l.E || n >= N) return;
  const uint16_t* w = v + ((int64_t)e * N + n) * l.r;
  const float* tr = t + m * l.r;
  float s = 0.f;
  for (int j = 0; j < l.r; j += 8) {
    const u32x4 b = *reinterpret_cast<const u32x4*>(w + j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = __builtin_fmaf(bf16_lo(b[i]), tr[j + 2 * i], s);
      s = __builtin_fmaf(bf16_hi(b[i]), tr[j + 2 * i + 1], s);
    }
  }
  uint16_t* o = y + m * N + n;
  *o = (uint16_t)f32_to_bf16_rne(__builtin_fmaf(scales[e], s, bf16_bits_to_f32(*o)));
}

// ---- g_e = s sum P^T t ---------------------------------------------------------------

// Byte offset of a 32-row tile's row in LDS: 16 columns of the 16 rows that the quarters of a wave read at
// once (rows 8 q .. + 4) fall into all banks twice, the least that 512 bytes take.
__device__ __forceinline__ int tile_row(int row) { return row * 288 + (row >> 3) * 128; }
constexpr int kTileBytes = 32 * 288 + 4 * 128;

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
__device__ __forceinline__ int64_t slot_of(const Run& r, int64_t chunk) { return r.lo / chunk * 2; }

// Block: 128 columns of P and all of the rank, over a part of adapter e's rows in steps of 32.
template <int RT, bool ROWS_R>
__global__ __launch_bounds__(256) void lora_outer_kernel(LoraRows l, const uint16_t* __restrict__ p,
                                                         int64_t ldp, int64_t C, const float* __restrict__ t,
                                                         int splits, const float* __restrict__ scales,
                                                         int64_t chunk, float* __restrict__ g,
                                                         float* __restrict__ part) {
  constexpr int UP = RT * 32 + 32;  // bytes of a row of t
  __shared__ __attribute__((aligned(16))) uint8_t ps[kTileBytes];
  __shared__ __attribute__((aligned(16))) uint8_t us[2][32 * UP];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t c0 = (int64_t)blockIdx.x * 128, e = blockIdx.z;
  const Run run = run_of(l, e);
  const int64_t begin = run.lo + blockIdx.y * chunk;
  if (begin >= run.hi && blockIdx.y > 0) return;
  const int64_t end = begin + chunk < run.hi ? begin + chunk : run.hi;
  const bool alone = run.hi - run.lo <= chunk;
  float* out = alone ? g + e * C * l.r : part + (slot_of(run, chunk) + blockIdx.y) * C * l.r;
  const float s = scales[e];
  f32x4 acc[2][RT];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row = tid >> 3, cc = tid & 7;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int64_t b = begin; b < end; b += 32) {
    // P: two chunks of 8 columns a thread.  (Without an order the one adapter's rows are
    // those that name it.)
    auto valid = [&](int64_t pos) { return pos < end && (l.offsets || l.adapters[pos] == 0); };
    const bool on = valid(b + row);
    const int64_t m = on ? (l.order ? (int64_t)l.order[b + row] : b + row) : 0;
    u32x4 pv[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t c = c0 + 8 * (cc + 8 * k);
      pv[k] = on && c < C ? *reinterpret_cast<const u32x4*>(p + m * ldp + c) : zero;
    }
    // t: 4 values at a time.
    constexpr int TU = 32 * RT * 4 / 256 > 0 ? 32 * RT * 4 / 256 : 1;
    u32x2 uh[TU], ul[TU];
#pragma unroll
    for (int k = 0; k < TU; ++k) {
      const int u = tid + 256 * k, ur = u / (RT * 4), j = u % (RT * 4) * 4;
      f32x4 f = {0.f, 0.f, 0.f, 0.f};
      if (ur < 32 && j < l.r && valid(b + ur))
        for (int i = 0; i < splits; ++i)
          f += *reinterpret_cast<const f32x4*>(t + ((int64_t)i * l.M + b + ur) * l.r + j);
      f *= s;
      const uint32_t h0 = pack_bf16x2(f[0], f[1]), h1 = pack_bf16x2(f[2], f[3]);
      uh[k] = u32x2{h0, h1};
      ul[k] = u32x2{pack_bf16x2(f[0] - bf16_lo(h0), f[1] - bf16_hi(h0)),
                    pack_bf16x2(f[2] - bf16_lo(h1), f[3] - bf16_hi(h1))};
    }
    __syncthreads();  // the step before has been read
#pragma unroll
    for (int k = 0; k < 2; ++k)
      *reinterpret_cast<u32x4*>(ps + tile_row(row) + 16 * (cc + 8 * k)) = pv[k];
#pragma unroll
    for (int k = 0; k < TU; ++k) {
      const int u = tid + 256 * k, ur = u / (RT * 4), j = u % (RT * 4) * 4;
      if (ur < 32) {
        *reinterpret_cast<u32x2*>(us[0] + ur * UP + 2 * j) = uh[k];
        *reinterpret_cast<u32x2*>(us[1] + ur * UP + 2 * j) = ul[k];
      }
    }
    __syncthreads();
    const int tr = 8 * q4 + (r16 >> 2), at = 8 * (r16 & 3);
    u32x4 pf[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int col = 2 * (32 * wave + 16 * k) + at;
      pf[k] = turned(ps + tile_row(tr) + col, ps + tile_row(tr + 4) + col);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* q = us[x] + tr * UP + 32 * i + at;
        const u32x4 uf = turned(q, q + 4 * UP);
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[k][i] = ROWS_R ? mfma(uf, pf[k], acc[k][i]) : mfma(pf[k], uf, acc[k][i]);
      }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int64_t c = c0 + 32 * wave + 16 * k + (ROWS_R ? r16 : 4 * q4 + x);
        const int j = 16 * i + (ROWS_R ? 4 * q4 + x : r16);
        if (c < C && j < l.r) out[ROWS_R ? j * C + c : c * l.r + j] = acc[k][i][x];
      }
}

// The sums of parts, of the adapters that have several.
__global__ __launch_bounds__(256) void lora_outer_sum_kernel(LoraRows l, int64_t size, int64_t chunk,
                                                             const float* __restrict__ part,
                                                             float* __restrict__ g) {
  const int64_t e = blockIdx.y;
  const Run run = run_of(l, e);
  if (run.hi - run.lo <= chunk) return;
  const int64_t parts = (run.hi - run.lo + chunk - 1) / chunk;
  const float* from = part + slot_of(run, chunk) * size;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 1024) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int64_t k = 0; k < parts; ++k) s += *reinterpret_cast<const f32x4*>(from + k * size + i);
    *reinterpret_cast<f32x4*>(g + e * size + i) = s;
  }
}

// ---- turned matrices -------------------------------------------------------------------

__global__ __launch_bounds__(256) void lora_turn_kernel(LoraRows l, const uint16_t* __restrict__ in,
                                                        uint16_t* __restrict__ out, int64_t R, int64_t C,
                                                        int64_t ldo) {
  __shared__ uint16_t s[32][33];
  const int64_t e = blockIdx.y;
  if (l.offsets && l.offsets[e] == l.offsets[e + 1]) return;
  const uint32_t tc = (uint32_t)((C + 31) / 32);
  const int64_t r0 = (int64_t)(blockIdx.x / tc) * 32, c0 = (int64_t)(blockIdx.x % tc) * 32;
  const int x = threadIdx.x & 31, yy = threadIdx.x >> 5;
  for (int i = yy; i < 32; i += 8)
    s[i][x] = r0 + i < R && c0 + x < C ? in[(e * R + r0 + i) * C + c0 + x] : 0;
  __syncthreads();
  for (int i = yy; i < 32; i += 8)
    if (c0 + i < C && r0 + x < ldo) out[(e * C + c0 + i) * ldo + r0 + x] = s[x][i];
}

bool rank_ok(int r) { return r >= 8 && r <= kLoraMaxRank && r % 8 == 0; }
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

// Enough blocks for two on each of 256 compute units, of 4 steps a wave at least.
int lora_splits(int64_t M, int64_t C) {
  const int64_t tiles = std::max<int64_t>(div_up(M, kTile), 1), want = 512 / tiles;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, C / (32 * 8 * 4), 8}));
}

hipError_t launch_lora_shrink(const LoraRows& l, const uint16_t* p, int64_t ldp, const uint16_t* v,
                              int64_t ldv, int64_t C, int splits, float* t, hipStream_t stream) {
  if (!rank_ok(l.r) || ldp % 8 || ldv % 8 || C % 8 || splits < 1) return hipErrorInvalidValue;
  if (l.M < 1) return hipSuccess;
  const dim3 grid((unsigned)div_up(l.M, kTile), (unsigned)splits);
  if (l.r <= 16) lora_shrink_kernel<1><<<grid, 512, 0, stream>>>(l, p, ldp, v, ldv, C, t);
  else if (l.r <= 32) lora_shrink_kernel<2><<<grid, 512, 0, stream>>>(l, p, ldp, v, ldv, C, t);
  else if (l.r <= 64) lora_shrink_kernel<4><<<grid, 512, 0, stream>>>(l, p, ldp, v, ldv, C, t);
  else lora_shrink_kernel<8><<<grid, 512, 0, stream>>>(l, p, ldp, v, ldv, C, t);
  return hipGetLastError();
}

hipError_t launch_lora_shrink_rows(const LoraRows& l, const uint16_t* p, int64_t ldp, const uint16_t* v,
                                   int64_t ldv, int64_t C, float* t, hipStream_t stream) {
  if (!rank_ok(l.r) || ldp % 8 || ldv % 8 || C % 8 || l.order) return hipErrorInvalidValue;
  if (l.M < 1) return hipSuccess;
  lora_shrink_rows_kernel<<<dim3((unsigned)l.M, (unsigned)(l.r / 4)), 256, 0, stream>>>(l, p, ldp, v, ldv,
                                                                                      C, t);
  return hipGetLastError();
}

hipError_t launch_lora_expand(const LoraRows& l, const float* t, int splits, const float* scales,
                              const uint16_t* v, uint16_t* y, int64_t N, hipStream_t stream) {
  const int64_t blocks = div_up(l.M, kTile) * div_up(N, 512);
  if (!rank_ok(l.r) || blocks >= kLoraMaxBlocks) return hipErrorInvalidValue;
  if (l.M < 1 || N < 1) return hipSuccess;
  const bool wide = N % 8 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
  const dim3 grid((unsigned)blocks);
  if (l.r <= 16) lora_expand_kernel<0><<<grid, 256, 0, stream>>>(l, t, splits, scales, v, y, N, wide);
  else if (l.r <= 32) lora_expand_kernel<1><<<grid, 256, 0, stream>>>(l, t, splits, scales, v, y, N, wide);
  else if (l.r <= 64) lora_expand_kernel<2><<<grid, 256, 0, stream>>>(l, t, splits, scales, v, y, N, wide);
  else lora_expand_kernel<4><<<grid, 256, 0, stream>>>(l, t, splits, scales, v, y, N, wide);
  return hipGetLastError();
}

hipError_t launch_lora_expand_rows(const LoraRows& l, const float* t, const float* scales,
                                   const uint16_t* v, uint16_t* y, int64_t N, hipStream_t stream) {
  if (!rank_ok(l.r) || l.order || l.M > 65535) return hipErrorInvalidValue;
  if (l.M < 1 || N < 1) return hipSuccess;
  lora_expand_rows_kernel<<<dim3((unsigned)div_up(N, 256), (unsigned)l.M), 256, 0, stream>>>(l, t, scales, v,
                                                                                            y, N);
  return hipGetLastError();
}

// Rows of a part: whole runs where the columns alone fill the chip (four blocks a compute unit),
// else as many parts as do, of 128 rows at least.
int64_t lora_outer_chunk(int64_t M, int64_t C) {
  const int64_t tiles = std::max<int64_t>(div_up(C, 128), 1), parts = std::max<int64_t>(1024 / tiles, 1);
  return std::max<int64_t>(div_up(div_up(M, parts), 32) * 32, 128);
}
int64_t lora_outer_floats(int64_t M, int64_t C, int r) {
  const int64_t chunk = lora_outer_chunk(M, C);
  return M > chunk ? 2 * (M / chunk + 1) * C * r : 0;
}

int64_t lora_outer_blocks(int64_t M, int64_t C, int64_t E) {
  return div_up(C, 128) * std::max<int64_t>(div_up(M, lora_outer_chunk(M, C)), 1) * E;
}

template <bool ROWS_R>
static hipError_t launch_outer(const LoraRows& l, const uint16_t* p, int64_t ldp, int64_t C, const float* t,
                               int splits, const float* scales, float* g, float* part, hipStream_t stream) {
  const int64_t chunk = lora_outer_chunk(l.M, C), parts = std::max<int64_t>(div_up(l.M, chunk), 1);
  const dim3 grid((unsigned)div_up(C, 128), (unsigned)parts, (unsigned)l.E);
  if ((int64_t)grid.x * grid.y * grid.z >= kLoraMaxBlocks) return hipErrorInvalidValue;
  if (l.r <= 16) lora_outer_kernel<1, ROWS_R><<<grid, 256, 0, stream>>>(l, p, ldp, C, t, splits, scales, chunk, g, part);
  else if (l.r <= 32) lora_outer_kernel<2, ROWS_R><<<grid, 256, 0, stream>>>(l, p, ldp, C, t, splits, scales, chunk, g, part);
  else if (l.r <= 64) lora_outer_kernel<4, ROWS_R><<<grid, 256, 0, stream>>>(l, p, ldp, C, t, splits, scales, chunk, g, part);
  else lora_outer_kernel<8, ROWS_R><<<grid, 256, 0, stream>>>(l, p, ldp, C, t, splits, scales, chunk, g, part);
  if (hipError_t e = hipGetLastError()) return e;
  if (parts == 1) return hipSuccess;
  const int64_t size = C * l.r;
  const dim3 sum((unsigned)std::min<int64_t>(div_up(size, 1024), 1024), (unsigned)l.E);
  lora_outer_sum_kernel<<<sum, 256, 0, stream>>>(l, size, chunk, part, g);
  return hipGetLastError();
}

hipError_t launch_lora_outer(const LoraRows& l, const uint16_t* p, int64_t ldp, int64_t C, const float* t,
                             int splits, const float* scales, bool rows_r, float* g, float* part,
                             hipStream_t stream) {
  if (!rank_ok(l.r) || ldp % 8 || l.E < 1 || (!l.offsets && l.E != 1)) return hipErrorInvalidValue;
  if (C < 1) return hipSuccess;
  return rows_r ? launch_outer<true>(l, p, ldp, C, t, splits, scales, g, part, stream)
                : launch_outer<false>(l, p, ldp, C, t, splits, scales, g, part, stream);
}

hipError_t launch_lora_turn(const LoraRows& l, const uint16_t* in, uint16_t* out, int64_t R, int64_t C,
                            int64_t ldo, hipStream_t stream) {
  const int64_t tiles = div_up(C, 32) * div_up(ldo, 32);
  if (R < 1 || C < 1 || l.E < 1 || tiles * l.E >= kLoraMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid((unsigned)tiles, (unsigned)l.E);
  lora_turn_kernel<<<grid, 256, 0, stream>>>(l, in, out, R, C, ldo);
  return hipGetLastError();
}

}  // namespace fmxq
