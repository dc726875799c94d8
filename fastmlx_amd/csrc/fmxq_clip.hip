// fmxq_clip.hip -- the norm over many gradients, and the gradients clipped to it:
//   norm = sqrt(sum g^2),   out = g min(1, max_norm / norm).
//
// A launch takes the tensors of one table (ClipTable, in its arguments: no copy from the host, so a
// graph can hold it) as tiles of 32 KB that its blocks walk.  Squares are added in 64 bits, in
// which those of the largest fp32 value have room, in an order that the sizes alone decide: a
// thread's, a block's, then the blocks' sums.  Every block of the second pass adds the blocks'
// sums up again (8 KB from the cache), which costs less than a launch between the passes.
// Bound: HBM (448 fp32 tensors of 0.34 GB 194 us, 5.2 TB/s of the three passes over them; bf16 99 us,
// 5.1), and the two launches where there is little (14 tensors of one layer 10 us).  The second pass walks
// a table's tiles from the last to the first, because what the first pass read last is what the last-level
// cache still holds: of one table, that is; with more of them it begins with the first table again.
#include "fmxq_common.hpp"
#include "fmxq_train.hpp"

namespace fmxq {
namespace {

constexpr int kT = 256;

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// The block's sum, in every thread; red: kT / 64 words.
__device__ __forceinline__ double block_sum64(double v, double* red) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// The entry of tile t.
__device__ __forceinline__ int entry_of(const ClipTable& t, uint32_t tile) {
  int lo = 0, hi = (int)t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.tile[mid] <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A tile: elements i0 .. i1 of an entry.
struct Tile {
  uint64_t src, dst;
  uint32_t i0, i1;
  bool bf16;
};
__device__ __forceinline__ Tile tile_of(const ClipTable& t, uint32_t tile) {
  const int e = entry_of(t, tile);
  Tile r;
  r.bf16 = t.src[e] & 1;
  r.src = t.src[e] & ~1ull;
  r.dst = t.dst[e];
  const uint32_t per = (uint32_t)kClipTileBytes / (r.bf16 ? 2 : 4);
  r.i0 = (tile - t.tile[e]) * per;
  r.i1 = t.count[e] - r.i0 < per ? t.count[e] : r.i0 + per;
  return r;
}

constexpr int kLoads = (int)(kClipTileBytes / 16 / kT);  // 16-byte loads of a thread in a tile

__device__ __forceinline__ double square(float v, double s) { return __builtin_fma((double)v, (double)v, s); }

__global__ __launch_bounds__(kT) void clip_squares_kernel(ClipTable t, double* __restrict__ sums, bool add) {
  __shared__ double red[kT / 64];
  const uint32_t tid = threadIdx.x;
  double s0 = 0., s1 = 0.;
  for (uint32_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const Tile r = tile_of(t, tile);
    const uint32_t n = r.i1 - r.i0;
    if ((r.src & 15) == 0) {
      const u32x4* p = reinterpret_cast<const u32x4*>(r.src + (uint64_t)r.i0 * (r.bf16 ? 2 : 4));
      const uint32_t units = n / (r.bf16 ? 8 : 4);
      u32x4 v[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        v[i] = tid + i * kT < units ? p[tid + i * kT] : u32x4{0u, 0u, 0u, 0u};
      if (r.bf16) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s0 = square(bf16_lo(v[i][j]), s0);
            s1 = square(bf16_hi(v[i][j]), s1);
          }
      } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s0 = square(__uint_as_float(v[i][2 * j]), s0);
            s1 = square(__uint_as_float(v[i][2 * j + 1]), s1);
          }
      }
      const uint32_t at = units * (r.bf16 ? 8 : 4) + tid;
      if (at < n)
        s0 = square(r.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(r.src)[r.i0 + at])
                           : reinterpret_cast<const float*>(r.src)[r.i0 + at],
                    s0);
    } else {
      for (uint32_t i = r.i0 + tid; i < r.i1; i += kT)
        s0 = square(r.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(r.src)[i])
                           : reinterpret_cast<const float*>(r.src)[i],
                    s0);
    }
  }
  const double s = block_sum64(s0 + s1, red);
  if (tid == 0) sums[blockIdx.x] = add ? sums[blockIdx.x] + s : s;
}

__device__ __forceinline__ double norm_of(const double* sums, double* red) {
  double s = 0.;
#pragma unroll
  for (int i = 0; i < kClipBlocks / kT; ++i) s += sums[threadIdx.x + i * kT];
  return sqrt(block_sum64(s, red));
}

__global__ __launch_bounds__(kT) void clip_norm_kernel(const double* __restrict__ sums, float* norm) {
  __shared__ double red[kT / 64];
  const double v = norm_of(sums, red);
  if (threadIdx.x == 0) *norm = (float)v;
}

__global__ __launch_bounds__(kT) void clip_scale_kernel(ClipTable t, const double* __restrict__ sums,
                                                        float max_norm, float* norm) {
  __shared__ double red[kT / 64];
  const uint32_t tid = threadIdx.x;
  const double v = norm_of(sums, red);
  if (norm && blockIdx.x == 0 && tid == 0) *norm = (float)v;
  // A norm of zero, infinity or NaN says nothing about a scale: the gradients stay as they are.  (In 64
  // bits: finite gradients whose norm is past fp32's range are scaled by it.)
  const double c = (double)max_norm / v;
  const float f = v > 0. && v < __builtin_huge_val() && c < 1. ? (float)c : 1.f;
  for (uint32_t k = blockIdx.x; k < t.tiles; k += gridDim.x) {
    const Tile r = tile_of(t, t.tiles - 1 - k);
    if (f == 1.f && r.src == r.dst) continue;
    const uint32_t n = r.i1 - r.i0;
    const uint64_t off = (uint64_t)r.i0 * (r.bf16 ? 2 : 4);
    uint32_t done = 0;
    if (((r.src | r.dst) & 15) == 0) {
      const u32x4* p = reinterpret_cast<const u32x4*>(r.src + off);
      u32x4* o = reinterpret_cast<u32x4*>(r.dst + off);
      const uint32_t units = n / (r.bf16 ? 8 : 4);
      u32x4 w[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        w[i] = tid + i * kT < units ? p[tid + i * kT] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[i][j] = r.bf16 ? pack_bf16x2(bf16_lo(w[i][j]) * f, bf16_hi(w[i][j]) * f)
                           : __float_as_uint(__uint_as_float(w[i][j]) * f);
        if (tid + i * kT < units) __builtin_nontemporal_store(w[i], o + tid + i * kT);
      }
      done = units * (r.bf16 ? 8 : 4);
    }
    for (uint32_t i = done + tid; i < n; i += kT) {
      if (r.bf16) {
        const float g = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(r.src + off)[i]);
        reinterpret_cast<uint16_t*>(r.dst + off)[i] = (uint16_t)f32_to_bf16_rne(g * f);
      } else {
        reinterpret_cast<float*>(r.dst + off)[i] = reinterpret_cast<const float*>(r.src + off)[i] * f;
      }
    }
  }
}

}  // namespace

hipError_t launch_clip_squares(const ClipTable& t, double* sums, bool add, hipStream_t stream) {
  clip_squares_kernel<<<kClipBlocks, kT, 0, stream>>>(t, sums, add);
  return hipGetLastError();
}

hipError_t launch_clip_norm(const double* sums, float* norm, hipStream_t stream) {
  clip_norm_kernel<<<1, kT, 0, stream>>>(sums, norm);
  return hipGetLastError();
}

hipError_t launch_clip_scale(const ClipTable& t, const double* sums, float max_norm, float* norm,
                             hipStream_t stream) {
  const unsigned blocks = t.tiles < 2048 ? (t.tiles > 0 ? t.tiles : 1) : 2048;
  clip_scale_kernel<<<blocks, kT, 0, stream>>>(t, sums, max_norm, norm);
  return hipGetLastError();
}

}  // namespace fmxq
