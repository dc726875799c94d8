// fmxq_rows.hip -- token rows sorted by expert and back, for MoE layers whose expert
// products run over sorted rows, with the gradients of both directions.
//
// The sort is a stable counting sort of the S = T k routing slots: order is the one a stable
// argsort of the ids gives, pos its inverse, offsets[e] the first sorted position of expert
// e.  Ids >= E sort behind offsets[E]; their rows are zero and they raise the error flag.
// The row kernels work by token: x (or dout) is read once for its k slots, and the sums of a
// token are fp32, rounded once.
//
// Bound: HBM; a call of few rows by its launch.  Measured for 8192 tokens of 8 slots, 7168 wide:
// the sort 16 us and its rows 183 us (5.8 TB/s), the sums 189 us (5.6 TB/s), the gradients of
// rows and weights 375 us (5.3 TB/s); a large copy ran at 4.5 to 5.0 TB/s.
#include <algorithm>

#include "fmxq_common.hpp"
#include "fmxq_grad.hpp"

namespace fmxq {
namespace {

// Slots of a block of the sort, in 4 waves of consecutive slots each: 1024, and more where there
// would be over kSortBlocks blocks, because each of them reads the histograms of all.  (2^23 slots
// over 256 experts: 5.4 ms in 8192 blocks, 0.84 in 512, 0.86 in 256 or 1024; 2^20 over 2048 experts
// 0.85 ms in 1024, 0.30 in 512.)
constexpr int kSortSlots = 1024;
constexpr int64_t kSortBlocks = 512;
int sort_slots(int64_t S) {
  return kSortSlots * (int)((S + kSortSlots * kSortBlocks - 1) / (kSortSlots * kSortBlocks));
}
int64_t sort_blocks(int64_t S) { return (S + sort_slots(S) - 1) / sort_slots(S); }

__device__ __forceinline__ uint32_t bucket_of(uint32_t e, int64_t E) {
  return e < (uint64_t)E ? e : (uint32_t)E;
}

// hist[block][e]: slots of each expert (bucket E: ids out of range) in the block's range.
__global__ __launch_bounds__(256) void sort_hist_kernel(MoeSort a, int64_t S, int slots) {
  extern __shared__ uint32_t cnt[];
  const int64_t nb = a.E + 1, s0 = (int64_t)blockIdx.x * slots;
  for (int64_t i = threadIdx.x; i < nb; i += 256) cnt[i] = 0;
  __syncthreads();
  for (int64_t s = s0 + threadIdx.x; s < s0 + slots && s < S; s += 256)
    atomicAdd(&cnt[bucket_of(a.inds[s], a.E)], 1u);
  __syncthreads();
  for (int64_t i = threadIdx.x; i < nb; i += 256) a.hist[blockIdx.x * nb + i] = cnt[i];
}

// Exclusive prefix sum over 256 threads.
__device__ __forceinline__ uint32_t scan256(uint32_t v, uint32_t* wsum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_up((int)inc, o, 64);
    if (lane >= o) inc += t;
  }
  __syncthreads();
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  uint32_t r = inc - v;
  for (int i = 0; i < wave; ++i) r += wsum[i];
  return r;
}

// Lanes of the wave with the same bucket: one ballot per bit of the bucket.
__device__ __forceinline__ uint64_t same_bucket(uint32_t b, bool on, int bits) {
  uint64_t m = __ballot(on);
  for (int i = 0; i < bits; ++i) {
    const uint64_t set = __ballot((b >> i) & 1u);
    m &= (b >> i) & 1u ? set : ~set;
  }
  return m;
}

// Orders the wave's own LDS accesses (no instruction; the LDS serves a wave in order).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Each block adds up the histograms before its own (every block reads the tables again, 512 at
// most, which costs less than a launch for the scan), then its waves place their slots in order.
__global__ __launch_bounds__(256) void sort_place_kernel(MoeSort a, int64_t S, int slots, int bits) {
  extern __shared__ uint32_t lds[];  // E + 1 cursors of each wave, then two tables more
  __shared__ uint32_t wsum[4];
  const int64_t nb = a.E + 1, s0 = (int64_t)blockIdx.x * slots;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t* cur = lds;
  // Per-wave counts of the block's slots.
  for (int64_t i = tid; i < 4 * nb; i += 256) cur[i] = 0;
  __syncthreads();
  const int64_t w0 = s0 + wave * (slots / 4), w1 = w0 + slots / 4 < S ? w0 + slots / 4 : S;
  for (int64_t s = w0 + lane; s < w1; s += 64)
    atomicAdd(&cur[wave * nb + bucket_of(a.inds[s], a.E)], 1u);
  __syncthreads();
  // Each bucket's slots in all blocks and in the earlier ones, then the buckets' first
  // positions, then each wave's cursors.
  uint32_t *all = lds + 4 * nb, *before = lds + 5 * nb;
  for (int64_t e = tid; e < nb; e += 256) {
    uint32_t n = 0, m = 0;
#pragma unroll 8
    for (unsigned k = 0; k < gridDim.x; ++k) {
      const uint32_t v = a.hist[k * nb + e];
      n += v;
      m += k < blockIdx.x ? v : 0u;
    }
    all[e] = n;
    before[e] = m;
  }
  __syncthreads();
  const int64_t per = (nb + 255) / 256;
  const int64_t b0 = tid * per < nb ? tid * per : nb, b1 = b0 + per < nb ? b0 + per : nb;
  uint32_t total = 0;
  for (int64_t e = b0; e < b1; ++e) total += all[e];
  uint32_t base = scan256(total, wsum);
  for (int64_t e = b0; e < b1; ++e) {
    if (blockIdx.x == 0) {
      a.offsets[e] = base;
      if (e == a.E && base < S) atomicOr(a.flag, 1u);
    }
    uint32_t at = base + before[e];
    for (int w = 0; w < 4; ++w) {
      const uint32_t n = cur[w * nb + e];
      cur[w * nb + e] = at;
      at += n;
    }
    base += all[e];
  }
  __syncthreads();
  for (int64_t s = w0 + lane; s - lane < w1; s += 64) {
    const bool on = s < w1;
    const uint32_t b = on ? bucket_of(a.inds[s], a.E) : 0u;
    const uint64_t same = same_bucket(b, on, bits);
    if (on) {
      const uint32_t p = cur[wave * nb + b] + (uint32_t)__popcll(same & ((1ull << lane) - 1));
      a.order[p] = (uint32_t)s;
      a.pos[s] = p;
    }
    wave_fence();
    if (on && (same & ((1ull << lane) - 1)) == 0)
      cur[wave * nb + b] += (uint32_t)__popcll(same);
    wave_fence();
  }
}

// 8 (or 1) bf16 values.
template <int VEC>
struct Row;
template <>
struct Row<8> {
  u32x4 v;
  __device__ __forceinline__ static Row load(const uint16_t* p) {
    return {*reinterpret_cast<const u32x4*>(p)};
  }
  __device__ __forceinline__ static Row stream(const uint16_t* p) {
    return {__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p))};
  }
  __device__ __forceinline__ void store(uint16_t* p) const { *reinterpret_cast<u32x4*>(p) = v; }
  __device__ __forceinline__ float at(int i) const {
    return i & 1 ? bf16_hi(v[i >> 1]) : bf16_lo(v[i >> 1]);
  }
  __device__ __forceinline__ static Row of(const float* f) {
    return {u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                  pack_bf16x2(f[6], f[7])}};
  }
};
template <>
struct Row<1> {
  uint16_t v;
  __device__ __forceinline__ static Row load(const uint16_t* p) { return {*p}; }
  __device__ __forceinline__ static Row stream(const uint16_t* p) { return load(p); }
  __device__ __forceinline__ void store(uint16_t* p) const { *p = v; }
  __device__ __forceinline__ float at(int) const { return bf16_bits_to_f32(v); }
  __device__ __forceinline__ static Row of(const float* f) {
    return {(uint16_t)f32_to_bf16_rne(f[0])};
  }
};

__device__ __forceinline__ float weight_of(const void* w, bool bf16, int64_t i) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(w)[i])
              : reinterpret_cast<const float*>(w)[i];
}

// xs[pos[t, j]] = x[t], or zeros for ids out of range.
template <int VEC>
__global__ __launch_bounds__(256) void rows_out_kernel(MoeSort a) {
  const int64_t t = blockIdx.x;
  const uint32_t valid = a.offsets[a.E];
  for (int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VEC; c < a.D;
       c += (int64_t)gridDim.y * 256 * VEC) {
    const Row<VEC> x = Row<VEC>::load(a.x + t * a.D + c);
    for (int64_t j = 0; j < a.k; ++j) {
      const uint32_t p = a.pos[t * a.k + j];
      (p < valid ? x : Row<VEC>{}).store(a.xs + (int64_t)p * a.D + c);
    }
  }
}

// Few slots: the whole sort in one launch.  Block t + 1 counts, for each slot of token t, the
// slots that sort before it (a smaller bucket, or the same one earlier), then writes the
// token's rows; block 0 counts the buckets for the offsets.  Every block reads all the ids.
// (160 slots over 512 experts 7.5 us against 11 us of three launches; from about 1100 slots
// on the three are quicker.)
constexpr int kSmallK = 16, kSmallBits = 10;
constexpr int64_t kSmallSlots = 1024;
template <int VEC>
__global__ __launch_bounds__(256) void sort_small_kernel(MoeSort a, int S) {
  extern __shared__ uint32_t cnt[];  // E + 1
  __shared__ uint32_t before[4][kSmallK], all[4], wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t t = (int64_t)blockIdx.x - 1;
  const int nb = (int)a.E + 1, k = (int)a.k;
  if (t < 0) {
    for (int i = tid; i < nb; i += 256) cnt[i] = 0;
    __syncthreads();
    for (int s = tid; s < S; s += 256) atomicAdd(&cnt[bucket_of(a.inds[s], a.E)], 1u);
    __syncthreads();
    const int per = (nb + 255) / 256;
    const int b0 = tid * per < nb ? tid * per : nb, b1 = b0 + per < nb ? b0 + per : nb;
    uint32_t n = 0;
    for (int e = b0; e < b1; ++e) n += cnt[e];
    uint32_t at = scan256(n, wsum);
    for (int e = b0; e < b1; ++e) {
      a.offsets[e] = at;
      if (e == nb - 1 && at < (uint32_t)S) atomicOr(a.flag, 1u);
      at += cnt[e];
    }
    return;
  }
  // A slot's key: its bucket, then its number.  Counted by ballots, so that a wave's totals need
  // no sum over its lanes; eight loads of ids are in flight at a time.
  const uint32_t none = ~0u, last = (uint32_t)a.E << kSmallBits;
  uint32_t mine[kSmallK], n[kSmallK], valid = 0;
#pragma unroll
  for (int j = 0; j < kSmallK; ++j) {
    const uint32_t s = (uint32_t)(t * k + j);
    mine[j] = j < k ? bucket_of(a.inds[s], a.E) << kSmallBits | s : 0u;
    n[j] = 0;
  }
  for (int s0 = 64 * wave; s0 < S; s0 += 8 * 256) {
    uint32_t key[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + 256 * i + lane;
      key[i] = s < S ? bucket_of(a.inds[s], a.E) << kSmallBits | (uint32_t)s : none;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s0 + 256 * i >= S) break;
      valid += __popcll(__ballot(key[i] < last));
#pragma unroll
      for (int j = 0; j < kSmallK; ++j)
        if (j < k) n[j] += __popcll(__ballot(key[i] < mine[j]));
    }
  }
#pragma unroll
  for (int j = 0; j < kSmallK; ++j)
    if (j < k && lane == 0) before[wave][j] = n[j];
  if (lane == 0) all[wave] = valid;
  __syncthreads();
  valid = all[0] + all[1] + all[2] + all[3];
  uint32_t p[kSmallK];
#pragma unroll
  for (int j = 0; j < kSmallK; ++j)
    p[j] = j < k ? before[0][j] + before[1][j] + before[2][j] + before[3][j] : 0u;
  if (tid == 0) {
#pragma unroll
    for (int j = 0; j < kSmallK; ++j)
      if (j < k) {
        a.pos[t * k + j] = p[j];
        a.order[p[j]] = (uint32_t)(t * k + j);
      }
  }
  for (int64_t c = (int64_t)tid * VEC; c < a.D; c += 256 * VEC) {
    const Row<VEC> x = Row<VEC>::load(a.x + t * a.D + c);
#pragma unroll
    for (int j = 0; j < kSmallK; ++j)
      if (j < k) (p[j] < valid ? x : Row<VEC>{}).store(a.xs + (int64_t)p[j] * a.D + c);
  }
}

constexpr int64_t kCacheBytes = 256 << 20;  // the last-level cache

// out[t] = sum_j w[t, j] y[pos[t, j]] in the order of j; a position outside the rows adds
// nothing.  Eight rows are requested before any is added.
template <int VEC, bool STREAM>
__global__ __launch_bounds__(256) void rows_sum_kernel(const uint16_t* __restrict__ y,
                                                       const uint32_t* __restrict__ pos,
                                                       const void* __restrict__ weights,
                                                       bool wbf16, uint16_t* __restrict__ out,
                                                       int64_t S, int64_t k, int64_t D,
                                                       uint32_t* flag) {
  const int64_t t = blockIdx.x;
  for (int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VEC; c < D;
       c += (int64_t)gridDim.y * 256 * VEC) {
    float s[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[i] = 0.f;
    for (int64_t j0 = 0; j0 < k; j0 += 8) {
      Row<VEC> v[8];
      float w[8];
      bool on[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = j0 + j < k;
        const int64_t p = in ? pos[t * k + j0 + j] : S;
        on[j] = p < S;
        v[j] = Row<VEC>{};
        w[j] = 0.f;
        if (on[j]) {
          v[j] = STREAM ? Row<VEC>::stream(y + p * D + c) : Row<VEC>::load(y + p * D + c);
          w[j] = weights ? weight_of(weights, wbf16, t * k + j0 + j) : 1.f;
        } else if (in && c == 0) {
          atomicOr(flag, 1u);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (on[j])
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[i] = __builtin_fmaf(w[j], v[j].at(i), s[i]);
    }
    Row<VEC>::of(s).store(out + t * D + c);
  }
}

// One wave per slot: dy[pos] = w dout, dweights = <dout, y[pos]>.  The waves of a block take
// neighbouring slots, which mostly share a token's dout.
template <int VEC>
__global__ __launch_bounds__(256) void rows_grad_kernel(const uint16_t* __restrict__ dout,
                                                        const uint16_t* __restrict__ y,
                                                        const uint32_t* __restrict__ pos,
                                                        const void* __restrict__ weights,
                                                        bool wbf16, uint16_t* __restrict__ dy,
                                                        void* __restrict__ dweights, int64_t S,
                                                        int64_t k, int64_t D, uint32_t* flag) {
  const int lane = threadIdx.x & 63;
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= S) return;
  const int64_t t = s / k, p = pos[s];
  const float w = weight_of(weights, wbf16, s);
  float dot = 0.f;
  if (p < S) {
    const uint16_t *dr = dout + t * D, *yr = y + p * D;
    uint16_t* o = dy + p * D;
#pragma unroll 4
    for (int64_t c = (int64_t)lane * VEC; c < D; c += 64 * VEC) {
      const Row<VEC> d = Row<VEC>::load(dr + c), v = Row<VEC>::load(yr + c);
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        dot = __builtin_fmaf(d.at(i), v.at(i), dot);
        f[i] = w * d.at(i);
      }
      Row<VEC>::of(f).store(o + c);
    }
  } else if (lane == 0) {
    atomicOr(flag, 1u);
  }
  dot = wave_sum(dot);
  if (lane == 0) {
    if (wbf16) reinterpret_cast<uint16_t*>(dweights)[s] = (uint16_t)f32_to_bf16_rne(dot);
    else reinterpret_cast<float*>(dweights)[s] = dot;
  }
}

bool vec8(int64_t D, const void* a, const void* b, const void* c) {
  return D % 8 == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
                         reinterpret_cast<uintptr_t>(c)) & 15) == 0;
}

dim3 row_grid(int64_t T, int64_t D, int vec) {
  const int64_t y = (D + 256 * vec - 1) / (256 * vec);
  return dim3((unsigned)T, (unsigned)std::min<int64_t>(std::max<int64_t>(y, 1), 1024));
}

}  // namespace

size_t moe_sort_hist_bytes(int64_t S, int64_t E) {
  return S == 0 ? 0 : (size_t)sort_blocks(S) * (E + 1) * sizeof(uint32_t);
}

hipError_t launch_moe_sort(const MoeSort& a, hipStream_t stream) {
  const int64_t S = a.T * a.k, nb = a.E + 1;
  const bool vec = vec8(a.D, a.x, a.xs, nullptr);
  if (S <= kSmallSlots && a.k <= kSmallK) {
    const dim3 grid((unsigned)a.T + 1);
    if (vec) sort_small_kernel<8><<<grid, 256, nb * sizeof(uint32_t), stream>>>(a, (int)S);
    else sort_small_kernel<1><<<grid, 256, nb * sizeof(uint32_t), stream>>>(a, (int)S);
    return hipGetLastError();
  }
  int bits = 1;
  while (nb > ((int64_t)1 << bits)) ++bits;
  const int slots = sort_slots(S);
  const unsigned blocks = (unsigned)sort_blocks(S);
  sort_hist_kernel<<<blocks, 256, nb * sizeof(uint32_t), stream>>>(a, S, slots);
  if (hipError_t e = hipGetLastError()) return e;
  sort_place_kernel<<<blocks, 256, 6 * nb * sizeof(uint32_t), stream>>>(a, S, slots, bits);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.D == 0) return hipSuccess;
  if (vec)
    rows_out_kernel<8><<<row_grid(a.T, a.D, 8), 256, 0, stream>>>(a);
  else
    rows_out_kernel<1><<<row_grid(a.T, a.D, 1), 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_moe_unsort(const uint16_t* y, const uint32_t* pos, const void* weights,
                             bool weights_bf16, uint16_t* out, int64_t T, int64_t k, int64_t D,
                             uint32_t* flag, hipStream_t stream) {
  // Rows that do not fit the last-level cache are read past it (8192 x 8 rows 7168 wide 189
  // against 216 us); smaller ones are read again by the gradients (all four calls of 4096 x 4
  // rows 2048 wide 74 us, 76 with such reads).
  const dim3 grid = row_grid(T, D, vec8(D, y, out, nullptr) ? 8 : 1);
  if (!vec8(D, y, out, nullptr))
    rows_sum_kernel<1, false><<<grid, 256, 0, stream>>>(y, pos, weights, weights_bf16, out, T * k, k, D, flag);
  else if (T * k * D * 2 > kCacheBytes)
    rows_sum_kernel<8, true><<<grid, 256, 0, stream>>>(y, pos, weights, weights_bf16, out, T * k, k, D, flag);
  else
    rows_sum_kernel<8, false><<<grid, 256, 0, stream>>>(y, pos, weights, weights_bf16, out, T * k, k, D, flag);
  return hipGetLastError();
}

hipError_t launch_moe_unsort_grad(const uint16_t* dout, const uint16_t* y, const uint32_t* pos,
                                  const void* weights, bool weights_bf16, uint16_t* dy,
                                  void* dweights, int64_t T, int64_t k, int64_t D, uint32_t* flag,
                                  hipStream_t stream) {
  if (vec8(D, dout, y, dy))
    rows_grad_kernel<8><<<(unsigned)((T * k + 3) / 4), 256, 0, stream>>>(dout, y, pos, weights, weights_bf16, dy,
                                                         dweights, T * k, k, D, flag);
  else
    rows_grad_kernel<1><<<(unsigned)((T * k + 3) / 4), 256, 0, stream>>>(dout, y, pos, weights, weights_bf16, dy,
                                                         dweights, T * k, k, D, flag);
  return hipGetLastError();
}

}  // namespace fmxq
