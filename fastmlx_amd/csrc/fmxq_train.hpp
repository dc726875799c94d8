// fmxq_train.hpp -- launchers of the adapters beside quantized products and of gradient
// clipping (fmxq_lora.hip, fmxq_clip.hip), shared with their C ABI (fmxq_train_capi.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmxq {

// ---- the norm over many tensors ----
// Tensors travel in the launch's arguments, which hold this many (an argument block is 4 KB).
constexpr int kClipTensors = 160;
struct ClipTable {
  // A tensor's address, with bit 0 set where it is bf16 (elements are 2 bytes at least), and
  // where its scaled values go.
  uint64_t src[kClipTensors];
  uint64_t dst[kClipTensors];
  uint32_t count[kClipTensors];   // elements
  uint32_t tile[kClipTensors];    // the first tile; tiles of a tensor follow each other
  uint32_t n, tiles;
};
// Source bytes of a tile, and the elements that a table's entry holds at most (a larger tensor
// takes several entries).
constexpr int64_t kClipTileBytes = 32768;
constexpr int64_t kClipMaxCount = (int64_t)1 << 30;
// Partial sums, one a block.
constexpr int kClipBlocks = 1024;
// sums [kClipBlocks] get (or, with add, are added to) the squares of the table's tensors.
hipError_t launch_clip_squares(const ClipTable& t, double* sums, bool add, hipStream_t stream);
// norm = the root of the sums' sum.
hipError_t launch_clip_norm(const double* sums, float* norm, hipStream_t stream);
// dst = src min(1, max_norm / norm); norm (null: not written) as above.
hipError_t launch_clip_scale(const ClipTable& t, const double* sums, float max_norm, float* norm,
                             hipStream_t stream);

// ---- low-rank adapters ----
// Rows m of adapter e = adapters[m] (none where it is outside 0 .. E - 1).  Position p of the rows'
// order is row order[p]; null: p itself.  With offsets, adapter e has positions offsets[e] ..
// offsets[e + 1] and those from offsets[E] on have none.
struct LoraRows {
  const int32_t* adapters;
  const uint32_t* order;
  const uint32_t* offsets;
  int64_t M, E;
  int r;           // rank, a multiple of 8
  uint32_t* flag;  // raised by shrinks for an adapter of E or more
};
constexpr int kLoraMaxRank = 128;
constexpr int64_t kLoraMaxAdapters = 2048;
constexpr int64_t kLoraMaxBlocks = 1 << 23;  // of a launch
// Parts of the shrink's contraction of C values, for M rows in tiles.
int lora_splits(int64_t M, int64_t C);
// t [splits][M][r] = P . V_e^T by position: P [M, C] (rows of ldp values), V [E][r] rows of ldv
// values; C, ldp and ldv multiples of 8.  Positions without adapter are not written.
hipError_t launch_lora_shrink(const LoraRows& l, const uint16_t* p, int64_t ldp, const uint16_t* v,
                              int64_t ldv, int64_t C, int splits, float* t, hipStream_t stream);
// The same a row at a time (order null, one part).
hipError_t launch_lora_shrink_rows(const LoraRows& l, const uint16_t* p, int64_t ldp, const uint16_t* v,
                                   int64_t ldv, int64_t C, float* t, hipStream_t stream);
// y [M, N] += scales[e] t . V_e^T, V [E][N][r].
hipError_t launch_lora_expand(const LoraRows& l, const float* t, int splits, const float* scales,
                              const uint16_t* v, uint16_t* y, int64_t N, hipStream_t stream);
hipError_t launch_lora_expand_rows(const LoraRows& l, const float* t, const float* scales,
                                   const uint16_t* v, uint16_t* y, int64_t N, hipStream_t stream);
// g [E][C][r] (or [E][r][C] with rows_r) = scales[e] sum over e's rows of P^T t; P's rows of ldp
// values, C of them used.  part: lora_outer_floats of scratch.
int64_t lora_outer_chunk(int64_t M, int64_t C);
int64_t lora_outer_floats(int64_t M, int64_t C, int r);
int64_t lora_outer_blocks(int64_t M, int64_t C, int64_t E);
hipError_t launch_lora_outer(const LoraRows& l, const uint16_t* p, int64_t ldp, int64_t C, const float* t,
                             int splits, const float* scales, bool rows_r, float* g, float* part,
                             hipStream_t stream);
// out [E][C][ldo] = in [E][R][C] turned, zeros from R to ldo; adapters without rows are left out.
hipError_t launch_lora_turn(const LoraRows& l, const uint16_t* in, uint16_t* out, int64_t R, int64_t C,
                            int64_t ldo, hipStream_t stream);

}  // namespace fmxq
