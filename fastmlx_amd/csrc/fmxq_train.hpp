// fmxq_train.hpp -- launchers of the adapters beside quantized products and of gradient
// clipping (fmxq_lora.hip, fmxq_clip.hip), shared with their C ABI (fmxq_train_capi.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fmxq_grad.hpp"

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
// u rows: the bf16 parts whose sum stands for a value of t (LoraAdd takes two, products of
// fp32 results three).
constexpr int kLoraParts = 3;

// t [splits][M][r] = P . V_e^T by position: P [M, C] (rows of ldp values), V [E][r] rows of ldv
// values; C, ldp and ldv multiples of 8.  Positions without adapter are not written.
struct LoraShrink {
  const uint16_t* p;
  int64_t ldp;
  const uint16_t* v;
  int64_t ldv, C;
  int splits;
  float* t;
  uint16_t* u;  // launch_lora_parts: [M][parts][r] by row, lora_scales[e] t
};
int lora_splits(int64_t M, int64_t C);
// order [M] and offsets [E + 1] of up to 16384 rows and 511 adapters.
bool lora_sort_supported(int64_t M, int64_t E);
hipError_t launch_lora_sort(const int32_t* adapters, int64_t M, int64_t E, uint32_t* order, uint32_t* offsets,
                            hipStream_t stream);
// Words that the last launch before a product clears for it.
struct Zeros {
  uint32_t* p;
  int64_t n;
};
// One or two at once, then their parts.
hipError_t launch_lora_shrink(const LoraRows& l, const LoraShrink* s, int n, hipStream_t stream);
hipError_t launch_lora_parts(const LoraRows& l, const LoraShrink* s, int n, int parts, const float* scales,
                             const Zeros& z, hipStream_t stream);
// Few rows: u (two parts) of one shrink at once, in any order (l.order null).
hipError_t launch_lora_shrink_rows(const LoraRows& l, const LoraShrink& s, const float* scales,
                                   const Zeros& z, hipStream_t stream);
// g [E][C][r] (or [E][r][C] with rows_r) = sum over e's rows of P^T u, u in kLoraParts parts.  part:
// lora_outer_floats of scratch.
struct LoraOuter {
  const uint16_t* p;
  int64_t ldp, C;
  const uint16_t* u;
  bool rows_r;
  float *g, *part;
};
int64_t lora_outer_floats(int64_t M, int64_t C, int r);
int64_t lora_outer_blocks(int64_t M, int64_t C, int64_t E);
hipError_t launch_lora_outer(const LoraRows& l, const LoraOuter* o, int n, hipStream_t stream);
// out [E][C][ldo] = in [E][R][C] turned, zeros from R to ldo; adapters without rows are left out.
struct LoraTurn {
  const uint16_t* in;
  uint16_t* out;
  int64_t R, C, ldo;
};
int64_t lora_turn_blocks(int64_t C, int64_t ldo, int64_t E);
hipError_t launch_lora_turn(const LoraRows& l, const LoraTurn* t, int n, hipStream_t stream);

// y [M, N] = x [M, K] . deq(W)^T with fmxq_dequantize's bits and an adapter's part, rounded once.
struct OutPlan {
  bool thin, skinny, wide, panel;
  int bm, splits;
  int64_t c_split, piece;  // piece: outputs of one panel
  int64_t counters;        // wide: words at count_at that have to be zero
  size_t slices, count_at, panel_at, xp, bytes;
};
OutPlan out_plan(int64_t M, int64_t N, int64_t K);
hipError_t launch_out(const uint16_t* x, const uint32_t* w, const uint16_t* scales, const uint16_t* biases,
                      const LoraAdd& lora, uint16_t* y, int64_t M, int64_t N, int64_t K, int group_size,
                      int bits, const OutPlan& p, void* ws, uint32_t* flag, hipStream_t stream);

}  // namespace fmxq
