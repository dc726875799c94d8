// fmxq_grad.hpp -- launchers of the losses over a quantized head, the input gradients of
// the quantized products and the sorted expert rows (fmxq_grad_gemm.hip, fmxq_head.hip,
// fmxq_rows.hip), shared with their C ABI (fmxq_grad_capi.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmxq {

// One product D [M, N] = A [M, C] . B with B the dequantized weights (the bits of
// fmxq_dequantize):
//   nn = false: B = deq(W)^T, W [N, C] packed along the contraction (logits);
//   nn = true:  B = deq(W),   W [C, N] packed along the outputs (input gradients).
// A's rows are 16-byte aligned and lda a multiple of 8; columns of A from a_cols (a multiple
// of 8) on are read as zero.
struct GradGemm {
  const uint16_t* a = nullptr;
  int64_t lda = 0, a_cols = 0;
  int64_t M = 0, N = 0, C = 0;
  const uint32_t* w = nullptr;
  const uint16_t* scales = nullptr;
  const uint16_t* biases = nullptr;
  int group_size = 64, bits = 4;
  // launch_panel_gemm: the weights as bf16 rows of ldp values (a multiple of 8), [N][C] for the
  // logits and [C][N] for input gradients.
  const uint16_t* panel = nullptr;
  int64_t ldp = 0;
  // launch_skinny_gemm (nt): skinny_pack_bytes of memory for x, or null to read it as it is.
  void* xp = nullptr;
  // The contraction in `splits` parts of c_split (a multiple of 64) values; part p goes to
  // slice p of out.
  int splits = 1;
  int64_t c_split = 0;
  // nn: fp32 slices out [splits][M][N], added to what is there (with add) times factor[row] (where
  // it is given); or, with y, bf16 rows y [M][ldy] (one part only).
  float* out = nullptr;
  bool add = false;
  const float* factor = nullptr;
  uint16_t* y = nullptr;
  int64_t ldy = 0;
  // nt: what a softmax needs of the logits l = D * logit_scale (in units of log 2) by
  // tiles of the kernel's stat width: stats[row][tile] = (m, sum 2^(l - m)) with m the multiple of
  // 64 nearest to the tile's largest l, and, with e, e[row][col] = bf16(2^(l - m)), which reaches
  // 2^32; zeros from column N to the next multiple of the stat width (what lies behind, up to
  // lde, may be anything: a product over e reads a_cols of it).
  // The row's wanted tokens take no part (their e is 0): ids wanted[row][0 .. wanted_k] of tokens
  // counted from -first_token on, other than wanted_none.
  float2* stats = nullptr;
  int64_t stat_tiles = 0;
  const int32_t* wanted = nullptr;
  int wanted_k = 0;
  int32_t wanted_none = -1;
  int64_t first_token = 0;
  uint16_t* e = nullptr;
  int64_t lde = 0;
  float logit_scale = 1.f;
  // Expert runs (nn only, into y): rows offsets[e] .. offsets[e + 1] of M take expert e, whose
  // weights are C rows into w; other rows get zeros.  max_tiles: grad_gemm_run_tiles.  *flag
  // is raised where the offsets decrease or leave 0 .. M (all rows are zero then).
  const int32_t* offsets = nullptr;
  int64_t experts = 0, max_tiles = 0;
  uint32_t* flag = nullptr;
};

// A launch has fewer blocks of these products: 2^32 threads.
constexpr int64_t kMaxBlocks = 1 << 23;
// Rows of a block's tile, for M rows (or expert runs of about that many).
int grad_gemm_rows(int64_t M);
constexpr int kGradStatWidth = 64;  // columns of a tile of the statistics (128 rows and more)
constexpr int kGradTileCols = 256;
constexpr int kLogitCols = 256, kGradCols = 128;  // of launch_grad_gemm's tiles
// Tiles of bm rows that cover any runs of S rows and one more that none does, in eights.
inline int64_t grad_gemm_run_tiles(int64_t S, int64_t E, int bm) {
  return (S / bm + (E < S ? E : S) + 8) / 8 * 8;
}
// Blocks of the gradient of `tiles` row tiles of bm rows, N columns.
inline int64_t grad_gemm_blocks(int64_t tiles, int bm, int64_t N) {
  const int64_t bn = bm < 256 ? kGradCols : kLogitCols;
  return tiles * ((N + bn - 1) / bn);
}
// What a tile's 32-bit offsets into its rows of A hold: lda of launch_grad_gemm and launch_panel_gemm.
constexpr int64_t kMaxLda = 0x7ffffff0LL / 512 - 1;
hipError_t launch_grad_gemm(const GradGemm& g, bool nn, int bm, hipStream_t stream);

// The same products where reading the weights is the work (fmxq_grad_skinny.hip): logits
// of up to kSkinnyRows rows or in chunks of as many, gradients of up to kGradSkinnyRows.  weight_rows: rows of
// a part of the contraction (nn).
constexpr int64_t kSkinnyRows = 64;
// ... and of gradients: 64 rows through 14336 x 4096 took 43 us there, 65 in tiles 37.
constexpr int64_t kGradSkinnyRows = 48;
constexpr int kSkinnyStatWidth = 32;
constexpr int kSkinnyCols = 128;  // outputs of a block (nn)
// Rows from which the logits' x is packed beforehand, and the bytes that takes.
constexpr int64_t kSkinnyPackRows = 17;
inline int64_t skinny_pack_bytes(int64_t M, int64_t K) {
  if (M < kSkinnyPackRows) return 0;
  return (K + 63) / 64 * 4096 * (M <= 32 ? 1 : 2) * ((M + kSkinnyRows - 1) / kSkinnyRows);
}
bool skinny_gemm_supported(int64_t lda, int64_t weight_rows, int64_t weight_cols);
hipError_t launch_skinny_gemm(const GradGemm& g, bool nn, hipStream_t stream);

// The same products over a panel of weights dequantized beforehand (fmxq_grad_panel.hip), in
// tiles of kPanelRows rows.
constexpr int kPanelRows = 256;
constexpr int kPanelStatWidth = 128;
// Whether a tile's 32-bit offsets into a panel of rows of ld values hold it.
inline bool panel_gemm_supported(int64_t ld) { return (kGradTileCols + 1) * ld * 2 < 0x7ffffff0LL; }
hipError_t launch_panel_gemm(const GradGemm& g, bool nn, hipStream_t stream);
// bf16 y [M, N] = the sum of the slices of out [splits][M][N].
hipError_t launch_sum_slices(const float* slices, int splits, uint16_t* y, int64_t M, int64_t N,
                             hipStream_t stream);
// dst [M, ld] = src [M, N] with zeros in columns N .. ld.
hipError_t launch_pad_rows(const uint16_t* src, uint16_t* dst, int64_t M, int64_t N, int64_t ld,
                           hipStream_t stream);
// A loss over a quantized head (fmxq_head.hip).  ids [M, k]: the targets (k = 1, teacher
// null) or the teacher's entries.  An id that names no token: `ignore` for targets, below
// zero for a teacher.
struct HeadLoss {
  const uint16_t* h;
  const uint32_t* w;
  const uint16_t *scales, *biases;
  const int32_t* ids;
  const void* teacher;  // null: cross entropy
  bool teacher_bf16;
  const float* grad_loss;
  float *loss, *lse;
  uint16_t* dh;  // null: no gradient
  int64_t M, V, K;
  int k;
  int32_t ignore;
  float temperature;
  int group_size, bits;
  uint32_t* flag;
};
struct HeadPlan {
  int bm, grad_bm, stat_width, pieces, splits;
  int64_t piece, c_split, stat_tiles;
  // The products run over panels of dequantized weights; the logits, the gradient on the
  // kernels that read the weights once.
  bool panel, skinny, grad_skinny;
  size_t stats, e, slices, state, factor, sel, panel_at, xp, bytes;  // in the workspace
};
HeadPlan head_plan(int64_t M, int64_t V, int64_t K, int k, bool grad, int cus);
hipError_t launch_head_loss(const HeadLoss& a, const HeadPlan& p, void* ws, hipStream_t stream);

// Rows sorted by expert and back (fmxq_rows.hip); S = T k slots, slot s of token s / k.
struct MoeSort {
  const uint16_t* x;     // [T, D]
  const uint32_t* inds;  // [S]
  uint16_t* xs;          // [S, D]
  uint32_t *order, *pos; // [S]
  uint32_t* offsets;     // [E + 1]
  int64_t T, k, E, D;
  uint32_t* hist;        // moe_sort_hist_bytes
  uint32_t* flag;
};
size_t moe_sort_hist_bytes(int64_t S, int64_t E);
hipError_t launch_moe_sort(const MoeSort& a, hipStream_t stream);
// out[t] = sum_j weights[t, j] y[pos[t, j]], weights bf16, fp32 or null (ones).
hipError_t launch_moe_unsort(const uint16_t* y, const uint32_t* pos, const void* weights,
                             bool weights_bf16, uint16_t* out, int64_t T, int64_t k, int64_t D,
                             uint32_t* flag, hipStream_t stream);
hipError_t launch_moe_unsort_grad(const uint16_t* dout, const uint16_t* y, const uint32_t* pos,
                                  const void* weights, bool weights_bf16, uint16_t* dy,
                                  void* dweights, int64_t T, int64_t k, int64_t D, uint32_t* flag,
                                  hipStream_t stream);

}  // namespace fmxq
