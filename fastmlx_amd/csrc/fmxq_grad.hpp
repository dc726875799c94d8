// fmxq_grad.hpp -- launchers of the losses over a quantized head, the input gradients of
// the quantized products and the sorted expert rows (fmxq_grad_gemm.hip, fmxq_head.hip,
// fmxq_rows.hip), shared with their C ABI (fmxq_grad_capi.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmxq {

// What a product leaves.  Logits (nt): the softmax statistics of the losses, those of log
// probabilities, the logits' gradient, or itself.  Input gradients (nn): itself.  The product
// itself (kEpiOut) takes a low-rank adapter's part.
enum Epilogue { kEpiStats = 0, kEpiScores = 1, kEpiCoef = 2, kEpiOut = 3 };
// The adapter's part of row m, output n: sum_j (u0 + u1)[m][j] v[e][n][j] with e = ids[m], none
// where it is outside 0 .. E - 1.  u: `parts` rows of r bf16 values for each m, of which the first two
// are taken (their sum holds the value to 16 bits); v [E][n][r].
struct LoraAdd {
  const uint16_t* u = nullptr;
  const uint16_t* v = nullptr;
  const int32_t* ids = nullptr;
  int64_t E = 0, n = 0;  // n: rows of v an adapter (N, or of more outputs than this product's)
  int r = 0, parts = 0;
};
// A tile of a row's logits for log probabilities (store_scores).
struct HeadTile {
  float top, sum, low;
  uint32_t first;
};

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
  // epi: kEpiScores writes score[row][tile] in place of stats (no wanted tokens); kEpiCoef writes e
  // from rows[row] = (lse, a, c, -) in units of log 2 (store_coef).
  Epilogue epi = kEpiStats;
  HeadTile* score = nullptr;
  const float* rows = nullptr;
  // kEpiOut: as nn into y or out (of one part y, any N), with the adapter's part in the first.
  LoraAdd lora;
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

// Logits or outputs (kEpiScores in tiles of kThinStatWidth, kEpiOut) of up to kThinRows rows, where every
// load of the weights is whole lines (fmxq_thin.hip), and where that is the quicker product: it reads x
// once for every 16 outputs, the one for few rows packs it first and works on 64 of them (us, outputs with
// an adapter's part: 4096 x 4096, 16 rows 14.5, on the other 17 rows 19; 14336 x 4096, 8 rows 28.4, 16 rows
// 41, on the other 17 rows 30.  Scores of 128256 x 4096: 1 row 124 on either, 16 rows 284 and 146).
constexpr int64_t kThinRows = 16;
constexpr int kThinStatWidth = 16;
bool thin_supported(int64_t M, int64_t N, int64_t K);
hipError_t launch_thin_gemm(const GradGemm& g, hipStream_t stream);

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
// fmxq_quantized_matmul_grad, its checks included, with an adapter's part (fmxq_grad_capi.cpp).  ld: the
// values from one row of dy to the next, N, or where N is no multiple of 8 also that next one, 16-byte
// aligned and zero past N: such a copy may lie where the workspace begins, where the call would put its own.
int input_grad(const uint16_t* dy, int64_t ld, const uint32_t* w, const uint16_t* scales, const uint16_t* biases,
               const LoraAdd& lora, uint16_t* dx, int64_t M, int64_t N, int64_t K, int group_size, int bits,
               void* workspace, size_t workspace_bytes, void* stream, const char* op);
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
// Few tokens for many rows: launch_skinny_gemm takes them in chunks.
bool few_tokens(int64_t M, int64_t V, int bm, int cus);
HeadPlan head_plan(int64_t M, int64_t V, int64_t K, int k, bool grad, int cus);
// Whether the operands of a product's logits are there.
inline bool logits_operands(const GradGemm& g) {
  switch (g.epi) {
    case kEpiStats: return g.stats && g.wanted;
    case kEpiScores: return g.score != nullptr;
    case kEpiCoef: return g.rows && g.wanted && g.e;
    case kEpiOut: return g.y || g.out;
  }
  return false;
}
hipError_t launch_head_loss(const HeadLoss& a, const HeadPlan& p, void* ws, hipStream_t stream);

// Log probabilities through a quantized head (fmxq_logprobs.hip).
struct HeadScore {
  const uint16_t* h;
  const uint32_t* w;
  const uint16_t *scales, *biases;
  const int32_t* ids;  // [M, k], below zero for an absent entry
  float *logp, *entropy, *lse;
  int32_t* top_ids;  // [M, top]
  float* top_logp;
  int64_t M, V, K;
  int k, top;
  float temperature;
  int group_size, bits;
  uint32_t* flag;
};
size_t head_score_bytes(int64_t M, int64_t V, int64_t K, int k, int top, int cus);
hipError_t launch_head_score(const HeadScore& a, int cus, void* ws, hipStream_t stream);
// Their gradient: dh from grad_logp [M, k] and grad_entropy [M] (or null), with the logp, entropy
// and lse that the scores gave.
struct HeadScoreGrad {
  const uint16_t* h;
  const uint32_t* w;
  const uint16_t *scales, *biases;
  const int32_t* ids;
  const float *logp, *entropy, *lse, *grad_logp, *grad_entropy;
  uint16_t* dh;
  int64_t M, V, K;
  int k;
  float temperature;
  int group_size, bits;
  uint32_t* flag;
};
size_t head_score_grad_bytes(int64_t M, int64_t V, int64_t K, int k, int cus);
hipError_t launch_head_score_grad(const HeadScoreGrad& a, int cus, void* ws, hipStream_t stream);

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
