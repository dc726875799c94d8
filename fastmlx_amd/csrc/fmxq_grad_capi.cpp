// fmxq_grad_capi.cpp -- extern "C" entry points for training and scoring over quantized
// weights (declared in include/fmxq.h): losses of a quantized head, input gradients of the
// quantized products, rows sorted by expert.
//
// As in fmxq_capi.cpp every check comes before anything is enqueued.  The workspaces are the
// caller's, so no call allocates, and none shares memory with another.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/fmxq.h"
#include "fmxq_grad.hpp"
#include "fmxq_host.hpp"
#include "fmxq_internal.hpp"

using fmxq::check_quant;
using fmxq::device_flag;
using fmxq::fail;
using fmxq::hip_status;

namespace {

// Compute units the plans are made for.  A plan depends on the sizes alone, so that the
// workspace functions need no device.
constexpr int kCus = 256;
constexpr int kHeadMaxTopK = 64;
constexpr int64_t kSortMaxExperts = 2048;
constexpr int64_t kMaxCount = 0x7fffffff;
// Rows of a call: a launch has at most 2^32 threads, 256 a row.
constexpr int64_t kMaxRows = (1 << 24) - 1;
// Widths: the products' offsets into 256 rows of bf16 are 32 bits.
constexpr int64_t kMaxWidth = (1 << 22) - 8;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// The gradient of M rows, K wide, in one launch.
bool outputs_ok(int64_t M, int64_t K) {
  return fmxq::grad_gemm_blocks((M + fmxq::kPanelRows - 1) / fmxq::kPanelRows, fmxq::kPanelRows, K) <
         fmxq::kMaxBlocks;
}

// a * b within 62 bits (a, b >= 0).
bool product_ok(int64_t a, int64_t b) { return a == 0 || b <= ((int64_t)1 << 62) / a; }

int check_workspace(const void* ws, size_t have, size_t need, const char* op) {
  if (need == 0) return FMXQ_OK;
  if (have < need)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu are needed", op, have,
                need);
  if (!ws || !aligned16(ws))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", op);
  return FMXQ_OK;
}

// ---- losses ---------------------------------------------------------------------

int head_sizes(int64_t M, int64_t V, int64_t K, int k, bool grad, const char* op) {
  if (M < 0 || V < 0 || K < 0)
    return fail(FMXQ_ERR_SHAPE, "%s: negative size M=%lld V=%lld K=%lld", op, (long long)M,
                (long long)V, (long long)K);
  if (k < 1 || k > kHeadMaxTopK)
    return fail(FMXQ_ERR_SHAPE, "%s: top_k=%d outside 1..%d", op, k, kHeadMaxTopK);
  if (M > 0 && V == 0) return fail(FMXQ_ERR_SHAPE, "%s: %lld rows over no tokens", op, (long long)M);
  if (M > 0 && K == 0) return fail(FMXQ_ERR_SHAPE, "%s: %lld rows of no width", op, (long long)M);
  if (M > kMaxRows || V > kMaxCount || K > kMaxWidth)
    return fail(FMXQ_ERR_SHAPE, "%s: M=%lld, V=%lld or K=%lld too large", op, (long long)M,
                (long long)V, (long long)K);
  if (grad && !outputs_ok(M, K))
    return fail(FMXQ_ERR_SHAPE, "%s: %lld rows of %lld are too many", op, (long long)M, (long long)K);
  return FMXQ_OK;
}

int head_loss(fmxq::HeadLoss a, void* ws, size_t ws_bytes, void* stream, const char* op) {
  if (int rc = check_quant(a.group_size, a.bits, a.K, true, op)) return rc;
  if (int rc = head_sizes(a.M, a.V, a.K, a.k, a.dh != nullptr, op)) return rc;
  if (a.grad_loss && !a.dh)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: grad_loss without dh", op);
  if (a.M == 0) return FMXQ_OK;
  if (!a.h || !a.w || !a.scales || !a.biases || !a.ids || !a.loss || !a.lse)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned16(a.h) || !aligned16(a.w) || !aligned16(a.dh))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: h, w and dh must be 16-byte aligned", op);
  if (!aligned(a.ids, 4) || !aligned(a.loss, 4) || !aligned(a.lse, 4) || !aligned(a.grad_loss, 4) ||
      !aligned(a.scales, 2) || !aligned(a.biases, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  const fmxq::HeadPlan p = fmxq::head_plan(a.M, a.V, a.K, a.k, a.dh != nullptr, kCus);
  if (int rc = check_workspace(ws, ws_bytes, p.bytes, op)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = device_flag(s, &a.flag)) return rc;
  return hip_status(fmxq::launch_head_loss(a, p, ws, s), op);
}

int score_sizes(int64_t M, int64_t V, int64_t K, int k, int top, const char* op) {
  if (int rc = head_sizes(M, V, K, std::max(k, 1), false, op)) return rc;
  if (k < 0) return fail(FMXQ_ERR_SHAPE, "%s: k=%d outside 0..%d", op, k, kHeadMaxTopK);
  if (top < 0 || top > kHeadMaxTopK || (M > 0 && top > V))
    return fail(FMXQ_ERR_SHAPE, "%s: top=%d outside 0..%d, or of %lld tokens", op, top, kHeadMaxTopK,
                (long long)V);
  return FMXQ_OK;
}
bool temperature_ok(float t) { return t >= 1e-30f && t <= 1e30f; }

// ---- input gradients --------------------------------------------------------------

struct GradPlan {
  int bm, splits;
  int64_t c_split, piece;  // piece: rows of the weight of one panel (N without panels)
  bool panel, skinny;
  size_t slices, panel_at, bytes;
};
// Rows from which the weights are dequantized to a panel beforehand: 14336 x 4096, four tiles of
// 256 rows take 149 us without, five 175 us with it.
constexpr int64_t kGradPanelRows = 1025;
// Most bytes of a panel: a larger weight is walked in pieces whose products are added in fp32, so
// that a call needs no bf16 copy of it.  (2048 rows, 128256 x 4096, in one panel of 1 GB 1.94 ms, in two
// pieces 1.97, in four of 256 MB 2.05: each piece reads the sums again and ends in a tail.)
constexpr int64_t kGradPanelBytes = 512 << 20;

// The rows of dy are copied to a stride of 8 values where N is not one, and where dy's address is
// not 16-byte aligned: for that, which the sizes do not show, a call takes moved_bytes more.
int64_t pad_cols(int64_t N) { return up(N, 8); }
size_t pad_bytes(int64_t M, int64_t N) { return N % 8 ? (size_t)up(M * pad_cols(N) * 2, 256) : 0; }
size_t moved_bytes(const void* dy, int64_t M, int64_t N) {
  return N % 8 == 0 && !aligned16(dy) ? (size_t)(M * N * 2) : 0;
}
// A call with rows needs some workspace at any size, so that a missing one is an error at every
// size and not at some.
constexpr size_t kLeastBytes = 256;

GradPlan grad_plan(int64_t M, int64_t N, int64_t K) {
  GradPlan p{};
  p.panel = M >= kGradPanelRows && fmxq::panel_gemm_supported(K);
  p.piece = N;
  if (p.panel) {
    const int64_t most = std::max<int64_t>(kGradPanelBytes / 2 / std::max<int64_t>(K, 1), 256);
    const int64_t pieces = std::max<int64_t>(1, (N + most - 1) / most);
    p.piece = up((N + pieces - 1) / pieces, 64);
  }
  p.bm = p.panel ? fmxq::kPanelRows : fmxq::grad_gemm_rows(M);
  p.skinny = M <= fmxq::kGradSkinnyRows && fmxq::skinny_gemm_supported(pad_cols(N), N + 64, K);
  const int64_t cols = p.skinny ? fmxq::kSkinnyCols : p.bm > 128 ? fmxq::kGradTileCols : fmxq::kGradCols;
  const int64_t tiles = (p.skinny ? M > 0 : (M + p.bm - 1) / p.bm) * ((K + cols - 1) / cols);
  // Parts of the contraction where the tiles leave compute units idle, of 256 values at
  // least.
  const int64_t want = tiles ? (p.bm > 128 ? kCus : 2 * kCus) / tiles : 1;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, p.piece / 256));
  p.c_split = up((p.piece + p.splits - 1) / p.splits, 64);
  p.splits = (int)std::max<int64_t>(1, (p.piece + p.c_split - 1) / std::max<int64_t>(p.c_split, 1));
  p.slices = pad_bytes(M, N);
  p.panel_at = p.slices + (p.splits > 1 || p.piece < N ? up(p.splits * M * K * 4, 256) : 0);
  p.bytes = M == 0 ? 0 : std::max(p.panel_at + (p.panel ? std::min(p.piece, N) * K * 2 : 0), kLeastBytes);
  return p;
}

// dy (rows of ld values) as the product reads it: itself, or a copy with padded rows in the workspace.
int grad_operand(const uint16_t* dy, int64_t ld, void* pad, int64_t M, int64_t N, hipStream_t s,
                 fmxq::GradGemm* g, const char* op) {
  g->a = dy;
  g->lda = g->a_cols = ld;
  if (ld % 8 == 0 && aligned16(dy)) return FMXQ_OK;
  g->a = static_cast<uint16_t*>(pad);
  g->lda = g->a_cols = pad_cols(N);
  return hip_status(fmxq::launch_pad_rows(dy, static_cast<uint16_t*>(pad), M, N, g->lda, s), op);
}

int grad_sizes(int64_t M, int64_t N, int64_t K, const char* op) {
  if (M < 0 || N < 0 || K < 0)
    return fail(FMXQ_ERR_SHAPE, "%s: negative size M=%lld N=%lld K=%lld", op, (long long)M,
                (long long)N, (long long)K);
  if (M > kMaxRows || N > kMaxWidth || K > kMaxWidth)
    return fail(FMXQ_ERR_SHAPE, "%s: M=%lld, N=%lld or K=%lld too large", op, (long long)M,
                (long long)N, (long long)K);
  if (!outputs_ok(M, K))
    return fail(FMXQ_ERR_SHAPE, "%s: %lld rows of %lld are too many", op, (long long)M, (long long)K);
  return FMXQ_OK;
}

int bytes_out(size_t v, size_t* out, const char* op) {
  if (!out) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null result", op);
  *out = v;
  return FMXQ_OK;
}

int run_rows(int64_t S, int64_t E) { return fmxq::grad_gemm_rows(E > 0 ? (S + E - 1) / E : S); }

int run_sizes(int64_t S, int64_t E, int64_t N, int64_t K, const char* op) {
  if (int rc = grad_sizes(S, N, K, op)) return rc;
  if (E < 0) return fail(FMXQ_ERR_SHAPE, "%s: negative size E=%lld", op, (long long)E);
  if (E > kMaxCount) return fail(FMXQ_ERR_SHAPE, "%s: %lld experts are too many", op, (long long)E);
  const int bm = run_rows(S, E);
  if (fmxq::grad_gemm_blocks(fmxq::grad_gemm_run_tiles(S, E, bm), bm, K) >= fmxq::kMaxBlocks)
    return fail(FMXQ_ERR_SHAPE, "%s: %lld rows of %lld in %lld runs are too many", op, (long long)S,
                (long long)K, (long long)E);
  return FMXQ_OK;
}

// ---- sorted rows --------------------------------------------------------------------

int row_sizes(int64_t T, int64_t k, int64_t D, const char* op) {
  if (T < 0 || k < 1 || D < 0)
    return fail(FMXQ_ERR_SHAPE, "%s: need T >= 0, top_k >= 1 and D >= 0 (got %lld %lld %lld)", op,
                (long long)T, (long long)k, (long long)D);
  if (T > kMaxRows || !product_ok(T, k) || T * k > 4 * kMaxRows)
    return fail(FMXQ_ERR_SHAPE, "%s: %lld x %lld slots are too many", op, (long long)T, (long long)k);
  return FMXQ_OK;
}

}  // namespace

int fmxq::input_grad(const uint16_t* dy, int64_t ld, const uint32_t* w, const uint16_t* scales,
                     const uint16_t* biases, const LoraAdd& lora, uint16_t* dx, int64_t M, int64_t N,
                     int64_t K, int group_size, int bits, void* workspace, size_t workspace_bytes,
                     void* stream, const char* op) {
  if (int rc = check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = grad_sizes(M, N, K, op)) return rc;
  if (M == 0) return FMXQ_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!dx || !aligned16(dx))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: dx must be 16-byte aligned", op);
  if (N == 0)
    return hip_status(fmxq::launch_fill_u32(reinterpret_cast<uint32_t*>(dx), 0u, M * K / 2, s), op);
  if (!dy || !w || !scales || !biases) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned16(w)) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: w must be 16-byte aligned", op);
  if (!aligned(dy, 2) || !aligned(scales, 2) || !aligned(biases, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  const GradPlan p = grad_plan(M, N, K);
  const size_t moved = moved_bytes(dy, M, N), moved_at = moved ? up(p.bytes, 256) : 0;
  if (int rc = check_workspace(workspace, workspace_bytes, moved ? moved_at + moved : p.bytes, op))
    return rc;
  char* ws = static_cast<char*>(workspace);
  fmxq::GradGemm g;
  if (int rc = grad_operand(dy, ld, ws + moved_at, M, N, s, &g, op)) return rc;
  g.M = M;
  g.N = K;
  g.C = N;
  g.w = w;
  g.scales = scales;
  g.biases = biases;
  g.group_size = group_size;
  g.bits = bits;
  g.splits = p.splits;
  g.lora = lora;
  g.c_split = p.c_split;
  float* slices = reinterpret_cast<float*>(ws + p.slices);
  if (p.splits > 1 || p.piece < N) {
    g.out = slices;
  } else {
    g.y = dx;
    g.ldy = K;
  }
  if (p.panel) {
    uint16_t* panel = reinterpret_cast<uint16_t*>(ws + p.panel_at);
    g.panel = panel;
    g.ldp = K;
    for (int64_t n0 = 0; n0 < N; n0 += p.piece) {
      fmxq::GradGemm d = g;
      d.C = std::min(p.piece, N - n0);
      d.a = g.a + n0;
      d.a_cols = std::min(p.piece, g.a_cols - n0);
      d.add = n0 > 0;
      if (d.add) d.lora = fmxq::LoraAdd{};
      const int64_t at = n0 * (K / group_size);
      if (int rc = hip_status(fmxq::launch_dequantize(w + n0 * (K * bits / 32), scales + at, biases + at,
                                                      panel, d.C, K, group_size, bits, s),
                              op))
        return rc;
      if (int rc = hip_status(fmxq::launch_panel_gemm(d, true, s), op)) return rc;
    }
  } else if (int rc = hip_status(p.skinny ? fmxq::launch_skinny_gemm(g, true, s)
                                          : fmxq::launch_grad_gemm(g, true, p.bm, s),
                                 op)) {
    return rc;
  }
  if (!g.out) return FMXQ_OK;
  return hip_status(fmxq::launch_sum_slices(slices, p.splits, dx, M, K, s), op);
}

extern "C" {

int fmxq_head_workspace(int64_t M, int64_t V, int64_t K, int top_k, bool with_grad, size_t* bytes) {
  const char* op = "head_workspace";
  if (int rc = head_sizes(M, V, K, top_k, with_grad, op)) return rc;
  return bytes_out(M == 0 ? 0 : fmxq::head_plan(M, V, K, top_k, with_grad, kCus).bytes, bytes, op);
}

int fmxq_head_cross_entropy(const uint16_t* h, const uint32_t* w, const uint16_t* scales,
                            const uint16_t* biases, const int32_t* targets,
                            const float* grad_loss, float* loss, float* lse, uint16_t* dh,
                            int64_t M, int64_t V, int64_t K, int32_t ignore_index, int group_size,
                            int bits, void* workspace, size_t workspace_bytes, void* stream) {
  fmxq::HeadLoss a{h,   w,    scales, biases, targets, nullptr, false, grad_loss, loss, lse, dh, M, V,
                   K,   1,    ignore_index, 1.f, group_size, bits, nullptr};
  return head_loss(a, workspace, workspace_bytes, stream, "head_cross_entropy");
}

int fmxq_head_distill(const uint16_t* h, const uint32_t* w, const uint16_t* scales,
                      const uint16_t* biases, const int32_t* ids, const void* teacher,
                      int teacher_bf16, const float* grad_loss, float* loss, float* lse,
                      uint16_t* dh, int64_t M, int64_t V, int64_t K, int top_k, float temperature,
                      int group_size, int bits, void* workspace, size_t workspace_bytes,
                      void* stream) {
  const char* op = "head_distill";
  if (!(temperature > 0.f) || temperature > 1e30f || temperature < 1e-30f)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: temperature %g must be a positive number", op,
                (double)temperature);
  if (M > 0 && !teacher) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(teacher, teacher_bf16 ? 2 : 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: teacher must be aligned to its element size", op);
  fmxq::HeadLoss a{h, w, scales, biases, ids, teacher, teacher_bf16 != 0, grad_loss, loss, lse, dh, M,
                   V, K, top_k, 0, temperature, group_size, bits, nullptr};
  return head_loss(a, workspace, workspace_bytes, stream, op);
}

int fmxq_head_logprobs_workspace(int64_t M, int64_t V, int64_t K, int k, int top, size_t* bytes) {
  const char* op = "head_logprobs_workspace";
  if (int rc = score_sizes(M, V, K, k, top, op)) return rc;
  return bytes_out(M == 0 ? 0 : fmxq::head_score_bytes(M, V, K, k, top, kCus), bytes, op);
}

int fmxq_head_logprobs(const uint16_t* h, const uint32_t* w, const uint16_t* scales,
                       const uint16_t* biases, const int32_t* ids, float* logp, float* entropy, float* lse,
                       int32_t* top_ids, float* top_logp, int64_t M, int64_t V, int64_t K, int k, int top,
                       float temperature, int group_size, int bits, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const char* op = "head_logprobs";
  if (int rc = check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = score_sizes(M, V, K, k, top, op)) return rc;
  if (!temperature_ok(temperature))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: temperature %g must be a positive number", op,
                (double)temperature);
  if (M == 0) return FMXQ_OK;
  if (!h || !w || !scales || !biases || !entropy || !lse || (k > 0 && (!ids || !logp)) ||
      (top > 0 && (!top_ids || !top_logp)))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned16(h) || !aligned16(w))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: h and w must be 16-byte aligned", op);
  if (!aligned(ids, 4) || !aligned(logp, 4) || !aligned(entropy, 4) || !aligned(lse, 4) ||
      !aligned(top_ids, 4) || !aligned(top_logp, 4) || !aligned(scales, 2) || !aligned(biases, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  if (int rc = check_workspace(workspace, workspace_bytes, fmxq::head_score_bytes(M, V, K, k, top, kCus), op))
    return rc;
  fmxq::HeadScore a{h, w, scales, biases, ids, logp, entropy, lse, top_ids, top_logp, M, V, K, k, top,
                    temperature, group_size, bits, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = device_flag(s, &a.flag)) return rc;
  return hip_status(fmxq::launch_head_score(a, kCus, workspace, s), op);
}

int fmxq_head_logprobs_grad_workspace(int64_t M, int64_t V, int64_t K, int k, size_t* bytes) {
  const char* op = "head_logprobs_grad_workspace";
  if (int rc = head_sizes(M, V, K, k, true, op)) return rc;
  return bytes_out(M == 0 ? 0 : fmxq::head_score_grad_bytes(M, V, K, k, kCus), bytes, op);
}

int fmxq_head_logprobs_grad(const uint16_t* h, const uint32_t* w, const uint16_t* scales,
                            const uint16_t* biases, const int32_t* ids, const float* logp,
                            const float* entropy, const float* lse, const float* grad_logp,
                            const float* grad_entropy, uint16_t* dh, int64_t M, int64_t V, int64_t K, int k,
                            float temperature, int group_size, int bits, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* op = "head_logprobs_grad";
  if (int rc = check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = head_sizes(M, V, K, k, true, op)) return rc;
  if (!temperature_ok(temperature))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: temperature %g must be a positive number", op,
                (double)temperature);
  if (M == 0) return FMXQ_OK;
  if (!h || !w || !scales || !biases || !ids || !logp || !entropy || !lse || !grad_logp || !dh)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned16(h) || !aligned16(w) || !aligned16(dh))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: h, w and dh must be 16-byte aligned", op);
  if (!aligned(ids, 4) || !aligned(logp, 4) || !aligned(entropy, 4) || !aligned(lse, 4) ||
      !aligned(grad_logp, 4) || !aligned(grad_entropy, 4) || !aligned(scales, 2) || !aligned(biases, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  if (int rc = check_workspace(workspace, workspace_bytes, fmxq::head_score_grad_bytes(M, V, K, k, kCus), op))
    return rc;
  fmxq::HeadScoreGrad a{h, w, scales, biases, ids, logp, entropy, lse, grad_logp, grad_entropy, dh, M, V, K,
                        k, temperature, group_size, bits, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = device_flag(s, &a.flag)) return rc;
  return hip_status(fmxq::launch_head_score_grad(a, kCus, workspace, s), op);
}

int fmxq_quantized_matmul_grad_workspace(int64_t M, int64_t N, int64_t K, size_t* bytes) {
  const char* op = "quantized_matmul_grad_workspace";
  if (int rc = grad_sizes(M, N, K, op)) return rc;
  return bytes_out(grad_plan(M, N, K).bytes, bytes, op);
}

int fmxq_quantized_matmul_grad(const uint16_t* dy, const uint32_t* w, const uint16_t* scales,
                               const uint16_t* biases, uint16_t* dx, int64_t M, int64_t N,
                               int64_t K, int group_size, int bits, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return fmxq::input_grad(dy, N, w, scales, biases, fmxq::LoraAdd{}, dx, M, N, K, group_size, bits, workspace,
                          workspace_bytes, stream, "quantized_matmul_grad");
}

int fmxq_gather_qmm_grad_workspace(int64_t S, int64_t E, int64_t N, int64_t K, size_t* bytes) {
  const char* op = "gather_qmm_grad_workspace";
  if (int rc = run_sizes(S, E, N, K, op)) return rc;
  return bytes_out(S == 0 ? 0 : std::max(pad_bytes(S, N), kLeastBytes), bytes, op);
}

int fmxq_gather_qmm_grad(const uint16_t* dy, const uint32_t* w, const uint16_t* scales,
                         const uint16_t* biases, const int32_t* offsets, uint16_t* dx, int64_t S,
                         int64_t E, int64_t N, int64_t K, int group_size, int bits,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "gather_qmm_grad";
  if (int rc = check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = run_sizes(S, E, N, K, op)) return rc;
  if (S == 0) return FMXQ_OK;
  if (E == 0) return fail(FMXQ_ERR_SHAPE, "%s: %lld rows but no experts", op, (long long)S);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!dx || !aligned16(dx))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: dx must be 16-byte aligned", op);
  if (N == 0)
    return hip_status(fmxq::launch_fill_u32(reinterpret_cast<uint32_t*>(dx), 0u, S * K / 2, s), op);
  if (!dy || !w || !scales || !biases || !offsets)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(offsets, 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  if (!aligned16(w)) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: w must be 16-byte aligned", op);
  if (!aligned(dy, 2) || !aligned(scales, 2) || !aligned(biases, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  const size_t need = std::max(pad_bytes(S, N), kLeastBytes) + moved_bytes(dy, S, N);
  if (int rc = check_workspace(workspace, workspace_bytes, need, op)) return rc;
  uint32_t* flag = nullptr;
  if (int rc = device_flag(s, &flag)) return rc;
  fmxq::GradGemm g;
  if (int rc = grad_operand(dy, N, workspace, S, N, s, &g, op)) return rc;
  g.M = S;
  g.N = K;
  g.C = N;
  g.w = w;
  g.scales = scales;
  g.biases = biases;
  g.group_size = group_size;
  g.bits = bits;
  g.c_split = up(N, 64);
  g.y = dx;
  g.ldy = K;
  const int bm = run_rows(S, E);
  g.offsets = offsets;
  g.experts = E;
  g.max_tiles = fmxq::grad_gemm_run_tiles(S, E, bm);
  g.flag = flag;
  return hip_status(fmxq::launch_grad_gemm(g, true, bm, s), op);
}

int fmxq_moe_sort_workspace(int64_t T, int64_t top_k, int64_t E, size_t* bytes) {
  const char* op = "moe_sort_workspace";
  if (int rc = row_sizes(T, top_k, 0, op)) return rc;
  if (E < 1 || E > kSortMaxExperts)
    return fail(FMXQ_ERR_UNSUPPORTED, "%s: %lld experts (1..%lld supported)", op, (long long)E,
                (long long)kSortMaxExperts);
  return bytes_out(fmxq::moe_sort_hist_bytes(T * top_k, E), bytes, op);
}

int fmxq_moe_sort(const uint16_t* x, const uint32_t* inds, uint16_t* xs, uint32_t* order,
                  uint32_t* pos, uint32_t* offsets, int64_t T, int64_t top_k, int64_t E, int64_t D,
                  void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "moe_sort";
  if (int rc = row_sizes(T, top_k, D, op)) return rc;
  if (E < 1 || E > kSortMaxExperts)
    return fail(FMXQ_ERR_UNSUPPORTED, "%s: %lld experts (1..%lld supported)", op, (long long)E,
                (long long)kSortMaxExperts);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!offsets || !aligned(offsets, 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null or misaligned offsets", op);
  if (T == 0) return hip_status(fmxq::launch_fill_u32(offsets, 0u, E + 1, s), op);
  if (!inds || !order || !pos || (D > 0 && (!x || !xs)))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(inds, 4) || !aligned(order, 4) || !aligned(pos, 4) || !aligned(x, 2) || !aligned(xs, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  if (int rc = check_workspace(workspace, workspace_bytes,
                               fmxq::moe_sort_hist_bytes(T * top_k, E), op))
    return rc;
  uint32_t* flag = nullptr;
  if (int rc = device_flag(s, &flag)) return rc;
  const fmxq::MoeSort a{x, inds, xs, order, pos, offsets, T, top_k, E, D,
                        static_cast<uint32_t*>(workspace), flag};
  return hip_status(fmxq::launch_moe_sort(a, s), op);
}

int fmxq_moe_sort_grad(const uint16_t* dxs, const uint32_t* pos, uint16_t* dx, int64_t T,
                       int64_t top_k, int64_t D, void* stream) {
  const char* op = "moe_sort_grad";
  if (int rc = row_sizes(T, top_k, D, op)) return rc;
  if (T == 0 || D == 0) return FMXQ_OK;
  if (!dxs || !pos || !dx) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(dxs, 2) || !aligned(pos, 4) || !aligned(dx, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint32_t* flag = nullptr;
  if (int rc = device_flag(s, &flag)) return rc;
  return hip_status(fmxq::launch_moe_unsort(dxs, pos, nullptr, false, dx, T, top_k, D, flag, s), op);
}

int fmxq_moe_unsort(const uint16_t* y, const uint32_t* pos, const void* weights, int weights_bf16,
                    uint16_t* out, int64_t T, int64_t top_k, int64_t D, void* stream) {
  const char* op = "moe_unsort";
  if (int rc = row_sizes(T, top_k, D, op)) return rc;
  if (T == 0 || D == 0) return FMXQ_OK;
  if (!y || !pos || !weights || !out) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(y, 2) || !aligned(pos, 4) || !aligned(weights, weights_bf16 ? 2 : 4) || !aligned(out, 2))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint32_t* flag = nullptr;
  if (int rc = device_flag(s, &flag)) return rc;
  return hip_status(
      fmxq::launch_moe_unsort(y, pos, weights, weights_bf16 != 0, out, T, top_k, D, flag, s), op);
}

int fmxq_moe_unsort_grad(const uint16_t* dout, const uint16_t* y, const uint32_t* pos,
                         const void* weights, int weights_bf16, uint16_t* dy, void* dweights,
                         int64_t T, int64_t top_k, int64_t D, void* stream) {
  const char* op = "moe_unsort_grad";
  if (int rc = row_sizes(T, top_k, D, op)) return rc;
  if (T == 0) return FMXQ_OK;
  if (!pos || !weights || !dweights || (D > 0 && (!dout || !y || !dy)))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  const uintptr_t we = weights_bf16 ? 2 : 4;
  if (!aligned(dout, 2) || !aligned(y, 2) || !aligned(pos, 4) || !aligned(weights, we) ||
      !aligned(dy, 2) || !aligned(dweights, we))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint32_t* flag = nullptr;
  if (int rc = device_flag(s, &flag)) return rc;
  return hip_status(fmxq::launch_moe_unsort_grad(dout, y, pos, weights, weights_bf16 != 0, dy, dweights,
                                                 T, top_k, D, flag, s),
                    op);
}

}  // extern "C"
