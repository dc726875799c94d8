// fmxq_train_capi.cpp -- extern "C" entry points of gradient clipping and of adapters beside
// quantized products (declared in include/fmxq.h).
//
// As in fmxq_capi.cpp every check comes before anything is enqueued.  The workspaces are the
// caller's, so no call allocates device memory, and none shares memory with another.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/fmxq.h"
#include "fmxq_grad.hpp"
#include "fmxq_host.hpp"
#include "fmxq_internal.hpp"
#include "fmxq_train.hpp"

using fmxq::fail;
using fmxq::hip_status;

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_workspace(const void* ws, size_t have, size_t need, const char* op) {
  if (have < need)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu are needed", op, have,
                need);
  if (need && (!ws || !aligned(ws, 16)))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", op);
  return FMXQ_OK;
}

// ---- the norm over many tensors -------------------------------------------------------

constexpr int64_t kMaxTensors = 1 << 20;

// A result must not share memory with another result, nor with a gradient other than its own.
int check_outs(const void* const* grads, void* const* outs, const int64_t* counts, const int* bf16,
               int64_t n, const char* op) {
  struct Range {
    uintptr_t at, end;
    int64_t i;
  };
  std::vector<Range> r;
  r.reserve((size_t)n);
  for (int64_t i = 0; i < n; ++i)
    if (counts[i]) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(outs[i]);
      r.push_back({p, p + (uintptr_t)counts[i] * (bf16[i] ? 2 : 4), i});
    }
  const auto less = [](const Range& a, const Range& b) { return a.at < b.at; };
  if (!std::is_sorted(r.begin(), r.end(), less)) std::sort(r.begin(), r.end(), less);
  for (size_t k = 1; k < r.size(); ++k)
    if (r[k].at < r[k - 1].end)
      return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: results %lld and %lld overlap", op,
                  (long long)r[k - 1].i, (long long)r[k].i);
  for (int64_t i = 0; i < n; ++i) {
    if (!counts[i] || grads[i] == outs[i]) continue;
    const uintptr_t p = reinterpret_cast<uintptr_t>(grads[i]), e = p + (uintptr_t)counts[i] * (bf16[i] ? 2 : 4);
    // The results end in the order in which they begin.
    auto at = std::upper_bound(r.begin(), r.end(), p, [](uintptr_t v, const Range& b) { return v < b.end; });
    if (at != r.end() && at->at < e)
      return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: gradient %lld overlaps result %lld", op, (long long)i,
                  (long long)at->i);
  }
  // A gradient that is its own result shares no memory with another's, by the first check; one
  // listed twice in place is the first check's error as well.
  return FMXQ_OK;
}

int clip(const void* const* grads, void* const* outs, const int64_t* counts, const int* bf16, int64_t n,
         float max_norm, float* norm, void* ws, size_t ws_bytes, void* stream, const char* op) {
  if (n < 0 || n > kMaxTensors)
    return fail(FMXQ_ERR_SHAPE, "%s: %lld tensors (0..%lld supported)", op, (long long)n,
                (long long)kMaxTensors);
  if (n > 0 && (!grads || !counts || !bf16))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!norm || !aligned(norm, 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null or misaligned norm", op);
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] < 0 || counts[i] > (int64_t)1 << 40)
      return fail(FMXQ_ERR_SHAPE, "%s: tensor %lld has %lld elements", op, (long long)i, (long long)counts[i]);
    if (counts[i] == 0) continue;
    const uintptr_t size = bf16[i] ? 2 : 4;
    if (!grads[i] || !aligned(grads[i], size) || (outs && (!outs[i] || !aligned(outs[i], size))))
      return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: tensor %lld is null or misaligned", op, (long long)i);
  }
  if (int rc = check_workspace(ws, ws_bytes, fmxq::kClipBlocks * sizeof(double), op)) return rc;
  if (outs)
    if (int rc = check_outs(grads, outs, counts, bf16, n, op)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* sums = static_cast<double*>(ws);
  // Every table of tensors to f(table, whether it is the first): the squares, then the scaling.
  auto tables = [&](auto&& f) -> int {
    fmxq::ClipTable t;
    t.n = t.tiles = 0;
    bool first = true;
    auto flush = [&]() -> int {
      const int rc = hip_status(f(t, first), op);
      first = false;
      t.n = t.tiles = 0;
      return rc;
    };
    for (int64_t i = 0; i < n; ++i)
      for (int64_t at = 0; at < counts[i]; at += fmxq::kClipMaxCount) {
        if (t.n == fmxq::kClipTensors || t.tiles > 0x7fffffffu - (1u << 18))
          if (int rc = flush()) return rc;
        const int64_t size = bf16[i] ? 2 : 4, c = std::min(counts[i] - at, fmxq::kClipMaxCount);
        t.src[t.n] = (reinterpret_cast<uint64_t>(grads[i]) + at * size) | (bf16[i] ? 1u : 0u);
        t.dst[t.n] = outs ? reinterpret_cast<uint64_t>(outs[i]) + at * size : 0;
        t.count[t.n] = (uint32_t)c;
        t.tile[t.n] = t.tiles;
        t.tiles += (uint32_t)((c * size + fmxq::kClipTileBytes - 1) / fmxq::kClipTileBytes);
        ++t.n;
      }
    return t.n || first ? flush() : (int)FMXQ_OK;
  };
  if (int rc = tables([&](const fmxq::ClipTable& t, bool first) {
        return fmxq::launch_clip_squares(t, sums, !first, s);
      }))
    return rc;
  if (!outs) return hip_status(fmxq::launch_clip_norm(sums, norm, s), op);
  return tables([&](const fmxq::ClipTable& t, bool first) {
    return fmxq::launch_clip_scale(t, sums, max_norm, first ? norm : nullptr, s);
  });
}

// ---- adapters -----------------------------------------------------------------------

constexpr int64_t kMaxRows = (1 << 24) - 1, kMaxWidth = (1 << 22) - 8;
// Up to here the rows' shrinks are taken one at a time, in any order: one launch, which reads an adapter and x
// again for every value; above, the sort, the shrink and its parts, three launches, which read an adapter once for
// 32 rows that share it.  (us that way and the other, 4 bits, 14336 x 4096.  128 rows: one adapter of rank 16
// 46 and 51, of rank 128 69 and 73; 8 adapters in any order, rank 16 64 and 79, rank 128 167 and 194.  256 rows:
// 61 and 64, 92 and 86; 77 and 90, 198 and 203.  Of 14336 values a row, 4096 outputs, 128 rows of one adapter of
// rank 128 100 and 84, of 8 200 and 214; rank 64 and lower as above.  So depth times rank decides nearer to the
// border than rows alone do.)
constexpr int64_t kLoraFewRows = 128;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct LoraPlan {
  bool few, sort;
  int64_t n8;
  int splits, splits_dy;
  fmxq::OutPlan out;
  size_t u, t, order, pos, offsets, hist, none, du, dt, at, bt, part_a, part_b, product, bytes;
};

// Workspace of the forward pass (product: that of x . deq(W)^T) or of the gradients (of dy . deq(W)).
LoraPlan lora_plan(int64_t M, int64_t N, int64_t K, int64_t E, int r, bool grad, size_t product) {
  LoraPlan p{};
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
  };
  p.n8 = up(N, 8);
  p.few = !grad && M <= kLoraFewRows;
  p.sort = !p.few && E > 1;
  p.splits = fmxq::lora_splits(M, K);
  p.splits_dy = fmxq::lora_splits(M, p.n8);
  p.u = take(M * (grad ? fmxq::kLoraParts : 2) * r * 2);
  p.t = take(p.few ? 0 : p.splits * M * r * 4);
  if (p.sort) {
    p.order = take(M * 4);
    p.pos = take(M * 4);
    p.offsets = take((E + 1) * 4);
    p.hist = take((int64_t)fmxq::moe_sort_hist_bytes(M, E));
    p.none = take(16);
  }
  if (grad) {
    p.du = take(M * fmxq::kLoraParts * r * 2);
    p.dt = take(p.splits_dy * M * r * 4);
    p.at = take(E * K * r * 2);
    p.bt = take(E * r * p.n8 * 2);
    p.part_a = take(fmxq::lora_outer_floats(M, K, r) * 4);
    p.part_b = take(fmxq::lora_outer_floats(M, N, r) * 4);
  } else {
    p.out = fmxq::out_plan(M, N, K);
    product = p.out.bytes;
  }
  p.product = take((int64_t)product);
  p.bytes = at;  // (an aligned copy of dy may follow)
  return p;
}

int lora_sizes(int64_t M, int64_t N, int64_t K, int64_t E, int r, bool grad, const char* op) {
  if (M < 0 || N < 0 || K < 0)
    return fail(FMXQ_ERR_SHAPE, "%s: negative size M=%lld N=%lld K=%lld", op, (long long)M,
                (long long)N, (long long)K);
  if (E < 1 || E > fmxq::kLoraMaxAdapters)
    return fail(FMXQ_ERR_UNSUPPORTED, "%s: %lld adapters (1..%lld supported)", op, (long long)E,
                (long long)fmxq::kLoraMaxAdapters);
  if (r < 8 || r > fmxq::kLoraMaxRank || r % 8)
    return fail(FMXQ_ERR_UNSUPPORTED, "%s: rank %d (multiples of 8 up to %d supported: zeros may fill it)",
                op, r, fmxq::kLoraMaxRank);
  if (M > kMaxRows || N > kMaxWidth || K > kMaxWidth)
    return fail(FMXQ_ERR_SHAPE, "%s: M=%lld, N=%lld or K=%lld too large", op, (long long)M,
                (long long)N, (long long)K);
  // (A and B, and both outer products, share a launch.)
  const int64_t rows = (M + 127) / 128, cols = (std::max(N, K) + 255) / 256;
  if (rows * cols >= fmxq::kLoraMaxBlocks ||
      (grad && (fmxq::lora_turn_blocks(K, r, E) + fmxq::lora_turn_blocks(r, up(N, 8), E) >=
                    fmxq::kLoraMaxBlocks ||
                fmxq::lora_outer_blocks(M, N, E) + fmxq::lora_outer_blocks(M, K, E) >= fmxq::kLoraMaxBlocks)))
    return fail(FMXQ_ERR_SHAPE, "%s: %lld rows of %lld and %lld for %lld adapters are too many", op,
                (long long)M, (long long)N, (long long)K, (long long)E);
  return FMXQ_OK;
}

// The rows' order by adapter, where the plan wants one.
int lora_rows(const LoraPlan& p, char* ws, const int32_t* adapters, int64_t M, int64_t E, int r,
              hipStream_t s, fmxq::LoraRows* l, const char* op) {
  *l = fmxq::LoraRows{adapters, nullptr, nullptr, M, E, r, nullptr};
  if (int rc = fmxq::device_flag(s, &l->flag)) return rc;
  if (!p.sort) return FMXQ_OK;
  l->order = reinterpret_cast<uint32_t*>(ws + p.order);
  l->offsets = reinterpret_cast<uint32_t*>(ws + p.offsets);
  if (fmxq::lora_sort_supported(M, E))
    return hip_status(fmxq::launch_lora_sort(adapters, M, E, reinterpret_cast<uint32_t*>(ws + p.order),
                                             reinterpret_cast<uint32_t*>(ws + p.offsets), s),
                      op);
  fmxq::MoeSort m{};
  m.inds = reinterpret_cast<const uint32_t*>(adapters);
  m.order = reinterpret_cast<uint32_t*>(ws + p.order);
  m.pos = reinterpret_cast<uint32_t*>(ws + p.pos);
  m.offsets = reinterpret_cast<uint32_t*>(ws + p.offsets);
  m.T = M;
  m.k = 1;
  m.E = E;
  m.hist = reinterpret_cast<uint32_t*>(ws + p.hist);
  m.flag = reinterpret_cast<uint32_t*>(ws + p.none);  // rows without adapter are no error
  return hip_status(fmxq::launch_moe_sort(m, s), op);
}

}  // namespace

extern "C" {

int fmxq_quantized_matmul_lora_workspace(int64_t M, int64_t N, int64_t K, int64_t E, int r, size_t* bytes) {
  const char* op = "quantized_matmul_lora_workspace";
  if (int rc = lora_sizes(M, N, K, E, r, false, op)) return rc;
  if (!bytes) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null result", op);
  *bytes = M == 0 || N == 0 ? 0 : lora_plan(M, N, K, E, r, false, 0).bytes;
  return FMXQ_OK;
}

int fmxq_quantized_matmul_lora(const uint16_t* x, const uint32_t* w, const uint16_t* scales,
                               const uint16_t* biases, const uint16_t* a, const uint16_t* b,
                               const int32_t* adapters, const float* lora_scales, uint16_t* y, int64_t M,
                               int64_t N, int64_t K, int64_t E, int r, int group_size, int bits,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "quantized_matmul_lora";
  if (int rc = fmxq::check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = lora_sizes(M, N, K, E, r, false, op)) return rc;
  if (M == 0 || N == 0) return FMXQ_OK;
  if (!x || !w || !scales || !biases || !a || !b || !adapters || !lora_scales || !y)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(a, 16) || !aligned(b, 16) || !aligned(y, 16))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: x, w, a, b and y must be 16-byte aligned", op);
  if (!aligned(scales, 2) || !aligned(biases, 2) || !aligned(adapters, 4) ||
      !aligned(lora_scales, 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  const LoraPlan p = lora_plan(M, N, K, E, r, false, 0);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, op)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  fmxq::LoraRows l;
  if (int rc = lora_rows(p, ws, adapters, M, E, r, s, &l, op)) return rc;
  const fmxq::LoraShrink xa{x, K, a, K, K, p.splits, reinterpret_cast<float*>(ws + p.t),
                            reinterpret_cast<uint16_t*>(ws + p.u)};
  const fmxq::Zeros zeros{reinterpret_cast<uint32_t*>(ws + p.product + p.out.count_at), p.out.counters};
  if (p.few) {
    if (int rc = hip_status(fmxq::launch_lora_shrink_rows(l, xa, lora_scales, zeros, s), op)) return rc;
  } else {
    if (int rc = hip_status(fmxq::launch_lora_shrink(l, &xa, 1, s), op)) return rc;
    if (int rc = hip_status(fmxq::launch_lora_parts(l, &xa, 1, 2, lora_scales, zeros, s), op)) return rc;
  }
  const fmxq::LoraAdd add{xa.u, b, adapters, E, N, r, 2};
  return hip_status(fmxq::launch_out(x, w, scales, biases, add, y, M, N, K, group_size, bits, p.out,
                                     ws + p.product, l.flag, s),
                    op);
}

int fmxq_quantized_matmul_lora_grad_workspace(int64_t M, int64_t N, int64_t K, int64_t E, int r,
                                              size_t* bytes) {
  const char* op = "quantized_matmul_lora_grad_workspace";
  if (int rc = lora_sizes(M, N, K, E, r, true, op)) return rc;
  size_t base = 0;
  if (int rc = fmxq_quantized_matmul_grad_workspace(M, N, K, &base)) return rc;
  if (!bytes) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null result", op);
  *bytes = M == 0 || N == 0 ? 0 : lora_plan(M, N, K, E, r, true, base).bytes;
  return FMXQ_OK;
}

int fmxq_quantized_matmul_lora_grad(const uint16_t* dy, const uint16_t* x, const uint32_t* w,
                                    const uint16_t* scales, const uint16_t* biases, const uint16_t* a,
                                    const uint16_t* b, const int32_t* adapters, const float* lora_scales,
                                    uint16_t* dx, float* da, float* db, int64_t M, int64_t N, int64_t K,
                                    int64_t E, int r, int group_size, int bits, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* op = "quantized_matmul_lora_grad";
  if (int rc = fmxq::check_quant(group_size, bits, K, true, op)) return rc;
  if (int rc = lora_sizes(M, N, K, E, r, true, op)) return rc;
  size_t base = 0;
  if (int rc = fmxq_quantized_matmul_grad_workspace(M, N, K, &base)) return rc;
  if (!da || !aligned(da, 16) || (N > 0 && (!db || !aligned(db, 16))))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: da and db must be 16-byte aligned", op);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (M > 0 && (!dx || !aligned(dx, 16)))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: dx must be 16-byte aligned", op);
  if (M == 0 || N == 0) {
    auto zero = [&](void* p, int64_t words) -> int {
      constexpr int64_t kMost = (int64_t)1 << 30;  // of a launch
      for (int64_t at = 0; at < words; at += kMost)
        if (int rc = hip_status(fmxq::launch_fill_u32(static_cast<uint32_t*>(p) + at, 0u,
                                                      std::min(words - at, kMost), s),
                                op))
          return rc;
      return FMXQ_OK;
    };
    if (int rc = zero(dx, M * K / 2)) return rc;
    if (int rc = zero(da, E * r * K)) return rc;
    return zero(db, E * r * N);
  }
  if (!dy || !x || !w || !scales || !biases || !a || !b || !adapters || !lora_scales)
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(a, 16) || !aligned(b, 16))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: x, w, a and b must be 16-byte aligned", op);
  if (!aligned(dy, 2) || !aligned(scales, 2) || !aligned(biases, 2) || !aligned(adapters, 4) ||
      !aligned(lora_scales, 4))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their element size", op);
  const LoraPlan p = lora_plan(M, N, K, E, r, true, base);
  const bool moved = N % 8 == 0 && !aligned(dy, 16);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes + (moved ? (size_t)(M * N * 2) : 0), op))
    return rc;
  char* ws = static_cast<char*>(workspace);
  // dy in rows of 16-byte units: a copy, where it takes one, serves all that reads dy.
  const uint16_t* g = dy;
  if (moved || N % 8) {
    uint16_t* pad = reinterpret_cast<uint16_t*>(ws + (moved ? p.bytes : p.product));
    if (int rc = hip_status(fmxq::launch_pad_rows(dy, pad, M, N, p.n8, s), op)) return rc;
    g = pad;
  }
  fmxq::LoraRows l;
  if (int rc = lora_rows(p, ws, adapters, M, E, r, s, &l, op)) return rc;
  uint16_t *at = reinterpret_cast<uint16_t*>(ws + p.at), *bt = reinterpret_cast<uint16_t*>(ws + p.bt);
  const fmxq::LoraTurn turns[2] = {{a, at, r, K, r}, {b, bt, N, r, p.n8}};
  const fmxq::LoraShrink shrinks[2] = {
      {x, K, a, K, K, p.splits, reinterpret_cast<float*>(ws + p.t), reinterpret_cast<uint16_t*>(ws + p.u)},
      {g, p.n8, bt, p.n8, p.n8, p.splits_dy, reinterpret_cast<float*>(ws + p.dt),
       reinterpret_cast<uint16_t*>(ws + p.du)}};
  const fmxq::LoraOuter outers[2] = {
      {g, p.n8, N, shrinks[0].u, false, db, reinterpret_cast<float*>(ws + p.part_b)},
      {x, K, K, shrinks[1].u, true, da, reinterpret_cast<float*>(ws + p.part_a)}};
  if (int rc = hip_status(fmxq::launch_lora_turn(l, turns, 2, s), op)) return rc;
  if (int rc = hip_status(fmxq::launch_lora_shrink(l, shrinks, 2, s), op)) return rc;
  if (int rc = hip_status(fmxq::launch_lora_parts(l, shrinks, 2, fmxq::kLoraParts, lora_scales, fmxq::Zeros{}, s), op))
    return rc;
  if (int rc = hip_status(fmxq::launch_lora_outer(l, outers, 2, s), op)) return rc;
  const fmxq::LoraAdd add{shrinks[1].u, at, adapters, E, K, r, fmxq::kLoraParts};
  return fmxq::input_grad(g, p.n8, w, scales, biases, add, dx, M, N, K, group_size, bits,
                          ws + p.product, base, stream, op);
}

int fmxq_grad_norm_workspace(size_t* bytes) {
  if (!bytes) return fail(FMXQ_ERR_INVALID_ARGUMENT, "grad_norm_workspace: null result");
  *bytes = fmxq::kClipBlocks * sizeof(double);
  return FMXQ_OK;
}

int fmxq_grad_norm(const void* const* grads, const int64_t* counts, const int* bf16, int64_t n,
                   float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  return clip(grads, nullptr, counts, bf16, n, 0.f, norm, workspace, workspace_bytes, stream, "grad_norm");
}

int fmxq_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* counts,
                        const int* bf16, int64_t n, float max_norm, float* norm, void* workspace,
                        size_t workspace_bytes, void* stream) {
  const char* op = "clip_grad_norm";
  if (!(max_norm >= 0.f))
    return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: max_norm %g must not be negative", op, (double)max_norm);
  if (n > 0 && !outs) return fail(FMXQ_ERR_INVALID_ARGUMENT, "%s: null operand", op);
  void* none = nullptr;
  try {
    return clip(grads, outs ? outs : &none, counts, bf16, n, max_norm, norm, workspace, workspace_bytes,
                stream, op);
  } catch (const std::bad_alloc&) {
    return fail(FMXQ_ERR_DEVICE, "%s: out of host memory", op);
  }
}

}  // extern "C"
