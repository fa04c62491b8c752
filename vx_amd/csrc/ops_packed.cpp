/*
 * ops_packed.cpp -- the ops of a packed batch in 8 bits (include/vx_hip_ops.h):
 * argument checks, then launches on the caller stream. Checks and devices as in
 * ops_batch.cpp.
 */
#include "../../include/vx_hip_ops.h"
#include "op_checks.h"
#include "vx_hip_common.h"
#include "vx_packed_kernels.h"

#include <cmath>

namespace {

using namespace vxops;

bool aligned_to(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int32_t norm(const char *op, const vxk::NormArgs &a, int64_t dim) {
  const size_t size = a.f32 ? 4 : 2;
  if (!a.x || (!a.y && !a.q) || !a.q != !a.q_scale) {
    return refuse(VX_OP_EINVAL, op, "x, one of y and q, and q_scale with q must not be NULL");
  }
  if (!within({a.rows, dim}, 1) || a.stride < dim || a.stride > kMaxExtent) {
    return refuse(VX_OP_EINVAL, op, "extents must be positive and the stride at least dim");
  }
  if (!(a.eps >= 0.0f) || !std::isfinite(a.eps)) {
    return refuse(VX_OP_EINVAL, op, "eps must be finite and not negative");
  }
  /* 1024 threads a row: their number is 32-bit */
  if (dim > vxk::kNormMaxDim || a.rows > (int64_t(1) << 21)) {
    return refuse(VX_OP_EUNSUPP, op, "more than 2^21 rows, or rows of more than 32768 elements");
  }
  if (!aligned_to(a.x, size) || !aligned_to(a.residual, size) || !aligned_to(a.sum, size) ||
      !aligned_to(a.y, 2) || !aligned4({a.weight, a.q_scale})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be aligned to their elements");
  }
  const OnDeviceOf on(op, {a.x, a.residual, a.weight, a.sum, a.y, a.q, a.q_scale});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  vxk::rms_norm_launch(a, stream());
  launched(op);
  return VX_OP_OK;
}

/* VX_OP_OK, or why the product takes no call of these extents. */
int32_t gemm_extents(int64_t tokens, int64_t rows, int64_t cols, const char **why) {
  if (!within({tokens, rows, cols}, 1)) {
    *why = "extents must be positive";
    return VX_OP_EINVAL;
  }
  if (cols % 16 != 0 || cols > vxk::kGemmI8MaxCols) {
    *why = "cols must be a multiple of 16 and at most 131056";
    return VX_OP_EUNSUPP;
  }
  if (tokens > (int64_t(1) << 24) || rows > (int64_t(1) << 24) ||
      ((tokens + 63) / 64) * ((rows + 63) / 64) > (int64_t(1) << 22)) {
    *why = "more than 2^24 tokens or rows, or 2^22 tiles of 64 x 64 outputs";
    return VX_OP_EUNSUPP;
  }
  return VX_OP_OK;
}

int32_t gemm(const char *op, bool f32, const int8_t *x, const float *x_scale, const int8_t *w,
             const float *w_scale, void *y, int64_t tokens, int64_t rows, int64_t cols,
             int64_t stride, void *workspace, int64_t workspace_bytes) {
  const char *why = nullptr;
  const int32_t code = gemm_extents(tokens, rows, cols, &why);
  if (code != VX_OP_OK) {
    return refuse(code, op, why);
  }
  if (!x || !x_scale || !w || !w_scale || !y) {
    return refuse(VX_OP_EINVAL, op, "a pointer is NULL");
  }
  if (stride < rows || stride > kMaxExtent) {
    return refuse(VX_OP_EINVAL, op, "the stride must be at least rows");
  }
  if (workspace && workspace_bytes < vx_nn_gemm_i8_workspace(tokens, rows, cols)) {
    return refuse(VX_OP_EINVAL, op, "the workspace is smaller than vx_nn_gemm_i8_workspace()");
  }
  if (!aligned16({x, w, workspace}) || !aligned4({x_scale, w_scale}) ||
      !aligned_to(y, f32 ? 4 : 2)) {
    return refuse(VX_OP_EUNSUPP, op, "x, w and the workspace must be 16-byte aligned, the others "
                                     "to their elements");
  }
  const OnDeviceOf on(op, {x, x_scale, w, w_scale, y, workspace});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  auto plan = [&](bool may_split) {
    return vxk::gemm_i8_plan(tokens, rows, cols, vxk::device_cu_count(), may_split);
  };
  const Space space(workspace, plan(true).ws_bytes);
  vxk::gemm_i8_launch(vxk::GemmI8Args{x, x_scale, w, w_scale, y, tokens, rows, (int)cols, stride, f32},
                      plan(space.enough), space.base, stream());
  launched(op);
  return VX_OP_OK;
}

int32_t logprobs(const char *op, bool f32, const void *logits, const int32_t *given, float *logprob,
                 float *entropy, int32_t *top_tokens, float *top_logprob, int64_t rows,
                 int64_t vocab, int64_t stride, int64_t n_given, int64_t n_top, void *workspace,
                 int64_t workspace_bytes) {
  const int64_t need = vx_nn_token_logprobs_workspace(rows, vocab, n_top);
  if (need < 0 || stride < vocab || stride > kMaxExtent) {
    return refuse(VX_OP_EINVAL, op,
                  "rows must be 1..2^21, vocab 1..2^30, n_top 0..64 and stride at least vocab");
  }
  if (n_given < 0 || n_given > (int64_t(1) << 20)) {
    return refuse(VX_OP_EINVAL, op, "n_given must be 0..2^20");
  }
  if (!logits || (n_given > 0 && (!given || !logprob)) || (n_top > 0 && !top_tokens) ||
      (n_given == 0 && n_top == 0 && !entropy)) {
    return refuse(VX_OP_EINVAL, op, "logits and what is asked for must not be NULL");
  }
  if (workspace && workspace_bytes < need) {
    return refuse(VX_OP_EINVAL, op, "the workspace is smaller than vx_nn_token_logprobs_workspace()");
  }
  if (!aligned4({given, logprob, entropy, top_tokens, top_logprob}) ||
      !aligned_to(logits, f32 ? 4 : 2) || !aligned16({workspace})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be aligned to their elements "
                                     "(the workspace to 16 bytes)");
  }
  const OnDeviceOf on(op, {logits, n_given ? given : nullptr, n_given ? logprob : nullptr, entropy,
                           n_top ? top_tokens : nullptr, n_top ? top_logprob : nullptr, workspace});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  const Space space(workspace, need);
  vxk::logprobs_launch(vxk::LogprobArgs{logits, given, logprob, entropy, top_tokens, top_logprob,
                                        (int)rows, (int)vocab, (int)n_given, (int)n_top, stride, f32},
                       vxk::logprobs_plan(rows, vocab, n_top, space.enough), space.base, stream());
  launched(op);
  return VX_OP_OK;
}

} // namespace

extern "C" {

int32_t vx_nn_rms_norm_bf16(const uint16_t *x, const uint16_t *residual, const float *weight,
                            uint16_t *sum, uint16_t *y, int8_t *q, float *q_scale, int64_t rows,
                            int64_t dim, int64_t stride, float eps) {
  return norm("vx_nn_rms_norm_bf16",
              vxk::NormArgs{x, residual, weight, sum, y, q, q_scale, rows, (int)dim, stride, eps,
                            false, true},
              dim);
}

int32_t vx_nn_rms_norm_f32(const float *x, const float *residual, const float *weight, float *sum,
                           uint16_t *y, int8_t *q, float *q_scale, int64_t rows, int64_t dim,
                           int64_t stride, float eps) {
  return norm("vx_nn_rms_norm_f32",
              vxk::NormArgs{x, residual, weight, sum, y, q, q_scale, rows, (int)dim, stride, eps,
                            true, true},
              dim);
}

int32_t vx_nn_quantize_i8_bf16(const uint16_t *x, int8_t *q, float *q_scale, int64_t rows,
                               int64_t dim, int64_t stride) {
  return norm("vx_nn_quantize_i8_bf16",
              vxk::NormArgs{x, nullptr, nullptr, nullptr, nullptr, q, q_scale, rows, (int)dim,
                            stride, 0.0f, false, false},
              dim);
}

int32_t vx_nn_quantize_i8_f32(const float *x, int8_t *q, float *q_scale, int64_t rows, int64_t dim,
                              int64_t stride) {
  return norm("vx_nn_quantize_i8_f32",
              vxk::NormArgs{x, nullptr, nullptr, nullptr, nullptr, q, q_scale, rows, (int)dim,
                            stride, 0.0f, true, false},
              dim);
}

int64_t vx_nn_gemm_i8_workspace(int64_t tokens, int64_t rows, int64_t cols) {
  const char *why = nullptr;
  const int32_t code = gemm_extents(tokens, rows, cols, &why);
  return code != VX_OP_OK
             ? code
             : vxk::gemm_i8_plan(tokens, rows, cols, vxk::device_cu_count(), true).ws_bytes;
}

int32_t vx_nn_gemm_i8_bf16(const int8_t *x, const float *x_scale, const int8_t *w,
                           const float *w_scale, uint16_t *y, int64_t tokens, int64_t rows,
                           int64_t cols, int64_t stride, void *workspace, int64_t workspace_bytes) {
  return gemm("vx_nn_gemm_i8_bf16", false, x, x_scale, w, w_scale, y, tokens, rows, cols, stride,
              workspace, workspace_bytes);
}

int32_t vx_nn_gemm_i8_f32(const int8_t *x, const float *x_scale, const int8_t *w,
                          const float *w_scale, float *y, int64_t tokens, int64_t rows,
                          int64_t cols, int64_t stride, void *workspace, int64_t workspace_bytes) {
  return gemm("vx_nn_gemm_i8_f32", true, x, x_scale, w, w_scale, y, tokens, rows, cols, stride,
              workspace, workspace_bytes);
}

int32_t vx_nn_flash_attention_packed_bf16(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                          const int32_t *offsets, uint16_t *o, float *lse,
                                          int64_t total, int64_t sequences, int64_t heads,
                                          int64_t kv_heads, int64_t head_dim, int64_t q_row,
                                          int64_t q_head, int64_t kv_row, int64_t kv_head,
                                          int64_t o_row, int64_t o_head, float scale,
                                          int32_t causal) {
  static const char op[] = "vx_nn_flash_attention_packed_bf16";
  if (!q || !k || !v || !offsets || !o) {
    return refuse(VX_OP_EINVAL, op, "q, k, v, offsets and o must not be NULL");
  }
  if (!within({total, sequences, heads, kv_heads}, 1) || heads % kv_heads != 0) {
    return refuse(VX_OP_EINVAL, op, "extents must be positive and heads a multiple of kv_heads");
  }
  if (head_dim != 64 && head_dim != 128) {
    return refuse(VX_OP_EUNSUPP, op, "head_dim must be 64 or 128");
  }
  if (!std::isfinite(scale * 1.4426950408889634f)) { /* the exponentials are of base 2 */
    return refuse(VX_OP_EINVAL, op, "scale must be finite, and times log2(e) too");
  }
  for (int64_t stride : {q_row, q_head, kv_row, kv_head, o_row, o_head}) {
    if (stride < head_dim || stride > kMaxExtent) {
      return refuse(VX_OP_EINVAL, op, "strides must be at least head_dim");
    }
    if (stride % 8 != 0) {
      return refuse(VX_OP_EUNSUPP, op, "strides must be multiples of 8");
    }
  }
  /* Rows of a sequence's queries, threads of a launch, and byte offsets within a
   * block of keys are 31-bit. */
  const int64_t rows = product({total, heads});
  if (rows < 0 || rows > (int64_t(1) << 28) || sequences > 65536 ||
      sequences * kv_heads > (int64_t(1) << 22) || kv_row > (int64_t(1) << 22)) {
    return refuse(VX_OP_EUNSUPP, op, "more than 2^28 queries of all heads, 65536 sequences or 2^22 "
                                     "sequences of a KV head, or kv_row above 2^22");
  }
  if (!aligned16({q, k, v, o}) || !aligned4({offsets, lse})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be 16-byte aligned (offsets and lse 4-byte)");
  }
  const OnDeviceOf on(op, {q, k, v, offsets, o, lse});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  vxk::flash_packed_launch(vxk::PackedAttnArgs{q, k, v, offsets, o, lse, (int)total, (int)sequences,
                                               (int)heads, (int)kv_heads, q_row, q_head, kv_row,
                                               kv_head, o_row, o_head, scale, causal != 0},
                           (int)head_dim, stream());
  launched(op);
  return VX_OP_OK;
}

int64_t vx_nn_token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t n_top) {
  /* 1024 threads a row: their number is 32-bit */
  if (rows < 1 || rows > (int64_t(1) << 21) || vocab < 1 || vocab > (int64_t(1) << 30) ||
      n_top < 0 || n_top > 64) {
    return VX_OP_EINVAL;
  }
  return vxk::logprobs_plan(rows, vocab, n_top, true).ws_bytes;
}

int32_t vx_nn_token_logprobs_f32(const float *logits, const int32_t *given, float *logprob,
                                 float *entropy, int32_t *top_tokens, float *top_logprob,
                                 int64_t rows, int64_t vocab, int64_t stride, int64_t n_given,
                                 int64_t n_top, void *workspace, int64_t workspace_bytes) {
  return logprobs("vx_nn_token_logprobs_f32", true, logits, given, logprob, entropy, top_tokens,
                  top_logprob, rows, vocab, stride, n_given, n_top, workspace, workspace_bytes);
}

int32_t vx_nn_token_logprobs_bf16(const uint16_t *logits, const int32_t *given, float *logprob,
                                  float *entropy, int32_t *top_tokens, float *top_logprob,
                                  int64_t rows, int64_t vocab, int64_t stride, int64_t n_given,
                                  int64_t n_top, void *workspace, int64_t workspace_bytes) {
  return logprobs("vx_nn_token_logprobs_bf16", false, logits, given, logprob, entropy, top_tokens,
                  top_logprob, rows, vocab, stride, n_given, n_top, workspace, workspace_bytes);
}

} // extern "C"
