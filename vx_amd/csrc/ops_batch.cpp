/*
 * ops_batch.cpp -- the ops of a batch that shares a prompt
 * (include/vx_hip_ops.h): argument checks, then launches on the caller stream.
 *
 * Arguments are checked before the GPU is looked for, so a refusal does not
 * depend on the machine. Every operand must be memory of one GPU, which is
 * the one the kernels run on whichever is current.
 */
#include "../../include/vx_hip_ops.h"
#include "op_checks.h"
#include "vx_batch_kernels.h"
#include "vx_hip_common.h"

#include <cmath>

namespace {

using namespace vxops;

int32_t rope_append(const char *op, bool f32, const void *qkv, const float *rope,
                    const int32_t *lens, uint16_t *q, uint16_t *k_cache, uint16_t *v_cache,
                    int64_t batch, int64_t seq_q, int64_t heads, int64_t kv_heads,
                    int64_t head_dim, int64_t shared_len, int64_t capacity, int64_t rope_len) {
  if (!qkv || !q || !k_cache || !v_cache) {
    return refuse(VX_OP_EINVAL, op, "qkv, q, k_cache and v_cache must not be NULL");
  }
  if (!within({batch, seq_q, heads, kv_heads, head_dim, capacity}, 1) || !within({shared_len}, 0)) {
    return refuse(VX_OP_EINVAL, op, "extents must be positive (shared_len may be 0)");
  }
  if (rope && rope_len < shared_len + capacity) {
    return refuse(VX_OP_EINVAL, op, "the table has fewer rows than shared_len + capacity");
  }
  if (head_dim % 8 != 0 || head_dim > 512) {
    return refuse(VX_OP_EUNSUPP, op, "head_dim must be a multiple of 8 and at most 512");
  }
  const int64_t units = product({batch, seq_q, heads + 2 * kv_heads, head_dim / 8});
  /* a thread a unit: their number is 31-bit */
  if (units < 0 || units > INT32_MAX || seq_q > INT32_MAX ||
      heads > INT32_MAX / 4 || kv_heads > INT32_MAX / 4 || capacity > INT32_MAX ||
      product({batch, kv_heads, capacity, head_dim}) < 0) {
    return refuse(VX_OP_EUNSUPP, op, "extents past 2^31");
  }
  if (!aligned16({qkv, rope, q, k_cache, v_cache}) || !aligned4({lens})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be 16-byte aligned (lens 4-byte)");
  }
  const OnDeviceOf on(op, {qkv, rope, lens, q, k_cache, v_cache});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  vxk::rope_append_launch(vxk::RopeAppendArgs{qkv, rope, lens, q, k_cache, v_cache, batch,
                                              (int)seq_q, (int)heads, (int)kv_heads,
                                              (int)head_dim, shared_len, capacity, f32},
                          vxops::stream());
  vxops::launched(op);
  return VX_OP_OK;
}

int32_t sample(const char *op, bool f32, const void *logits, const float *temperature,
               const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
               int32_t *tokens, float *logprob, int64_t rows, int64_t vocab, int64_t stride,
               void *workspace, int64_t workspace_bytes) {
  if (!logits || !u || !tokens) {
    return refuse(VX_OP_EINVAL, op, "logits, u and tokens must not be NULL");
  }
  const int64_t need = vx_nn_sample_workspace(rows, vocab);
  if (need < 0 || stride < vocab || stride > kMaxExtent) {
    return refuse(VX_OP_EINVAL, op,
                  "rows must be 1..2^21, vocab 1..2^30 and stride at least vocab");
  }
  if (workspace && workspace_bytes < need) {
    return refuse(VX_OP_EINVAL, op, "the workspace is smaller than vx_nn_sample_workspace()");
  }
  if (!aligned4({temperature, top_k, top_p, min_p, u, tokens, logprob}) ||
      (reinterpret_cast<uintptr_t>(logits) & (f32 ? 3 : 1)) || !aligned16({workspace})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be aligned to their elements "
                                     "(the workspace to 16 bytes)");
  }
  const OnDeviceOf on(op, {logits, temperature, top_k, top_p, min_p, u, tokens, logprob, workspace});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  const bool borders = top_k || top_p;
  const Space space(workspace, vxk::sample_plan(rows, vocab, borders, true).ws_bytes);
  vxk::sample_launch(vxk::SampleArgs{logits, temperature, top_k, top_p, min_p, u, tokens, logprob,
                                     (int)rows, (int)vocab, stride, f32},
                     vxk::sample_plan(rows, vocab, borders, space.enough), space.base,
                     vxops::stream());
  vxops::launched(op);
  return VX_OP_OK;
}

/* VX_OP_OK, or why the attention takes no call of these extents. */
int32_t shared_extents(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
                       int64_t shared_len, int64_t capacity, int64_t head_dim, const char **why) {
  if (!within({batch, heads, kv_heads, seq_q}, 1) || !within({shared_len, capacity}, 0) ||
      shared_len + capacity < 1 || heads % kv_heads != 0) {
    *why = "extents must be positive (one of shared_len and capacity may be 0) and heads a "
           "multiple of kv_heads";
    return VX_OP_EINVAL;
  }
  if (head_dim != 64 && head_dim != 128) {
    *why = "head_dim must be 64 or 128";
    return VX_OP_EUNSUPP;
  }
  const int64_t rows = product({batch, heads, seq_q, head_dim});
  /* Byte offsets within a KV head's keys and within a KV head's queries, and
   * workgroup counts, are 31-bit. */
  if (rows < 0 || rows / head_dim > INT32_MAX / 512 || shared_len + capacity > INT32_MAX / 256 ||
      product({batch, kv_heads, capacity, head_dim}) < 0) {
    *why = "more than 2^22 queries of all heads, or more than 2^23 keys";
    return VX_OP_EUNSUPP;
  }
  return VX_OP_OK;
}

} // namespace

extern "C" {

int32_t vx_nn_rope_append_bf16(const uint16_t *qkv, const float *rope, const int32_t *lens,
                               uint16_t *q, uint16_t *k_cache, uint16_t *v_cache, int64_t batch,
                               int64_t seq_q, int64_t heads, int64_t kv_heads, int64_t head_dim,
                               int64_t shared_len, int64_t capacity, int64_t rope_len) {
  return rope_append("vx_nn_rope_append_bf16", false, qkv, rope, lens, q, k_cache, v_cache, batch,
                     seq_q, heads, kv_heads, head_dim, shared_len, capacity, rope_len);
}

int32_t vx_nn_rope_append_f32(const float *qkv, const float *rope, const int32_t *lens,
                              uint16_t *q, uint16_t *k_cache, uint16_t *v_cache, int64_t batch,
                              int64_t seq_q, int64_t heads, int64_t kv_heads, int64_t head_dim,
                              int64_t shared_len, int64_t capacity, int64_t rope_len) {
  return rope_append("vx_nn_rope_append_f32", true, qkv, rope, lens, q, k_cache, v_cache, batch,
                     seq_q, heads, kv_heads, head_dim, shared_len, capacity, rope_len);
}

int64_t vx_nn_flash_attention_shared_workspace(int64_t batch, int64_t heads, int64_t kv_heads,
                                               int64_t seq_q, int64_t shared_len,
                                               int64_t capacity, int64_t head_dim) {
  const char *why = nullptr;
  const int32_t code = shared_extents(batch, heads, kv_heads, seq_q, shared_len, capacity,
                                      head_dim, &why);
  if (code != VX_OP_OK) {
    return code;
  }
  return vxk::flash_shared_plan(batch, (int)heads, (int)kv_heads, (int)seq_q, (int)shared_len,
                                (int)capacity, (int)head_dim, vxk::device_cu_count(), true)
      .ws_bytes;
}

int32_t vx_nn_flash_attention_shared_bf16(
    const uint16_t *q, const uint16_t *k_shared, const uint16_t *v_shared, const uint16_t *k,
    const uint16_t *v, const int32_t *lens, uint16_t *o, float *lse, int64_t batch, int64_t heads,
    int64_t kv_heads, int64_t seq_q, int64_t shared_len, int64_t shared_capacity,
    int64_t capacity, int64_t head_dim, float scale, int32_t causal, void *workspace,
    int64_t workspace_bytes) {
  static const char op[] = "vx_nn_flash_attention_shared_bf16";
  const char *why = nullptr;
  const int32_t code = shared_extents(batch, heads, kv_heads, seq_q, shared_len, capacity,
                                      head_dim, &why);
  if (code != VX_OP_OK) {
    return refuse(code, op, why);
  }
  if (!q || !o || (shared_len > 0 && (!k_shared || !v_shared)) || (capacity > 0 && (!k || !v))) {
    return refuse(VX_OP_EINVAL, op, "q, o and the keys and values of what is not empty must not "
                                    "be NULL");
  }
  if (!std::isfinite(scale * 1.4426950408889634f)) { /* the exponentials are of base 2 */
    return refuse(VX_OP_EINVAL, op, "scale must be finite, and times log2(e) too");
  }
  if (shared_capacity < shared_len || shared_capacity > INT32_MAX / 256) {
    return refuse(VX_OP_EINVAL, op, "shared_capacity must be at least shared_len and below 2^23");
  }
  if (workspace && workspace_bytes < vx_nn_flash_attention_shared_workspace(
                                         batch, heads, kv_heads, seq_q, shared_len, capacity,
                                         head_dim)) {
    return refuse(VX_OP_EINVAL, op, "the workspace is smaller than "
                                    "vx_nn_flash_attention_shared_workspace()");
  }
  if (!aligned16({q, k_shared, v_shared, k, v, o, workspace}) || !aligned4({lens, lse})) {
    return refuse(VX_OP_EUNSUPP, op, "operands must be 16-byte aligned (lens and lse 4-byte)");
  }
  const OnDeviceOf on(op, {q, shared_len ? k_shared : nullptr, shared_len ? v_shared : nullptr,
                           capacity ? k : nullptr, capacity ? v : nullptr, lens, o, lse,
                           static_cast<const uint16_t *>(workspace)});
  if (on.code != VX_OP_OK) {
    return on.code;
  }
  const vxk::SharedAttnArgs args{q, k_shared, v_shared, k, v, lens, o, lse, (int)batch,
                                 (int)heads, (int)kv_heads, (int)seq_q, (int)shared_len,
                                 shared_capacity, (int)capacity, scale, causal != 0};
  auto plan = [&](bool may_split) {
    return vxk::flash_shared_plan(batch, (int)heads, (int)kv_heads, (int)seq_q, (int)shared_len,
                                  (int)capacity, (int)head_dim, vxk::device_cu_count(),
                                  may_split);
  };
  const Space space(workspace, plan(true).ws_bytes);
  vxk::flash_shared_launch(args, plan(space.enough), (int)head_dim, space.base, vxops::stream());
  vxops::launched(op);
  return VX_OP_OK;
}

int64_t vx_nn_sample_workspace(int64_t rows, int64_t vocab) {
  /* 1024 threads a row: their number is 32-bit */
  if (rows < 1 || rows > (int64_t(1) << 21) || vocab < 1 || vocab > (int64_t(1) << 30)) {
    return VX_OP_EINVAL;
  }
  return vxk::sample_plan(rows, vocab, true, true).ws_bytes;
}

int32_t vx_nn_sample_f32(const float *logits, const float *temperature, const int32_t *top_k,
                         const float *top_p, const float *min_p, const float *u, int32_t *tokens,
                         float *logprob, int64_t rows, int64_t vocab, int64_t stride,
                         void *workspace, int64_t workspace_bytes) {
  return sample("vx_nn_sample_f32", true, logits, temperature, top_k, top_p, min_p, u, tokens,
                logprob, rows, vocab, stride, workspace, workspace_bytes);
}

int32_t vx_nn_sample_bf16(const uint16_t *logits, const float *temperature, const int32_t *top_k,
                          const float *top_p, const float *min_p, const float *u,
                          int32_t *tokens, float *logprob, int64_t rows, int64_t vocab,
                          int64_t stride, void *workspace, int64_t workspace_bytes) {
  return sample("vx_nn_sample_bf16", false, logits, temperature, top_k, top_p, min_p, u, tokens,
                logprob, rows, vocab, stride, workspace, workspace_bytes);
}

} // extern "C"
