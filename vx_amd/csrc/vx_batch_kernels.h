/*
 * vx_batch_kernels.h -- launchers of the kernels of a batch that shares a
 * prompt (ops_batch.cpp calls them after validating arguments): rope_append,
 * attention over a shared prefix, sampling.
 */
#ifndef VX_AMD_BATCH_KERNELS_H
#define VX_AMD_BATCH_KERNELS_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vxk {

struct RopeAppendArgs {
  const void *qkv; /* bf16, or f32 where `f32` */
  const float *rope;
  const int32_t *lens;
  uint16_t *q, *k_cache, *v_cache;
  int64_t batch;
  int seq_q, heads, kv_heads, head_dim;
  int64_t shared_len, capacity;
  bool f32;
};
void rope_append_launch(const RopeAppendArgs &a, hipStream_t stream);

struct SharedAttnArgs {
  const uint16_t *q, *k_shared, *v_shared, *k, *v;
  const int32_t *lens;
  uint16_t *o;
  float *lse;
  int batch, heads, kv_heads, seq_q;
  int shared_len;
  int64_t shared_capacity;
  int capacity;
  float scale;
  bool causal;
};
void flash_shared_launch(const SharedAttnArgs &a, int head_dim, hipStream_t stream);

struct SampleArgs {
  const void *logits; /* bf16, or f32 where `f32` */
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p, *u;
  int32_t *tokens;
  float *logprob;
  int rows, vocab;
  int64_t stride;
  bool f32;
};
void sample_launch(const SampleArgs &a, hipStream_t stream);

} // namespace vxk

#endif /* VX_AMD_BATCH_KERNELS_H */
