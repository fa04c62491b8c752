/*
 * vx_batch_kernels.h -- launchers of the kernels of a batch that shares a
 * prompt (ops_batch.cpp calls them after validating arguments): rope_append,
 * attention over a shared prefix, sampling.
 */
#ifndef VX_AMD_BATCH_KERNELS_H
#define VX_AMD_BATCH_KERNELS_H

#include "kernels/flash_shared.h"

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
void flash_shared_launch(const SharedAttnArgs &a, const SharedPlan &plan, int head_dim, char *ws,
                         hipStream_t stream);

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
  /* Where not NULL, the one row's uniform number is u[*step - step0] (u[0]
   * before step0). */
  const int *step = nullptr;
  int step0 = 0;
};
/* `slices` workgroups a row of `slice` logits each (1: one a row, which needs no
 * workspace). */
struct SamplePlan {
  int slices, slice;
  int64_t ws_bytes;
};
/* Plain host arithmetic; `borders`: top_k or top_p may be on in a row;
 * `may_split` false: a plan without a workspace. */
SamplePlan sample_plan(int64_t rows, int64_t vocab, bool borders, bool may_split);
void sample_launch(const SampleArgs &a, const SamplePlan &plan, char *ws, hipStream_t stream);

} // namespace vxk

#endif /* VX_AMD_BATCH_KERNELS_H */
