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
/* How a call is divided: `shared_groups` workgroups over the shared keys of
 * all sequences' queries, `own_groups` over own keys (`together`: over shared
 * and own ones), parts merged from `ws_bytes` of workspace. */
struct SharedPlan {
  int rows;        /* queries of all heads */
  int parts;       /* partial results of each (1: none, the result itself) */
  int shared_splits, own_splits; /* workgroups that divide a tile's keys */
  int shared_groups, own_groups;
  int own_tiles;   /* tiles of a sequence's queries of a KV head */
  int tile;        /* rows of a wide tile: 64 or 128 */
  bool together;
  bool shared_rows, own_rows; /* 16-row tiles */
  int64_t ws_bytes;
};
/* Plain host arithmetic; `may_split` false: a plan without a workspace. */
SharedPlan flash_shared_plan(int64_t batch, int heads, int kv_heads, int seq_q, int shared_len,
                             int capacity, int head_dim, int cus, bool may_split);
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
