/*
 * vx_packed_kernels.h -- launchers of the kernels of a packed batch in 8 bits
 * (ops_packed.cpp calls them after validating arguments): RMS norm and
 * quantization, int8 products, packed attention, log probabilities.
 */
#ifndef VX_AMD_PACKED_KERNELS_H
#define VX_AMD_PACKED_KERNELS_H

#include "kernels/gemm_i8.h"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vxk {

/* Widest rows of rms_norm and quantize_i8: a workgroup keeps one in registers. */
constexpr int64_t kNormMaxDim = 32768;

struct NormArgs {
  const void *x, *residual; /* bf16, or f32 where `f32`; residual may be null */
  const float *weight;      /* may be null */
  void *sum;                /* as x; may be null */
  uint16_t *y;              /* may be null */
  int8_t *q;                /* may be null, with q_scale */
  float *q_scale;
  int64_t rows;
  int dim;
  int64_t stride; /* of x */
  float eps;
  bool f32, norm; /* norm false: no division by the root mean square */
};
void rms_norm_launch(const NormArgs &a, hipStream_t stream);

struct GemmI8Args {
  const int8_t *x;
  const float *x_scale;
  const int8_t *w;
  const float *w_scale;
  void *y; /* bf16, or f32 where `f32` */
  int64_t tokens, rows;
  int cols;
  int64_t stride; /* of y */
  bool f32;
};
void gemm_i8_launch(const GemmI8Args &a, const GemmI8Plan &plan, char *ws, hipStream_t stream);

struct PackedAttnArgs {
  const uint16_t *q, *k, *v;
  const int32_t *offsets;
  uint16_t *o;
  float *lse; /* may be null */
  int total, sequences, heads, kv_heads;
  int64_t q_row, q_head, kv_row, kv_head, o_row, o_head; /* elements */
  float scale;
  bool causal;
};
void flash_packed_launch(const PackedAttnArgs &a, int head_dim, hipStream_t stream);

struct LogprobArgs {
  const void *logits; /* bf16, or f32 where `f32` */
  const int32_t *given;
  float *logprob, *entropy; /* entropy may be null */
  int32_t *top_tokens;
  float *top_logprob;
  int rows, vocab, n_given, n_top;
  int64_t stride;
  bool f32;
};
/* `slices` workgroups a row (1: one, which needs no workspace). */
struct LogprobPlan {
  int slices, slice;
  int64_t ws_bytes;
};
/* Plain host arithmetic; `may_split` false: a plan without a workspace. */
LogprobPlan logprobs_plan(int64_t rows, int64_t vocab, int64_t n_top, bool may_split);
void logprobs_launch(const LogprobArgs &a, const LogprobPlan &plan, char *ws, hipStream_t stream);

} // namespace vxk

#endif /* VX_AMD_PACKED_KERNELS_H */
