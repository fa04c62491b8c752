/*
 * vx_hip_ops.h -- library ops of the MI355X dispatch library that have no
 * `kind=` route, called from Vx through `extern "C"` blocks.
 *
 * The reference has no flash-attention op and no int8 GEMV
 * (packages/vx_nn/lib.vx:1 is a placeholder; packages/README.md:10-19), and
 * the compiler has no AMDGPU image pipeline, so these ops are exported by the
 * dispatch library and declared in Vx the way `std::collective` declares its
 * entry points (reference stdlib/std/collective.vx:14-29,
 * runtime/cuda_dispatch.cpp:2064-2123). A tensor cannot cross an `extern`
 * (E3022, reference docs/lang/abi.md section 2), so every op takes element
 * pointers plus extents. Pointers are HBM allocations from
 * vx_plugin_alloc_and_transfer on Topology::GPU[i]; the op runs on the device
 * that owns them, on the calling thread's stream (vx_cuda_set_stream), and
 * returns before the GPU finishes, like a routed GEMM.
 *
 * Each op returns 0 on success and a negative VX_OP_E* code (with a
 * `[Vx HIP]` line on stderr) for arguments it cannot take. A device fault is
 * fatal, as everywhere in the plugin ABI.
 *
 * bf16 and f16 elements travel as uint16_t bit patterns.
 */
#ifndef VX_HIP_OPS_H
#define VX_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  VX_OP_OK = 0,
  VX_OP_EINVAL = -1,   /* an extent, stride or argument is out of range */
  VX_OP_ENODEV = -2,   /* no GPU: this library has no host copy of the op */
  VX_OP_ENOTDEV = -3,  /* a pointer is not device memory */
  VX_OP_EUNSUPP = -4,  /* a shape the kernels do not take */
  VX_OP_ENOMEM = -5    /* host or device memory ran out */
};

/* Flash-attention forward (the op packages/vx_nn/lib.vx declares).
 *
 * q: [batch, heads, seq_q, head_dim] bf16; k, v: [batch, kv_heads, seq_k,
 * head_dim] bf16; o: like q; lse: [batch, heads, seq_q] f32 (may be NULL).
 * All dense row-major. Query head h reads kv head h / (heads / kv_heads).
 * o = softmax(scale * q k^T) v with f32 accumulation, o rounded to bf16 once;
 * lse = natural-log sum of exp of the scaled scores of each row. With
 * `causal`, query i sees key j iff j <= i + (seq_k - seq_q) (the queries are
 * the last seq_q positions). head_dim must be 64 or 128.
 *
 * A launch whose query blocks fill less than one round of the GPU (for
 * example 512 queries of 32 heads over a long cache) may cut the key range
 * into splits and merge them in f32 (same result to within f32 rounding
 * before the one bf16 rounding). The split partials live in HBM the
 * library keeps per (device, stream): at most 8 x batch x heads x seq_q x
 * (head_dim + 1) x 4 bytes, taken in the stream's order. A stream's block
 * is freed, in its order, when the calling thread's stream is set to
 * another one (so set another stream, or NULL, before destroying one); the
 * default stream's block stays until the process ends. A stream that is
 * capturing a graph gets the unsplit launch. */
int32_t vx_nn_flash_attention_fwd_bf16(const uint16_t *q, const uint16_t *k,
                                       const uint16_t *v, uint16_t *o,
                                       float *lse, int64_t batch, int64_t heads,
                                       int64_t kv_heads, int64_t seq_q,
                                       int64_t seq_k, int64_t head_dim,
                                       float scale, int32_t causal);

/* int8 weight-only GEMV / skinny GEMM.
 *
 * w: [rows, cols] int8 row-major; scale: [rows] f32; x: [batch, cols] bf16;
 * y: [batch, rows] f32. y[b, r] = scale[r] * sum_c w[r, c] * x[b, c], the sum
 * in f32. batch 1..16; cols a multiple of 16 and at most 2^24. */
int32_t vx_nn_gemv_i8_bf16(const int8_t *w, const float *scale,
                           const uint16_t *x, float *y, int64_t rows,
                           int64_t cols, int64_t batch);

/* ---- Many answers to one prompt ----------------------------------------
 *
 * A step of a batch of sequences that begin with the same prompt: the prompt's
 * keys and values are stored once, each sequence has a cache of its own for
 * what follows. vx_nn_rope_append_* turns a fused projection into rotated
 * queries and new cache rows, vx_nn_flash_attention_shared_bf16 attends over
 * the shared prefix and the own cache, and vx_nn_sample_* draws the next
 * tokens from the classifier's logits. No counterpart in the reference.
 *
 * lens (device memory, int32 [batch]) says how many rows of its own cache each
 * sequence has, the step's seq_q new ones among them: query i of sequence b is
 * at position shared_len + lens[b] - seq_q + i. It is read when the kernels
 * run, so a captured graph follows it. lens NULL: capacity for all. A slot
 * whose lens[b] is negative or above capacity holds no sequence: what it has
 * for queries and cache does not matter, and its outputs and cache stay as they
 * were.
 *
 * Arguments are checked before the GPU is looked for, so a refusal is the same
 * without one. Every pointer must be memory of one GPU; the ops run on that
 * GPU, whichever is current.
 *
 * `workspace`: GPU memory for partial results, 16-byte aligned, its contents
 * of no account before and after. The calls work with NULL: then the library
 * keeps a block of up to 128 MiB per (device, stream), taken and freed as
 * attention's split workspaces are. A call that needs more has it for itself, in
 * the stream's order, which costs it 25 us, or 0.4 ms where the GPU was waited for
 * before. A stream that is capturing a graph, or hipStreamPerThread, gets a launch
 * that needs none (slower: each sequence reads the shared keys itself, one
 * workgroup draws each row). A captured call that shall divide its
 * work is given one of at least *_workspace() bytes (a smaller one is refused),
 * which two launches that may run at the same time must not share. Sampling
 * uses at most 1024 x (45 KiB + 8.2 KiB per begun 32768 logits), attention 4 *
 * (head_dim + 2) bytes a query of a head for each part of the keys (of each
 * part up to 8 more). */

/* Splits, rotates and appends. qkv: [batch, seq_q, heads + 2 * kv_heads,
 * head_dim] (a token's queries, keys and values together, as one projection
 * leaves them), bf16 or f32. rope: [rope_len, head_dim / 2, 2] f32 of (cos,
 * sin), at least shared_len + capacity rows; NULL: no rotation. q: [batch,
 * heads, seq_q, head_dim] bf16; k_cache, v_cache: [batch, kv_heads, capacity,
 * head_dim] bf16.
 * With at = lens[b] - seq_q + i, the query and key of token i turn by row
 * shared_len + at of the table, pairs (2 j, 2 j + 1), in f32, rounded to bf16
 * once; q gets the query, row `at` of the caches the key and value. A token
 * whose `at` is below 0 belongs to the shared prefix: its query is turned
 * alike (zeros if it lies before the prefix's begin), its key and value are
 * not stored. head_dim a multiple of 8, at most 512; pointers 16-byte
 * aligned; outputs must not overlap qkv. */
int32_t vx_nn_rope_append_bf16(const uint16_t *qkv, const float *rope,
                               const int32_t *lens, uint16_t *q,
                               uint16_t *k_cache, uint16_t *v_cache,
                               int64_t batch, int64_t seq_q, int64_t heads,
                               int64_t kv_heads, int64_t head_dim,
                               int64_t shared_len, int64_t capacity,
                               int64_t rope_len);
int32_t vx_nn_rope_append_f32(const float *qkv, const float *rope,
                              const int32_t *lens, uint16_t *q,
                              uint16_t *k_cache, uint16_t *v_cache,
                              int64_t batch, int64_t seq_q, int64_t heads,
                              int64_t kv_heads, int64_t head_dim,
                              int64_t shared_len, int64_t capacity,
                              int64_t rope_len);

/* Attention over a shared prefix and own caches: what
 * vx_nn_flash_attention_fwd_bf16 computes for each sequence over the shared
 * keys followed by its own, with the shared keys read for many sequences at
 * once.
 * q: [batch, heads, seq_q, head_dim] bf16; k_shared, v_shared: the first
 * shared_len rows of [kv_heads, shared_capacity, head_dim] bf16; k, v:
 * [batch, kv_heads, capacity, head_dim] bf16, of which lens[b] rows count
 * (what the others hold is never looked at); o: like q; lse: [batch, heads,
 * seq_q] f32 (may be NULL). With `causal`, query i of sequence b sees key j
 * of shared ++ own iff j <= shared_len + lens[b] - seq_q + i; else all
 * shared_len + lens[b]. The softmax weights are rounded to bf16 for their product
 * with v, as in vx_nn_flash_attention_fwd_bf16; scores, maxima and sums are f32 (o
 * is off by 2.3e-3 of its size in the root mean square, where the rounding of o
 * itself makes 1.7e-3). A key that a query does not see does not reach its
 * result, whatever its values; a query that sees none gets o = 0 and lse =
 * -inf. k_shared and v_shared may be NULL where shared_len is 0, k and v
 * where capacity is 0. head_dim 64 or 128; pointers 16-byte aligned; scale and
 * scale * log2(e) finite. */
int32_t vx_nn_flash_attention_shared_bf16(
    const uint16_t *q, const uint16_t *k_shared, const uint16_t *v_shared,
    const uint16_t *k, const uint16_t *v, const int32_t *lens, uint16_t *o,
    float *lse, int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q,
    int64_t shared_len, int64_t shared_capacity, int64_t capacity,
    int64_t head_dim, float scale, int32_t causal, void *workspace,
    int64_t workspace_bytes);
/* Bytes of workspace that such a call uses (0: none); a negative VX_OP_E*
 * code for extents it does not take. */
int64_t vx_nn_flash_attention_shared_workspace(int64_t batch, int64_t heads,
                                               int64_t kv_heads, int64_t seq_q,
                                               int64_t shared_len,
                                               int64_t capacity,
                                               int64_t head_dim);

/* Next tokens from logits: temperature, top-k, top-p, min-p and one given
 * uniform number a row.
 * logits: [rows, vocab] f32 or bf16, rows `stride` elements apart (at least
 * vocab); u: [rows] f32 in [0, 1); tokens: [rows] int32; logprob: [rows] f32
 * (may be NULL). The settings are arrays of a value per row, each of which may
 * be NULL: temperature (1), top_k (off), top_p (off), min_p (off).
 * With t = logit / temperature and w = exp(t - max t), tokens go in the order
 * of falling logits, the lower index first among equals. Of that order the
 * first token stays, and of the others those that every setting keeps:
 *   top_k: the first top_k (0 or less: all);
 *   top_p: those before which, of the tokens that top_k keeps, lies less than
 *     top_p of their weight (1 or more, or NaN: all);
 *   min_p: those with w >= min_p (0 or less, or NaN: all).
 * The row's token is the lowest index i of a kept token at which the sum of
 * the kept weights up to i exceeds u times their sum; logprob is the natural
 * logarithm of its share of that sum. temperature 0, negative or NaN: the
 * first token of the order. u outside [0, 1) counts as the nearest number
 * inside, NaN as 0.
 * A NaN logit counts as -inf, and what is -inf is never drawn; where a logit
 * is +inf, those are the only ones, with equal weights. A row without a logit
 * above -inf gets token -1 and logprob -inf.
 * Weights are 64-bit integers in units of at most 2^-32 of the row's largest
 * one (2^-45 at a vocabulary of 131072), so sums are exact and a result does
 * not depend on how the work is divided; a token whose weight rounds to 0 is
 * not drawn. rows at most 2^21, vocab at most 2^30. */
int32_t vx_nn_sample_f32(const float *logits, const float *temperature,
                         const int32_t *top_k, const float *top_p,
                         const float *min_p, const float *u, int32_t *tokens,
                         float *logprob, int64_t rows, int64_t vocab,
                         int64_t stride, void *workspace,
                         int64_t workspace_bytes);
int32_t vx_nn_sample_bf16(const uint16_t *logits, const float *temperature,
                          const int32_t *top_k, const float *top_p,
                          const float *min_p, const float *u, int32_t *tokens,
                          float *logprob, int64_t rows, int64_t vocab,
                          int64_t stride, void *workspace,
                          int64_t workspace_bytes);
/* Bytes of workspace that such a call uses (0: none); VX_OP_EINVAL for
 * extents it does not take. */
int64_t vx_nn_sample_workspace(int64_t rows, int64_t vocab);

/* ---- A packed batch in 8 bits --------------------------------------------
 *
 * Texts of different lengths in one run, their tokens one behind the other
 * without padding, and activations in 8 bits against int8 weights: the norm (or
 * plain quantization) that makes them, the product that reads them, attention
 * that keeps the texts apart, and what the classifier's logits say of given
 * tokens. vx_nn_rope_append_* turns a packed projection's heads as one sequence
 * whose table has a row a token. No counterpart in the reference.
 *
 * Arguments, devices and `workspace` as for many answers to one prompt above
 * (log probabilities use at most 132 KiB, the product 64 KiB a CU, 16 MiB on 256).
 * Outputs must not overlap inputs but where it is said. */

/* The residual's addition and RMS norm of rows: s = x + residual, y = s *
 * (mean s^2 + eps)^-1/2 * weight, the mean in 64 bits.
 * x: [rows, dim], rows `stride` elements apart; residual: [rows, dim] (NULL: 0);
 * weight: [dim] f32 (NULL: 1). Outputs, each of which may be NULL, one of y and
 * q not: sum: [rows, dim], s rounded to x's type (the norm is of s itself); y:
 * [rows, dim] bf16; q: [rows, dim] int8 with q_scale: [rows] f32, y in 8 bits: with
 * t = s * weight in f32 and u = max |t| / 127 (1 where that is 0), q = t / u rounded
 * to the nearest, half to even, and q_scale = u * (mean s^2 + eps)^-1/2.
 * A row in which a t is not finite gets q = 0 and q_scale = NaN. sum may be x
 * (where stride is dim) or residual itself. dim at most 32768, rows 2^21. */
int32_t vx_nn_rms_norm_bf16(const uint16_t *x, const uint16_t *residual,
                            const float *weight, uint16_t *sum, uint16_t *y,
                            int8_t *q, float *q_scale, int64_t rows,
                            int64_t dim, int64_t stride, float eps);
int32_t vx_nn_rms_norm_f32(const float *x, const float *residual,
                           const float *weight, float *sum, uint16_t *y,
                           int8_t *q, float *q_scale, int64_t rows, int64_t dim,
                           int64_t stride, float eps);

/* Rows in 8 bits: q = x / u rounded to the nearest, half to even, q_scale = u =
 * max |x| / 127 of the row (1 where that is 0). As above otherwise. */
int32_t vx_nn_quantize_i8_bf16(const uint16_t *x, int8_t *q, float *q_scale,
                               int64_t rows, int64_t dim, int64_t stride);
int32_t vx_nn_quantize_i8_f32(const float *x, int8_t *q, float *q_scale,
                              int64_t rows, int64_t dim, int64_t stride);

/* int8 activations times int8 weights: y[t, r] = x_scale[t] * w_scale[r] *
 * sum_c x[t, c] * w[r, c].
 * x: [tokens, cols] int8; x_scale: [tokens] f32; w: [rows, cols] int8; w_scale:
 * [rows] f32 (the weights of vx_nn_gemv_i8_bf16); y: [tokens, rows], rows
 * `stride` elements apart (at least `rows`), bf16 or f32. The sum is exact; it
 * is rounded to f32, multiplied by x_scale, then by w_scale, in f32, and rounded
 * to y's type. cols a multiple of 16, at most 131056; x and w 16-byte aligned;
 * tokens and rows at most 2^24, and at most 2^22 tiles of 64 x 64 outputs. */
int32_t vx_nn_gemm_i8_bf16(const int8_t *x, const float *x_scale,
                           const int8_t *w, const float *w_scale, uint16_t *y,
                           int64_t tokens, int64_t rows, int64_t cols,
                           int64_t stride, void *workspace,
                           int64_t workspace_bytes);
int32_t vx_nn_gemm_i8_f32(const int8_t *x, const float *x_scale,
                          const int8_t *w, const float *w_scale, float *y,
                          int64_t tokens, int64_t rows, int64_t cols,
                          int64_t stride, void *workspace,
                          int64_t workspace_bytes);
/* Bytes of workspace that such a call uses (0: none); a negative VX_OP_E* code
 * for extents it does not take. */
int64_t vx_nn_gemm_i8_workspace(int64_t tokens, int64_t rows, int64_t cols);

/* Attention of packed sequences, each over its own keys.
 * q, o: `total` rows of `heads` heads of head_dim bf16; k, v: the same of
 * kv_heads heads. Row i of head h lies i * q_row + h * q_head elements from q
 * (o_row and o_head from o, kv_row and kv_head from k and v alike): [heads,
 * total, head_dim] as well as slices of a projection [total, heads + 2 *
 * kv_heads, head_dim]. offsets (device memory, int32 [sequences + 1], read when
 * the kernels run): sequence s has rows offsets[s] .. offsets[s + 1] - 1, none
 * where those are equal. Rows before the first and from the last offset on
 * belong to no sequence: they are not read, and their outputs stay as they
 * were. offsets must not fall; where they do or lie outside 0 .. total, nothing
 * outside the tensors is read or written, but which outputs are is not said.
 * lse: [heads, total] f32 (may be NULL), natural logarithm.
 * With `causal`, a query sees its sequence's keys up to its own row; else all.
 * Numerics (the weights' rounding to bf16 among them: o is off by 1.8e-3 to
 * 2.0e-3 of its size, where the rounding of o itself makes 1.5e-3 to 1.6e-3),
 * `scale` and what hidden keys may hold as in
 * vx_nn_flash_attention_shared_bf16. head_dim 64 or 128; strides multiples of
 * 8, at least head_dim; kv_row at most 2^22; pointers 16-byte aligned; at most
 * 65536 sequences, 2^22 sequences * kv_heads and 2^28 queries of all heads. */
int32_t vx_nn_flash_attention_packed_bf16(
    const uint16_t *q, const uint16_t *k, const uint16_t *v,
    const int32_t *offsets, uint16_t *o, float *lse, int64_t total,
    int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
    int64_t q_row, int64_t q_head, int64_t kv_row, int64_t kv_head,
    int64_t o_row, int64_t o_head, float scale, int32_t causal);

/* Log probabilities of given tokens, entropy, and the likeliest tokens of each
 * row of logits, of p = softmax(logits), natural logarithms.
 * logits: [rows, vocab] f32 or bf16, rows `stride` elements apart (at least
 * vocab); given: [rows, n_given] int32, logprob: [rows, n_given] f32 (a token
 * outside 0 .. vocab - 1 gets -inf); entropy: [rows] f32 (may be NULL), -sum p
 * ln p; top_tokens: [rows, n_top] int32, the tokens of the n_top largest logits,
 * falling, the lower index first among equals, and top_logprob: [rows, n_top]
 * f32 (may be NULL).
 * A NaN logit counts as -inf, and what is -inf is no alternative: where fewer
 * are left, the rest are token -1 with logprob -inf. Where a logit is +inf,
 * those alone have a probability, the same for each; the alternatives keep
 * their order. A row without a logit above -inf has logprob -inf and entropy 0.
 * n_top 0..64, n_given 0..2^20, rows at most 2^21, vocab at most 2^30. */
int32_t vx_nn_token_logprobs_f32(const float *logits, const int32_t *given,
                                 float *logprob, float *entropy,
                                 int32_t *top_tokens, float *top_logprob,
                                 int64_t rows, int64_t vocab, int64_t stride,
                                 int64_t n_given, int64_t n_top,
                                 void *workspace, int64_t workspace_bytes);
int32_t vx_nn_token_logprobs_bf16(const uint16_t *logits, const int32_t *given,
                                  float *logprob, float *entropy,
                                  int32_t *top_tokens, float *top_logprob,
                                  int64_t rows, int64_t vocab, int64_t stride,
                                  int64_t n_given, int64_t n_top,
                                  void *workspace, int64_t workspace_bytes);
/* Bytes of workspace that such a call uses (0: none); VX_OP_EINVAL for extents
 * it does not take. */
int64_t vx_nn_token_logprobs_workspace(int64_t rows, int64_t vocab,
                                       int64_t n_top);

/* Greedy int8 decode of a Llama-2-style model, resident in HBM.
 *
 * The token step of reference examples/llama.vx:173-420 (RMSNorm eps 1e-5,
 * Q/K/V, RoPE, KV cache, causal attention, Wo, SwiGLU FFN, residuals, final
 * RMSNorm, classifier sharing the embedding table, argmax with the lowest
 * index winning a tie) as GPU library ops: every linear is an int8
 * weight-only GEMV with per-row f32 scales; activations and everything else
 * are f32, as in the reference. The position and the next token stay on the GPU,
 * so a whole step is replayable as one hipGraph with no host round trip.
 *
 * Weights are host pointers in llama2.c order, matrices [out][in]:
 * tok [vocab, dim] (embedding and classifier); per layer wq [dim, dim],
 * wk/wv [kv_dim, dim], wo [dim, dim], w1/w3 [hidden, dim], w2 [dim, hidden],
 * each with one f32 scale per row; RMSNorm weights f32; `rope` the
 * [seq_len, head_size / 2] table of (cos, sin) of the rotary angles. */
typedef struct vx_llama_i8_config {
  int32_t dim, hidden_dim, n_layers, n_heads, n_kv_heads, vocab_size, seq_len;
} vx_llama_i8_config;

typedef struct vx_llama_i8_weights {
  const int8_t *tok_q;
  const float *tok_s;
  const float *rms_att; /* [layers, dim] */
  const int8_t *wq_q;
  const float *wq_s;
  const int8_t *wk_q;
  const float *wk_s;
  const int8_t *wv_q;
  const float *wv_s;
  const int8_t *wo_q;
  const float *wo_s;
  const float *rms_ffn; /* [layers, dim] */
  const int8_t *w1_q;
  const float *w1_s;
  const int8_t *w2_q;
  const float *w2_s;
  const int8_t *w3_q;
  const float *w3_s;
  const float *rms_final; /* [dim] */
  const float *rope;      /* [seq_len, head_size / 2, 2] */
} vx_llama_i8_weights;

/* Capture the token step as hipGraphs (8 steps, and 1 for the remainder;
 * one pair for positions whose attention takes the small rounds, one for
 * the rest) and replay them (else: stream launches, one by one). */
#define VX_LLAMA_GRAPH 1

/* Upload a model to GPU[topology_id - 500]; NULL (and a [Vx HIP] line) when
 * the config is not one the kernels take or there is no GPU. */
void *vx_llama_i8_create(const vx_llama_i8_config *cfg,
                         const vx_llama_i8_weights *w, uint32_t topology_id);

/* Feed prompt[0..n_prompt), then generate n_steps tokens greedily into
 * out_tokens; out_margin (may be NULL) gets each generated token's logit
 * lead over the runner-up. Returns 0, or a VX_OP_E* code. */
int32_t vx_llama_i8_generate(void *model, const int32_t *prompt,
                             int32_t n_prompt, int32_t n_steps,
                             int32_t *out_tokens, float *out_margin,
                             int32_t flags);

/* The same with tokens drawn as vx_nn_sample_f32 draws them, by the given
 * settings (values that turn a setting off: temperature 1, top_k 0, top_p 1,
 * min_p 0; temperature 0 is greedy) and u[i] for the i-th generated token.
 * out_logprob (may be NULL) gets the natural logarithm of each token's share of
 * the kept weight; where every logit is NaN the token is -1 and generation goes
 * on from token 0. */
typedef struct vx_llama_sampling {
  float temperature;
  int32_t top_k;
  float top_p, min_p;
} vx_llama_sampling;
int32_t vx_llama_i8_sample(void *model, const int32_t *prompt, int32_t n_prompt,
                           int32_t n_steps, const vx_llama_sampling *how,
                           const float *u, int32_t *out_tokens,
                           float *out_logprob, int32_t flags);

/* Feed tokens[0..n) at positions 0..n-1 and copy the logits after each
 * position to logits[n, vocab]. Returns 0 or a VX_OP_E* code. */
int32_t vx_llama_i8_logits(void *model, const int32_t *tokens, int32_t n,
                           float *logits);

void vx_llama_i8_destroy(void *model);

/* ---- Model files (host side; no GPU needed) ----
 *
 * Two formats are read:
 *  - a llama2.c checkpoint, the file reference examples/llama.vx loads
 *    (stdlib/rust_core/src/ffi/llama.rs:10-45 reads it: seven int32 --
 *    dim, hidden_dim, n_layers, n_heads, n_kv_heads, vocab_size, seq_len --
 *    then the f32 arrays in the order of examples/llama.vx:80-120; the
 *    RoPE arrays llama2.c appends after rms_final may be present or not).
 *    Every matrix is quantized per output row on the way in (scale =
 *    max|w| / 127, q = round-half-even(w / scale));
 *  - the int8 file vx_llama_i8_save writes ("VXQ8" version 1: the config,
 *    then every array of vx_llama_i8_weights in field order, then a 64-bit
 *    FNV-1a of everything before it), so the quantization is done once.
 * Either way the RoPE table is computed from the config (base 10000), the
 * classifier is the token table (a negative vocab_size -- an unshared
 * classifier -- is refused), and the result feeds vx_llama_i8_create. */
typedef struct vx_llama_i8_host vx_llama_i8_host;

/* Read `path`; on VX_OP_OK, *cfg holds the config and *out the weights
 * (free with vx_llama_i8_host_free). VX_OP_EINVAL for an unreadable,
 * truncated or corrupt file, VX_OP_EUNSUPP for a layout this build does
 * not take. */
int32_t vx_llama_i8_read(const char *path, vx_llama_i8_config *cfg,
                         vx_llama_i8_host **out);
/* The weights of a read model, valid until vx_llama_i8_host_free. */
const vx_llama_i8_weights *vx_llama_i8_host_weights(const vx_llama_i8_host *h);
void vx_llama_i8_host_free(vx_llama_i8_host *h);
/* Write cfg and w as a "VXQ8" file. */
int32_t vx_llama_i8_save(const char *path, const vx_llama_i8_config *cfg,
                         const vx_llama_i8_weights *w);

/* ---- device images in the payload ------------------------------------
 *
 * vx_plugin_dispatch_async runs a region whose payload says `format=hsaco`
 * from the gfx950 code object in the payload's binary section (a bare ELF or
 * a clang offload bundle): one parameter per memref field (allocated,
 * aligned, offset, sizes, strides) and per scalar, as the reference's PTX
 * path marshals them (runtime/vx_kernel_launch.h:57-140); the launch shape
 * from `grid=`/`block=`/`grid_loops=` or `launch=`; `assert_flag=1` appends
 * a pointer to a cleared device int that a failed assert sets; `shared=`
 * bytes of dynamic LDS; `coop=1` launches cooperatively. Before the first
 * launch the count below is compared with what the arguments produce.
 *
 * How many of its own parameters (not the hidden ones the runtime appends)
 * `kernel` declares in the gfx950 code object `image`, read from the code
 * object's metadata; -1 when the image, its metadata or the kernel is
 * absent. Replaces, for AMDGPU images, the reference's
 * vx_launch_entry_param_count (runtime/vx_kernel_launch.h:206-222, PTX) and
 * vx_launch_entry_param_count_spirv (:248-315). */
int32_t vx_hip_image_param_count(const void *image, size_t image_size,
                                 const char *kernel);

/* ---- a routed GEMM that allocates nothing -----------------------------
 *
 * No counterpart in the reference. For callers that cannot allocate device
 * memory (tight serving loops, harnesses that forbid hipMalloc): the
 * kind=matmul dispatch of vx_plugin_dispatch_async, with the same payload,
 * arguments and result, except that host operands and a host result buffer
 * are staged through a fixed 16 MiB array per GPU (in this library's code
 * object) instead of the staging pool. Launches that divide a tile's K
 * between workgroups need a workspace (16-bit products of few rows, of grids
 * short of the CUs or ending in a partial round of 256x256 tiles, and f32 ones
 * of 2^30 multiply-adds and more on few tiles): such a product runs here
 * undivided, on the kernel that is the fastest then, as into a captured graph
 * and under hipStreamPerThread. The results agree with
 * vx_plugin_dispatch_async's to 1e-5 relative (one unit of a 16-bit output),
 * not bit for bit. Returns 1 when the GEMM was issued,
 * 0 (reason on stderr, nothing launched) for a region that is not a routed
 * GEMM, a result published through a slot (host memory the program frees),
 * staging beyond 16 MiB, or staging while the caller stream is capturing a
 * graph. Operands already in GPU memory need no staging. Calls on one GPU
 * share its array and take turns on it: a call that stages waits, in its
 * stream's order, for the GEMM of the previous such call (on any stream or
 * thread) before it overwrites the array. */
uint64_t vx_hip_dispatch_async_noalloc(const void *binary_payload,
                                       size_t payload_size, void **device_args,
                                       const int32_t *arg_tags,
                                       int64_t num_args);

#ifdef __cplusplus
}
#endif

#endif /* VX_HIP_OPS_H */
