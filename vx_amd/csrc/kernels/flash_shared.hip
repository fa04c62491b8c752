/*
 * flash_shared.hip -- attention over a prefix that all sequences share and
 * each sequence's own cache (vx_nn_flash_attention_shared_bf16).
 *
 * A wave per query: a lane scores one key of a block of 64, the block's
 * maximum and sum move the running ones, and each lane adds the block's
 * weighted values of its columns.
 */
#include "../vx_batch_kernels.h"
#include "../vx_hip_common.h"
#include "vx_wave_ops.hip.h"

#include <cmath>

namespace vxk {
namespace {

template <int kD> __global__ __launch_bounds__(64) void flash_shared_simple(SharedAttnArgs a) {
  constexpr int kCols = kD / 64;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x; /* of [batch, heads, seq_q] */
  const int i = (int)(row % a.seq_q);
  const int h = (int)(row / a.seq_q % a.heads);
  const int64_t b = row / a.seq_q / a.heads;
  const int len = a.lens ? a.lens[b] : a.capacity;
  if (len < 0 || len > a.capacity) {
    return;
  }
  const int kv = h / (a.heads / a.kv_heads);
  const int total = a.shared_len + len;
  const int end = a.causal ? min(total, total - a.seq_q + i + 1) : total;
  __shared__ float q[kD], p[64];
  for (int c = lane; c < kD; c += 64) {
    q[c] = bf16_to_f32(a.q[row * kD + c]);
  }
  __syncthreads();
  auto at = [&](const uint16_t *shared, const uint16_t *own, int key) {
    return key < a.shared_len
               ? shared + ((int64_t)kv * a.shared_capacity + key) * kD
               : own + ((b * a.kv_heads + kv) * a.capacity + key - a.shared_len) * kD;
  };
  float m = -INFINITY, l = 0.0f, o[kCols] = {};
  for (int k0 = 0; k0 < end; k0 += 64) {
    float s = -INFINITY;
    if (k0 + lane < end) {
      const uint16_t *k = at(a.k_shared, a.k, k0 + lane);
      s = 0.0f;
      for (int c = 0; c < kD; ++c) {
        s += q[c] * bf16_to_f32(k[c]);
      }
      s *= a.scale;
    }
    const float m_next = fmaxf(m, wave_max(s));
    const float base = m_next == -INFINITY ? 0.0f : m_next;
    const float w = expf(s - base);
    const float back = expf(m - base);
    m = m_next;
    l = l * back + wave_sum(w);
    p[lane] = w;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      o[j] *= back;
    }
    for (int key = k0; key < min(k0 + 64, end); ++key) {
      const uint16_t *v = at(a.v_shared, a.v, key);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        o[j] += p[key - k0] * bf16_to_f32(v[lane + 64 * j]);
      }
    }
    __syncthreads();
  }
  const float inv = end > 0 ? 1.0f / l : 0.0f;
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    a.o[row * kD + lane + 64 * j] = f32_to_bf16(o[j] * inv);
  }
  if (a.lse && lane == 0) {
    a.lse[row] = end > 0 ? m + logf(l) : -INFINITY;
  }
}

} // namespace

void flash_shared_launch(const SharedAttnArgs &a, int head_dim, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.heads * a.seq_q));
  if (head_dim == 128) {
    hipLaunchKernelGGL((flash_shared_simple<128>), grid, dim3(64), 0, stream, a);
  } else {
    hipLaunchKernelGGL((flash_shared_simple<64>), grid, dim3(64), 0, stream, a);
  }
  VX_HIP_CHECK(hipGetLastError());
}

} // namespace vxk
