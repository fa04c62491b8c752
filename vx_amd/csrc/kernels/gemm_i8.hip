/*
 * gemm_i8.hip -- products of int8 activations and int8 weights
 * (vx_nn_gemm_i8_*): y[t, r] = (sum_c x[t, c] w[r, c]) x_scale[t] w_scale[r].
 *
 * The sum is an int32 on v_mfma_i32_16x16x64_i8, exact for up to 131056 columns,
 * so a result does not depend on how the columns are divided. Both operands
 * have their columns together, so an MFMA operand is 16 bytes of a row: lane l
 * holds row l % 16, columns 16 (l / 16) .. + 15 of a stage of 64. The weights are
 * the first operand, so that a lane ends with 4 consecutive outputs of a token.
 */
#include "../vx_hip_common.h"
#include "../vx_packed_kernels.h"
#include "gemm_pp_layout.h"
#include "vx_lds_dma.hip.h"

#include <type_traits>

namespace vxk {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kStage = 64; /* columns of an MFMA */

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                               __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

/* Four outputs of token `t` from row `r` on. */
template <bool kF32>
__device__ __forceinline__ void put4(const GemmI8Args &a, int64_t t, int64_t r, i32x4 sum, float xs,
                                     f32x4 ws, bool vec) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = (float)sum[e] * xs * ws[e];
  }
  const int64_t at = t * a.stride + r;
  if constexpr (kF32) {
    float *y = static_cast<float *>(a.y) + at;
    if (vec) {
      *reinterpret_cast<f32x4 *>(y) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (r + e < a.rows) {
          y[e] = v[e];
        }
      }
    }
  } else {
    u32x2 h;
    h[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2));
    h[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2));
    uint16_t *y = static_cast<uint16_t *>(a.y) + at;
    if (vec) {
      *reinterpret_cast<u32x2 *>(y) = h;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (r + e < a.rows) {
          y[e] = (uint16_t)(h[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

/* Four outputs at once: their rows are all there, and the address allows it. */
template <bool kF32> __device__ __forceinline__ bool aligned_rows(const GemmI8Args &a) {
  return (a.stride & 3) == 0 && ((uintptr_t)a.y & (kF32 ? 15 : 7)) == 0;
}

__device__ __forceinline__ f32x4 scales4(const float *s, int64_t r, int64_t rows) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = s[min(r + e, rows - 1)];
  }
  return v;
}

__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0));
}

/* Up to 64 tokens: a workgroup has 16 rows of w and all tokens, its waves take
 * the stages in turn, each from memory into registers, and meet in LDS. */
constexpr uint32_t kPast = 0x7ffffff0u; /* an offset past any buffer's end: reads zeros */

template <bool kF32, int kTT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void gemm_i8_few(GemmI8Args a) {
  constexpr int kAhead = 4; /* stages whose loads are in flight together */
  __shared__ i32x4 part[kWaves][kTT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int64_t r0 = (int64_t)blockIdx.x * 16;
  const int cols = a.cols;
  const int rows_here = (int)min((int64_t)16, a.rows - r0);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t *>(a.w) + r0 * cols, (short)0, rows_here * cols, 0x00020000);
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t *>(a.x), (short)0, (int)a.tokens * cols, 0x00020000);
  i32x4 acc[kTT];
#pragma unroll
  for (int i = 0; i < kTT; ++i) {
    acc[i] = i32x4{0, 0, 0, 0};
  }
  const int stages = (cols + kStage - 1) / kStage;
  for (int s0 = wave; s0 < stages; s0 += kWaves * kAhead) {
    u32x4 wv[kAhead], xv[kAhead][kTT];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = (s0 + i * kWaves) * kStage + 16 * g;
      const bool in = c < cols;
      wv[i] = load16(wr, in ? (uint32_t)(l16 * cols + c) : kPast);
#pragma unroll
      for (int j = 0; j < kTT; ++j) {
        xv[i][j] = load16(xr, in ? (uint32_t)((16 * j + l16) * cols + c) : kPast);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int j = 0; j < kTT; ++j) {
        acc[j] = mfma_i8(wv[i], xv[i][j], acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kTT; ++j) {
    part[wave][j][lane] = acc[j];
  }
  __syncthreads();
  const bool aligned = aligned_rows<kF32>(a);
  for (int j = wave; j < kTT; j += kWaves) {
    i32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      sum += part[i][j][lane];
    }
    const int64_t t = 16 * j + l16, r = r0 + 4 * g;
    if (t < a.tokens && r < a.rows) {
      put4<kF32>(a, t, r, sum, a.x_scale[t], scales4(a.w_scale, r, a.rows), aligned && r + 4 <= a.rows);
    }
  }
}

/* Tiles of 128 tokens x 128 rows: four waves of 64x64, two workgroups to a CU,
 * stages of 64 columns through an LDS ring of five slots filled by
 * buffer-to-LDS loads. Planes are [128 rows][4 chunks of 16 columns], a chunk's
 * place XORed with the row's bits as in the 16-bit kernels. */
constexpr int kBM = 128, kBN = 128, kTM = 4, kTN = 4, kNS = 5;
constexpr int kUnitsA = kBM * 4, kUnitsB = kBN * 4;

template <bool kF32>
__global__ __launch_bounds__(256, 2) void gemm_i8_tiles(GemmI8Args a, int tiles_m, int tiles_n) {
  constexpr int kLA = kUnitsA / 256, kLB = kUnitsB / 256;
  __shared__ u32x4 ring[kNS][kUnitsA + kUnitsB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  const pp::Tile tile = pp::tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n);
  const int64_t m0 = (int64_t)tile.tm * kBM;
  const int64_t n0 = (int64_t)tile.tn * kBN;
  const int cols = a.cols;
  const int stages = (cols + kStage - 1) / kStage;
  const bool ragged = cols % kStage != 0;

  /* Rows past the end read zeros; columns past the end of a row belong to the
   * next one, and are left out on x's side. */
  uint32_t a_off[kLA], b_off[kLB];
  bool a_in[kLA]; /* in the last stage */
#pragma unroll
  for (int p = 0; p < kLA; ++p) {
    const int u = (wave * kLA + p) * 64 + lane;
    const int row = u >> 2, c = pp::dswz_a(row, u & 3) * 16;
    a_off[p] = (uint32_t)(row * cols + c);
    a_in[p] = (stages - 1) * kStage + c < cols;
  }
#pragma unroll
  for (int p = 0; p < kLB; ++p) {
    const int u = (wave * kLB + p) * 64 + lane;
    const int row = u >> 2;
    b_off[p] = (uint32_t)(row * cols + pp::dswz_a(row, u & 3) * 16);
  }
  const int a_end = (int)min((int64_t)kBM, a.tokens - m0) * cols;
  const int b_end = (int)min((int64_t)kBN, a.rows - n0) * cols;
  const uint32_t ring_base = (uint32_t)(uintptr_t)(VX_LDS void *)&ring[0][0];
  auto issue = [&](int st, int slot) {
    const int c0 = st * kStage;
    const i32x4 ra = buffer_rsrc(a.x + m0 * cols + c0, a_end - c0);
    const i32x4 rb = buffer_rsrc(a.w + n0 * cols + c0, b_end - c0);
    const uint32_t base = ring_base + (uint32_t)(slot * (kUnitsA + kUnitsB) * 16);
    const bool cut = ragged && st == stages - 1;
#pragma unroll
    for (int p = 0; p < kLA; ++p) {
      dma16(ra, cut && !a_in[p] ? kPast : a_off[p], base + (uint32_t)((wave * kLA + p) * 1024));
    }
#pragma unroll
    for (int p = 0; p < kLB; ++p) {
      dma16(rb, b_off[p], base + (uint32_t)(kUnitsA * 16 + (wave * kLB + p) * 1024));
    }
  };

  struct Frags {
    u32x4 a[kTM], b[kTN];
  };
  auto read = [&](int slot, Frags &f) {
    const u32x4 *la = ring[slot], *lb = la + kUnitsA;
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
      const int row = (wn * kTN + j) * 16 + l16;
      f.b[j] = lb[row * 4 + pp::dswz_a(row, g)];
    }
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      const int row = (wm * kTM + i) * 16 + l16;
      f.a[i] = la[row * 4 + pp::dswz_a(row, g)];
    }
  };
  i32x4 acc[kTM][kTN];
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
      acc[i][j] = i32x4{0, 0, 0, 0};
    }
  }
  auto multiply = [&](const Frags &f) {
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
#pragma unroll
      for (int i0 = 0; i0 < kTM; ++i0) {
        const int i = (j & 1) ? kTM - 1 - i0 : i0;
        acc[i][j] = mfma_i8(f.b[j], f.a[i], acc[i][j]);
      }
    }
  };

#pragma unroll
  for (int s = 0; s < kNS; ++s) {
    if (s < stages) {
      issue(s, s);
    }
  }
  wait_stages<kNS - 1, kLA + kLB>(min(stages, kNS) - 1);
  lds_barrier();
  Frags f0, f1;
  read(0, f0);
  /* Entering stage s: its operands are in `f`, and every wave's reads of them
   * end before the barrier, after which its slot takes stage s + kNS. The
   * next stage's reads run beside this one's MFMAs. */
  int slot = 0;
  auto stage = [&](int s, const Frags &f, Frags &next) {
    wait_stages<kNS - 2, kLA + kLB>(min(stages - 2 - s, kNS - 2));
    lds_barrier();
    if (s + kNS < stages) {
      issue(s + kNS, slot);
    }
    slot = slot == kNS - 1 ? 0 : slot + 1;
    read(slot, next);
    multiply(f);
  };
  int s = 0;
  for (; s + 2 < stages; s += 2) {
    stage(s, f0, f1);
    stage(s + 1, f1, f0);
  }
  if (s + 1 < stages) {
    stage(s, f0, f1);
    multiply(f1);
  } else {
    multiply(f0);
  }

  const bool aligned = aligned_rows<kF32>(a);
#pragma unroll
  for (int j = 0; j < kTN; ++j) {
    const int64_t r = n0 + (wn * kTN + j) * 16 + 4 * g;
    if (r >= a.rows) {
      continue;
    }
    const f32x4 ws = scales4(a.w_scale, r, a.rows);
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
      const int64_t t = m0 + (wm * kTM + i) * 16 + l16;
      if (t < a.tokens) {
        put4<kF32>(a, t, r, acc[i][j], a.x_scale[t], ws, aligned && r + 4 <= a.rows);
      }
    }
  }
}

template <bool kF32, int kTT> void few(const GemmI8Args &a, int waves, hipStream_t stream) {
  const dim3 grid((unsigned)((a.rows + 15) / 16));
  if (waves == 4) {
    hipLaunchKernelGGL((gemm_i8_few<kF32, kTT, 4>), grid, dim3(256), 0, stream, a);
  } else if (waves == 8) {
    hipLaunchKernelGGL((gemm_i8_few<kF32, kTT, 8>), grid, dim3(512), 0, stream, a);
  } else {
    hipLaunchKernelGGL((gemm_i8_few<kF32, kTT, 16>), grid, dim3(1024), 0, stream, a);
  }
}

template <bool kF32> void launch(const GemmI8Args &a, const GemmI8Plan &p, hipStream_t stream) {
  if (p.kind == GemmI8Plan::kFew) {
    if (a.tokens <= 16) {
      few<kF32, 1>(a, p.waves, stream);
    } else if (a.tokens <= 32) {
      few<kF32, 2>(a, p.waves, stream);
    } else {
      few<kF32, 4>(a, p.waves, stream);
    }
    return;
  }
  const int tm = (int)((a.tokens + kBM - 1) / kBM), tn = (int)((a.rows + kBN - 1) / kBN);
  hipLaunchKernelGGL((gemm_i8_tiles<kF32>), dim3((unsigned)(tm * tn)), dim3(256), 0, stream, a, tm, tn);
}

} // namespace

void gemm_i8_launch(const GemmI8Args &a, const GemmI8Plan &plan, char *, hipStream_t stream) {
  a.f32 ? launch<true>(a, plan, stream) : launch<false>(a, plan, stream);
}

} // namespace vxk
