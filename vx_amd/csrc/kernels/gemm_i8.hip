/*
 * gemm_i8.hip -- products of int8 activations and int8 weights
 * (vx_nn_gemm_i8_*): y[t, r] = (sum_c x[t, c] w[r, c]) x_scale[t] w_scale[r].
 *
 * The sum is an int32 on v_mfma_i32_16x16x64_i8, exact for up to 131056 columns,
 * so a result does not depend on how the columns are divided. Both operands
 * have their columns together, so an MFMA operand is 16 bytes of a row: lane l
 * holds row l % 16, columns 16 (l / 16) .. + 15 of a stage of 64. The weights are
 * the first operand, so that a lane ends with 4 consecutive outputs of a token.
 *
 * Three kernels by the number of tokens (gemm_i8.h has the rules): one, few, and
 * tiles. A tile's stage is 128 columns, since loads that take 64 of a row fetch
 * each cache line in two turns (4096 x 11008 x 4096 266 us, whole lines and tiles
 * of 256 x 256 163-168). That shape is 2.2-2.3 POP/s, of 8192^3 2.4-2.7: there MFMAs
 * are busy 59% of the cycles, at a clock that the power limit holds at 1.75-1.93 GHz;
 * no LDS conflicts. 777 x 6144 x 4096 takes 27: 224 tiles of 128 x 192, one round in
 * which 32 CUs have none and a seventh of the last tile row is empty. 48 x 11008 x
 * 4096, 172 workgroups that read 45 MB, takes 10.4 where the last-level cache holds
 * the weights and 13.9 from HBM.
 */
#include "../vx_hip_common.h"
#include "../vx_packed_kernels.h"
#include "gemm_pp_layout.h"
#include "vx_lds_dma.hip.h"
#include "vx_wave_ops.hip.h"

#include <type_traits>

namespace vxk {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                               __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x2 bf16x4_of(f32x4 v) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2)),
               __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2))};
}

/* Element `at` of `to` from that of `from`, of kEsz bytes. */
template <int kEsz> __device__ __forceinline__ void put_bits(char *to, int at, const char *from) {
  if constexpr (kEsz == 4) {
    reinterpret_cast<uint32_t *>(to)[at] = reinterpret_cast<const uint32_t *>(from)[at];
  } else {
    reinterpret_cast<uint16_t *>(to)[at] = reinterpret_cast<const uint16_t *>(from)[at];
  }
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
    const u32x2 h = bf16x4_of(f32x4{v[0], v[1], v[2], v[3]});
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

/* One token: a wave has 4 rows of w, whose bytes it reads 1 KiB at a time of
 * each, and adds up the products of its columns on v_dot4. With kSplit the four
 * waves of a workgroup have the same rows and take the pieces in turn. Bound by HBM:
 * 32000 x 768 6.2 us (4.0 TB/s), 11008 x 4096 8.9 (5.1 TB/s), and where the last-level
 * cache holds the weights 4.9 and 7.1. Of 2 rows 6.7 and 8.7, of 8 6.5 and 9.4. */
constexpr int kRowsEach = 4;

template <bool kF32, bool kSplit>
__global__ __launch_bounds__(256) void gemm_i8_row(GemmI8Args a) {
  constexpr int kPiece = 1024;
  constexpr int kAhead = 2; /* pieces whose loads are in flight together */
  __shared__ int part[kSplit ? 4 : 1][kRowsEach];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r0 = ((int64_t)blockIdx.x * (kSplit ? 1 : 4) + (kSplit ? 0 : wave)) * kRowsEach;
  if (r0 >= a.rows) {
    return; /* (not with kSplit) */
  }
  const int cols = a.cols;
  const int rows_here = (int)min((int64_t)kRowsEach, a.rows - r0);
  int acc[kRowsEach] = {};
  constexpr int kStep = kSplit ? 4 : 1;
  const int pieces = (cols + kPiece - 1) / kPiece;
  for (int p0 = kSplit ? wave : 0; p0 < pieces; p0 += kStep * kAhead) {
    u32x4 w[kAhead][kRowsEach], x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = (p0 + i * kStep) * kPiece + 16 * lane;
      const bool in = c < cols;
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r) {
        w[i][r] = u32x4{0, 0, 0, 0};
        if (in) {
          w[i][r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
              a.w + (r0 + min(r, rows_here - 1)) * cols + c));
        }
      }
      x[i] = u32x4{0, 0, 0, 0};
      if (in) {
        x[i] = *reinterpret_cast<const u32x4 *>(a.x + c);
      }
    }
    __builtin_amdgcn_sched_barrier(0); /* all loads before the first product */
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r) {
        for (int e = 0; e < 4; ++e) {
          acc[r] = __builtin_amdgcn_sdot4((int)w[i][r][e], (int)x[i][e], acc[r], false);
        }
      }
    }
  }
  /* lane r stores row r's output */
  int mine = 0;
#pragma unroll
  for (int r = 0; r < kRowsEach; ++r) {
    const int sum = wave_sum_int(acc[r]);
    mine = lane == r ? sum : mine;
  }
  if constexpr (kSplit) {
    if (lane < kRowsEach) {
      part[wave][lane] = mine;
    }
    __syncthreads();
    if (wave != 0 || lane >= kRowsEach) {
      return;
    }
    mine = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  }
  if (lane < rows_here) {
    const float v = (float)mine * a.x_scale[0] * a.w_scale[r0 + lane];
    if constexpr (kF32) {
      static_cast<float *>(a.y)[r0 + lane] = v;
    } else {
      static_cast<uint16_t *>(a.y)[r0 + lane] = f32_to_bf16(v);
    }
  }
}

/* Few tokens: a workgroup has 16 rows of w and all tokens, its waves take lines
 * of 128 columns in turn, kAhead at once, from memory into registers, and meet in
 * LDS. 8 waves: 16 tokens x 32000 x 768 8.3 us, and 8.8 in 4, 12.7 in 16. 16 x 11008
 * x 4096 14.0, 3.2 TB/s of weights, and as many bytes of x through the caches. */
constexpr int kFewWaves = 8;
constexpr uint32_t kPast = 0x7ffffff0u; /* an offset past any buffer's end: reads zeros */
using i8::kLine;

template <bool kF32, int kTT, int kAhead>
__global__ __launch_bounds__(64 * kFewWaves) void gemm_i8_few(GemmI8Args a) {
  constexpr int kWaves = kFewWaves;
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
  const int lines = (cols + kLine - 1) / kLine;
  for (int s0 = wave; s0 < lines; s0 += kWaves * kAhead) {
    u32x4 wv[kAhead][2], xv[kAhead][2][kTT];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = (s0 + i * kWaves) * kLine + 64 * h + 16 * g;
        const bool in = c < cols;
        wv[i][h] = load16(wr, in ? (uint32_t)(l16 * cols + c) : kPast);
#pragma unroll
        for (int j = 0; j < kTT; ++j) {
          xv[i][h][j] = load16(xr, in ? (uint32_t)((16 * j + l16) * cols + c) : kPast);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0); /* all loads before the first product */
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < kTT; ++j) {
          acc[j] = mfma_i8(wv[i][h], xv[i][h][j], acc[j]);
        }
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

/* A wave's kTM x kTN blocks of outputs from token t0 and row r0 on, 16 tokens at
 * a time through LDS (`mine`, the wave's own), so that a store has whole lines of a
 * token's row: 16 lanes with 4 rows each, as the products leave them, would store
 * 32 bytes of each (4096 x 32000 x 768 in bf16 208 us, and 144-149 this way: six
 * stages a tile, and one workgroup a CU, whose stores nothing overlaps). */
template <bool kF32, int kTM, int kTN>
__device__ __forceinline__ void store_blocks(const GemmI8Args &a, const i32x4 (&acc)[kTM][kTN],
                                             int64_t t0, int64_t r0, char *mine) {
  constexpr int kEsz = kF32 ? 4 : 2;
  constexpr int kRows = 16 * kTN, kPitch = kRows * kEsz + 16;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint32_t at = (uint32_t)(a.stride * kEsz) | (uint32_t)(uintptr_t)a.y; /* alignment */
  f32x4 ws[kTN];
#pragma unroll
  for (int j = 0; j < kTN; ++j) {
    ws[j] = scales4(a.w_scale, min(r0 + 16 * j + 4 * g, a.rows - 1), a.rows);
  }
  const int rows_here = (int)min((int64_t)kRows, a.rows - r0);
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
    const int64_t t = t0 + 16 * i;
    const float xs = a.x_scale[min(t + l16, a.tokens - 1)];
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = (float)acc[i][j][e] * xs * ws[j][e];
      }
      char *to = mine + l16 * kPitch + (16 * j + 4 * g) * kEsz;
      if constexpr (kF32) {
        *reinterpret_cast<f32x4 *>(to) = v;
      } else {
        *reinterpret_cast<u32x2 *>(to) = bf16x4_of(v);
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int tokens_here = (int)min((int64_t)16, a.tokens - t);
    auto pieces = [&](auto bytes) {
      constexpr int kBytes = decltype(bytes)::value;
      typedef uint32_t piece __attribute__((ext_vector_type(kBytes < 4 ? 1 : kBytes / 4)));
      constexpr int kEach = kBytes / kEsz, kChunks = kRows / kEach;
#pragma unroll 4
      for (int u = lane; u < 16 * kChunks; u += 64) {
        const int row = u / kChunks, c = u % kChunks * kEach;
        const char *from = mine + row * kPitch + c * kEsz;
        char *to = static_cast<char *>(a.y) + ((t + row) * a.stride + r0 + c) * kEsz;
        if (row >= tokens_here) {
        } else if (kEach > 1 && c + kEach <= rows_here) {
          *reinterpret_cast<piece *>(to) = *reinterpret_cast<const piece *>(from);
        } else {
          for (int e = 0; e < kEach && c + e < rows_here; ++e) {
            put_bits<kEsz>(to, e, from);
          }
        }
      }
    };
    if ((at & 15) == 0) {
      pieces(std::integral_constant<int, 16>{});
    } else if (kEsz == 2 && (at & 7) == 0) {
      pieces(std::integral_constant<int, 8>{});
    } else {
      pieces(std::integral_constant<int, kEsz>{});
    }
    __builtin_amdgcn_wave_barrier();
  }
}

/* Tiles of kBM tokens x kBN rows on kWM x kWN waves: stages of 128 columns (a
 * whole cache line of each row) through an LDS ring of kNS slots filled by
 * buffer-to-LDS loads. Planes are [rows][8 chunks of 16 columns], chunk c of a row
 * at place c ^ (row % 8), so that reads of 16 rows at one chunk meet every bank.
 * With kMid a slot's plane of w is filled again from the middle of its stage on,
 * when all of it is in registers. With kSplits several workgroups may divide a tile's
 * stages, whose sums gemm_i8_join adds up. */
template <bool kF32, int kBM, int kBN, int kWM, int kWN, int kNS, bool kMid, int kPerCu, bool kSplits>
__global__ __launch_bounds__(64 * kWM * kWN, kPerCu * kWM * kWN / 4) void gemm_i8_tiles(
    GemmI8Args a, int tiles_m, int tiles_n, int splits, i32x4 *__restrict__ parts) {
  constexpr int kThreads = 64 * kWM * kWN;
  constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16; /* 16x16 blocks of a wave */
  constexpr int kUnitsA = kBM * 8, kUnitsB = kBN * 8;       /* 16-byte units per stage */
  constexpr int kLA = kUnitsA / kThreads, kLB = kUnitsB / kThreads;
  constexpr int kLead = 2;        /* steps that A's reads run ahead */
  constexpr int kSteps = 2 * kTM; /* of kTN products, a stage's */
  static_assert(kUnitsA % kThreads == 0 && kUnitsB % kThreads == 0 && kLead <= kTM, "whole loads");
  __shared__ u32x4 ring[kNS][kUnitsA + kUnitsB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int wm = wave / kWN, wn = wave % kWN;
  const int tiles = tiles_m * tiles_n;
  const int split = kSplits ? (int)blockIdx.x / tiles : 0;
  const int id = (int)blockIdx.x - split * tiles;
  const pp::Tile tile = pp::tile_of(id, tiles, tiles_m, tiles_n);
  const int64_t m0 = (int64_t)tile.tm * kBM;
  const int64_t n0 = (int64_t)tile.tn * kBN;
  /* this workgroup's stages */
  const int all = (a.cols + kLine - 1) / kLine;
  const int first = kSplits ? (int)((int64_t)all * split / splits) : 0;
  const int stages = kSplits ? (int)((int64_t)all * (split + 1) / splits) - first : all;
  const int cols = a.cols;

  /* Load p of a wave fills rows (wave * kLA + p) * 8 + lane / 8 of a plane; its
   * offset is that of p = 0 and 8 p rows. Rows past the end read zeros; columns
   * past the end of a row belong to the next one, and are left out on x's side. */
  const int at_chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  const uint32_t a_off = (uint32_t)((wave * kLA * 8 + (lane >> 3)) * cols + at_chunk);
  const uint32_t b_off = (uint32_t)((wave * kLB * 8 + (lane >> 3)) * cols + at_chunk);
  const bool cut = (all - 1) * kLine + at_chunk >= cols; /* in the row's last stage */
  const int a_end = (int)min((int64_t)kBM, a.tokens - m0) * cols;
  const int b_end = (int)min((int64_t)kBN, a.rows - n0) * cols;
  const uint32_t ring_base = (uint32_t)(uintptr_t)(VX_LDS void *)&ring[0][0];
  auto issue_a = [&](int st, int slot) {
    const int c0 = (first + st) * kLine;
    const i32x4 rs = buffer_rsrc(a.x + m0 * cols + c0, a_end - c0);
    const uint32_t to = ring_base + (uint32_t)(slot * (kUnitsA + kUnitsB) * 16 + wave * kLA * 1024);
    const bool last = first + st == all - 1;
#pragma unroll
    for (int p = 0; p < kLA; ++p) {
      dma16(rs, cut && last ? kPast : a_off + (uint32_t)(8 * p * cols), to + (uint32_t)(p * 1024));
    }
  };
  auto issue_b = [&](int st, int slot) {
    const int c0 = (first + st) * kLine;
    const i32x4 rs = buffer_rsrc(a.w + n0 * cols + c0, b_end - c0);
    const uint32_t to =
        ring_base + (uint32_t)((slot * (kUnitsA + kUnitsB) + kUnitsA) * 16 + wave * kLB * 1024);
#pragma unroll
    for (int p = 0; p < kLB; ++p) {
      dma16(rs, b_off + (uint32_t)(8 * p * cols), to + (uint32_t)(p * 1024));
    }
  };

  /* Blocks are 16 rows apart, so that their chunks' places are the same. */
  const int at0 = l16 * 8 + (g ^ (l16 & 7)), at1 = l16 * 8 + ((4 + g) ^ (l16 & 7));
  auto read_a = [&](int slot, int ks, int i) {
    return ring[slot][(wm * kTM + i) * 128 + (ks ? at1 : at0)];
  };
  auto read_b = [&](int slot, int ks, int j) {
    return ring[slot][kUnitsA + (wn * kTN + j) * 128 + (ks ? at1 : at0)];
  };
  i32x4 acc[kTM][kTN];
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
      acc[i][j] = i32x4{0, 0, 0, 0};
    }
  }

#pragma unroll
  for (int s = 0; s < kNS; ++s) {
    if (s < stages) {
      issue_a(s, s);
      issue_b(s, s);
    }
  }
  wait_stages<kNS - 1, kLA + kLB>(min(stages, kNS) - 1);
  lds_barrier();
  u32x4 b0[kTN], b1[kTN], av[kLead];
#pragma unroll
  for (int j = 0; j < kTN; ++j) {
    b0[j] = read_b(0, 0, j);
  }
#pragma unroll
  for (int i = 0; i < kLead; ++i) {
    av[i] = read_a(0, 0, i);
  }
  /* Entering stage s, its first B operands are in b0 and its first A operands in
   * av. kLead steps before its end every wave has read all of it: the next stage's
   * loads are waited for, and past the barrier its first operands are read and the
   * slot takes stage s + kNS. (kMid: its plane of w was read by the middle.) */
  int slot = 0;
  for (int s = 0; s < stages; ++s) {
    const int after = slot == kNS - 1 ? 0 : slot + 1;
    const bool more = s + kNS < stages;
#pragma unroll
    for (int r = 0; r < kSteps; ++r) {
      const int ks = r / kTM, i = r % kTM;
      __builtin_amdgcn_sched_barrier(0);
      if (kMid && r == kTM) {
        lds_barrier();
        if (more) {
          issue_b(s + kNS, slot);
        }
      }
      if (r == kSteps - kLead) {
        if constexpr (kMid) {
          /* newer than stage s + 1: whole stages, and the plane just issued */
          if (more) {
            wait_vm<(kNS - 2) * (kLA + kLB) + kLB>();
          } else {
            wait_stages<kNS - 2, kLA + kLB>(min(stages - 2 - s, kNS - 2));
          }
        } else {
          wait_stages<kNS - 2, kLA + kLB>(min(stages - 2 - s, kNS - 2));
        }
        lds_barrier();
        if (more) {
          issue_a(s + kNS, slot);
          if (!kMid) {
            issue_b(s + kNS, slot);
          }
        }
      }
      const int n = r + kLead; /* the step that this one's read is for */
      const u32x4 an = n < kSteps ? read_a(slot, n / kTM, n % kTM) : read_a(after, 0, n - kSteps);
      if (ks == 0) {
        constexpr int kPer = (kTN + kTM - 1) / kTM;
#pragma unroll
        for (int j = i * kPer; j < min((i + 1) * kPer, kTN); ++j) {
          b1[j] = read_b(slot, 1, j);
        }
      } else if (r >= kSteps - kLead) {
        /* in place of those that this step's products no longer need */
        constexpr int kPer = (kTN + kLead - 1) / kLead;
        const int e = r - (kSteps - kLead);
#pragma unroll
        for (int j = e * kPer; j < min((e + 1) * kPer, kTN); ++j) {
          b0[j] = read_b(after, 0, j);
        }
      }
#pragma unroll
      for (int j0 = 0; j0 < kTN; ++j0) {
        const int j = (i & 1) ? kTN - 1 - j0 : j0;
        acc[i][j] = mfma_i8(ks ? b1[j] : b0[j], av[0], acc[i][j]);
      }
#pragma unroll
      for (int e = 0; e + 1 < kLead; ++e) {
        av[e] = av[e + 1];
      }
      av[kLead - 1] = an;
    }
    slot = after;
  }

  if (kSplits && splits > 1) {
    i32x4 *to = parts + ((int64_t)blockIdx.x * kTM * kTN) * kThreads + threadIdx.x;
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
#pragma unroll
      for (int j = 0; j < kTN; ++j) {
        to[(i * kTN + j) * kThreads] = acc[i][j];
      }
    }
    return;
  }
  lds_barrier(); /* the ring is free */
  store_blocks<kF32, kTM, kTN>(a, acc, m0 + wm * kTM * 16, n0 + wn * kTN * 16,
                               reinterpret_cast<char *>(&ring[0][0]) +
                                   wave * 16 * (16 * kTN * (kF32 ? 4 : 2) + 16));
}

/* The sums of a tile's splits, a thread a register of the kernel that left them. */
template <bool kF32, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(256) void gemm_i8_join(GemmI8Args a, int tiles_m, int tiles_n,
                                                    int splits, const i32x4 *__restrict__ parts) {
  constexpr int kThreads = 64 * kWM * kWN;
  constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16;
  constexpr int kPart = kTM * kTN * kThreads; /* of a tile */
  const int tiles = tiles_m * tiles_n;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int id = (int)(at / kPart), u = (int)(at % kPart);
  if (id >= tiles) {
    return;
  }
  const pp::Tile tile = pp::tile_of(id, tiles, tiles_m, tiles_n);
  const int block = u / kThreads, thread = u % kThreads;
  const int wave = thread >> 6, l16 = thread & 15, g = (thread & 63) >> 4;
  const int64_t r = (int64_t)tile.tn * kBN + (wave % kWN * kTN + block % kTN) * 16 + 4 * g;
  const int64_t t = (int64_t)tile.tm * kBM + (wave / kWN * kTM + block / kTN) * 16 + l16;
  if (r >= a.rows || t >= a.tokens) {
    return;
  }
  i32x4 sum = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s) {
    sum += parts[((int64_t)s * tiles + id) * kPart + u];
  }
  put4<kF32>(a, t, r, sum, a.x_scale[t], scales4(a.w_scale, r, a.rows),
             aligned_rows<kF32>(a) && r + 4 <= a.rows);
}

template <bool kF32> void row(const GemmI8Args &a, hipStream_t stream) {
  const unsigned groups = (unsigned)((a.rows + kRowsEach - 1) / kRowsEach);
  /* 11008 x 4096 12.7 us undivided, 8.9 divided; 16384 x 2048 7.2 and 7.7 */
  if (a.cols > 2048) {
    hipLaunchKernelGGL((gemm_i8_row<kF32, true>), dim3(groups), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((gemm_i8_row<kF32, false>), dim3((groups + 3) / 4), dim3(256), 0, stream, a);
  }
}

template <bool kF32, int kTT, int kAhead> void few_ahead(const GemmI8Args &a, hipStream_t stream) {
  hipLaunchKernelGGL((gemm_i8_few<kF32, kTT, kAhead>), dim3((unsigned)((a.rows + 15) / 16)),
                     dim3(64 * kFewWaves), 0, stream, a);
}
/* A wave's lines at once, 1 and 4: 16 tokens x 32000 x 1024 10.1 us and 16.5, 4096 x
 * 4096 7.2 and 6.7, 11008 x 4096 14.9 and 14.0; 24 x 4096 x 4096 7.7 and 8.0, 16000 x
 * 1024 7.7 and 11.9. */
template <bool kF32, int kTT> void few(const GemmI8Args &a, hipStream_t stream) {
  if (kTT == 1 && a.cols > kFewWaves * kLine) {
    few_ahead<kF32, kTT, kTT == 1 ? 4 : 1>(a, stream);
  } else {
    few_ahead<kF32, kTT, 1>(a, stream);
  }
}

template <bool kF32, int kBM, int kBN, int kWM, int kWN, int kNS, bool kMid, int kPerCu, bool kSplits>
void tiles(const GemmI8Args &a, int splits, char *ws, hipStream_t stream) {
  const int tm = (int)((a.tokens + kBM - 1) / kBM), tn = (int)((a.rows + kBN - 1) / kBN);
  hipLaunchKernelGGL((gemm_i8_tiles<kF32, kBM, kBN, kWM, kWN, kNS, kMid, kPerCu, kSplits>),
                     dim3((unsigned)(tm * tn * splits)), dim3(64 * kWM * kWN), 0, stream, a, tm, tn,
                     splits, reinterpret_cast<i32x4 *>(ws));
  if constexpr (kSplits) {
    if (splits > 1) {
      const int64_t all = (int64_t)tm * tn * (kBM * kBN / 4);
      hipLaunchKernelGGL((gemm_i8_join<kF32, kBM, kBN, kWM, kWN>), dim3((unsigned)((all + 255) / 256)),
                         dim3(256), 0, stream, a, tm, tn, splits, reinterpret_cast<const i32x4 *>(ws));
    }
  }
}

template <bool kF32>
void launch(const GemmI8Args &a, const GemmI8Plan &p, char *ws, hipStream_t stream) {
  if (p.kind == GemmI8Plan::kRow) {
    row<kF32>(a, stream);
  } else if (p.kind == GemmI8Plan::kFew) {
    a.tokens <= 16 ? few<kF32, 1>(a, stream) : few<kF32, 2>(a, stream);
  } else if (p.tile == 0) { /* i8::kSplitTiles of them may be split */
    tiles<kF32, 64, 64, 2, 2, 4, false, 2, true>(a, p.splits, ws, stream);
  } else if (p.tile == 1) {
    tiles<kF32, 128, 128, 4, 2, 4, false, 1, true>(a, p.splits, ws, stream);
  } else if (p.tile == 2) {
    tiles<kF32, 128, 128, 4, 2, 2, true, 2, false>(a, 1, nullptr, stream);
  } else if (p.tile == 3) {
    tiles<kF32, 128, 192, 4, 2, 3, false, 1, false>(a, 1, nullptr, stream);
  } else if (p.tile == 4) {
    tiles<kF32, 256, 128, 4, 2, 3, false, 1, false>(a, 1, nullptr, stream);
  } else {
    tiles<kF32, 256, 256, 4, 2, 2, true, 1, false>(a, 1, nullptr, stream);
  }
}

} // namespace

void gemm_i8_launch(const GemmI8Args &a, const GemmI8Plan &plan, char *ws, hipStream_t stream) {
  a.f32 ? launch<true>(a, plan, ws, stream) : launch<false>(a, plan, ws, stream);
}

} // namespace vxk
