/*
 * rms_norm.hip -- the residual's addition, RMS norm and quantization of rows
 * (vx_nn_rms_norm_*, vx_nn_quantize_i8_*).
 *
 * s = x + residual, r = (mean s^2 + eps)^-1/2, y = s r w, and in 8 bits q =
 * rint(t / u) of t = s w with u = max|t| / 127, q_scale = u r: r cancels in q, so
 * q does not depend on the order of the squares' sum. The sum is taken in 64
 * bits: squares of any f32 fit.
 *
 * A workgroup has a row in registers, so that each element is read once and
 * written once; two reductions over LDS at once (the sum and the largest |t|).
 * 4096 x 4096 in bf16 with a residual, to 8 bits, 25.0 us, 4.7 TB/s, and in f32 49.4,
 * 4.4 TB/s (218 MB): bound by HBM.
 */
#include "../vx_hip_common.h"
#include "../vx_packed_kernels.h"
#include "vx_wave_ops.hip.h"

#include <type_traits>

namespace vxk {
namespace {

typedef uint32_t u32;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int kO> __device__ __forceinline__ void meet(double &sum, u32 &top) {
  const uint64_t b = __builtin_bit_cast(uint64_t, sum);
  const uint64_t o = (uint64_t)partner_word<kO>((u32)(b >> 32)) << 32 | partner_word<kO>((u32)b);
  sum += __builtin_bit_cast(double, o);
  top = max(top, partner_word<kO>(top));
}

__device__ __forceinline__ u32 bf16_pair(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

/* Inputs that do not stay in the L2 caches (kPast) are read past them: 4096 x 4096
 * with a residual, 67 MB in, 25.0 us, and 27.8 through them; 777 x 11008, 17 MB, 9.3
 * and 8.9. */
constexpr int64_t kCaches = (int64_t)32 << 20;

/* kVec: 8 elements from (j * kThreads + thread) * 8 on, by vector loads; else
 * element (j * 8 + e) * kThreads + thread. */
template <bool kF32, bool kVec, bool kPast, int kThreads, int kUnits>
__global__ __launch_bounds__(kThreads) void rms_norm(NormArgs a) {
  constexpr int kWaves = kThreads / 64;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  auto at = [&](int j, int e) { return kVec ? (j * kThreads + t) * 8 + e : (j * 8 + e) * kThreads + t; };
  auto vector = [&](auto *src) { return kPast ? __builtin_nontemporal_load(src) : *src; };
  auto load = [&](const void *p, int64_t base, int j, float (&v)[8]) {
    if constexpr (kVec) {
      const bool in = at(j, 0) < a.dim;
      if constexpr (kF32) {
        const f32x4 *src = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + base + at(j, 0));
        const f32x4 lo = in ? vector(src) : f32x4{0, 0, 0, 0}, hi = in ? vector(src + 1) : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = lo[e];
          v[4 + e] = hi[e];
        }
      } else {
        const u32x4 w = in ? vector(reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + base + at(j, 0)))
                           : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[2 * e] = __uint_as_float(w[e] << 16);
          v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = at(j, e);
        v[e] = 0.0f;
        if (i < a.dim) {
          v[e] = kF32 ? static_cast<const float *>(p)[base + i]
                      : bf16_to_f32(static_cast<const uint16_t *>(p)[base + i]);
        }
      }
    }
  };

  /* read again where they are used: from the caches, they cost no registers */
  auto weights = [&](int j, float (&v)[8]) {
    if (!a.weight) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = 1.0f;
      }
    } else if constexpr (kVec) {
      const bool in = at(j, 0) < a.dim;
      const f32x4 *src = reinterpret_cast<const f32x4 *>(a.weight + at(j, 0));
      const f32x4 lo = in ? src[0] : f32x4{0, 0, 0, 0}, hi = in ? src[1] : f32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = lo[e];
        v[4 + e] = hi[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = at(j, e) < a.dim ? a.weight[at(j, e)] : 0.0f;
      }
    }
  };

  float s[kUnits][8];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    load(a.x, row * a.stride, j, s[j]);
  }
  if (a.residual) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      float r[8];
      load(a.residual, row * a.dim, j, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[j][e] += r[e];
      }
    }
  }
  if (a.sum) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      if constexpr (kVec) {
        if (at(j, 0) < a.dim) {
          const int64_t to = row * a.dim + at(j, 0);
          if constexpr (kF32) {
            f32x4 *dst = reinterpret_cast<f32x4 *>(static_cast<float *>(a.sum) + to);
            dst[0] = f32x4{s[j][0], s[j][1], s[j][2], s[j][3]};
            dst[1] = f32x4{s[j][4], s[j][5], s[j][6], s[j][7]};
          } else {
            *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.sum) + to) =
                u32x4{bf16_pair(s[j][0], s[j][1]), bf16_pair(s[j][2], s[j][3]),
                      bf16_pair(s[j][4], s[j][5]), bf16_pair(s[j][6], s[j][7])};
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = at(j, e);
          if (i < a.dim) {
            if constexpr (kF32) {
              static_cast<float *>(a.sum)[row * a.dim + i] = s[j][e];
            } else {
              static_cast<uint16_t *>(a.sum)[row * a.dim + i] = f32_to_bf16(s[j][e]);
            }
          }
        }
      }
    }
  }

  /* Bits of |t| order as the values do, a NaN above all. */
  double sum = 0.0;
  u32 top = 0;
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    float w[8];
    weights(j, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (a.norm) {
        sum = fma((double)s[j][e], (double)s[j][e], sum);
      }
      top = max(top, __float_as_uint(s[j][e] * w[e]) & 0x7fffffffu);
    }
  }
  meet<32>(sum, top);
  meet<16>(sum, top);
  meet<8>(sum, top);
  meet<4>(sum, top);
  meet<2>(sum, top);
  meet<1>(sum, top);
  if constexpr (kWaves > 1) {
    __shared__ double sums[kWaves];
    __shared__ u32 tops[kWaves];
    if ((t & 63) == 0) {
      sums[t >> 6] = sum;
      tops[t >> 6] = top;
    }
    __syncthreads();
    sum = 0.0;
    top = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      sum += sums[i];
      top = max(top, tops[i]);
    }
  }

  /* r as a fraction and a power of two: it may lie outside the range of f32 */
  const double root = a.norm ? 1.0 / sqrt(sum / a.dim + (double)a.eps) : 1.0;
  int power;
  const float r = (float)frexp(root, &power);
  if (a.y) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      float y[8];
      weights(j, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] *= ldexpf(s[j][e], power) * r;
      }
      if constexpr (kVec) {
        if (at(j, 0) < a.dim) {
          *reinterpret_cast<u32x4 *>(a.y + row * a.dim + at(j, 0)) =
              u32x4{bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3]), bf16_pair(y[4], y[5]),
                    bf16_pair(y[6], y[7])};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (at(j, e) < a.dim) {
            a.y[row * a.dim + at(j, e)] = f32_to_bf16(y[e]);
          }
        }
      }
    }
  }
  if (!a.q) {
    return;
  }
  /* A row with an infinity or a NaN: zeros of scale NaN. */
  const bool finite = top < 0x7f800000u;
  float unit = __uint_as_float(top) / 127.0f;
  unit = unit > 0.0f ? unit : 1.0f;
  if (t == 0) {
    a.q_scale[row] = finite ? (float)(unit * root) : NAN;
  }
  /* t / unit by the reciprocal is within 1.5 * 2^-23 of its size (127), 2.3e-5, of
   * the rounded quotient: where it is further than that from a half, both round
   * alike; the few others are divided. Reciprocals of units near the smallest f32 are
   * infinite: those rows divide throughout. Adding 1.5 * 2^23 rounds to the
   * nearest, half to even, and leaves the integer in the low bits. */
  constexpr float kRound = 12582912.0f;
  const float inv = 1.0f / unit;
  const float far = unit > 1e-30f ? 0.49997f : -1.0f;
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    float v[8], n[8];
    weights(j, v);
    float off = 0.0f; /* the furthest from an integer */
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= s[j][e];
      const float f = v[e] * inv;
      n[e] = f + kRound;
      off = fmaxf(off, fabsf(f - (n[e] - kRound)));
    }
    if (off > far) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[e] = fminf(fmaxf(rintf(v[e] / unit), -127.0f), 127.0f) + kRound;
      }
    }
    if (!finite) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[e] = kRound;
      }
    }
    if constexpr (kVec) {
      u32 four[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32 two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          two[i] = __builtin_amdgcn_perm(__float_as_uint(n[4 * h + 2 * i + 1]),
                                         __float_as_uint(n[4 * h + 2 * i]), 0x0c0c0400u);
        }
        four[h] = two[0] | two[1] << 16;
      }
      if (at(j, 0) < a.dim) {
        *reinterpret_cast<u32x2 *>(a.q + row * a.dim + at(j, 0)) = u32x2{four[0], four[1]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (at(j, e) < a.dim) {
          a.q[row * a.dim + at(j, e)] = (int8_t)(__float_as_uint(n[e]) & 0xff);
        }
      }
    }
  }
}

template <bool kF32, bool kVec, bool kPast, int kThreads, int kUnits>
void launch_row(const NormArgs &a, hipStream_t stream) {
  hipLaunchKernelGGL((rms_norm<kF32, kVec, kPast, kThreads, kUnits>), dim3((unsigned)a.rows),
                     dim3(kThreads), 0, stream, a);
}

/* As few threads as hold a row in two units: 777 x 11008 in 8 bits 9.3 us in 768
 * threads, 10.4 in 1024 or in 256 of six units, 9.6 in 512 of three; 4096 x 4096
 * 28.1 in 256, 29.1 in 512 of one unit, 29.8 in 128 of four. */
template <bool kF32, bool kVec, bool kPast> void launch(const NormArgs &a, hipStream_t stream) {
  if (a.dim <= 512) {
    launch_row<kF32, kVec, kPast, 64, 1>(a, stream);
  } else if (a.dim <= 1024) {
    launch_row<kF32, kVec, kPast, 128, 1>(a, stream);
  } else if (a.dim <= 2048) {
    launch_row<kF32, kVec, kPast, 256, 1>(a, stream);
  } else if (a.dim <= 4096) {
    launch_row<kF32, kVec, kPast, 256, 2>(a, stream);
  } else if (a.dim <= 8192) {
    launch_row<kF32, kVec, kPast, 512, 2>(a, stream);
  } else if (a.dim <= 12288) {
    launch_row<kF32, kVec, kPast, 768, 2>(a, stream);
  } else if (a.dim <= 16384) {
    launch_row<kF32, kVec, kPast, 1024, 2>(a, stream);
  } else {
    launch_row<kF32, kVec, kPast, 1024, 4>(a, stream);
  }
}

} // namespace

void rms_norm_launch(const NormArgs &a, hipStream_t stream) {
  auto on16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.dim % 8 == 0 && a.stride % 8 == 0 && on16(a.x) && on16(a.residual) &&
                   on16(a.weight) && on16(a.sum) && on16(a.y) &&
                   (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
  const int64_t in = a.rows * a.dim * (a.f32 ? 4 : 2) * (a.residual ? 2 : 1);
  auto with = [&](auto f32) {
    constexpr bool kF32 = decltype(f32)::value;
    if (!vec) {
      launch<kF32, false, false>(a, stream);
    } else if (in > kCaches) {
      launch<kF32, true, true>(a, stream);
    } else {
      launch<kF32, true, false>(a, stream);
    }
  };
  a.f32 ? with(std::true_type{}) : with(std::false_type{});
}

} // namespace vxk
