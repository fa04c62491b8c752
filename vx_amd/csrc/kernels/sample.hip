/*
 * sample.hip -- next tokens from logits (vx_nn_sample_*): temperature, top-k,
 * top-p, min-p and one uniform number a row.
 *
 * With tokens in the order of falling logits (the lower index first among
 * equals), each setting keeps a first part of the order, so the kept tokens
 * are one: those whose logit is above a border, and the first few of those at
 * it. The draw then goes over the kept tokens by rising index and needs no
 * sort.
 *
 * Weights 2^((l - top) c), with c = log2(e) / T and top the largest logit, are
 * taken in 64 bits and kept as 64-bit integers of unit 2^-shift, so many that
 * a row's sum stays within 2^62. Integer sums do not
 * depend on their order: LDS atomics and any division of the row give the
 * same bits.
 *
 * sample_rows: a workgroup a row. A border is found digit by digit (11, 11 and
 * 10 bits) of the logits' order-preserving 32-bit keys, each digit by a
 * histogram of counts and weights over the row.
 */
#include "../vx_batch_kernels.h"
#include "../vx_hip_common.h"

#include <cmath>

namespace vxk {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

/* A row's logit in f32; -0 as +0. */
template <bool kF32> __device__ __forceinline__ float logit(const void *row, int i) {
  if constexpr (kF32) {
    return static_cast<const float *>(row)[i] + 0.0f;
  } else {
    return bf16_to_f32(static_cast<const uint16_t *>(row)[i]) + 0.0f;
  }
}

/* Rises with l; 0 for NaN and -inf, which are never drawn. */
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l);
  const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return l > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

/* 2^d for d <= 0 to 2^-52: 2^(d - k) = e^(ln2 (d - k)) by its Taylor sum to the
 * 12th power (the next term is below 2^-53 at |d - k| = 1/2), times 2^k. */
__device__ __forceinline__ double exp2_neg(double d) {
  d = fmax(d, -1000.0);
  const double k = rint(d);
  const double x = (d - k) * 0.69314718055994530942;
  double y = 1.0 / 479001600.0;
  y = fma(y, x, 1.0 / 39916800.0);
  y = fma(y, x, 1.0 / 3628800.0);
  y = fma(y, x, 1.0 / 362880.0);
  y = fma(y, x, 1.0 / 40320.0);
  y = fma(y, x, 1.0 / 5040.0);
  y = fma(y, x, 1.0 / 720.0);
  y = fma(y, x, 1.0 / 120.0);
  y = fma(y, x, 1.0 / 24.0);
  y = fma(y, x, 1.0 / 6.0);
  y = fma(y, x, 0.5);
  y = fma(y, x, 1.0);
  y = fma(y, x, 1.0);
  return ldexp(y, (int)k);
}

/* How a row's logits become weights. */
struct Scale {
  double c, top; /* 2^((l - top) c) */
  double unit; /* 2^shift */
  bool inf;    /* a logit is +inf: those alone */
};

__device__ __forceinline__ double ratio(const Scale &s, float l) {
  if (s.inf) {
    return l == INFINITY ? 1.0 : 0.0;
  }
  return l > -INFINITY ? exp2_neg(((double)l - s.top) * s.c) : 0.0;
}
__device__ __forceinline__ u64 weight(const Scale &s, float l) {
  return (u64)rint(ratio(s, l) * s.unit);
}

__device__ __forceinline__ u64 wave_max64(u64 v) {
  for (int o = 32; o; o >>= 1) {
    const u64 w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
  for (int o = 32; o; o >>= 1) {
    v += __shfl_xor(v, o);
  }
  return v;
}
/* Inclusive, over the wave's lanes up to this one. */
__device__ __forceinline__ u64 wave_scan64(u64 v) {
  const int lane = threadIdx.x & 63;
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(v, o);
    v += lane >= o ? w : 0;
  }
  return v;
}

/* floor(x total) and, with kUp, ceil(x total) of x in (0, 1), exactly: x is 24
 * bits times a power of two. A border that falls between two tokens (equal
 * logits, a half) falls on the side that the definition says. */
template <bool kUp> __device__ __forceinline__ u64 part_of(float x, u64 total) {
  const uint32_t b = __float_as_uint(x);
  const int e = (int)(b >> 23);
  const uint32_t m = (b & 0x7fffffu) | (e ? 0x800000u : 0u);
  const int down = e ? 150 - e : 149; /* 24 .. 149 */
  const unsigned __int128 p = (unsigned __int128)m * total;
  if (down >= 128) {
    return kUp && p ? 1 : 0;
  }
  const u64 q = (u64)(p >> down);
  return q + (kUp && ((unsigned __int128)q << down) != p ? 1 : 0);
}

/* The border of a setting: tokens of a key above `key` stay, and the first
 * `ties` of those that have it. */
struct Border {
  uint32_t key;
  u64 ties;
  u64 mass; /* of all that stay */
};

struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 wave[kWaves], wave2[kWaves];
  int bin;
  u64 above_mass, above_count, bin_mass, bin_count;
};

template <bool kF32, typename F>
__device__ __forceinline__ void each(const void *row, int vocab, F f) {
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    f(i, logit<kF32>(row, i));
  }
}

/* The border at the `want`-th token (kMass false) or the token whose weights
 * from the first on reach `want`. Every thread calls it and gets the same. */
template <bool kF32, bool kMass>
__device__ Border find_border(Shared &sh, const void *row, int vocab, const Scale &s, u64 want) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint32_t prefix = 0, mask = 0;
  u64 above_mass = 0, above_count = 0, mass = 0, count = 0;
  constexpr int kShift[3] = {21, 10, 0};
  for (int level = 0; level < 3; ++level) {
    const int shift = kShift[level];
    const uint32_t digits = level == 2 ? 1023 : 2047;
    for (int b = t; b < kBins; b += kThreads) {
      sh.mass[b] = 0;
      sh.count[b] = 0;
    }
    __syncthreads();
    each<kF32>(row, vocab, [&](int, float l) {
      const uint32_t k = key_of(l);
      if (k && (k & mask) == prefix) {
        const int b = (int)(k >> shift & digits);
        atomicAdd(&sh.mass[b], weight(s, l));
        atomicAdd(&sh.count[b], 1u);
      }
    });
    __syncthreads();
    /* From the highest digit down, two a thread. */
    const int hi = kBins - 1 - 2 * t;
    const u64 m0 = sh.mass[hi], m1 = sh.mass[hi - 1];
    const u64 c0 = sh.count[hi], c1 = sh.count[hi - 1];
    const u64 ms = wave_scan64(m0 + m1), cs = wave_scan64(c0 + c1);
    if (lane == 63) {
      sh.wave[wave] = ms;
      sh.wave2[wave] = cs;
    }
    __syncthreads();
    u64 mb = above_mass + ms - m0 - m1, cb = above_count + cs - c0 - c1;
    for (int w = 0; w < wave; ++w) {
      mb += sh.wave[w];
      cb += sh.wave2[w];
    }
    const u64 before = kMass ? mb : cb, own0 = kMass ? m0 : c0, own1 = kMass ? m1 : c1;
    if (before < want && want <= before + own0) {
      sh.bin = hi;
      sh.above_mass = mb;
      sh.above_count = cb;
      sh.bin_mass = m0;
      sh.bin_count = c0;
    } else if (before + own0 < want && want <= before + own0 + own1) {
      sh.bin = hi - 1;
      sh.above_mass = mb + m0;
      sh.above_count = cb + c0;
      sh.bin_mass = m1;
      sh.bin_count = c1;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.bin << shift;
    mask |= digits << shift;
    above_mass = sh.above_mass;
    above_count = sh.above_count;
    mass = sh.bin_mass;
    count = sh.bin_count;
    __syncthreads();
  }
  const u64 each_mass = mass / count; /* equal keys, equal weights */
  u64 ties = kMass ? (want - above_mass + each_mass - 1) / each_mass : want - above_count;
  ties = ties < count ? ties : count;
  return Border{prefix, ties, above_mass + ties * each_mass};
}

template <bool kF32> __global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a) {
  __shared__ Shared sh;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int r = blockIdx.x;
  const void *row = kF32 ? (const void *)(static_cast<const float *>(a.logits) + r * a.stride)
                         : (const void *)(static_cast<const uint16_t *>(a.logits) + r * a.stride);
  const float heat = a.temperature ? a.temperature[r] : 1.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f;
  const float min_p = a.min_p ? a.min_p[r] : 0.0f;

  /* The first token: the largest key, its lowest index. */
  u64 best = 0;
  each<kF32>(row, a.vocab, [&](int i, float l) {
    const uint32_t k = key_of(l);
    const u64 v = k ? (u64)k << 32 | (uint32_t)~i : 0;
    best = v > best ? v : best;
  });
  best = wave_max64(best);
  if (lane == 0) {
    sh.wave[wave] = best;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    best = sh.wave[w] > best ? sh.wave[w] : best;
  }
  __syncthreads();
  const bool first_alone = !(heat > 0.0f) || top_k == 1 || top_p <= 0.0f;
  if (!best || first_alone) {
    if (t == 0) {
      a.tokens[r] = best ? (int)~(uint32_t)best : -1;
      if (a.logprob) {
        a.logprob[r] = best ? 0.0f : -INFINITY;
      }
    }
    return;
  }

  const float top = logit_of((uint32_t)(best >> 32));
  Scale s;
  s.inf = top == INFINITY;
  s.c = 1.4426950408889634074 / (double)heat;
  s.top = (double)top;
  const int shift = 62 - (a.vocab > 1 ? 32 - __clz(a.vocab - 1) : 0);
  s.unit = ldexp(1.0, shift);

  Border border{0, ~0ull, 0};
  if (top_k > 0 && top_k < a.vocab) {
    /* as many as there are above -inf: all of them */
    u64 some = 0;
    each<kF32>(row, a.vocab, [&](int, float l) { some += l > -INFINITY; });
    some = wave_sum64(some);
    if (lane == 0) {
      sh.wave[wave] = some;
    }
    __syncthreads();
    some = 0;
    for (int w = 0; w < kWaves; ++w) {
      some += sh.wave[w];
    }
    __syncthreads();
    if ((u64)top_k < some) {
      border = find_border<kF32, false>(sh, row, a.vocab, s, (u64)top_k);
    }
  }
  if (top_p < 1.0f) {
    u64 mass = border.mass;
    if (!border.key) {
      each<kF32>(row, a.vocab, [&](int, float l) { mass += weight(s, l); });
      mass = wave_sum64(mass);
      if (lane == 0) {
        sh.wave[wave] = mass;
      }
      __syncthreads();
      mass = 0;
      for (int w = 0; w < kWaves; ++w) {
        mass += sh.wave[w];
      }
      __syncthreads();
    }
    const u64 want = part_of<true>(top_p, mass);
    border = find_border<kF32, true>(sh, row, a.vocab, s, want);
  }

  /* A wave's part of the row: its kept weight above the border, and its ties. */
  const double least = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
  auto stays = [&](float l, uint32_t k) { return k >= border.key && ratio(s, l) >= least; };
  const int per = ((a.vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int i0 = min(a.vocab, wave * per), i1 = min(a.vocab, i0 + per);
  u64 mass = 0, ties = 0;
  for (int i = i0 + lane; i < i1; i += 64) {
    const float l = logit<kF32>(row, i);
    const uint32_t k = key_of(l);
    if (k && stays(l, k)) {
      if (k == border.key) {
        ++ties;
      } else {
        mass += weight(s, l);
      }
    }
  }
  mass = wave_sum64(mass);
  ties = wave_sum64(ties);
  if (lane == 0) {
    sh.wave[wave] = mass;
    sh.wave2[wave] = ties;
  }
  __syncthreads();
  const u64 tie_weight = border.key ? weight(s, logit_of(border.key)) : 0;
  u64 total = 0, before = 0, left = border.ties, my_left = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) {
      before = total;
      my_left = left;
    }
    const u64 n = sh.wave2[w] < left ? sh.wave2[w] : left;
    total += sh.wave[w] + n * tie_weight;
    left -= n;
  }
  float u = a.u[r];
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
  u64 target = part_of<false>(u, total);
  const u64 mine = mass + (ties < my_left ? ties : my_left) * tie_weight;
  if (target < before || target >= before + mine) {
    return;
  }
  target -= before;
  for (int i = i0; i < i1; i += 64) {
    const bool in = i + lane < i1;
    const float l = in ? logit<kF32>(row, i + lane) : -INFINITY;
    const uint32_t k = key_of(l);
    const bool kept = k && stays(l, k);
    const bool tie = kept && k == border.key;
    const u64 tied = __ballot(tie);
    const bool over = tie && (u64)__popcll(tied & ((1ull << lane) - 1)) >= my_left;
    const u64 w = kept && !over ? weight(s, l) : 0;
    const u64 sum = wave_scan64(w);
    const u64 hit = __ballot(sum > target);
    if (hit) {
      if (lane == __ffsll((long long)hit) - 1) {
        a.tokens[r] = i + lane;
        if (a.logprob) {
          a.logprob[r] = (float)log((double)w / (double)total);
        }
      }
      return;
    }
    target -= __shfl(sum, 63);
    const u64 n = (u64)__popcll(tied);
    my_left -= n < my_left ? n : my_left;
  }
}

} // namespace

void sample_launch(const SampleArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)a.rows);
  if (a.f32) {
    hipLaunchKernelGGL((sample_rows<true>), grid, dim3(kThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((sample_rows<false>), grid, dim3(kThreads), 0, stream, a);
  }
  VX_HIP_CHECK(hipGetLastError());
}

} // namespace vxk
