/*
 * sample.hip -- next tokens from logits (vx_nn_sample_*): temperature, top-k,
 * top-p, min-p and one uniform number a row.
 *
 * With tokens in the order of falling logits (the lower index first among
 * equals), each setting keeps a first part of the order, so the kept tokens
 * are those above a border: a logit, and among the tokens that have it an
 * index. The draw then goes over the kept tokens by rising index. Nothing is
 * sorted: a border, or the drawn token, is where a running count or weight
 * reaches some amount, found by histograms over ever smaller ranges of an
 * order-preserving 32-bit key (`descend`).
 *
 * Weights 2^((l - top) c), with c = log2(e) / T and top the largest logit, are
 * taken in 64 bits and kept as 64-bit integers of unit 2^-shift, so many that
 * a row's sum stays within 2^62 (and at most 51). Integer sums do not depend on their order:
 * LDS atomics and any division of the row give the same bits.
 *
 * A first histogram over (top - l) c finds the bin of the border of top-k (by
 * count, no weight is taken) or of top-p (by weight). The tokens down to that
 * bin, mostly a few dozen, then go into LDS and everything else happens there;
 * where they are many, `descend` and the draw go over the row again.
 *
 * sample_rows: a workgroup a row, which it keeps in LDS up to 128 KiB of it. sample_tops and sample_parts: several workgroups a row find its
 * top, then its histogram or weight, in a workspace; the last of a row to
 * finish does the rest.
 */
#include "../vx_batch_kernels.h"
#include "../vx_hip_common.h"
#include "vx_lds_dma.hip.h"
#include "vx_wave_ops.hip.h"

#include <algorithm>
#include <cmath>

namespace vxk {
namespace {

typedef unsigned long long u64;
typedef uint32_t u32;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 1024;      /* one a thread */
constexpr int kChunk = 4 * kThreads; /* logits of a vector load of every thread */
constexpr int kList = kThreads;  /* tokens in LDS, one a thread */
constexpr int kFew = 256;        /* of them, each compared with each */
constexpr float kPerOctave = 16.0f; /* bins per factor of two of the weight: 2^64 in all */

/* Rises with l; 0 for -inf (and what counts as it), which is never drawn. */
__device__ __forceinline__ u32 key_of(float l) {
  const u32 b = __float_as_uint(l);
  const u32 k = b ^ ((u32)((int32_t)b >> 31) | 0x80000000u);
  return l > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float logit_of(u32 key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

/* floor(x total) and, with kUp, ceil(x total) of x in (0, 1), exactly: x is 24
 * bits times a power of two. A border that falls between two tokens (equal
 * logits, a half) falls on the side that the definition says. */
template <bool kUp> __device__ __forceinline__ u64 part_of(float x, u64 total) {
  const u32 b = __float_as_uint(x);
  const int e = (int)(b >> 23);
  const u32 m = (b & 0x7fffffu) | (e ? 0x800000u : 0u);
  const int down = e ? 150 - e : 149; /* 24 .. 149 */
  const unsigned __int128 p = (unsigned __int128)m * total;
  if (down >= 128) {
    return kUp && p ? 1 : 0;
  }
  const u64 q = (u64)(p >> down);
  return q + (kUp && ((unsigned __int128)q << down) != p ? 1 : 0);
}

/* A row's settings, as the kernels use them. */
struct Settings {
  int top_k; /* 0: off */
  float top_p, min_p;
  bool first; /* only the first token of the order stays */
  double c;
  float per; /* bins per unit of logit */
};
__device__ __forceinline__ Settings settings_of(const SampleArgs &a, int r) {
  const float heat = a.temperature ? a.temperature[r] : 1.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f;
  const float min_p = a.min_p ? a.min_p[r] : 0.0f;
  Settings s;
  s.first = !(heat > 0.0f) || top_k == 1 || top_p <= 0.0f;
  s.top_k = top_k > 0 && top_k < a.vocab ? top_k : 0;
  s.top_p = top_p < 1.0f ? top_p : 1.0f;
  s.min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  s.c = 1.4426950408889634074 / (double)heat;
  s.per = (float)fmin(s.c * (double)kPerOctave, 1e30);
  return s;
}

/* How a row's logits become weights. Where a logit is +inf, those count as 0
 * and the others as -inf.
 * 2^d, d <= 0, in units: with k the integer next to 64 d, 2^(k / 64) comes from a
 * table of 64 powers and the exponent, and 2^(d - k / 64) = e^x, |x| <= ln(2) /
 * 128, from its Taylor sum to the 5th power: what is left out is below 2^-54. */
struct Scale {
  double c64, top, unit; /* 64 c */
  const double *table;   /* 2^(i / 64) units, in LDS */
  float ftop, per;
  bool inf;

  __device__ __forceinline__ float logit(float l) const {
    return !inf ? l : l == INFINITY ? 0.0f : -INFINITY;
  }
  /* of what logit() gives, in units, not rounded */
  __device__ __forceinline__ double units(float l) const {
    const double d = fmax(((double)l - top) * c64, -8192.0); /* 2^-128: 0 units */
    const double k = rint(d);
    const double x = (d - k) * (0.69314718055994530942 / 64.0);
    double y = fma(x, 1.0 / 120.0, 1.0 / 24.0);
    y = fma(y, x, 1.0 / 6.0);
    y = fma(y, x, 0.5);
    y = fma(y, x, 1.0);
    y = fma(y, x, 1.0);
    const int i = (int)k;
    return ldexp(y * table[i & 63], i >> 6);
  }
  /* to the nearest integer: units stay within 2^51, where adding 2^52 leaves it
   * in the low bits */
  static __device__ __forceinline__ u64 whole(double units) {
    return (u64)__double_as_longlong(units + 0x1p52) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 weight(float l) const { return whole(units(l)); }
  /* Falls with l; the last bin's weights are 0. */
  __device__ __forceinline__ int bin(float l) const {
    return (int)fminf(fminf(ftop - l, 3.4028234664e38f) * per, (float)(kBins - 1));
  }
  /* No logit of a bin up to `b` is lower. */
  __device__ __forceinline__ float least(int b) const {
    return per > 0.0f ? ftop - (float)(b + 2) / per : -INFINITY;
  }
};
/* Threads 0 .. 63 fill the table; the caller synchronises. */
__device__ __forceinline__ Scale scale_of(const SampleArgs &a, const Settings &s, float top,
                                          double *table) {
  Scale x;
  x.inf = top == INFINITY;
  x.ftop = x.inf ? 0.0f : top;
  x.top = (double)x.ftop;
  x.c64 = s.c * 64.0;
  x.per = s.per;
  x.unit = ldexp(1.0, min(51, 62 - (a.vocab > 1 ? 32 - __clz(a.vocab - 1) : 0)));
  x.table = table;
  if (threadIdx.x < 64) {
    table[threadIdx.x] = exp2((double)threadIdx.x / 64.0) * x.unit;
  }
  return x;
}

__device__ __forceinline__ u64 wave_sum64(u64 v) {
  for (int o = 32; o; o >>= 1) {
    v += __shfl_xor(v, o);
  }
  return v;
}
/* Inclusive, over the wave's lanes up to this one. */
template <typename T> __device__ __forceinline__ T wave_scan(T v) {
  const int lane = threadIdx.x & 63;
  for (int o = 1; o < 64; o <<= 1) {
    const T w = __shfl_up(v, o);
    v += lane >= o ? w : 0;
  }
  return v;
}

struct Found {
  u64 above_mass, mass;
  u32 above_count, count;
  int bin;
};

struct Shared {
  u64 mass[kBins];
  u64 list_w[kList];
  u64 list_k[kList]; /* key, then the index's complement */
  u32 count[kBins];
  u64 wave_m[kWaves];
  u32 wave_c[kWaves];
  u32 n;
  Found found;
  double table[64];
};

__device__ __forceinline__ u64 block_sum(Shared &sh, u64 v) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) {
    sh.wave_m[threadIdx.x >> 6] = v;
  }
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sum += sh.wave_m[w];
  }
  __syncthreads();
  return sum;
}
__device__ __forceinline__ float block_max(Shared &sh, float v) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) {
    sh.wave_c[threadIdx.x >> 6] = __float_as_uint(v);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    v = fmaxf(v, __uint_as_float(sh.wave_c[w]));
  }
  __syncthreads();
  return v;
}

/* Which bin a running count or weight over the threads' bins, from thread 0 on,
 * starts at from `above_*` and reaches `want` in; .bin -1 where none does. By
 * count, weights are not looked at. */
template <bool kMass>
__device__ Found find_bin(Shared &sh, u64 mass, u32 count, u64 above_mass, u32 above_count,
                          u64 want) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 ms = kMass ? wave_scan(mass) : 0;
  const u32 cs = wave_scan(count);
  if (lane == 63) {
    sh.wave_m[wave] = ms;
    sh.wave_c[wave] = cs;
  }
  if (threadIdx.x == 0) {
    sh.found.bin = -1;
  }
  __syncthreads();
  u64 mb = above_mass + ms - (kMass ? mass : 0);
  u32 cb = above_count + cs - count;
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w) {
    mb += kMass && w < wave ? sh.wave_m[w] : 0;
    cb += w < wave ? sh.wave_c[w] : 0;
  }
  const u64 before = kMass ? mb : cb, own = kMass ? mass : count;
  if (before < want && want <= before + own) {
    sh.found = Found{mb, mass, cb, count, (int)threadIdx.x};
  }
  __syncthreads();
  const Found f = sh.found;
  __syncthreads();
  return f;
}

/* Over the items that `each` gives to its callback (a key, and what makes its
 * weight), in the order of falling keys: the key at which the running count
 * (kMass: weight), `above` items above `hi` included, reaches `want`; with the
 * sums above it and at it. Keys outside [lo, hi] are passed over. */
struct Point {
  u32 key;
  Found f;
};
template <bool kMass, typename Each>
__device__ Point descend(Shared &sh, Each each, u32 lo, u32 hi, u64 above_mass, u32 above_count,
                         u64 want) {
  const int t = threadIdx.x;
  for (;;) {
    const u32 width = hi - lo;
    const int shift = max(0, 32 - (width ? __clz((int)width) : 32) - 10);
    sh.mass[t] = 0;
    sh.count[t] = 0;
    __syncthreads();
    each([&](u32 key, auto weight) {
      if (key >= lo && key <= hi) {
        const u32 b = (hi - key) >> shift;
        if constexpr (kMass) {
          atomicAdd(&sh.mass[b], weight());
        }
        atomicAdd(&sh.count[b], 1u);
      }
    });
    __syncthreads();
    const Found f = find_bin<kMass>(sh, sh.mass[t], sh.count[t], above_mass, above_count, want);
    hi -= (u32)f.bin << shift;
    if (shift == 0) {
      return Point{hi, f};
    }
    const u32 span = (1u << shift) - 1;
    lo = hi - lo > span ? hi - span : lo;
    above_mass = f.above_mass;
    above_count = f.above_count;
  }
}

/* Tokens that stay: keys above `key`, and those that have it up to index
 * `last`. */
struct Border {
  u32 key, last;
  __device__ __forceinline__ bool keeps(u32 k, u32 i) const {
    return k > key || (k == key && i <= last);
  }
};

/* The border at `point`, whose first `ties` tokens stay. */
template <typename Each>
__device__ Border border_at(Shared &sh, Each each, const Point &point, u64 ties, int vocab) {
  if (ties >= point.f.count) {
    return Border{point.key, 0xffffffffu};
  }
  const Point p = descend<false>(
      sh,
      [&](auto take) {
        each([&](u32 key, u32 i, auto) {
          if (key == point.key) {
            take(~i, [] { return u64(0); });
          }
        });
      },
      ~(u32)(vocab - 1), 0xffffffffu, 0, 0, ties);
  return Border{point.key, ~p.key};
}

/* How many of the tokens at a point stay where a running weight stops at
 * `want`: those before which it is less. */
__device__ __forceinline__ u64 ties_of(const Found &f, u64 want) {
  const u64 each = f.mass / f.count; /* equal keys, equal weights */
  return (want - f.above_mass + each - 1) / each;
}

__device__ __forceinline__ u64 target_of(const SampleArgs &a, int r, u64 total) {
  const float u = a.u[r];
  return part_of<false>(u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f, total);
}

__device__ __forceinline__ void put(const SampleArgs &a, int r, int token, u64 w, u64 total) {
  a.tokens[r] = token;
  if (a.logprob) {
    a.logprob[r] = (float)log((double)w / (double)total);
  }
}

/* Everything that is left to do for at most kFew tokens in the list: a token's
 * place in the order, and the weight before it there and by index, by comparing
 * it with each, kSlices threads a token. `mass`: the weight that top_p is a
 * share of, where no top_k is on. */
__device__ void finish_few(const SampleArgs &a, Shared &sh, int r, const Settings &s,
                           const Scale &x, int n, u64 mass) {
  constexpr int kSlices = kThreads / kFew;
  const int t = threadIdx.x, e = t % kFew, slice = t / kFew;
  const bool real = e < n;
  const u64 k = real ? sh.list_k[e] : 0;
  const u32 i = ~(u32)k;
  /* sums over the slices meet in mass[e] and count[e] */
  if (t < kFew) {
    sh.mass[t] = 0;
    sh.count[t] = 0;
    sh.mass[kFew + t] = 0;
  }
  __syncthreads();
  if (real) {
    u64 before = 0;
    u32 rank = 0;
#pragma unroll 4
    for (int j = slice; j < n; j += kSlices) {
      const bool over = sh.list_k[j] > k;
      rank += over ? 1u : 0u;
      before += over ? sh.list_w[j] : 0;
    }
    atomicAdd(&sh.count[e], rank);
    atomicAdd(&sh.mass[e], before);
  }
  __syncthreads();
  bool in = real;
  u64 w = real ? sh.list_w[e] : 0;
  if (s.top_k) {
    in = in && sh.count[e] < (u32)s.top_k;
    mass = s.top_p < 1.0f ? block_sum(sh, in && slice == 0 ? w : 0) : 0;
  }
  if (s.top_p < 1.0f) {
    in = in && sh.mass[e] < part_of<true>(s.top_p, mass);
  }
  if (s.min_p > 0.0f) {
    in = in && x.units(logit_of((u32)(k >> 32))) >= (double)s.min_p * x.unit;
  }
  w = in ? w : 0;
  const u64 total = block_sum(sh, slice == 0 ? w : 0);
  const u64 target = target_of(a, r, total);
  if (slice == 0 && real) {
    sh.list_w[e] = w;
  }
  __syncthreads();
  if (real) {
    u64 before = 0;
#pragma unroll 4
    for (int j = slice; j < n; j += kSlices) {
      before += ~(u32)sh.list_k[j] < i ? sh.list_w[j] : 0;
    }
    atomicAdd(&sh.mass[kFew + e], before);
  }
  __syncthreads();
  if (in && slice == 0) {
    const u64 before = sh.mass[kFew + e];
    if (before <= target && target < before + w) {
      put(a, r, (int)i, w, total);
    }
  }
}

/* The same for up to kList tokens, one a thread, of bins up to `bin`. */
__device__ void finish_list(const SampleArgs &a, Shared &sh, int r, const Settings &s,
                            const Scale &x, int n, u64 mass, int bin) {
  const int t = threadIdx.x;
  const bool mine = t < n;
  const u64 kw = mine ? sh.list_k[t] : 0;
  const u64 w = mine ? sh.list_w[t] : 0;
  const u32 key = (u32)(kw >> 32), i = ~(u32)kw;
  bool in = mine;
  const u32 hi = key_of(x.ftop);
  const u32 lo = max(key_of(x.least(bin)), 1u);
  auto by_key = [&](auto take) {
    if (in) {
      take(key, [&] { return w; });
    }
  };
  auto both = [&](auto take) {
    if (in) {
      take(key, i, [&] { return w; });
    }
  };
  if (s.top_k) {
    const Point p = descend<false>(sh, by_key, lo, hi, 0, 0, (u64)s.top_k);
    const Border b = border_at(sh, both, p, (u64)s.top_k - p.f.above_count, a.vocab);
    in = mine && b.keeps(key, i);
    mass = s.top_p < 1.0f ? block_sum(sh, in ? w : 0) : 0;
  }
  if (s.top_p < 1.0f) {
    const u64 want = part_of<true>(s.top_p, mass);
    const Point p = descend<true>(sh, by_key, lo, hi, 0, 0, want);
    const Border b = border_at(sh, both, p, ties_of(p.f, want), a.vocab);
    in = in && b.keeps(key, i);
  }
  if (s.min_p > 0.0f) {
    in = in && x.units(logit_of(key)) >= (double)s.min_p * x.unit;
  }
  const u64 total = block_sum(sh, in ? w : 0);
  const u64 target = target_of(a, r, total);
  const Point p = descend<true>(
      sh,
      [&](auto take) {
        if (in) {
          take(~i, [&] { return w; });
        }
      },
      ~(u32)(a.vocab - 1), 0xffffffffu, 0, 0, target + 1);
  if (in && i == ~p.key) {
    put(a, r, (int)i, w, total);
  }
}

/* Four logits from index i on (NaN as -inf, -0 as +0), -inf from `end` on. */
template <bool kF32> struct Four;
template <> struct Four<true> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  typedef float whole __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ float value(float v) { return v; }
};
template <> struct Four<false> {
  typedef unsigned short type __attribute__((ext_vector_type(4), aligned(2)));
  typedef unsigned short whole __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ float value(unsigned short v) { return bf16_to_f32(v); }
};

/* A row, in memory or (kLds bytes, room for all of it) in LDS. */
template <bool kF32, int kLds> struct Row {
  typedef typename Four<kF32>::type V;
  typedef typename Four<kF32>::whole VA;
  static constexpr int kSize = kF32 ? 4 : 2;
  const char *p;
  int vocab;
  u32 lds; /* where LDS holds it */

  __device__ __forceinline__ Row(const SampleArgs &a, int r, const char *buffer)
      : p(static_cast<const char *>(a.logits) + (int64_t)r * a.stride * kSize), vocab(a.vocab),
        lds(kLds ? (u32)(uintptr_t)(const VX_LDS char *)buffer : 0u) {}

  static __device__ __forceinline__ float clean(float l) {
    return l > -INFINITY ? l + 0.0f : -INFINITY;
  }
  __device__ __forceinline__ void from_memory(int64_t i, int64_t end, float (&l)[4]) const {
    if (i + 3 < end) {
      const V v = *reinterpret_cast<const V *>(p + i * kSize);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] = clean(Four<kF32>::value(v[e]));
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      l[e] = -INFINITY;
      if (i + e < end) {
        if constexpr (kF32) {
          l[e] = clean(reinterpret_cast<const float *>(p)[i + e]);
        } else {
          l[e] = clean(bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i + e]));
        }
      }
    }
  }
  __device__ __forceinline__ void load4(int64_t i, int64_t end, float (&l)[4]) const {
    if constexpr (kLds > 0) {
      const VA v = *(const VX_LDS VA *)(uintptr_t)(lds + (u32)i * kSize);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] = i + e < end ? clean(Four<kF32>::value(v[e])) : -INFINITY;
      }
    } else {
      from_memory(i, end, l);
    }
  }
  /* The row's first reading: its largest logit, and into LDS. */
  __device__ __forceinline__ float take() const {
    float top = -INFINITY;
#pragma unroll 4
    for (int64_t i = 4 * threadIdx.x; i < vocab; i += kChunk) {
      float l[4];
      from_memory(i, vocab, l);
      VA v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        top = fmaxf(top, l[e]);
        if constexpr (kF32) {
          v[e] = l[e];
        } else {
          v[e] = (unsigned short)(__float_as_uint(l[e]) >> 16); /* as it was, but for NaN */
        }
      }
      if constexpr (kLds > 0) {
        *(VX_LDS VA *)(uintptr_t)(lds + (u32)i * kSize) = v;
      }
    }
    return top;
  }
  /* f(index, logit), in no order. */
  template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int64_t i = 4 * threadIdx.x; i < vocab; i += kChunk) {
      float v[4];
      load4(i, vocab, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f((u32)i + e, v[e]);
      }
    }
  }
};

/* The draw over a row, `weight` giving a token's (0 if it does not stay). The
 * row, then the part of it that the sum falls in, is cut into a part for each
 * wave until it is a chunk. */
template <typename R, typename W>
__device__ void draw(const SampleArgs &a, Shared &sh, int r, const R &row, W weight) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int64_t begin = 0, end = row.vocab;
  u64 total = 0, target = 0;
  while (end - begin > kChunk) {
    const int64_t per = ((end - begin + kWaves - 1) / kWaves + 3) / 4 * 4;
    const int64_t i0 = begin + wave * per, i1 = i0 + per < end ? i0 + per : end;
    u64 sum = 0;
#pragma unroll 1
    for (int64_t i = i0 + 4 * lane; i < i1; i += 256) {
      float v[4];
      row.load4(i, i1, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum += weight((u32)(i + e), v[e]);
      }
    }
    sum = wave_sum64(sum);
    if (lane == 0) {
      sh.wave_m[wave] = sum;
    }
    __syncthreads();
    if (total == 0) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        total += sh.wave_m[w];
      }
      target = target_of(a, r, total);
    }
    int at = 0;
    for (; at + 1 < kWaves && target >= sh.wave_m[at]; ++at) {
      target -= sh.wave_m[at];
    }
    __syncthreads();
    begin += at * per;
    end = begin + per < end ? begin + per : end;
  }
  float v[4];
  u64 w[4], sum = 0;
  const int64_t i = begin + 4 * t;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = -INFINITY;
  }
  if (i < end) {
    row.load4(i, end, v);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = weight((u32)(i + e), v[e]);
    sum += w[e];
  }
  if (total == 0) {
    total = block_sum(sh, sum);
    target = target_of(a, r, total);
  }
  const Found f = find_bin<true>(sh, sum, 0, 0, 0, target + 1);
  if (f.bin == t) {
    target -= f.above_mass;
    for (int e = 0; e < 4; ++e) {
      if (target < w[e]) {
        put(a, r, (int)(i + e), w[e], total);
        return;
      }
      target -= w[e];
    }
  }
}

/* The row's tokens of bins up to `bin` into the list; how many there are, which
 * may be more than it holds. */
template <typename R>
__device__ int gather(Shared &sh, const R &row, const Scale &x, int bin) {
  if (threadIdx.x == 0) {
    sh.n = 0;
  }
  __syncthreads();
  const float least = x.inf ? INFINITY : x.least(bin);
  row.each([&](u32 i, float l) {
    if (l >= least) { /* one of a few, mostly */
      l = x.logit(l);
      if (l > -INFINITY && x.bin(l) <= bin) {
        const u32 at = atomicAdd(&sh.n, 1u);
        if (at < (u32)kList) {
          sh.list_k[at] = (u64)key_of(l) << 32 | (u32)~i;
        }
      }
    }
  });
  __syncthreads();
  return (int)sh.n;
}

/* The result from the list's n tokens, those of bins up to `bin`. */
__device__ void finish(const SampleArgs &a, Shared &sh, int r, const Settings &s, const Scale &x,
                       int n, u64 mass, int bin) {
  const int t = threadIdx.x;
  if (t < n) {
    sh.list_w[t] = x.weight(logit_of((u32)(sh.list_k[t] >> 32)));
  }
  __syncthreads();
  if (n <= kFew) {
    finish_few(a, sh, r, s, x, n, mass);
  } else {
    finish_list(a, sh, r, s, x, n, mass, bin);
  }
}

/* What is left to do once the row's histogram is in the threads' registers
 * (`mass` only where no top_k is on; all of the row's bins). */
template <typename R>
__device__ void finish_bins(const SampleArgs &a, Shared &sh, int r, const R &row, Settings s,
                            const Scale &x, u64 mass, u32 count) {
  const int t = threadIdx.x;
  u64 sum = 0;
  Found f;
  if (s.top_k) {
    f = find_bin<false>(sh, 0, t == kBins - 1 ? 0 : count, 0, 0, (u64)s.top_k);
    if (f.bin < 0) {
      /* more than there are above -inf, or into the weights of 0: all of them */
      s.top_k = 0;
      if (s.top_p < 1.0f) {
        sh.mass[t] = 0;
        __syncthreads();
        row.each([&](u32, float l) {
          l = x.logit(l);
          if (l > -INFINITY) {
            atomicAdd(&sh.mass[x.bin(l)], x.weight(l));
          }
        });
        __syncthreads();
        mass = sh.mass[t];
      }
    }
  }
  if (!s.top_k && s.top_p < 1.0f) {
    sum = block_sum(sh, mass);
    f = find_bin<true>(sh, mass, count, 0, 0, part_of<true>(s.top_p, sum));
  }
  const bool bordered = s.top_k || s.top_p < 1.0f;
  if (bordered && f.above_count + f.count <= (u32)kList) {
    finish(a, sh, r, s, x, gather(sh, row, x, f.bin), sum, f.bin);
    return;
  }
  Border border{0, 0xffffffffu};
  if (bordered) {
    auto by_key = [&](auto take) {
      row.each([&](u32 i, float l) {
        l = x.logit(l);
        const u32 k = key_of(l);
        if (k && border.keeps(k, i)) {
          take(k, [&] { return x.weight(l); });
        }
      });
    };
    auto both = [&](auto take) {
      row.each([&](u32 i, float l) {
        l = x.logit(l);
        const u32 k = key_of(l);
        if (k && border.keeps(k, i)) {
          take(k, i, [&] { return x.weight(l); });
        }
      });
    };
    /* from the top to a bin below the border's */
    const u32 lo = max(key_of(x.least(f.bin)), 1u);
    const u32 hi = key_of(x.ftop);
    if (s.top_k) {
      const Point p = descend<false>(sh, by_key, lo, hi, 0, 0, (u64)s.top_k);
      border = border_at(sh, both, p, (u64)s.top_k - p.f.above_count, a.vocab);
      if (s.top_p < 1.0f) {
        by_key([&](u32, auto weight) { sum += weight(); });
        sum = block_sum(sh, sum);
      }
    }
    if (s.top_p < 1.0f) {
      const u64 want = part_of<true>(s.top_p, sum);
      const Point p = descend<true>(sh, by_key, lo, hi, 0, 0, want);
      border = border_at(sh, both, p, ties_of(p.f, want), a.vocab);
    }
  }
  const double least = (double)s.min_p * x.unit;
  auto weight = [&](u32 i, float l) {
    l = x.logit(l);
    const u32 k = key_of(l);
    if (!k || !border.keeps(k, i)) {
      return u64(0);
    }
    const double q = x.units(l);
    return q >= least ? Scale::whole(q) : u64(0);
  };
  draw(a, sh, r, row, weight);
}

/* The largest logit, or, where only the first token stays or there is none
 * above -inf, the result: true. */
__device__ __forceinline__ bool first_only(const SampleArgs &a, int r, const Settings &s,
                                           float top, u32 first_index) {
  const bool none = top == -INFINITY;
  if (!none && !s.first) {
    return false;
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = none ? -1 : (int)first_index;
    if (a.logprob) {
      a.logprob[r] = none ? -INFINITY : 0.0f;
    }
  }
  return true;
}

template <bool kF32, int kLds>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a) {
  __shared__ Shared sh;
  __shared__ __align__(16) char buffer[std::max(kLds, 16)];
  const int t = threadIdx.x, r = blockIdx.x;
  const Row<kF32, kLds> row(a, r, buffer);
  const Settings s = settings_of(a, r);
  const float own = row.take();
  const float top = block_max(sh, own);
  u32 index = 0xffffffffu;
  if (s.first) {
    row.each([&](u32 i, float l) { index = l == top && i < index ? i : index; });
    for (int o = 32; o; o >>= 1) {
      const u32 other = (u32)__shfl_xor((int)index, o);
      index = other < index ? other : index;
    }
    if ((t & 63) == 0) {
      sh.wave_c[t >> 6] = index;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
      index = sh.wave_c[w] < index ? sh.wave_c[w] : index;
    }
  }
  if (first_only(a, r, s, top, index)) {
    return;
  }
  const Scale x = scale_of(a, s, top, sh.table);
  u64 mass = 0;
  u32 count = 0;
  if (s.top_k || s.top_p < 1.0f) {
    sh.mass[t] = 0;
    sh.count[t] = 0;
    __syncthreads();
    if (s.top_k) {
      /* The top_k largest lie down to the bin of the top_k-th largest of the
       * threads' own maxima; mostly there are few more. */
      const float l = x.logit(own);
      if (l > -INFINITY) {
        atomicAdd(&sh.count[x.bin(l)], 1u);
      }
      __syncthreads();
      const Found f = find_bin<false>(sh, 0, sh.count[t], 0, 0, (u64)s.top_k);
      if (f.bin >= 0 && f.bin < kBins - 1) {
        const int n = gather(sh, row, x, f.bin);
        if (n <= kList) {
          finish(a, sh, r, s, x, n, 0, f.bin);
          return;
        }
      }
      sh.count[t] = 0;
      __syncthreads();
    }
    row.each([&](u32, float l) {
      l = x.logit(l);
      if (l > -INFINITY) {
        const int b = x.bin(l);
        atomicAdd(&sh.count[b], 1u);
        if (!s.top_k) {
          atomicAdd(&sh.mass[b], x.weight(l));
        }
      }
    });
    __syncthreads();
    mass = sh.mass[t];
    count = sh.count[t];
  }
  __syncthreads();
  finish_bins(a, sh, r, row, s, x, mass, count);
}

template <bool kF32> void launch(const SampleArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)a.rows), block(kThreads);
  /* the row in LDS where it fits, in two sizes: the smaller leaves room for a
   * second workgroup on a CU */
  constexpr int kSize = kF32 ? 4 : 2;
  if (a.vocab <= 32768 / kSize) {
    hipLaunchKernelGGL((sample_rows<kF32, 32768>), grid, block, 0, stream, a);
  } else if (a.vocab <= 131072 / kSize) {
    hipLaunchKernelGGL((sample_rows<kF32, 131072>), grid, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL((sample_rows<kF32, 0>), grid, block, 0, stream, a);
  }
}

} // namespace

void sample_launch(const SampleArgs &a, hipStream_t stream) {
  if (a.f32) {
    launch<true>(a, stream);
  } else {
    launch<false>(a, stream);
  }
  VX_HIP_CHECK(hipGetLastError());
}

} // namespace vxk
