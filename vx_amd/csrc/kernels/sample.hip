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
 * a row's sum stays within 2^62 (and at most 51). Integer sums do not depend on
 * their order: LDS atomics and any division of the row give the same bits.
 *
 * A first histogram over (top - l) c finds the bin of the border of top-k (by
 * count, no weight is taken) or of top-p (by weight). The tokens down to that
 * bin, mostly a few dozen, then go into LDS and everything else happens there;
 * where they are many, `descend` and the draw go over the row again.
 *
 * sample_rows: a workgroup a row, which it keeps in LDS up to 128 KiB of it.
 * sample_tops, sample_weigh, sample_settle: several workgroups a row, each of a
 * slice of it, find its top, then its histogram or weight, in a workspace; the
 * slice that the draw falls in, or the last to leave its few tokens, does the
 * rest.
 *
 * Latency bounds the small calls. 1 x 32000 f32 by top-k 11.6 us (10.2 at best),
 * of which 2.7 for the row's 128 KB into LDS and its largest logit by one
 * workgroup, 1.4 for the threads' maxima and their bin, 3.1 for the list and 3.1
 * for the rest; 48 x 32000 with every setting in use 23, of which the 64-bit
 * weights of rows with top-p alone, 32 a thread, take 11 (atomics for the tokens
 * near the border alone save nothing). 8 x 131072 by top-p 30 a call, its three
 * launches 4.5, 8.8 and 14 (3.9, 8.2 and 12.6 at best). 256 x 131071 without a
 * border 64: the row out of memory twice and a sixteenth of it a third time, 276
 * MB at 4.3 TB/s, and 128 64-bit weights a thread, 33 us on one CU; by top-p 160,
 * the row three times and the histogram's weights.
 */
#include "../vx_batch_kernels.h"
#include "../vx_hip_common.h"
#include "sample_list.h"
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
  float u;   /* in [0, 1) */
};
__device__ __forceinline__ Settings settings_of(const SampleArgs &a, int r) {
  /* one of the pointers is always good to read, so that all loads go together */
  auto value = [&](const float *p, float none) {
    const float v = (p ? p : a.u)[p ? r : 0];
    return p ? v : none;
  };
  const int *steps = a.step ? a.step : reinterpret_cast<const int *>(a.u);
  const int at = steps[0];
  const float heat = value(a.temperature, 1.0f);
  const int top_k = __float_as_int(value(reinterpret_cast<const float *>(a.top_k), 0.0f));
  const float top_p = value(a.top_p, 1.0f);
  const float min_p = value(a.min_p, 0.0f);
  const float u = a.u[a.step ? max(at - a.step0, 0) : r];
  Settings s;
  s.u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
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
 * 2^d, d <= 0, in units: with k the integer next to d, 2^(d - k) by the
 * polynomial of degree 10 that meets 2^f at the 11 Chebyshev nodes of [-1/2, 1/2]
 * (off by at most 2^-51.5), and 2^k by an addition to the exponent. Adding 1.5 *
 * 2^52 to d leaves k in the low bits: conversions and roundings of 64 bits take
 * four times an addition's cycles, and a table in LDS twice a longer sum's. */
struct Scale {
  double c, top;
  float ftop, per;
  int shift; /* a unit is 2^-shift of the largest weight */
  bool inf;

  /* in units, not rounded */
  __device__ __forceinline__ double units(float l) const {
    const double d = fmax(((double)l - top) * c, -128.0); /* 0 units */
    const double t = d + 0x1.8p52;
    const double f = d - (t - 0x1.8p52);
    double y = 0x1.e6063f7217bc6p-28;
    y = fma(y, f, 0x1.b675bca4eeebbp-24);
    y = fma(y, f, 0x1.62bfd47773353p-20);
    y = fma(y, f, 0x1.ffcb54062e698p-17);
    y = fma(y, f, 0x1.430913096fd9fp-13);
    y = fma(y, f, 0x1.5d87fe9d7a584p-10);
    y = fma(y, f, 0x1.3b2ab6fba1ddap-7);
    y = fma(y, f, 0x1.c6b08d703ce49p-5);
    y = fma(y, f, 0x1.ebfbdff82c598p-3);
    y = fma(y, f, 0x1.62e42fefa3a19p-1);
    y = fma(y, f, 1.0);
    const int k = (int)(u32)__double_as_longlong(t) + shift;
    return __hiloint2double(__double2hiint(y) + (k << 20), __double2loint(y));
  }
  /* to the nearest integer: units stay within 2^51, where adding 2^52 leaves it
   * in the low bits */
  static __device__ __forceinline__ u64 whole(double units) {
    return (u64)__double_as_longlong(units + 0x1p52) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 weight(float l) const { return whole(units(l)); }
  /* `min_p` in units. */
  __device__ __forceinline__ double share(float min_p) const { return ldexp((double)min_p, shift); }
  /* Falls with l; the last bin's weights are 0. */
  __device__ __forceinline__ int bin(float l) const {
    return (int)fminf(fminf(ftop - l, 3.4028234664e38f) * per, (float)(kBins - 1));
  }
  /* No logit of a bin up to `b` is lower. */
  __device__ __forceinline__ float least(int b) const {
    return per > 0.0f ? ftop - (float)(b + 2) / per : -INFINITY;
  }
};
__device__ __forceinline__ Scale scale_of(const SampleArgs &a, const Settings &s, float top) {
  Scale x;
  x.inf = top == INFINITY;
  x.ftop = x.inf ? 0.0f : top;
  x.top = (double)x.ftop;
  x.c = s.c;
  x.per = s.per;
  x.shift = min(51, 62 - (a.vocab > 1 ? 32 - __clz(a.vocab - 1) : 0));
  return x;
}

/* A value of another lane by VALU data movement; 0 where there is none. */
template <int kCtrl, int kRows> __device__ __forceinline__ u32 dpp(u32 v) {
  return (u32)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, false);
}
template <int kCtrl, int kRows> __device__ __forceinline__ u64 dpp(u64 v) {
  return (u64)dpp<kCtrl, kRows>((u32)(v >> 32)) << 32 | dpp<kCtrl, kRows>((u32)v);
}
/* Inclusive sum over the wave's lanes up to this one: within rows of 16 lanes by
 * shifts of 1, 2, 4 and 8, then the last lanes of rows and of halves. */
template <typename T> __device__ __forceinline__ T wave_scan(T v) {
  v += dpp<0x111, 0xf>(v);
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v); /* lane 15 of rows 0 and 2 to the next row */
  v += dpp<0x143, 0xc>(v); /* lane 31 to rows 2 and 3 */
  return v;
}
__device__ __forceinline__ u64 lane63(u64 v) {
  return (u64)(u32)__builtin_amdgcn_readlane((int)(u32)(v >> 32), 63) << 32 |
         (u32)__builtin_amdgcn_readlane((int)(u32)v, 63);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane63(wave_scan(v)); }
/* The wave's largest, of values above 0 or 0. */
__device__ __forceinline__ u64 wave_max64(u64 v) {
  auto up = [&](u64 w) { v = w > v ? w : v; };
  up(dpp<0x111, 0xf>(v));
  up(dpp<0x112, 0xf>(v));
  up(dpp<0x114, 0xf>(v));
  up(dpp<0x118, 0xf>(v));
  up(dpp<0x142, 0xa>(v));
  up(dpp<0x143, 0xc>(v));
  return lane63(v);
}

struct Found {
  u64 above_mass, mass;
  u32 above_count, count;
  int bin;
};

/* Which thread's `own` the draw falls in, by rising thread; with the row's weight,
 * and where in that part it does. */
struct Drawn {
  u64 total, target;
  int at;
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
  Drawn drawn;
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
__device__ __forceinline__ Found find_bin(Shared &sh, u64 mass, u32 count, u64 above_mass, u32 above_count,
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
__device__ __forceinline__ Point descend(Shared &sh, Each each, u32 lo, u32 hi, u64 above_mass, u32 above_count,
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
__device__ __forceinline__ Border border_at(Shared &sh, Each each, const Point &point, u64 ties, int vocab) {
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

__device__ __forceinline__ Drawn draw_part(Shared &sh, u64 own, float u) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 upto = wave_scan(own);
  if (lane == 63) {
    sh.wave_m[wave] = upto;
  }
  __syncthreads();
  u64 total = 0, before = upto - own;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const u64 m = sh.wave_m[w];
    total += m;
    before += w < wave ? m : 0;
  }
  const u64 target = part_of<false>(u, total);
  if (before <= target && target < before + own) {
    sh.drawn = Drawn{total, target - before, (int)threadIdx.x};
  }
  __syncthreads();
  const Drawn d = sh.drawn;
  __syncthreads();
  return d;
}

__device__ __forceinline__ void put(const SampleArgs &a, int r, int token, u64 w, u64 total) {
  a.tokens[r] = token;
  if (a.logprob) {
    a.logprob[r] = (float)log((double)w / (double)total);
  }
}

/* Everything that is left to do for at most kFew tokens in the list: a token's
 * place in the order, and the weight before it there and by index, by comparing
 * it with each, 4 to 16 threads a token. `mass`: the weight that top_p is a
 * share of, where no top_k is on. */
__device__ __forceinline__ void finish_few(const SampleArgs &a, Shared &sh, int r, const Settings &s,
                           const Scale &x, int n, u64 mass) {
  const int room = n <= 64 ? 64 : n <= 128 ? 128 : kFew;
  const int slices = kThreads / room;
  const int t = threadIdx.x, e = t & (room - 1), slice = t / room;
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
    for (int j = slice; j < n; j += slices) {
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
    in = in && x.units(logit_of((u32)(k >> 32))) >= x.share(s.min_p);
  }
  w = in ? w : 0;
  const u64 total = block_sum(sh, slice == 0 ? w : 0);
  const u64 target = part_of<false>(s.u, total);
  if (slice == 0 && real) {
    sh.list_w[e] = w;
  }
  __syncthreads();
  if (real) {
    u64 before = 0;
#pragma unroll 4
    for (int j = slice; j < n; j += slices) {
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

/* The same for up to kList tokens, one a thread, of bins up to `bin`. Where min_p
 * leaves no more than those, the border of top_k or top_p may lie below them all. */
__device__ __forceinline__ void finish_list(const SampleArgs &a, Shared &sh, int r, const Settings &s,
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
    if (s.top_k < n) {
      const Point p = descend<false>(sh, by_key, lo, hi, 0, 0, (u64)s.top_k);
      const Border b = border_at(sh, both, p, (u64)s.top_k - p.f.above_count, a.vocab);
      in = mine && b.keeps(key, i);
    }
    mass = s.top_p < 1.0f ? block_sum(sh, in ? w : 0) : 0;
  }
  if (s.top_p < 1.0f) {
    const u64 want = part_of<true>(s.top_p, mass);
    if (want <= block_sum(sh, in ? w : 0)) {
      const Point p = descend<true>(sh, by_key, lo, hi, 0, 0, want);
      const Border b = border_at(sh, both, p, ties_of(p.f, want), a.vocab);
      in = in && b.keeps(key, i);
    }
  }
  if (s.min_p > 0.0f) {
    in = in && x.units(logit_of(key)) >= x.share(s.min_p);
  }
  const u64 total = block_sum(sh, in ? w : 0);
  const u64 target = part_of<false>(s.u, total);
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
  int begin, end; /* the part of it that is meant */
  u32 lds;        /* where LDS holds it (from index 0 on) */
  bool inf;       /* it holds +inf: those are 0, the others -inf */

  __device__ __forceinline__ Row(const SampleArgs &a, int r, const char *buffer)
      : p(static_cast<const char *>(a.logits) + (int64_t)r * a.stride * kSize), begin(0),
        end(a.vocab), lds(kLds ? (u32)(uintptr_t)(const VX_LDS char *)buffer : 0u),
        inf(false) {}

  static __device__ __forceinline__ float clean(float l) {
    return l > -INFINITY ? l + 0.0f : -INFINITY;
  }
  /* kRaw: as they are. */
  template <bool kRaw = false>
  __device__ __forceinline__ void from_memory(int i, int end, float (&l)[4]) const {
    if (i + 3 < end) {
      const V v = *reinterpret_cast<const V *>(p + (int64_t)i * kSize);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = Four<kF32>::value(v[e]);
        l[e] = kRaw ? x : clean(x);
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
  template <bool kRaw = false>
  __device__ __forceinline__ void load4(int i, int end, float (&l)[4]) const {
    load<kRaw>(i, end, l);
    if (inf) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] = l[e] == INFINITY ? 0.0f : -INFINITY;
      }
    }
  }
  template <bool kRaw>
  __device__ __forceinline__ void load(int i, int end, float (&l)[4]) const {
    if constexpr (kLds > 0) {
      if (i >= end) {
        l[0] = l[1] = l[2] = l[3] = -INFINITY;
        return;
      }
      const VA v = *(const VX_LDS VA *)(uintptr_t)(lds + (u32)i * kSize);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] = i + e < end ? Four<kF32>::value(v[e]) : -INFINITY; /* clean already */
      }
    } else {
      from_memory<kRaw>(i, end, l);
    }
  }
  /* The first reading: the thread's largest logit, and into LDS. */
  __device__ __forceinline__ float take() const {
    float top = -INFINITY;
#pragma unroll 8
    for (int i = begin + 4 * threadIdx.x; i < end; i += kChunk) {
      float l[4];
      from_memory(i, end, l);
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
  /* f(index, logit), in no order. Out of memory four loads a thread are in
   * flight, -inf past the end. */
  template <bool kRaw = false, typename F> __device__ __forceinline__ void each(F f) const {
    constexpr int kAhead = kLds > 0 ? 1 : 4;
#pragma unroll 1
    for (int i = begin + 4 * threadIdx.x; i < end; i += kAhead * kChunk) {
      float v[kAhead][4];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        load4<kRaw>(i + j * kChunk, end, v[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f((u32)(i + j * kChunk + e), v[j][e]);
        }
      }
    }
  }
};

/* The draw over a row's part, `weight` giving a token's (0 if it does not stay);
 * with `total`, the weight of the whole row, of the token in which the part's
 * sum passes `target`. The part, then the part of it that the sum falls in, is
 * cut into one for each wave until it is a chunk. */
template <typename R, typename W>
__device__ __forceinline__ void draw(const SampleArgs &a, Shared &sh, int r, const R &row, float u, W weight,
                     u64 total = 0, u64 target = 0) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int begin = row.begin, end = row.end;
  while (end - begin > kChunk) {
    const int per = ((end - begin + kWaves - 1) / kWaves + 3) / 4 * 4;
    const int i0 = min(begin + wave * per, end), i1 = min(i0 + per, end);
    u64 sum = 0;
    constexpr int kAhead = 4;
#pragma unroll 1
    for (int i = i0 + 4 * lane; i < i1; i += kAhead * 256) {
      float v[kAhead][4];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        row.template load4<W::kRaw>(i + j * 256, i1, v[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum += weight((u32)(i + j * 256 + e), v[j][e]);
        }
      }
    }
    sum = wave_sum64(sum);
    if (lane == 0) {
      sh.wave_m[wave] = sum;
    }
    __syncthreads();
    u64 part[kWaves];
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      part[w] = sh.wave_m[w];
      all += part[w];
    }
    if (total == 0) {
      total = all;
      target = part_of<false>(u, total);
    }
    int at = 0;
    u64 before = 0, run = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      run += part[w];
      at = target >= run ? w + 1 : at;
      before = target >= run ? run : before;
    }
    target -= before;
    __syncthreads();
    begin += at * per;
    end = min(begin + per, end);
  }
  float v[4];
  u64 w[4], sum = 0;
  const int i = begin + 4 * t;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = -INFINITY;
  }
  if (i < end) {
    row.template load4<W::kRaw>(i, end, v);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = weight((u32)(i + e), v[e]);
    sum += w[e];
  }
  int at;
  if (total == 0) {
    const Drawn d = draw_part(sh, sum, u);
    total = d.total;
    target = d.target;
    at = d.at;
  } else {
    const Found f = find_bin<true>(sh, sum, 0, 0, 0, target + 1);
    target -= f.above_mass;
    at = f.bin;
  }
  if (at == t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (target < w[e]) {
        put(a, r, i + e, w[e], total);
        return;
      }
      target -= w[e];
    }
  }
}

/* A workgroup's threads, for fill_list. */
struct Group {
  __device__ __forceinline__ int thread() const { return (int)threadIdx.x; }
  __device__ __forceinline__ void sync() const { __syncthreads(); }
  __device__ __forceinline__ u32 add(u32 &n) const { return atomicAdd(&n, 1u); }
};

/* The row's tokens of bins up to `bin` (kOne: of that bin) into the list; how
 * many there are, of which it holds the first kCap. */
template <bool kOne = false, int kCap, typename R>
__device__ __forceinline__ int gather(Shared &sh, const R &row, const Scale &x, int bin,
                                      u64 (&list)[kCap]) {
  const float least = x.least(bin);
  return fill_list(Group{}, sh.n, list, [&](auto take) {
    row.each([&](u32 i, float l) {
      if (l >= least) { /* one of a few, mostly */
        const int b = x.bin(l);
        if (l > -INFINITY && (kOne ? b == bin : b <= bin)) {
          take((u64)key_of(l) << 32 | (u32)~i);
        }
      }
    });
  });
}

/* The result from the list's n tokens, those of bins up to `bin`. */
__device__ __forceinline__ void finish(const SampleArgs &a, Shared &sh, int r, const Settings &s, const Scale &x,
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

/* A token's weight, 0 where min_p (kLeast) or a border (kBordered) hides it.
 * Without a border -0 and NaN need no care: units() makes nothing of either. */
template <bool kBordered, bool kLeast> struct Keep {
  static constexpr bool kRaw = !kBordered;
  const Scale &x;
  double least; /* units */
  Border border;

  __device__ __forceinline__ u64 operator()(u32 i, float l) const {
    const double q = x.units(l);
    u64 w = Scale::whole(q);
    if constexpr (kLeast) {
      w = q >= least ? w : u64(0);
    }
    return !kBordered || border.keeps(key_of(l), i) ? w : u64(0);
  }
};
/* f(a Keep without a border). */
template <typename F>
__device__ __forceinline__ void unbordered(const Scale &x, const Settings &s, F f) {
  if (s.min_p > 0.0f) {
    f(Keep<false, true>{x, x.share(s.min_p), {}});
  } else {
    f(Keep<false, false>{x, 0.0, {}});
  }
}

/* Where the border of top_k, or without it of top_p, lies in the row's histogram,
 * which is in the threads' registers (`mass` only where no top_k is on). */
struct Where {
  Found f;
  u64 sum; /* the row's weight, without top_k */
  int bin; /* the tokens of bins up to this one are enough to go on with */
  u32 n;   /* so many */
};
/* .f.bin -1: top_k is more than there are above -inf, or reaches the weights of
 * 0, so that it hides nothing. */
__device__ __forceinline__ Where locate(Shared &sh, const Settings &s, u64 mass, u32 count) {
  const int t = threadIdx.x;
  Where w;
  w.sum = 0;
  if (s.top_k) {
    w.f = find_bin<false>(sh, 0, t == kBins - 1 ? 0 : count, 0, 0, (u64)s.top_k);
  } else {
    w.sum = block_sum(sh, mass);
    w.f = find_bin<true>(sh, mass, count, 0, 0, part_of<true>(s.top_p, w.sum));
  }
  w.bin = w.f.bin;
  w.n = w.f.above_count + w.f.count;
  if (s.min_p > 0.0f && (!s.top_k || s.top_p >= 1.0f)) {
    /* weights from min_p on lie down to here; nothing below is needed unless
     * top_p is a share of what top_k keeps */
    const int bin = (int)fminf(-log2f(s.min_p) * kPerOctave + 2.0f, (float)(kBins - 2));
    if (bin < w.bin) {
      w.bin = bin;
      w.n = (u32)block_sum(sh, t <= bin ? count : 0);
    }
  }
  return w;
}

/* What is left to do once the row's histogram is known (without counts where no
 * top_k is on). */
template <typename R>
__device__ __forceinline__ void finish_bins(const SampleArgs &a, Shared &sh, int r, const R &row, Settings s,
                            const Scale &x, u64 mass, u32 count) {
  const int t = threadIdx.x;
  Where at;
  bool bordered = s.top_k || s.top_p < 1.0f;
  if (bordered) {
    at = locate(sh, s, mass, count);
    if (at.f.bin < 0) {
      s.top_k = 0;
      bordered = s.top_p < 1.0f;
      if (bordered) {
        sh.mass[t] = 0;
        __syncthreads();
        row.each([&](u32, float l) {
          if (l > -INFINITY) {
            atomicAdd(&sh.mass[x.bin(l)], x.weight(l));
          }
        });
        __syncthreads();
        at = locate(sh, s, sh.mass[t], count);
      }
    }
  }
  if (bordered && (!s.top_k || at.n <= (u32)kList)) {
    const int n = gather(sh, row, x, at.bin, sh.list_k);
    if (n <= kList) {
      finish(a, sh, r, s, x, n, at.sum, at.bin);
      return;
    }
  }
  if (!bordered) {
    unbordered(x, s, [&](auto keep) { draw(a, sh, r, row, s.u, keep); });
    return;
  }
  Keep<true, true> keep{x, x.share(s.min_p), {0, 0xffffffffu}};
  const u32 lo = max(key_of(x.least(at.f.bin)), 1u), hi = key_of(x.ftop);
  const int in_bin = s.top_k ? kList + 1 : gather<true>(sh, row, x, at.f.bin, sh.list_k);
  if (in_bin <= kList) {
    /* the border's bin alone, in the list */
    const bool mine = t < in_bin;
    const u64 kw = mine ? sh.list_k[t] : 0;
    const u64 w = mine ? x.weight(logit_of((u32)(kw >> 32))) : 0;
    auto both = [&](auto take) {
      if (mine) {
        take((u32)(kw >> 32), ~(u32)kw, [&] { return w; });
      }
    };
    auto by_key = [&](auto take) { both([&](u32 key, u32, auto weight) { take(key, weight); }); };
    const u64 want = part_of<true>(s.top_p, at.sum);
    const Point p = descend<true>(sh, by_key, lo, hi, at.f.above_mass, 0, want);
    keep.border = border_at(sh, both, p, ties_of(p.f, want), a.vocab);
  } else {
    /* the border's own bin, then, after top_k, what that keeps */
    bool all = false;
    auto passes = [&](u32 k, u32 i, float l) {
      return all ? k && keep.border.keeps(k, i) : k && x.bin(l) == at.f.bin;
    };
    auto by_key = [&](auto take) {
      row.each([&](u32 i, float l) {
        const u32 k = key_of(l);
        if (passes(k, i, l)) {
          take(k, [&] { return x.weight(l); });
        }
      });
    };
    auto both = [&](auto take) {
      row.each([&](u32 i, float l) {
        const u32 k = key_of(l);
        if (passes(k, i, l)) {
          take(k, i, [&] { return x.weight(l); });
        }
      });
    };
    if (s.top_k) {
      const Point p =
          descend<false>(sh, by_key, lo, hi, 0, at.f.above_count, (u64)s.top_k);
      keep.border = border_at(sh, both, p, (u64)s.top_k - p.f.above_count, a.vocab);
      if (s.top_p < 1.0f) {
        all = true;
        at.sum = 0;
        by_key([&](u32, auto weight) { at.sum += weight(); });
        at.sum = block_sum(sh, at.sum);
        at.f.above_mass = 0;
      }
    }
    if (s.top_p < 1.0f) {
      const u64 want = part_of<true>(s.top_p, at.sum);
      const Point p = descend<true>(sh, by_key, lo, hi, at.f.above_mass, 0, want);
      const Border b = border_at(sh, both, p, ties_of(p.f, want), a.vocab);
      /* of equal logits top_k may have kept fewer than there are */
      keep.border = Border{b.key, b.key == keep.border.key ? min(b.last, keep.border.last) : b.last};
    }
  }
  draw(a, sh, r, row, s.u, keep);
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
  Row<kF32, kLds> row(a, r, buffer);
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
  const Scale x = scale_of(a, s, top);
  row.inf = x.inf;
  u64 mass = 0;
  u32 count = 0;
  if (s.top_k || s.top_p < 1.0f) {
    sh.mass[t] = 0;
    sh.count[t] = 0;
    __syncthreads();
    if (s.top_k) {
      /* The top_k largest lie down to the bin of the top_k-th largest of the
       * threads' own maxima; mostly there are few more. */
      const float l = !x.inf ? own : own == INFINITY ? 0.0f : -INFINITY;
      if (l > -INFINITY) {
        atomicAdd(&sh.count[x.bin(l)], 1u);
      }
      __syncthreads();
      const Found f = find_bin<false>(sh, 0, sh.count[t], 0, 0, (u64)s.top_k);
      if (f.bin >= 0 && f.bin < kBins - 1) {
        const int n = gather(sh, row, x, f.bin, sh.list_k);
        if (n <= kList) {
          finish(a, sh, r, s, x, n, 0, f.bin);
          return;
        }
      }
      sh.count[t] = 0;
      __syncthreads();
    }
    row.each([&](u32, float l) {
      if (l > -INFINITY) {
        const int b = x.bin(l);
        if (s.top_k) {
          atomicAdd(&sh.count[b], 1u);
        } else {
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

/* ---- several workgroups a row ---- */

/* Tokens of one bin that are settled in LDS: at 16 bins per factor of two, a
 * bell of 131072 logits two units wide has up to 1100 in one. */
constexpr int kBinList = 4096;

/* A row's workspace, and after it for each slice its first token, its weight,
 * and (where top_p alone makes the border) its bins' weights. */
struct Shelf {
  u64 mass[kBins];
  u64 list[kBinList];
  u32 count[kBins];
  u32 n, ticket;

  __device__ __forceinline__ u64 *tops() { return reinterpret_cast<u64 *>(this + 1); }
  __device__ __forceinline__ u64 *sums(int slices) { return tops() + slices; }
  __device__ __forceinline__ u64 *bins(int slices, int slice) {
    return sums(slices) + slices + (int64_t)slice * kBins;
  }
};
static_assert(sizeof(Shelf) % 8 == 0, "what follows is of 64-bit words");

struct Split {
  int slices, slice; /* and logits of one */
  char *ws;
  int64_t shelf; /* bytes from one row's to the next */
};

__device__ __forceinline__ u64 load_far(const u64 *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_far(u64 *p, u64 v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

/* A slice's first token (its key, then the index's complement). */
template <bool kF32> __global__ __launch_bounds__(kThreads) void sample_tops(SampleArgs a, Split p) {
  __shared__ u64 wave_best[kWaves];
  const int t = threadIdx.x, r = blockIdx.x % a.rows, slice = blockIdx.x / a.rows;
  Row<kF32, 0> row(a, r, nullptr);
  row.begin = slice * p.slice;
  row.end = min(row.begin + p.slice, a.vocab);
  float top = -INFINITY;
  u32 at = 0;
  row.each([&](u32 i, float l) { /* indexes rise: the first of equals stays */
    at = l > top ? i : at;
    top = fmaxf(top, l);
  });
  const u32 k = key_of(top);
  u64 best = wave_max64(k ? (u64)k << 32 | (u32)~at : 0);
  if ((t & 63) == 0) {
    wave_best[t >> 6] = best;
  }
  __syncthreads();
  Shelf *shelf = reinterpret_cast<Shelf *>(p.ws + r * p.shelf);
  if (t == 0) {
    for (int w = 1; w < kWaves; ++w) {
      best = wave_best[w] > best ? wave_best[w] : best;
    }
    shelf->tops()[slice] = best;
  }
  if (slice == 0) {
    shelf->mass[t] = 0;
    shelf->count[t] = 0;
    if (t == 0) {
      shelf->n = 0;
      shelf->ticket = 0;
    }
  }
}

/* The row's first token, from its slices'. */
__device__ __forceinline__ u64 first_of(Shared &sh, Shelf *shelf, int slices) {
  const int t = threadIdx.x;
  u64 best = wave_max64(t < slices ? shelf->tops()[t] : 0);
  if ((t & 63) == 0) {
    sh.wave_m[t >> 6] = best;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    best = sh.wave_m[w] > best ? sh.wave_m[w] : best;
  }
  __syncthreads();
  return best;
}

/* A slice's weight, or its part of the row's histogram. */
template <bool kF32> __global__ __launch_bounds__(kThreads) void sample_weigh(SampleArgs a, Split p) {
  __shared__ Shared sh;
  const int t = threadIdx.x, r = blockIdx.x % a.rows, slice = blockIdx.x / a.rows;
  Shelf *shelf = reinterpret_cast<Shelf *>(p.ws + r * p.shelf);
  const Settings s = settings_of(a, r);
  const u64 first = first_of(sh, shelf, p.slices);
  if (!first || s.first) {
    return;
  }
  const Scale x = scale_of(a, s, logit_of((u32)(first >> 32)));
  Row<kF32, 0> row(a, r, nullptr);
  row.inf = x.inf;
  row.begin = slice * p.slice;
  row.end = min(row.begin + p.slice, a.vocab);
  sh.mass[t] = 0;
  sh.count[t] = 0;
  __syncthreads();
  if (!s.top_k && s.top_p >= 1.0f) {
    u64 sum = 0;
    unbordered(x, s, [&](auto keep) {
      row.template each<true>([&](u32 i, float l) { sum += keep(i, l); });
    });
    sum = block_sum(sh, sum);
    if (t == 0) {
      shelf->sums(p.slices)[slice] = sum;
    }
    return;
  }
  row.each([&](u32, float l) {
    if (l > -INFINITY) {
      const int b = x.bin(l);
      atomicAdd(&sh.count[b], 1u);
      if (!s.top_k) {
        atomicAdd(&sh.mass[b], x.weight(l));
      }
    }
  });
  __syncthreads();
  if (!s.top_k) {
    shelf->bins(p.slices, slice)[t] = sh.mass[t];
    if (sh.mass[t]) {
      __hip_atomic_fetch_add(&shelf->mass[t], sh.mass[t], __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (sh.count[t]) {
    __hip_atomic_fetch_add(&shelf->count[t], sh.count[t], __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
  }
}

/* The result of a row whose border top_p makes in a bin that is in the list,
 * with more tokens above it than a list holds: the border, then the slice that
 * the draw falls in, by the slices' bins, then the token. */
template <typename R>
__device__ __forceinline__ void finish_slices(const SampleArgs &a, Shared &sh, int r, R row, const Settings &s,
                              const Scale &x, const Where &at, const u64 *list, int n,
                              const Split &p, Shelf *shelf) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto both = [&](auto take) {
    for (int j = t; j < n; j += kThreads) {
      const u32 key = (u32)(list[j] >> 32);
      take(key, ~(u32)list[j], [&] { return x.weight(logit_of(key)); });
    }
  };
  auto by_key = [&](auto take) { both([&](u32 key, u32, auto weight) { take(key, weight); }); };
  const u64 want = part_of<true>(s.top_p, at.sum);
  const Point point = descend<true>(sh, by_key, max(key_of(x.least(at.f.bin)), 1u),
                                    key_of(x.ftop), at.f.above_mass, 0, want);
  const Keep<true, false> keep{x, 0.0, border_at(sh, both, point, ties_of(point.f, want), a.vocab)};
  /* the kept weight of each slice */
  __syncthreads();
  sh.mass[t] = 0;
  __syncthreads();
  both([&](u32 key, u32 i, auto weight) {
    if (keep.border.keeps(key, i)) {
      atomicAdd(&sh.mass[i / (u32)p.slice], weight());
    }
  });
  for (int sl = wave; sl < p.slices; sl += kWaves) {
    const u64 *bins = shelf->bins(p.slices, sl);
    u64 sum = 0;
    for (int b = lane; b < at.f.bin; b += 64) {
      sum += bins[b];
    }
    sum = wave_sum64(sum);
    if (lane == 0) {
      atomicAdd(&sh.mass[sl], sum);
    }
  }
  __syncthreads();
  const Drawn d = draw_part(sh, sh.mass[t], s.u);
  row.begin = d.at * p.slice;
  row.end = min(row.begin + p.slice, a.vocab);
  draw(a, sh, r, row, s.u, keep, d.total, d.target);
}

/* The rest: without a border the first slice finds the slice that the draw falls
 * in and its token; with one, the slices' tokens down to its bin (or, too many, of
 * that bin) meet in the workspace, and the last slice goes on with them. Where the
 * tokens are too many and top_k or min_p is on, one workgroup goes over the whole
 * row: 1 x 131072 f32 by top-k of 2000 123 us (133 undivided), by top-p 0.9999 with
 * min-p 1e-5 at a temperature of 1.5 113 (146), by that top-p alone 35 (146). */
template <bool kF32> __global__ __launch_bounds__(kThreads) void sample_settle(SampleArgs a, Split p) {
  __shared__ Shared sh;
  __shared__ u64 list[kBinList];
  __shared__ u32 base, last;
  const int t = threadIdx.x, r = blockIdx.x % a.rows, slice = blockIdx.x / a.rows;
  Shelf *shelf = reinterpret_cast<Shelf *>(p.ws + r * p.shelf);
  const Settings s = settings_of(a, r);
  if (slice != 0 && (s.first || (!s.top_k && s.top_p >= 1.0f))) {
    return; /* one workgroup is enough */
  }
  const u64 first = first_of(sh, shelf, p.slices);
  const float top = first ? logit_of((u32)(first >> 32)) : -INFINITY;
  if (!first || s.first) {
    if (slice == 0) {
      first_only(a, r, s, top, ~(u32)first);
    }
    return;
  }
  const Scale x = scale_of(a, s, top);
  Row<kF32, 0> row(a, r, nullptr);
  row.inf = x.inf;
  Row<kF32, 0> mine = row;
  mine.begin = slice * p.slice;
  mine.end = min(mine.begin + p.slice, a.vocab);
  __syncthreads();
  if (!s.top_k && s.top_p >= 1.0f) {
    const Drawn d = draw_part(sh, t < p.slices ? shelf->sums(p.slices)[t] : 0, s.u);
    mine.begin = d.at * p.slice;
    mine.end = min(mine.begin + p.slice, a.vocab);
    unbordered(x, s, [&](auto keep) { draw(a, sh, r, mine, s.u, keep, d.total, d.target); });
    return;
  }
  const Where at = locate(sh, s, shelf->mass[t], shelf->count[t]);
  const bool few = at.f.bin >= 0 && at.n <= (u32)kList;
  const bool one_bin = !few && !s.top_k && s.min_p == 0.0f && at.f.count <= (u32)kBinList;
  if (!few && !one_bin) {
    if (slice == 0) {
      finish_bins(a, sh, r, row, s, x, shelf->mass[t], shelf->count[t]);
    }
    return;
  }
  int n = few ? gather(sh, mine, x, at.bin, list) : gather<true>(sh, mine, x, at.f.bin, list);
  if (t == 0) {
    base = __hip_atomic_fetch_add(&shelf->n, (u32)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  for (int j = t; j < n; j += kThreads) {
    store_far(&shelf->list[base + j], list[j]);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (t == 0) {
    last = __hip_atomic_fetch_add(&shelf->ticket, 1u, __ATOMIC_RELAXED,
                                  __HIP_MEMORY_SCOPE_AGENT) == (u32)p.slices - 1;
  }
  __syncthreads();
  if (!last) {
    return;
  }
  n = few ? (int)at.n : (int)at.f.count; /* what the slices found in all */
  for (int j = t; j < n; j += kThreads) {
    (few ? sh.list_k : list)[j] = load_far(&shelf->list[j]);
  }
  __syncthreads();
  if (few) {
    finish(a, sh, r, s, x, n, at.sum, at.bin);
  } else {
    finish_slices(a, sh, r, row, s, x, at, list, n, p, shelf);
  }
}

template <bool kF32> void launch(const SampleArgs &a, const SamplePlan &plan, char *ws, hipStream_t stream) {
  const dim3 grid((unsigned)a.rows), block(kThreads);
  if (plan.slices > 1) {
    const Split p{plan.slices, plan.slice, ws, plan.ws_bytes / a.rows};
    const dim3 all((unsigned)(a.rows * plan.slices));
    hipLaunchKernelGGL((sample_tops<kF32>), all, block, 0, stream, a, p);
    hipLaunchKernelGGL((sample_weigh<kF32>), all, block, 0, stream, a, p);
    hipLaunchKernelGGL((sample_settle<kF32>), all, block, 0, stream, a, p);
    return;
  }
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

/* In us, several workgroups a row and one: 1 x 131072 f32 by top-k 22 and 25, by
 * top-p 23 and 69, without a border 20 and 48; 100 x 131072 without one 55 and
 * 59, 150 66 and 60, 256 92 and 73; 256 with one 190 and 226; 64 by top-k 38 and
 * 31, by top-p 60 and 122. At 50000 top-k 22 and 16, top-p 23 and 33. Up to 32768
 * one workgroup has the row in LDS (1 x 32000 12 and 23). */
SamplePlan sample_plan(int64_t rows, int64_t vocab, bool borders, bool may_split) {
  SamplePlan p{1, 0, 0};
  const int64_t chunks = (vocab + kChunk - 1) / kChunk;
  if (!may_split || vocab <= 32768 || rows > (borders ? 1024 : 128)) {
    return p;
  }
  /* slices of 1 to 8 chunks, as many as two workgroups a CU of 256 */
  const int64_t per = std::max<int64_t>(1, std::min<int64_t>(8, rows * chunks / 512));
  const int64_t slices = (chunks + per - 1) / per;
  if (slices > kThreads) {
    return p;
  }
  p.slices = (int)slices;
  p.slice = (int)(per * kChunk);
  p.ws_bytes = rows * (int64_t)(sizeof(Shelf) + slices * (16 + kBins * 8));
  return p;
}

void sample_launch(const SampleArgs &a, const SamplePlan &plan, char *ws, hipStream_t stream) {
  if (a.f32) {
    launch<true>(a, plan, ws, stream);
  } else {
    launch<false>(a, plan, ws, stream);
  }
  VX_HIP_CHECK(hipGetLastError());
}

} // namespace vxk
