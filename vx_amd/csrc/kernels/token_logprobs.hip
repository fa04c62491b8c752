/*
 * token_logprobs.hip -- log probabilities of given tokens, entropy, and the
 * likeliest tokens of rows of logits (vx_nn_token_logprobs_*).
 *
 * With m the largest logit, t = x - m and S = sum e^t: logprob = t - ln S, entropy
 * = ln S - (sum e^t t) / S. One pass over the row: each thread keeps sums against
 * a reference of its own, which moves only when a logit passes it by more than
 * kSlack, and the threads' sums meet at the end.
 *
 * The likeliest tokens: tokens have distinct 64-bit keys (the logit's order, then
 * the complement of the index), and each thread keeps the largest of its own. The
 * n largest of a row lie with the threads whose largest is at least the n-th of
 * the threads' largest: a few dozen threads, whose logits are read again, and
 * those not below that border go into a list in LDS, where each is compared with
 * all others. So ties need no case of their own.
 *
 * Rows fewer than CUs are divided: a workgroup a slice leaves its sums and its
 * likeliest in a workspace, logprobs_merge adds them up.
 *
 * 512 x 131071 bf16 with entropy and 20 alternatives 36 us, of which 31 without
 * alternatives (4.3 TB/s: the row's reading bounds it), 2048 x 32000 f32 44-47 (5.6-5.9
 * TB/s) and 55 with 5 alternatives. 1 x 32000 9.2: two launches, 6.5 for its two slices,
 * a chain of barriers and dependent loads, and 2.6 for the merge.
 */
#include "../vx_hip_common.h"
#include "../vx_packed_kernels.h"
#include "vx_wave_ops.hip.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace vxk {
namespace {

typedef unsigned long long u64;
typedef uint32_t u32;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;
constexpr float kFar = -1000.0f; /* e^kFar is 0 */
constexpr int kMostTop = 64;

/* Rises with l; 0 for -inf and NaN, which are no alternatives. */
__device__ __forceinline__ u32 order_of(float l) {
  const u32 b = __float_as_uint(l + 0.0f); /* -0 equals 0 */
  const u32 k = b ^ ((u32)((int32_t)b >> 31) | 0x80000000u);
  return l > -INFINITY ? k : 0u;
}
__device__ __forceinline__ u64 key_of(float l, int index) {
  const u32 k = order_of(l);
  return k ? (u64)k << 32 | (u32)~index : 0;
}
__device__ __forceinline__ float logit_of(u64 key) {
  const u32 k = (u32)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(u32)key; }

/* Sums against a reference m: s of e^(x - m), e of e^(x - m) (x - m). */
struct Sums {
  float m, s, e;
};
/* Against `top`, which is no lower than any logit in them. e^-1000 is 0 in f32, and s
 * times it too: the distance itself may be past the largest f32 (a part in which all
 * is masked by the type's lowest value), and 0 times infinity a NaN. */
__device__ __forceinline__ Sums against(Sums v, float top) {
  const float d = fmaxf(v.m - top, kFar);
  const float f = __builtin_amdgcn_exp2f(d * kLog2e);
  return v.s > 0.0f ? Sums{top, v.s * f, f * (v.e + v.s * d)} : Sums{top, 0.0f, 0.0f};
}

__device__ __forceinline__ u64 wave_min_key(u64 v) {
  auto meet = [&](auto step) {
    constexpr int kO = decltype(step)::value;
    const u64 o = (u64)partner_word<kO>((u32)(v >> 32)) << 32 | partner_word<kO>((u32)v);
    v = min(v, o);
  };
  meet(std::integral_constant<int, 1>{});
  meet(std::integral_constant<int, 2>{});
  meet(std::integral_constant<int, 4>{});
  meet(std::integral_constant<int, 8>{});
  meet(std::integral_constant<int, 16>{});
  meet(std::integral_constant<int, 32>{});
  return v;
}

template <bool kF32> struct Elements {
  static constexpr int kVec = kF32 ? 4 : 8; /* of a 16-byte load */
  const void *row;
  __device__ __forceinline__ float at(int64_t i) const {
    return kF32 ? static_cast<const float *>(row)[i] : bf16_to_f32(static_cast<const uint16_t *>(row)[i]);
  }
  __device__ __forceinline__ u32x4 raw(int64_t i) const {
    return *reinterpret_cast<const u32x4 *>(static_cast<const char *>(row) + i * (kF32 ? 4 : 2));
  }
  static __device__ __forceinline__ void open(u32x4 w, float (&x)[kVec]) {
    if constexpr (kF32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
};

/* What a row's parts come to. */
struct Row {
  float top, log_sum, entropy;
  bool inf; /* a logit is +inf: those alone count, equally */
};
/* From the sums against `top`, or how many are +inf. Rounding may leave an entropy
 * below 0; a NaN stays one. */
__device__ __forceinline__ Row row_of(float top, float s, float e, int infs) {
  if (top == INFINITY) {
    const float n = logf((float)infs);
    return Row{top, n, n, true};
  }
  if (!(top > -INFINITY)) {
    return Row{top, 0.0f, 0.0f, false};
  }
  const float log_sum = logf(s), entropy = log_sum - e / s;
  return Row{top, log_sum, entropy < 0.0f ? 0.0f : entropy, false};
}
__device__ __forceinline__ float logprob_of(const Row &r, float x) {
  if (r.inf) {
    return x == INFINITY ? -r.log_sum : -INFINITY;
  }
  return x > -INFINITY ? (x - r.top) - r.log_sum : -INFINITY;
}

/* A slice's result in the workspace: sums against its largest logit, how many
 * are +inf, then its likeliest keys in falling order (0: none). */
struct Part {
  float top, s, e;
  int infs;
  u64 keys[kMostTop];
};

template <int kThreads> struct Shared {
  static constexpr int kWaves = kThreads / 64;
  static constexpr int kList = kThreads < 256 ? 8 * kThreads : 2048; /* above 64 */
  float a[kWaves], b[kWaves];
  int n[kWaves];
  u64 best[kThreads];
  u64 border, list[kList];
  int threads, count;
  int which[64];
};

/* The n largest keys of the list, in falling order, to `put`; what is not there
 * is 0. Eight lanes compare a key with an eighth of the others each. */
template <int kThreads, typename Put>
__device__ __forceinline__ void in_order(const u64 *list, int count, int n, Put put) {
  const int part = threadIdx.x & 7;
  for (int i0 = 0; i0 < count; i0 += kThreads / 8) {
    const int i = i0 + (int)threadIdx.x / 8;
    const u64 mine = list[min(i, count - 1)];
    int above = 0;
#pragma unroll 4
    for (int j = part; j < count; j += 8) {
      above += list[j] > mine;
    }
    above += (int)partner_word<1>((u32)above);
    above += (int)partner_word<2>((u32)above);
    above += (int)partner_word<4>((u32)above);
    if (part == 0 && i < count && above < n) {
      put(above, mine);
    }
  }
  for (int i = count + threadIdx.x; i < n; i += kThreads) {
    put(i, 0);
  }
}

template <int kThreads>
__device__ __forceinline__ void write_given(const LogprobArgs &a, int64_t r, const Row &row) {
  for (int i = threadIdx.x; i < a.n_given; i += kThreads) {
    const int64_t at = r * a.n_given + i;
    const int token = a.given[at];
    float lp = -INFINITY;
    if (token >= 0 && token < a.vocab) {
      const Elements<true> f{static_cast<const float *>(a.logits) + (a.f32 ? r * a.stride : 0)};
      const Elements<false> h{static_cast<const uint16_t *>(a.logits) + (a.f32 ? 0 : r * a.stride)};
      lp = logprob_of(row, a.f32 ? f.at(token) : h.at(token));
    }
    a.logprob[at] = lp;
  }
}

template <bool kF32, int kThreads, bool kSliced>
__global__ __launch_bounds__(kThreads) void logprobs_rows(LogprobArgs a, LogprobPlan plan, Part *parts) {
  constexpr int kVec = Elements<kF32>::kVec;
  constexpr int kWaves = kThreads / 64;
  constexpr int kList = Shared<kThreads>::kList;
  __shared__ Shared<kThreads> sh;
  const int t = threadIdx.x;
  const int lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t r = kSliced ? blockIdx.x / plan.slices : blockIdx.x;
  const int slice = kSliced ? (int)(blockIdx.x - r * plan.slices) : 0;
  const Elements<kF32> x{static_cast<const char *>(a.logits) + r * a.stride * (kF32 ? 4 : 2)};
  const int begin = kSliced ? min(slice * plan.slice, a.vocab) : 0;
  const int end = kSliced ? min(begin + plan.slice, a.vocab) : a.vocab;
  /* [begin, lead) up to a 16-byte boundary and [tail, end) after the last whole
   * vector go element by element, a thread each */
  const int off = (int)(((uintptr_t)x.row / (kF32 ? 4 : 2) + begin) & (kVec - 1));
  const int lead = min(begin + (off ? kVec - off : 0), end);
  const int vectors = (end - lead) / kVec;
  const int tail = lead + vectors * kVec;
  const int singles = (lead - begin) + (end - tail);
  const int single = t < lead - begin ? begin + t : tail + (t - (lead - begin));

  Sums acc{-INFINITY, 0.0f, 0.0f};
  float best = -INFINITY;
  int best_at = 0;
  auto take = [&](auto &v, int first, auto count) {
    constexpr int kN = decltype(count)::value;
    float vm = v[0]; /* fmaxf leaves NaNs out */
#pragma unroll
    for (int e = 1; e < kN; ++e) {
      vm = fmaxf(vm, v[e]);
    }
    if (vm > best) {
      best = vm;
#pragma unroll
      for (int e = kN - 1; e >= 0; --e) {
        best_at = v[e] == vm ? first + e : best_at;
      }
    }
    if (vm > acc.m + kSlack || (acc.m == -INFINITY && vm > -INFINITY)) {
      acc = against(acc, vm);
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      /* -inf and NaN weigh nothing */
      const float d = fmaxf(v[e] - acc.m, kFar);
      const float w = __builtin_amdgcn_exp2f(d * kLog2e);
      acc.s += w;
      acc.e = __builtin_fmaf(w, d, acc.e);
    }
  };
  if (t < singles) {
    float v[1] = {x.at(single)};
    take(v, single, std::integral_constant<int, 1>{});
  }
  constexpr int kAhead = 4;
  for (int i0 = t; i0 < vectors; i0 += kAhead * kThreads) {
    u32x4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      w[i] = x.raw(lead + (int64_t)min(i0 + i * kThreads, vectors - 1) * kVec);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i * kThreads < vectors) {
        float v[kVec];
        Elements<kF32>::open(w[i], v);
        take(v, lead + (i0 + i * kThreads) * kVec, std::integral_constant<int, kVec>{});
      }
    }
  }
  /* A single of the tail comes before the thread's vectors above: a vector's
   * equal logit has the lower index. */
  if (t < singles && single >= tail && best_at == single) {
    for (int i = t; i < vectors; i += kThreads) {
      float v[kVec];
      Elements<kF32>::open(x.raw(lead + (int64_t)i * kVec), v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int at = lead + i * kVec + e;
        best_at = v[e] == best && at < best_at ? at : best_at;
      }
    }
  }

  /* the row's largest, then its sums against it */
  const float wm = wave_max(best);
  if (lane == 0) {
    sh.a[wave] = wm;
  }
  sh.best[t] = key_of(best, best_at);
  __syncthreads();
  float top = sh.a[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) {
    top = fmaxf(top, sh.a[i]);
  }
  __syncthreads();
  const bool none = !(top > -INFINITY), inf = top == INFINITY;
  int infs = 0;
  if (inf) {
    for (int i = begin + t; i < end; i += kThreads) {
      infs += x.at(i) == INFINITY;
    }
    infs = wave_sum_int(infs);
  }
  const Sums mine = none || inf ? Sums{0, 0, 0} : against(acc, top);
  const float ws = wave_sum(mine.s), we = wave_sum(mine.e);
  if (lane == 0) {
    sh.a[wave] = ws;
    sh.b[wave] = we;
    sh.n[wave] = infs;
  }
  __syncthreads();
  float s = 0.0f, e = 0.0f;
  infs = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    s += sh.a[i];
    e += sh.b[i];
    infs += sh.n[i];
  }
  const Row row = row_of(top, s, e, infs);
  if constexpr (kSliced) {
    if (t == 0) {
      Part &p = parts[blockIdx.x];
      p.top = top;
      p.s = s;
      p.e = e;
      p.infs = infs;
    }
  } else {
    write_given<kThreads>(a, r, row);
    if (a.entropy && t == 0) {
      a.entropy[r] = row.entropy;
    }
  }
  const int n = a.n_top;
  if (n == 0) {
    return;
  }

  /* A border with at least n threads' largest at or above it and not many more
   * (or all, where there are no n): one wave halves the keys' range. */
  if (wave == 0) {
    u64 k[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      k[i] = sh.best[i * 64 + lane];
    }
    auto from = [&](u64 b) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k[i] >= b));
      }
      return c;
    };
    /* from(lo) >= n > from(hi), if there are n: all from the least on */
    u64 lo = k[0], hi = key_of(top, 0) + 1;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
      lo = min(lo, k[i]);
    }
    lo = max(wave_min_key(lo), (u64)1);
    int c = from(lo);
    const int most = max(n, kThreads / 16);
    while (c > most) {
      const u64 mid = lo + (hi - lo) / 2;
      const int m = from(mid);
      if (m >= n) {
        lo = mid;
        c = m;
      } else {
        hi = mid;
      }
    }
    if (lane == 0) {
      sh.border = lo;
      sh.threads = c;
    }
    int at = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const u64 in = __builtin_amdgcn_ballot_w64(k[i] >= lo);
      if (k[i] >= lo) {
        sh.which[at + __builtin_popcountll(in & ((1ull << lane) - 1))] = i * 64 + lane;
      }
      at += __builtin_popcountll(in);
    }
  }
  __syncthreads();
  const int threads = sh.threads;
  u64 lo = sh.border, hi = 0;
  /* Their keys from the border on into the list; where they do not fit, a higher
   * border that still leaves n. */
  int count;
  for (;;) {
    if (t == 0) {
      sh.count = 0;
    }
    __syncthreads();
    auto add = [&](u64 key) {
      if (key >= lo) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) {
          sh.list[at] = key;
        }
      }
    };
    if (t < threads && sh.which[t] < singles) {
      const int owner = sh.which[t];
      const int at = owner < lead - begin ? begin + owner : tail + (owner - (lead - begin));
      add(key_of(x.at(at), at));
    }
    /* every vector of theirs, a thread one at a time */
    const int per = (vectors + kThreads - 1) / kThreads;
    for (int i = t; i < per * threads; i += kThreads) {
      const int v = sh.which[i % threads] + i / threads * kThreads;
      if (v < vectors) {
        float el[kVec];
        Elements<kF32>::open(x.raw(lead + (int64_t)v * kVec), el);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          add(key_of(el[j], lead + v * kVec + j));
        }
      }
    }
    __syncthreads();
    count = sh.count;
    __syncthreads();
    if (count <= kList && (count >= n || hi == 0)) {
      break;
    }
    /* the keys that are n-th or higher are between lo (too many) and hi (too few) */
    if (hi == 0) {
      hi = key_of(top, 0) + 1;
      sh.border = lo;
    }
    if (count > kList) {
      sh.border = lo;
    } else {
      hi = lo;
    }
    __syncthreads();
    lo = sh.border + (hi - sh.border) / 2;
    __syncthreads();
  }
  if constexpr (kSliced) {
    Part &p = parts[blockIdx.x];
    in_order<kThreads>(sh.list, count, n, [&](int i, u64 key) { p.keys[i] = key; });
  } else {
    in_order<kThreads>(sh.list, count, n, [&](int i, u64 key) {
      a.top_tokens[r * n + i] = key ? index_of(key) : -1;
      if (a.top_logprob) {
        a.top_logprob[r * n + i] = key ? logprob_of(row, logit_of(key)) : -INFINITY;
      }
    });
  }
}

constexpr int kMergeThreads = 256;
constexpr int kMostSlices = 16;

__global__ __launch_bounds__(kMergeThreads) void logprobs_merge(LogprobArgs a, LogprobPlan plan,
                                                               const Part *parts) {
  __shared__ u64 list[kMostSlices * kMostTop];
  __shared__ int real;
  const int64_t r = blockIdx.x;
  const Part *mine = parts + r * plan.slices;
  const int n = a.n_top, all = n * plan.slices;
  if (threadIdx.x == 0) {
    real = 0;
  }
  __syncthreads();
  /* keys of 0 are none */
  for (int i = threadIdx.x; i < all; i += kMergeThreads) {
    const u64 key = mine[i / n].keys[i % n];
    if (key) {
      list[atomicAdd(&real, 1)] = key;
    }
  }
  /* a lane a slice, on every wave */
  const int lane = threadIdx.x & 63;
  const bool has = lane < plan.slices;
  const Part &part = mine[min(lane, plan.slices - 1)];
  const Sums own{part.top, part.s, part.e};
  const float top = wave_max(own.m);
  const int infs = wave_sum_int(has ? part.infs : 0);
  const bool none = !(top > -INFINITY), inf = top == INFINITY;
  const Sums v = has && !none && !inf ? against(own, top) : Sums{0.0f, 0.0f, 0.0f};
  const float s = wave_sum(v.s), e = wave_sum(v.e);
  const Row row = row_of(top, s, e, infs);
  write_given<kMergeThreads>(a, r, row);
  if (a.entropy && threadIdx.x == 0) {
    a.entropy[r] = row.entropy;
  }
  __syncthreads();
  in_order<kMergeThreads>(list, real, n, [&](int i, u64 key) {
    a.top_tokens[r * n + i] = key ? index_of(key) : -1;
    if (a.top_logprob) {
      a.top_logprob[r * n + i] = key ? logprob_of(row, logit_of(key)) : -INFINITY;
    }
  });
}

template <bool kF32, int kThreads>
void launch_rows(const LogprobArgs &a, const LogprobPlan &plan, hipStream_t stream) {
  hipLaunchKernelGGL((logprobs_rows<kF32, kThreads, false>), dim3((unsigned)a.rows), dim3(kThreads), 0,
                     stream, a, plan, nullptr);
}

/* Threads by the row's length, in us: 4096 x 1000 9.0 by 64, 14.9 by 256; 4096 x
 * 4000 18.7 by 128, 19.9 by 64; 4096 x 8000 34 by 256, 39 by 128 or 512; 2048 x
 * 32000 55 by 512, 60 by 1024; 512 x 131071 37 by 1024, 41 by 512. */
template <bool kF32>
void launch(const LogprobArgs &a, const LogprobPlan &plan, Part *parts, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.rows * plan.slices));
  if (plan.slices > 1) {
    hipLaunchKernelGGL((logprobs_rows<kF32, 512, true>), grid, dim3(512), 0, stream, a, plan, parts);
    hipLaunchKernelGGL(logprobs_merge, dim3((unsigned)a.rows), dim3(kMergeThreads), 0, stream, a, plan,
                       parts);
  } else if (a.vocab <= 2048) {
    launch_rows<kF32, 64>(a, plan, stream);
  } else if (a.vocab <= 4096) {
    launch_rows<kF32, 128>(a, plan, stream);
  } else if (a.vocab <= 12288) {
    launch_rows<kF32, 256>(a, plan, stream);
  } else if (a.vocab <= 49152) {
    launch_rows<kF32, 512>(a, plan, stream);
  } else {
    launch_rows<kF32, 1024>(a, plan, stream);
  }
}

} // namespace

/* Slices of a row: as many as give 256 workgroups, of at least 12288 logits, and
 * with no more than 160 alternatives in all, which the merge compares each with
 * each. In us, undivided and in 2, 4, 8 and 16: 1 x 131072 with 5 alternatives 18,
 * 16.2, 11.8, 10.3 and 10.2; 1 x 50257 10.8, 10.8, 9.7, 9.6 and 10.4; 16 x 131072
 * with 20 17.7, 15.3, 13.2, 13.3 and 19.9; 64 rows 20.2, 19.4, 15.7, 17.2 and 25;
 * 128 rows 22.2, 21.5, 20.7, 22.9 and 32 (more workgroups than CUs gain 4% there, and
 * nothing with 64 rows). */
LogprobPlan logprobs_plan(int64_t rows, int64_t vocab, int64_t n_top, bool may_split) {
  LogprobPlan p{1, (int)vocab, 0};
  const int64_t want = std::min<int64_t>(
      {256 / rows, vocab / 12288, kMostSlices, 160 / std::max<int64_t>(n_top, 1)});
  if (may_split && want > 1) {
    p.slice = (int)(((vocab + want - 1) / want + 63) / 64 * 64);
    p.slices = (int)((vocab + p.slice - 1) / p.slice);
    p.ws_bytes = rows * p.slices * (int64_t)sizeof(Part);
  }
  return p;
}

void logprobs_launch(const LogprobArgs &a, const LogprobPlan &plan, char *ws, hipStream_t stream) {
  Part *parts = reinterpret_cast<Part *>(ws);
  a.f32 ? launch<true>(a, plan, parts, stream) : launch<false>(a, plan, parts, stream);
}

} // namespace vxk
