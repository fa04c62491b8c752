/*
 * flash_shared.hip -- attention over a prefix that all sequences share and
 * each sequence's own cache (vx_nn_flash_attention_shared_bf16), bf16 in, f32
 * accumulate, bf16 out, f32 log-sum-exp.
 *
 * A query's keys are two segments: the shared ones, the same for every
 * sequence, then its sequence's own. All queries of a KV head, of every
 * sequence and of the heads that read it, can so be rows of one product with
 * the shared keys. With few queries a sequence the shared keys are read by
 * tiles of such rows ("wide": 128 or 64 rows; up to 16 rows: "rows"), the own
 * keys by each sequence's queries alone, several workgroups divide either, and
 * flash_shared_merge adds the parts up. With many queries a sequence (or
 * without a workspace) a tile holds queries of one sequence and walks both
 * segments; nothing is left to merge.
 *
 * wide: 4 waves, K and V through a two-slot LDS ring by buffer-to-LDS loads;
 * as in flash_attn.hip the products are transposed, S^T = K Q^T and O^T += V^T
 * P^T (v_mfma_f32_32x32x16_bf16), so that a lane holds one query's scores and
 * P^T is the scores' accumulator rounded in place. 64 rows: two halves of the
 * workgroup divide the keys and meet in LDS.
 * The weights are rounded to bf16, off by at most 2^-8 each, because the second
 * product's operands are bf16 (f32 ones multiply at a sixteenth of the rate);
 * maxima, sums and partial results stay in f32, the sums over unrounded weights.
 * Outputs are so off by 2.3e-3 in the root mean square, where the rounding of an
 * output alone makes 1.7e-3.
 * rows: K and V straight from memory into v_mfma_f32_16x16x32_bf16 operands,
 * four waves dividing the keys, as flash_rows.hip.
 *
 * A block in which a key is hidden from one of a wave's queries and not from
 * another goes a key at a time where V there holds infinities or NaNs (0 x inf
 * is NaN), each key for the queries that see it.
 *
 * 16 sequences, 32 heads on 8 of 128, over 65536 shared keys and own caches of up
 * to 1024 (7176 keys in all): 58 us for 298 MB of keys, 5.1 TB/s, and 5 for the
 * merge: the keys' bytes bound it. 64 on 4 KV heads over 8192: 25 and 5.3, where 10
 * would read the keys and 7 multiply; a workgroup of 128 rows, one wave a SIMD,
 * spends 8 us of its 25 before its first and after its last block of 64 keys, and
 * 1.7 on each. 8 sequences of 256 queries, 32 heads on 8, over 4096 and 300 own,
 * causal: 172 to 187 us from one card to another, 830 to 760 TFLOP/s.
 */
#include "../vx_batch_kernels.h"
#include "../vx_hip_common.h"
#include "vx_lds_dma.hip.h"
#include "vx_mfma16.hip.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace vxk {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
using shared::kBK;
constexpr int kRK = 32;        /* keys per block of a rows tile */
constexpr float kSlack = 8.0f; /* base-2 headroom of the stale row max */
constexpr float kLn2 = 0.69314718055994531f;

struct KernelArgs {
  SharedAttnArgs a;
  float scale_log2; /* above 0 */
  uint32_t q_and, q_xor;
  int group, rows_seq; /* heads of a KV head; their queries of one sequence */
  SharedPlan p;
  char *ws;
};

/* The workspace's part `part`: [rows][kD] sums, then [rows] statistics (max in
 * base 2, weight). */
template <int kD> __device__ __forceinline__ float *part_of(const KernelArgs &p, int part) {
  return reinterpret_cast<float *>(p.ws) + part * shared::part_floats(p.p.rows, kD);
}

struct Segment {
  const uint16_t *k, *v;
  int keys;
};

/* What a tile works on: rows row0 .. of KV head kv (all sequences' where
 * `b` is -1, else sequence b's), blocks first .. last - 1 of its segments'
 * blocks one after the other, and the part they become (-1: the result). */
struct Item {
  int kv, b, row0, part;
  Segment seg[2];
  int blocks0, first, last;
  int end; /* the last block any query of the tile sees */

  __device__ __forceinline__ const uint16_t *k(int s) const { return s ? seg[1].k : seg[0].k; }
  __device__ __forceinline__ const uint16_t *v(int s) const { return s ? seg[1].v : seg[0].v; }
  __device__ __forceinline__ int keys(int s) const { return s ? seg[1].keys : seg[0].keys; }
};

__device__ __forceinline__ int own_keys(const SharedAttnArgs &a, int b) {
  const int n = a.lens ? a.lens[b] : a.capacity;
  return n > a.capacity ? -1 : n;
}

/* Row r of an item's tile: its place among all queries (-1: past the last),
 * the last key it sees, counted from the first shared one, and whether its
 * slot holds a sequence. */
struct Row {
  int place, limit;
  bool real;
};
__device__ __forceinline__ Row row_of(const KernelArgs &p, int kv, int b, int r) {
  const int rem = b >= 0 ? r : r % p.rows_seq;
  b = b >= 0 ? b : r / p.rows_seq;
  if (b >= p.a.batch || rem >= p.rows_seq) {
    return Row{-1, -1, false};
  }
  const int own = own_keys(p.a, b);
  const int total = p.a.shared_len + own;
  const int i = rem % p.a.seq_q;
  return Row{(b * p.a.heads + kv * p.group) * p.a.seq_q + rem,
             p.a.causal ? min(total - 1, total - p.a.seq_q + i) : total - 1, own >= 0};
}

/* Eight elements of a row's query, from column c on; of a row that is none they
 * stay in its own column of every product. The scale's sign goes into the query,
 * so that a hidden key's score is -inf whatever the scale. */
__device__ __forceinline__ u32x4 query(const KernelArgs &p, const Row &row, int head_dim, int c) {
  u32x4 q = {0, 0, 0, 0};
  if (row.place >= 0) {
    q = *reinterpret_cast<const u32x4 *>(p.a.q + (int64_t)row.place * head_dim + c);
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    q[w] = (q[w] & p.q_and) ^ p.q_xor;
  }
  return q;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

/* Not 0 where one of a word's two bf16 is infinite or NaN. */
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

/* The lane's number, read again: an address made from it where it is used needs
 * no register in between. */
__device__ __forceinline__ int lane_here() {
  int v;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(v));
  return v;
}

__device__ __forceinline__ int wave_min(int v) {
  for (int o = 32; o; o >>= 1) {
    v = min(v, __shfl_xor(v, o));
  }
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
  for (int o = 32; o; o >>= 1) {
    v = max(v, __shfl_xor(v, o));
  }
  return v;
}

/* The block (of `size` keys) that holds key `limit`; -1 for none. */
__device__ __forceinline__ int block_of(const Item &it, int limit, int size) {
  return limit == INT32_MAX        ? INT32_MAX
         : limit < 0               ? -1
         : limit < it.seg[0].keys ? limit / size
                                  : it.blocks0 + (limit - it.seg[0].keys) / size;
}

/* The least and the greatest limit of the wave's rows; of real ones only, and
 * INT32_MAX and -1 where there are none. */
struct Limits {
  int lo, hi;
};
__device__ __forceinline__ Limits limits_of(const KernelArgs &p, const Item &it, const Row &row) {
  const bool real = row.real;
  const int all = it.keys(0) + it.keys(1) - 1;
  /* most often every row sees all of the item's keys */
  if (__builtin_amdgcn_ballot_w64(real && row.limit < all) == 0) {
    return Limits{INT32_MAX, __builtin_amdgcn_ballot_w64(real) ? INT32_MAX : -1};
  }
  return Limits{__builtin_amdgcn_readfirstlane(wave_min(real ? row.limit : INT32_MAX)),
                __builtin_amdgcn_readfirstlane(wave_max(real ? row.limit : -1))};
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

/* x of lanes l and l ^ 32, in some order. */
__device__ __forceinline__ f32x2 halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

/* Where a 16-byte chunk c of key row `row` lies in its LDS plane: K so that a
 * read of 16 rows at one chunk meets every bank, V so that the transposing
 * read (4 rows x 32 bytes per 16 lanes) does. */
template <int kChunks> __device__ __forceinline__ int place_k(int row, int c) {
  if constexpr (kChunks == 16) {
    return c ^ (row & 15);
  } else {
    return c ^ (row & 7) ^ ((row >> 3) & 1);
  }
}
template <int kChunks> __device__ __forceinline__ int place_v(int key, int c) {
  const int q = key & 3;
  if constexpr (kChunks >= 16) {
    return c ^ ((q << 1) ^ (q << 2));
  } else {
    return c ^ (q << 1);
  }
}

/* The last d-step of a query waits in LDS where its registers would be spilled
 * (to memory, whose reload waits for the keys in flight). */
template <int kD, int kGroups> constexpr bool kParkQ = kD == 128 && kGroups == 1;
template <int kD, int kGroups> constexpr int wide_lds() {
  return 4 * kBK * kD * 2 + (kParkQ<kD, kGroups> ? kThreads * 16 : 0);
}

/* A tile of 128 / kGroups rows. */
template <int kD, int kGroups>
__device__ __forceinline__ void wide(const KernelArgs &p, const Item &it, char *lds) {
  constexpr int kTileKeys = kBK / kGroups; /* a group's block: kBK keys at one group */
  constexpr int kKT = kTileKeys / 32;
  constexpr int kKS = kTileKeys / 16;
  constexpr int kChunks = kD / 8;
  constexpr int kUnits = kTileKeys * kChunks;
  constexpr int kGroupThreads = kThreads / kGroups;
  constexpr int kWavesQ = 4 / kGroups;
  constexpr int kLoads = kUnits / kGroupThreads;
  constexpr int kDSteps = kD / 16;
  constexpr int kDTiles = kD / 32;
  constexpr int kRowBytes = kD * 2;

  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63;
  const int lq = lane & 31;
  const int g = lane >> 5;
  const int grp = kGroups == 1 ? 0 : wave / kWavesQ;
  const int wq = kGroups == 1 ? wave : wave % kWavesQ;

  /* Load l of a thread fills unit l * kGroupThreads + tg of a plane: key row
   * l * kRowsPer + tg / kChunks, whose place differs from l = 0's by an XOR. */
  constexpr int kRowsPer = kGroupThreads / kChunks;
  static_assert(kChunks == 16 ? 16 % kRowsPer == 0 && kRowsPer % 4 == 0 : kRowsPer % 16 == 0,
                "places of the loads of a thread");
  /* [group][slot][K|V][unit] */
  u32x4 *ring = reinterpret_cast<u32x4 *>(lds) + grp * 4 * kUnits;
  const uint32_t ring_base = (uint32_t)(uintptr_t)(VX_LDS void *)ring;
  struct At {
    int seg, key0;
  };
  auto at_turn = [&](int j) {
    const int blk = it.first + j * kGroups + grp;
    const int seg = blk < it.blocks0 ? 0 : 1;
    return At{seg, (blk - (seg ? it.blocks0 : 0)) * kTileKeys};
  };
  auto issue = [&](int j, int plane) {
    const At x = at_turn(j);
    const int bytes = max(0, min(kTileKeys, it.keys(x.seg) - x.key0)) * kRowBytes;
    const uint16_t *src = plane == 0 ? it.k(x.seg) : it.v(x.seg);
    i32x4 rs = buffer_rsrc(src + (int64_t)x.key0 * kD, bytes);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      rs[w] = __builtin_amdgcn_readfirstlane(rs[w]); /* uniform, which the compiler cannot tell */
    }
    const uint32_t base = ring_base + (uint32_t)((((j & 1) * 2 + plane) * kUnits + wq * 64) * 16);
    const uint32_t tg = (uint32_t)(wq * 64 + lane_here());
    const int row = (int)(tg / kChunks), c = (int)(tg % kChunks);
    const int off =
        row * kRowBytes + (plane == 0 ? place_k<kChunks>(row, c) : place_v<kChunks>(row, c)) * 16;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int turn = plane == 0 && kChunks == 16 ? (l * kRowsPer & 15) << 4 : 0;
      dma16(rs, (uint32_t)((off ^ turn) + l * kRowsPer * kRowBytes),
            base + (uint32_t)(l * kGroupThreads * 16));
    }
  };

  /* Turns: a group's j-th block is first + j * kGroups + grp. The first two of K
   * and the first of V are on their way before anything else is looked at. */
  const int end = min(it.last - 1, it.end) + 1;
  const int turns = end > it.first ? (end - it.first + kGroups - 1) / kGroups : 0;
  if (turns > 0) {
    issue(0, 0);
    issue(0, 1);
    if (turns > 1) {
      issue(1, 0);
    }
  }

  const Row row = row_of(p, it.kv, it.b, it.row0 + 32 * wq + lq);
  const bool real = row.real;
  u32x4 qf[kDSteps];
#pragma unroll
  for (int s = 0; s < kDSteps; ++s) {
    qf[s] = query(p, row, kD, 8 * g + 16 * s);
  }
  const Limits lim = limits_of(p, it, row);
  const int limit = real ? row.limit : lim.hi;
  const int lim_lo = lim.lo;
  /* the last block any of the wave's queries sees */
  const int wave_last = min(end - 1, block_of(it, lim.hi, kTileKeys));
  VX_LDS u32x4 *parked = (VX_LDS u32x4 *)(lds + 4 * kBK * kD * 2) + t;
  if constexpr (kParkQ<kD, kGroups>) {
    *parked = qf[kDSteps - 1];
  }


  /* Where the lane reads in a slot's K plane (row lq, chunk g: chunk 2 ds + g
   * of a place that is an XOR lies at the address XOR 32 ds) and, transposing,
   * in its V plane: key 4 g + i / 4 of a 16-key step, d 16 j + 4 (i % 4) of a
   * 32-wide tile, i = lane % 16, j = lane / 16 % 2, which hands it the 8 keys
   * of its k-slots at d = lane % 32; tile i lies at XOR 64 i. */
  auto keys_at = [&](int j) {
    const int l = lane_here();
    return ring_base + (uint32_t)((j & 1) * 2 * kUnits * 16 + (l & 31) * kRowBytes +
                                  place_k<kChunks>(l & 31, l >> 5) * 16);
  };
  auto values_at = [&](int j) {
    const int l = lane_here();
    const int key = 4 * (l >> 5) + ((l & 15) >> 2);
    const int d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
    return ring_base + (uint32_t)(((j & 1) * 2 + 1) * kUnits * 16 + key * kRowBytes +
                                  place_v<kChunks>(key, d >> 3) * 16 + (d & 7) * 2);
  };

  f32x16 o[kDTiles];
#pragma unroll
  for (int i = 0; i < kDTiles; ++i) {
    o[i] = f32x16{};
  }
  float m_run = -INFINITY, l_run = 0.0f;

  typedef f32x16 Scores[kKT];
  auto scores = [&](int j, Scores &st) {
    const uint32_t at = keys_at(j);
#pragma unroll
    for (int ds = 0; ds < kDSteps; ++ds) {
      const u32x4 q = kParkQ<kD, kGroups> && ds == kDSteps - 1 ? *parked : qf[ds];
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt) {
        const u32x4 a =
            *(const VX_LDS u32x4 *)(uintptr_t)((at ^ (uint32_t)(ds << 5)) + (uint32_t)(kt * 32 * kRowBytes));
        st[kt] = mfma32(a, q, ds == 0 ? f32x16{} : st[kt]);
      }
    }
  };

  const float scale = p.scale_log2;
  /* A hidden key's score is -inf, and its weight 2^-inf = 0. */
  auto softmax = [&](Scores &st, u32x4 (&pt)[kKS], float &alpha) -> bool {
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        mx = fmaxf(mx, st[kt][r]);
      }
    }
    const f32x2 m2 = halves(mx);
    mx = fmaxf(m2[0], m2[1]) * scale;
    /* The reference max moves only when a block's passes it by more than
     * kSlack, and always from -inf. */
    const bool bump = mx > m_run + kSlack;
    const float m_next = bump ? mx : m_run;
    const float m_use = m_next == -INFINITY ? 0.0f : m_next;
    alpha = bump ? __builtin_amdgcn_exp2f(m_run - m_use) : 1.0f;
    float sum = 0.0f;
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][8 * h + i], scale, -m_use));
          sum += e[i];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          pt[2 * kt + h][w] = pack2(e[2 * w], e[2 * w + 1]);
        }
      }
    }
    const f32x2 s2 = halves(sum);
    l_run = l_run * alpha + s2[0] + s2[1];
    m_run = m_next;
    return bump;
  };

  /* V^T's operand of 16-key step ks and d tile i of turn j. */
  auto values = [&](uint32_t at, int ks, int i) {
    u32x4 a;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 w = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (VX_LDS i16x4 *)(uintptr_t)((at ^ (uint32_t)(i << 6)) +
                                                 (uint32_t)((16 * ks + 8 * h) * kRowBytes))));
      a[2 * h] = w[0];
      a[2 * h + 1] = w[1];
    }
    return a;
  };
  auto accumulate = [&](int j, const u32x4 (&pt)[kKS]) {
    const uint32_t at = values_at(j);
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
        o[i] = mfma32(values(at, ks, i), pt[ks], o[i]);
      }
    }
    /* the transposing reads run ahead of the products that take them */
    constexpr int kLead = kKS * kDTiles >= 8 ? 8 : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, kLead, 0); /* DS read */
#pragma unroll
    for (int s = 0; s < (2 * kKS * kDTiles - kLead) / 2; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); /* MFMA */
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kLead / 2, 0);
  };
  /* The same a key at a time, each for the queries that see it: those whose
   * last key of the block, `seen`, is no lower. */
  auto accumulate_apart = [&](int j, const u32x4 (&pt)[kKS], int seen) {
    const uint32_t at = values_at(j);
    const int vg = lane_here() >> 5;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
#pragma unroll 1
      for (int n = 0; n < 16; ++n) {
        /* slot e of a lane: key 4 g + e of the step, from e = 4 on 8 more */
        const int e = (n & 3) + 4 * (n >> 3);
        const uint32_t half = ((n >> 2) & 1) != vg ? 0u : e & 1 ? 0xffff0000u : 0xffffu;
#pragma unroll
        for (int i = 0; i < kDTiles; ++i) {
          u32x4 one = values(at, ks, i);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            one[w] &= e >> 1 == w ? half : 0u;
          }
          const f32x16 add = mfma32(one, pt[ks], f32x16{});
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            o[i][r] += 16 * ks + n <= seen ? add[r] : 0.0f;
          }
          __builtin_amdgcn_sched_barrier(0); /* one product's registers at a time */
        }
      }
    }
  };

  /* One turn; entering it, K of it and the next and V of it are requested and
   * its scores are in `st`. */
  auto step = [&](int j, Scores &st, Scores &sn) {
    wait_vm<0>();
    lds_barrier();
    if (j + 2 < turns) {
      issue(j + 2, 0);
    }
    if (j + 1 < turns) {
      issue(j + 1, 1);
    }
    const int blk = it.first + j * kGroups + grp;
    if (blk > wave_last) {
      return;
    }
    const At x = at_turn(j);
    const int keys = it.keys(x.seg) - x.key0;        /* from the block's first on */
    const int base = x.seg ? it.seg[0].keys + x.key0 : x.key0;
    const bool hidden = base + min(keys, kTileKeys) - 1 > lim_lo;
    const bool need_mask = keys < kTileKeys || hidden;
    const bool next = j + 1 < turns && blk + kGroups <= wave_last;
    u32x4 pt[kKS];
    float alpha;
    bool bump;
    if (!need_mask && next) {
      scores(j + 1, sn);
      bump = softmax(st, pt, alpha);
      /* 64 sequences of 8 queries, 32 heads on 8, over 4000 keys: 65.5 us with 8
       * reads ahead and 6 VALU a product, 67.3 with 4 and 3 */
      constexpr int kProducts = kDSteps * kKT, kLead = kProducts >= 16 ? 8 : 4;
      __builtin_amdgcn_sched_group_barrier(0x100, kLead, 0); /* DS read */
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); /* MFMA */
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0); /* VALU */
        if (i < kProducts - kLead + (kParkQ<kD, kGroups> ? 1 : 0)) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      }
    } else {
      if (next) {
        scores(j + 1, sn);
      }
      if (need_mask) {
        /* the last key of the block it sees, against constants: keys that are
         * registers would be kept through the loop, and spilled */
        const int seen = min(limit - base, keys - 1) - 4 * (lane_here() >> 5);
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            st[kt][r] = 32 * kt + 8 * (r >> 2) + (r & 3) <= seen ? st[kt][r] : -INFINITY;
          }
        }
      }
      bump = softmax(st, pt, alpha);
    }
    if (__builtin_amdgcn_ballot_w64(bump) != 0) {
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          o[i][r] *= alpha;
        }
      }
    }
    if (hidden) {
      uint32_t any = 0;
      const uint32_t at = values_at(j);
#pragma unroll 1
      for (int ks = 0; ks < kKS; ++ks) {
#pragma unroll
        for (int i = 0; i < kDTiles; ++i) {
          const u32x4 a = values(at, ks, i);
          any |= not_finite(a[0]) | not_finite(a[1]) | not_finite(a[2]) | not_finite(a[3]);
        }
      }
      if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
        accumulate_apart(j, pt, min(limit - base, keys - 1));
        return;
      }
    }
    accumulate(j, pt);
  };

  Scores sa, sb;
  if (turns > 0) {
    wait_vm<0>();
    lds_barrier();
    if (it.first + grp <= wave_last) {
      scores(0, sa);
    }
  }
  for (int j = 0; j < turns; j += 2) {
    step(j, sa, sb);
    if (j + 1 < turns) {
      step(j + 1, sb, sa);
    }
  }

  if constexpr (kGroups == 2) {
    /* Group 1 leaves its part in LDS, lane by lane; group 0's wave of the same
     * queries takes it in. */
    f32x4 *so = reinterpret_cast<f32x4 *>(lds) + wq * (kDTiles * 4 + 1) * 64 + lane;
    __syncthreads();
    if (grp == 1) {
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          so[(4 * i + r4) * 64] =
              f32x4{o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]};
        }
      }
      so[kDTiles * 4 * 64] = f32x4{m_run, l_run, 0.0f, 0.0f};
    }
    __syncthreads();
    if (grp == 1) {
      return;
    }
    const f32x4 other = so[kDTiles * 4 * 64];
    const float mx = fmaxf(m_run, other[0]);
    const float m_use = mx == -INFINITY ? 0.0f : mx;
    const float f0 = __builtin_amdgcn_exp2f(m_run - m_use);
    const float f1 = __builtin_amdgcn_exp2f(other[0] - m_use);
    m_run = mx;
    l_run = l_run * f0 + other[1] * f1;
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 v = so[(4 * i + r4) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[i][4 * r4 + e] = o[i][4 * r4 + e] * f0 + v[e] * f1;
        }
      }
    }
  }
  if (!real) {
    return;
  }
  if (it.part >= 0) {
    float *sums = part_of<kD>(p, it.part) + (int64_t)row.place * kD;
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        *reinterpret_cast<f32x4 *>(sums + 32 * i + 8 * r4 + 4 * g) =
            f32x4{o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]};
      }
    }
    if (g == 0) {
      *reinterpret_cast<f32x2 *>(part_of<kD>(p, it.part) + (int64_t)p.p.rows * kD +
                                 (int64_t)row.place * 2) = f32x2{m_run, l_run};
    }
    return;
  }
  const bool seen = m_run > -INFINITY || l_run != 0.0f;
  const float inv = seen ? 1.0f / l_run : 0.0f;
  uint16_t *dst = p.a.o + (int64_t)row.place * kD;
#pragma unroll
  for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      *reinterpret_cast<u32x2 *>(dst + 32 * i + 8 * r4 + 4 * g) =
          u32x2{pack2(o[i][4 * r4] * inv, o[i][4 * r4 + 1] * inv),
                pack2(o[i][4 * r4 + 2] * inv, o[i][4 * r4 + 3] * inv)};
    }
  }
  if (p.a.lse && g == 0) {
    p.a.lse[row.place] = seen ? (m_run + log2f(l_run)) * kLn2 : -INFINITY;
  }
}

/* Over the four lanes that share lane % 16. */
__device__ __forceinline__ float over_g_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const f32x2 s = halves(v);
  return fmaxf(s[0], s[1]);
}
__device__ __forceinline__ float over_g_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const f32x2 s = halves(v);
  return s[0] + s[1];
}

template <int kD> constexpr int rows_lds() { return (4 * 16 * (kD + 4) + 4 * 16 * 2) * 4; }

/* A tile of 16 rows. */
template <int kD>
__device__ __forceinline__ void rows16(const KernelArgs &p, const Item &it, char *lds) {
  constexpr int kSteps = kD / 32; /* MFMA steps over d of a score tile */
  constexpr int kCols = kD / 16;  /* d per lane of V */
  constexpr int kVW = kCols / 2;  /* words of them */
  constexpr int kRow = kD * 2;
  constexpr int kPad = kD + 4;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;

  const Row row = row_of(p, it.kv, it.b, it.row0 + l16);
  const bool real = row.real;
  const Limits lim = limits_of(p, it, row);
  const int limit = real ? row.limit : lim.hi;
  const int lim_lo = lim.lo;
  const int last = min(min(it.last - 1, it.end), block_of(it, lim.hi, kRK));

  u32x4 qf[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    qf[s] = query(p, row, kD, 32 * s + 8 * g);
  }

  struct Keys {
    u32x4 f[2][kSteps];
  };
  struct Values {
    uint32_t f[8][kVW];
  };
  const uint32_t k_at = (uint32_t)(l16 * kRow + 16 * g);
  const uint32_t v_at = (uint32_t)(4 * g * kRow + l16 * (2 * kCols));
  /* Blocks past the last and keys past a segment's end load zeros. */
  auto source = [&](int b, bool value) {
    const int s = b < it.blocks0 ? 0 : 1;
    const int key0 = (b - (s ? it.blocks0 : 0)) * kRK;
    const int keys = b > last ? 0 : min(kRK, it.keys(s) - key0);
    const uint16_t *base = (value ? it.v(s) : it.k(s)) + (int64_t)(keys > 0 ? key0 : 0) * kD;
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, max(keys, 0) * kRow,
                                             0x00020000);
  };
  auto load_k = [&](Keys &d, int b) {
    const __amdgpu_buffer_rsrc_t r = source(b, false);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        d.f[h][s] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                       r, (int)(k_at + (uint32_t)(16 * h * kRow + 64 * s)), 0, 0));
      }
    }
  };
  auto load_v = [&](Values &d, int b) {
    const __amdgpu_buffer_rsrc_t r = source(b, true);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int off = (int)(v_at + (uint32_t)((16 * (e >> 2) + (e & 3)) * kRow));
      if constexpr (kVW == 4) {
        const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d.f[e][i] = w[i];
        }
      } else {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
        d.f[e][0] = w[0];
        d.f[e][1] = w[1];
      }
    }
  };

  f32x4 o[kCols];
  float m_run = -INFINITY, l_run = 0.0f; /* l: over this lane's keys */
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto step = [&](int b, Keys &kf, Values &vf) {
    f32x4 s[2];
#pragma unroll
    for (int d = 0; d < kSteps; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = mfma16<true>(kf.f[h][d], qf[d], d == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : s[h]);
      }
    }
    load_k(kf, b + 8);
    const int sg = b < it.blocks0 ? 0 : 1;
    const int key0 = (b - (sg ? it.blocks0 : 0)) * kRK;
    const int keys = it.keys(sg) - key0;
    const int base = sg ? it.seg[0].keys + key0 : key0;
    const bool hidden = base + min(keys, kRK) - 1 > lim_lo;
    const bool mask = keys < kRK || hidden;
    const int seen = min(limit - base, keys - 1); /* the last key of the block it sees */
    if (mask) { /* slot e: key 4 g + e, then 16 + 4 g + e - 4 */
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e >> 2][e & 3] =
            16 * (e >> 2) + 4 * g + (e & 3) <= seen ? s[e >> 2][e & 3] : -INFINITY;
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = over_g_max(mx) * p.scale_log2;
    const bool bump = mx > m_run + kSlack;
    const float m_next = bump ? mx : m_run;
    const float m_use = m_next == -INFINITY ? 0.0f : m_next;
    float x[8], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], p.scale_log2, -m_use));
      sum += x[e];
    }
    u32x4 pt;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      pt[w] = pack2(x[2 * w], x[2 * w + 1]);
    }
    const float alpha = bump ? __builtin_amdgcn_exp2f(m_run - m_use) : 1.0f;
    l_run = l_run * alpha + sum;
    m_run = m_next;
    if (__builtin_amdgcn_ballot_w64(bump) != 0) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          o[j][r] *= alpha;
        }
      }
    }
    bool apart = false;
    if (hidden) {
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int w = 0; w < kVW; ++w) {
          any |= not_finite(vf.f[e][w]);
        }
      }
      apart = __builtin_amdgcn_ballot_w64(any != 0) != 0;
    }
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      u32x4 vj;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        vj[d] = __builtin_amdgcn_perm(vf.f[2 * d + 1][j >> 1], vf.f[2 * d][j >> 1],
                                      j & 1 ? 0x07060302u : 0x05040100u);
      }
      if (!apart) {
        o[j] = mfma16<true>(vj, pt, o[j]);
        continue;
      }
      /* a key at a time, each for the queries that see it */
#pragma unroll 1
      for (int n = 0; n < kRK; ++n) {
        const int e = (n & 3) + 4 * (n >> 4);
        const uint32_t half = ((n >> 2) & 3) != g ? 0u : e & 1 ? 0xffff0000u : 0xffffu;
        u32x4 one = vj;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          one[w] &= e >> 1 == w ? half : 0u;
        }
        const f32x4 add = mfma16<true>(one, pt, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          o[j][r] += n <= seen ? add[r] : 0.0f;
        }
      }
    }
    load_v(vf, b + 8);
  };

  Keys ka, kb;
  Values va, vb;
  int blk = it.first + wave;
  load_k(ka, blk);
  load_v(va, blk);
  load_k(kb, blk + 4);
  load_v(vb, blk + 4);
  for (; blk <= last; blk += 8) {
    step(blk, ka, va);
    if (blk + 4 > last) {
      break;
    }
    step(blk + 4, kb, vb);
  }

  /* The four waves' results. o[j][r]: query l16, d = kCols (4 g + r) + j. */
  float(*so)[16][kPad] = reinterpret_cast<float(*)[16][kPad]>(lds);
  float(*sm)[16] = reinterpret_cast<float(*)[16]>(lds + 4 * 16 * kPad * 4);
  float(*sl)[16] = sm + 4;
  const float l_all = over_g_sum(l_run);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int h = 0; h < kCols / 4; ++h) {
      *reinterpret_cast<f32x4 *>(&so[wave][l16][kCols * (4 * g + r) + 4 * h]) =
          f32x4{o[4 * h][r], o[4 * h + 1][r], o[4 * h + 2][r], o[4 * h + 3][r]};
    }
  }
  if (g == 0) {
    sm[wave][l16] = m_run;
    sl[wave][l16] = l_all;
  }
  __syncthreads();
  /* Thread: four columns of a row, kPer rows apart by kStep. */
  constexpr int kQuads = kD / 4;
  constexpr int kStep = kThreads / kQuads;
  constexpr int kPer = 16 / kStep;
  const int c4 = threadIdx.x % kQuads * 4;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = threadIdx.x / kQuads + i * kStep;
    const Row to = row_of(p, it.kv, it.b, it.row0 + r);
    if (!to.real) {
      continue;
    }
    const float m = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
    const float m_use = m == -INFINITY ? 0.0f : m;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][r] - m_use); /* 0 where it saw none */
      l += sl[w][r] * f;
      const f32x4 v = *reinterpret_cast<const f32x4 *>(&so[w][r][c4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] += v[e] * f;
      }
    }
    if (it.part >= 0) {
      float *part = part_of<kD>(p, it.part);
      *reinterpret_cast<f32x4 *>(part + (int64_t)to.place * kD + c4) = acc;
      if (c4 == 0) {
        *reinterpret_cast<f32x2 *>(part + (int64_t)p.p.rows * kD + (int64_t)to.place * 2) =
            f32x2{m, l};
      }
      continue;
    }
    const bool seen = m > -INFINITY || l != 0.0f;
    const float inv = seen ? 1.0f / l : 0.0f;
    *reinterpret_cast<u32x2 *>(p.a.o + (int64_t)to.place * kD + c4) =
        u32x2{pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv)};
    if (p.a.lse && c4 == 0) {
      p.a.lse[to.place] = seen ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
  }
}

/* Workgroups 0 .. shared_groups - 1 take the shared keys, the others own ones
 * (with plan.together: both). */
template <int kD, bool kSharedRows, int kGroups, bool kOwnRows>
__global__ __launch_bounds__(kThreads, 2) void flash_shared(KernelArgs p) {
  constexpr int kLds = std::max(kSharedRows && kOwnRows ? 0 : wide_lds<kD, kGroups>(),
                            kSharedRows || kOwnRows ? rows_lds<kD>() : 0);
  __shared__ __align__(1024) char lds[kLds]; /* addresses in it are XORed */
  const SharedAttnArgs &a = p.a;
  Item it;
  const int id = blockIdx.x;
  const bool shared = id < p.p.shared_groups;
  constexpr int kSharedSize = kSharedRows ? kRK : kBK / kGroups;
  constexpr int kOwnSize = kOwnRows ? kRK : kBK / kGroups;
  if (shared) {
    /* the tiles of one reading far apart in the launch order, on one XCD where
     * the number of readings is a multiple of 8 */
    const int readings = a.kv_heads * p.p.shared_splits;
    const int reading = id % readings;
    it.kv = reading / p.p.shared_splits;
    const int split = reading % p.p.shared_splits;
    it.b = -1;
    it.row0 = id / readings * (kSharedRows ? 16 : 128 / kGroups);
    it.part = p.p.parts > 1 ? split : -1;
    it.seg[1] = Segment{nullptr, nullptr, 0};
    it.end = INT32_MAX;
    it.blocks0 = (a.shared_len + kSharedSize - 1) / kSharedSize;
    it.first = (int)((int64_t)it.blocks0 * split / p.p.shared_splits);
    it.last = (int)((int64_t)it.blocks0 * (split + 1) / p.p.shared_splits);
  } else {
    int at = id - p.p.shared_groups;
    const int split = at % p.p.own_splits;
    at /= p.p.own_splits;
    const int tile = p.p.own_tiles - 1 - at % p.p.own_tiles; /* the longest first */
    at /= p.p.own_tiles;
    it.kv = at % a.kv_heads;
    it.b = at / a.kv_heads;
    it.row0 = tile * (kOwnRows ? 16 : 128 / kGroups);
    it.part = p.p.parts > 1 ? p.p.shared_splits + split : -1;
    const int own = __builtin_amdgcn_readfirstlane(own_keys(a, it.b));
    if (own < 0) {
      return;
    }
    const int64_t mine = ((int64_t)it.b * a.kv_heads + it.kv) * a.capacity * kD;
    it.seg[1] = Segment{a.k + mine, a.v + mine, own};
    it.blocks0 = (a.shared_len + kOwnSize - 1) / kOwnSize;
    it.end = INT32_MAX;
    if (a.causal) { /* by the last of the tile's queries, all of one head or not */
      const int r1 = min(it.row0 + (kOwnRows ? 16 : 128 / kGroups), p.rows_seq) - 1;
      const int i1 = it.row0 / a.seq_q == r1 / a.seq_q ? r1 % a.seq_q : a.seq_q - 1;
      const int at = a.shared_len + own - a.seq_q + i1;
      it.end = at < 0                ? -1
               : at < a.shared_len ? at / kOwnSize
                                   : it.blocks0 + (at - a.shared_len) / kOwnSize;
    }
    /* all blocks, or those of the own keys */
    const int begin = p.p.together ? 0 : it.blocks0;
    const int blocks = it.blocks0 + (own + kOwnSize - 1) / kOwnSize - begin;
    it.first = begin + (int)((int64_t)blocks * split / p.p.own_splits);
    it.last = begin + (int)((int64_t)blocks * (split + 1) / p.p.own_splits);
  }
  const int64_t head = (int64_t)it.kv * a.shared_capacity * kD;
  it.seg[0] = Segment{a.k_shared + head, a.v_shared + head, a.shared_len};
  if constexpr (kSharedRows && kOwnRows) {
    rows16<kD>(p, it, lds);
  } else if constexpr (kOwnRows) {
    if (shared) {
      wide<kD, kGroups>(p, it, lds);
    } else {
      rows16<kD>(p, it, lds);
    }
  } else {
    wide<kD, kGroups>(p, it, lds);
  }
}

/* Four columns of a row, with the row's running maximum and weight. */
struct Sum {
  float m = -INFINITY, l = 0.0f;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};

  __device__ __forceinline__ void add(f32x2 ml, f32x4 w) {
    const float mx = fmaxf(m, ml[0]);
    const float m_use = mx == -INFINITY ? 0.0f : mx;
    const float back = __builtin_amdgcn_exp2f(m - m_use);
    const float f = __builtin_amdgcn_exp2f(ml[0] - m_use);
    m = mx;
    l = l * back + ml[1] * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = v[e] * back + w[e] * f;
    }
  }
  template <int kD>
  __device__ __forceinline__ void store(const SharedAttnArgs &a, int place, int c4) const {
    const bool seen = m > -INFINITY || l != 0.0f;
    const float inv = seen ? 1.0f / l : 0.0f;
    *reinterpret_cast<u32x2 *>(a.o + (int64_t)place * kD + c4) =
        u32x2{pack2(v[0] * inv, v[1] * inv), pack2(v[2] * inv, v[3] * inv)};
    if (a.lse && c4 == 0) {
      a.lse[place] = seen ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
  }
};

/* Parts first, first + step, .. of [0, parts), `get` giving one's statistics
 * and columns; kBatch of them in flight. */
template <int kBatch, typename F>
__device__ __forceinline__ void add_parts(Sum &sum, int first, int step, int parts, F get) {
  for (int s0 = first; s0 < parts; s0 += kBatch * step) {
    f32x2 ml[kBatch];
    f32x4 v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      get(min(s0 + u * step, parts - 1), ml[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (s0 + u * step < parts) {
        sum.add(ml[u], v[u]);
      }
    }
  }
}

/* kD / 4 threads a row, four columns each, and kSlices of those, which take
 * every kSlices-th part and meet in LDS. */
template <int kD, int kSlices>
__global__ __launch_bounds__(kThreads) void flash_shared_merge(KernelArgs p) {
  constexpr int kQuads = kD / 4;
  constexpr int kOne = kThreads / kSlices;
  const int slice = threadIdx.x / kOne, t = threadIdx.x % kOne;
  const int row = (int)blockIdx.x * (kOne / kQuads) + t / kQuads;
  const int c4 = t % kQuads * 4;
  const bool real = row < p.p.rows && own_keys(p.a, row / (p.a.heads * p.a.seq_q)) >= 0;
  Sum sum;
  if (real) {
    add_parts<kSlices == 1 ? 6 : 5>(sum, slice, kSlices, p.p.parts, [&](int s, f32x2 &ml, f32x4 &v) {
      const float *part = part_of<kD>(p, s);
      ml = *reinterpret_cast<const f32x2 *>(part + (int64_t)p.p.rows * kD + (int64_t)row * 2);
      v = *reinterpret_cast<const f32x4 *>(part + (int64_t)row * kD + c4);
    });
  }
  if constexpr (kSlices > 1) {
    __shared__ f32x4 sv[kSlices][kOne];
    __shared__ f32x2 sml[kSlices][kOne];
    sv[slice][t] = sum.v;
    sml[slice][t] = f32x2{sum.m, sum.l};
    __syncthreads();
    if (slice != 0) {
      return;
    }
#pragma unroll
    for (int s = 1; s < kSlices; ++s) {
      sum.add(sml[s][t], sv[s][t]);
    }
  }
  if (real) {
    sum.store<kD>(p.a, row, c4);
  }
}

template <int kD, int kSlices> void launch_merge(const KernelArgs &k, hipStream_t stream) {
  const int64_t threads = (int64_t)k.p.rows * (kD / 4) * kSlices;
  hipLaunchKernelGGL((flash_shared_merge<kD, kSlices>),
                     dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                     stream, k);
}

template <int kD, bool kSharedRows, int kGroups, bool kOwnRows>
void launch(const KernelArgs &k, hipStream_t stream) {
  hipLaunchKernelGGL((flash_shared<kD, kSharedRows, kGroups, kOwnRows>),
                     dim3((unsigned)(k.p.shared_groups + k.p.own_groups)), dim3(kThreads), 0,
                     stream, k);
}

template <int kD> void launch_all(const KernelArgs &k, hipStream_t stream) {
  if (k.p.shared_rows && k.p.own_rows) {
    launch<kD, true, 1, true>(k, stream);
  } else if (k.p.own_rows) {
    k.p.tile == 64 ? launch<kD, false, 2, true>(k, stream) : launch<kD, false, 1, true>(k, stream);
  } else {
    k.p.tile == 64 ? launch<kD, false, 2, false>(k, stream) : launch<kD, false, 1, false>(k, stream);
  }
  if (k.p.parts > 1) {
    /* 65 parts of 32 rows 14 -> 6 us, 5 of 4096 rows 5.2 against 9 */
    k.p.parts > 8 ? launch_merge<kD, 4>(k, stream) : launch_merge<kD, 1>(k, stream);
  }
}

} // namespace

void flash_shared_launch(const SharedAttnArgs &a, const SharedPlan &plan, int head_dim, char *ws,
                         hipStream_t stream) {
  KernelArgs k;
  k.a = a;
  /* a scale of 0 is a query of 0 */
  k.scale_log2 = a.scale != 0.0f ? std::fabs(a.scale) * 1.4426950408889634f : 1.0f;
  k.q_and = a.scale != 0.0f ? 0xffffffffu : 0u;
  k.q_xor = a.scale < 0.0f ? 0x80008000u : 0u;
  k.group = a.heads / a.kv_heads;
  k.rows_seq = k.group * a.seq_q;
  k.p = plan;
  k.ws = ws;
  if (head_dim == 128) {
    launch_all<128>(k, stream);
  } else {
    launch_all<64>(k, stream);
  }
  VX_HIP_CHECK(hipGetLastError());
}

} // namespace vxk
