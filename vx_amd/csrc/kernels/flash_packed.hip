/*
 * flash_packed.hip -- attention of sequences of different lengths packed one
 * behind the other (vx_nn_flash_attention_packed_bf16), bf16 in, f32 accumulate,
 * bf16 out, f32 log-sum-exp.
 *
 * The rows of a tile are queries of one sequence, position by position and for
 * each the heads that read one KV head, so that a tile of 128 rows covers 128 /
 * group positions: K and V are read once for all heads of the group, and short
 * sequences fill a tile. Workgroups find their tile from the offsets
 * themselves (tile_of); the launch has as many as there can be tiles, the others
 * end at once. So a captured launch follows the offsets in GPU memory, and no
 * workspace is needed.
 *
 * 4 waves; K and V through a two-slot LDS ring by buffer-to-LDS loads; as in
 * flash_attn.hip the products are transposed, S^T = K Q^T and O^T += V^T P^T
 * (v_mfma_f32_32x32x16_bf16), so that a lane holds one query's scores and P^T is
 * the scores' accumulator rounded in place. 64 rows: two halves of the workgroup
 * divide the keys and meet in LDS.
 * The weights are rounded to bf16, off by at most 2^-8 each, because the second
 * product's operands are bf16 (f32 ones multiply at a sixteenth of the rate);
 * maxima and sums stay in f32, the sums over unrounded weights. It takes o from
 * 1.5e-3-1.6e-3 of its 2-norm, its own rounding, to 1.8e-3-2.0e-3.
 *
 * Where V holds infinities or NaNs, a key hidden from a query reaches it all the
 * same (0 x inf is NaN): a workgroup whose outputs are not all finite goes over its
 * keys again and takes the blocks in which a key is hidden from one of a wave's
 * queries and not from another a key at a time, each for the queries that see it.
 * With that beside the loop instead of in it, the loop's registers stay in place:
 * 8192 and 91 tokens, 32 heads on 8, 627 -> 552 us.
 *
 * 537-550 us there, 1.0 PFLOP/s (without a mask 1136, 0.97), is bound by the CU's
 * parts taking turns: a turn of two workgroups (2.0 us) needs 0.86 of MFMAs, 0.95
 * of the softmax's VALU and 1.2 of LDS. 64 sequences of 1 to 1024 tokens take 90
 * (135 without a mask): a workgroup of 4.6 turns spends 2 us to find its tile, 3
 * until its first keys are there, and 2.6 after the last. Workgroups that go from
 * tile to tile and load the next one's keys in between needed registers that the
 * loop's values were then moved and spilled for: 116 us, and 590 for the long
 * one.
 */
#include "../vx_hip_common.h"
#include "../vx_packed_kernels.h"
#include "vx_lds_dma.hip.h"
#include "vx_mfma16.hip.h"
#include "vx_wave_ops.hip.h"

#include <algorithm>
#include <cmath>

namespace vxk {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBK = 64;        /* keys per turn of a workgroup */
constexpr float kSlack = 8.0f; /* base-2 headroom of the stale row max */
constexpr float kLn2 = 0.69314718055994531f;

struct KernelArgs {
  PackedAttnArgs a;
  float scale_log2; /* above 0 */
  uint32_t q_and, q_xor;
  int group; /* heads of a KV head */
  bool sorted;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

/* The lane's number, read again: an address made from it where it is used needs
 * no register in between. */
__device__ __forceinline__ int lane_here() {
  int v;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(v));
  return v;
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

/* A sequence's first row and length; offsets that fall or lie outside the
 * tensors are taken as the nearest that do not. */
struct Span {
  int begin, len;
};
__device__ __forceinline__ Span span_of(const PackedAttnArgs &a, int s) {
  const int begin = min(max(a.offsets[s], 0), a.total);
  return Span{begin, min(max(a.offsets[s + 1], begin), a.total) - begin};
}

struct Tile {
  Span span;
  int index; /* of the sequence's tiles; -1: none */
};

/* The launch's tile number `rank`, the same on every lane. `sorted`, for at most
 * 64 sequences: tiles of the highest index, which see the most keys, come first.
 * With n_s tiles in sequence s, sum max(n_s - b, 0) of them have an index of b or
 * more: the index is the highest b for which this exceeds `rank`. Else in the order
 * of the sequences, which read their keys at about the same time, each from its last
 * tile to its first; sequence s from floor(first row / rows of a tile) + s on, which
 * leaves each at least its tiles and is searched, not added up. */
__device__ __forceinline__ Tile tile_of(const PackedAttnArgs &a, int group, int tile, int rank,
                                        bool sorted) {
  const int lane = lane_here();
  auto tiles = [&](int len) { return (int)(((int64_t)len * group + tile - 1) / tile); };
  if (sorted) {
    const Span span = lane < a.sequences ? span_of(a, lane) : Span{0, 0};
    const int n = tiles(span.len);
    auto from = [&](int b) { return wave_sum_int(max(n - b, 0)); };
    if (from(0) <= rank) {
      return Tile{Span{0, 0}, -1};
    }
    int lo = 0, hi = 1; /* from(lo) > rank >= from(hi) */
    while (from(hi) > rank) {
      lo = hi;
      hi *= 2;
    }
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (from(mid) > rank) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    const int j = rank - from(lo + 1); /* among the sequences that have a tile `lo` */
    const uint64_t has = __builtin_amdgcn_ballot_w64(n > lo);
    const bool me = n > lo && __builtin_popcountll(has & ((1ull << lane) - 1)) == j;
    const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(me));
    return Tile{Span{__builtin_amdgcn_readlane(span.begin, who),
                     __builtin_amdgcn_readlane(span.len, who)},
                lo};
  }
  /* the last sequence that starts at `rank` or before: 64 of them, then 64 in between */
  auto first = [&](int s) {
    const int64_t row = min(max(a.offsets[s], 0), a.total);
    return (int)(row * group / tile) + s;
  };
  int at = 0;
  for (int n = a.sequences; n > 1;) { /* it is one of the n from `at` */
    const int step = (n + 63) / 64;
    const int s = at + lane * step;
    const bool past = lane * step >= n || first(min(s, a.sequences - 1)) > rank;
    const int before = 64 - __builtin_popcountll(__builtin_amdgcn_ballot_w64(past));
    const int skip = max(before - 1, 0) * step;
    at += skip;
    n = min(step, n - skip);
  }
  const Span span = span_of(a, at);
  const int n = tiles(span.len), index = n - 1 - (rank - first(at));
  return Tile{span, index < n ? index : -1};
}

/* Tiles of 128 / kGroups rows. */
template <int kD, int kGroups>
__global__ __launch_bounds__(kThreads, 2) void flash_packed(KernelArgs p) {
  constexpr int kTileRows = 128 / kGroups;
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
  __shared__ __align__(kRowBytes) char lds[4 * kBK * kD * 2]; /* addresses of a row are XORed */

  /* Workgroup i runs on XCD i % 8: where the KV heads are a multiple of 8, each
   * XCD has its own, whose keys its L2 then holds alone. */
  const int kv_heads = p.a.kv_heads;
  int kv, rank;
  if (kv_heads % 8 == 0) {
    const int local = (int)blockIdx.x >> 3, per = kv_heads >> 3;
    rank = local / per;
    kv = ((int)blockIdx.x & 7) + 8 * (local - rank * per);
  } else {
    rank = (int)blockIdx.x / kv_heads;
    kv = (int)blockIdx.x - rank * kv_heads;
  }
  const Tile tile = tile_of(p.a, p.group, kTileRows, rank, p.sorted);
  if (tile.index < 0) {
    return;
  }
  const int keys_all = tile.span.len;
  const int rows_all = keys_all * p.group;
  const int row0 = tile.index * kTileRows;
  /* the keys that any row of the tile sees, in blocks */
  const int pos_last = (min(row0 + kTileRows, rows_all) - 1) / p.group;
  const int turns = ((p.a.causal ? pos_last + 1 : keys_all) + kBK - 1) / kBK;

  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63;
  const int g = lane >> 5;
  const int grp = kGroups == 1 ? 0 : wave / kWavesQ;
  const int wq = kGroups == 1 ? wave : wave % kWavesQ;

  /* The lane's number where addresses are made of it: read again, they need no
   * registers in between, of which 128 rows of 128 have none to spare but for K's
   * (64 sequences of up to 1024, 32 heads on 8: 95.8 us, with K's kept 92.2, with
   * all, where values spill, 104; 1 x 512 in 64 rows 15.2, and kept 13.5). */
  constexpr bool kKeep = kD == 64 || kGroups == 2;
  auto lane_for = [&] { return kKeep ? lane : lane_here(); };

  /* Load l of a thread fills unit l * kGroupThreads + tg of a plane: key row
   * l * kRowsPer + tg / kChunks, whose place differs from l = 0's by an XOR. */
  constexpr int kRowsPer = kGroupThreads / kChunks;
  static_assert(kChunks == 16 ? 16 % kRowsPer == 0 && kRowsPer % 4 == 0 : kRowsPer % 16 == 0,
                "places of the loads of a thread");
  /* [group][slot][K|V][unit] */
  u32x4 *ring = reinterpret_cast<u32x4 *>(lds) + grp * 4 * kUnits;
  const uint32_t ring_base = (uint32_t)(uintptr_t)(VX_LDS void *)ring;
  const int kv_bytes = (int)p.a.kv_row * 2; /* from a key to the next */
  const int64_t kv_base = (int64_t)tile.span.begin * p.a.kv_row + kv * p.a.kv_head;
  /* A group's turn j has block j * kGroups + grp, in slot j % 2. */
  auto key_of = [&](int j) { return (j * kGroups + grp) * kTileKeys; };
  auto issue = [&](int j, int plane) {
    const int key0 = key_of(j);
    const int n = min(kTileKeys, keys_all - key0);
    const int bytes = n > 0 ? (n - 1) * kv_bytes + kRowBytes : 0;
    const uint16_t *src = plane == 0 ? p.a.k : p.a.v;
    i32x4 rs = buffer_rsrc(src + kv_base + (int64_t)key0 * p.a.kv_row, bytes);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      rs[e] = __builtin_amdgcn_readfirstlane(rs[e]); /* uniform, which the compiler cannot tell */
    }
    const uint32_t base = ring_base + (uint32_t)((((j & 1) * 2 + plane) * kUnits + wq * 64) * 16);
    const uint32_t tg = (uint32_t)(wq * 64 + lane_for());
    const int row = (int)(tg / kChunks), c = (int)(tg % kChunks);
    const int place = (plane == 0 ? place_k<kChunks>(row, c) : place_v<kChunks>(row, c)) * 16;
    const int off = row * kv_bytes;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int turn = plane == 0 && kChunks == 16 ? (l * kRowsPer & 15) << 4 : 0;
      dma16(rs, (uint32_t)(off + (place ^ turn) + l * kRowsPer * kv_bytes),
            base + (uint32_t)(l * kGroupThreads * 16));
    }
  };
  /* The lane's row: its place and position, and whether it is one (else the
   * sequence's last). */
  struct Row {
    int64_t at;
    int pos, head;
    bool real;
  };
  auto row_of = [&] {
    const int r = row0 + 32 * wq + (lane_here() & 31);
    const int in = min(r, rows_all - 1), pos = in / p.group;
    return Row{(int64_t)tile.span.begin + pos, pos, kv * p.group + (in - pos * p.group), r < rows_all};
  };
  u32x4 qf[kDSteps];
  auto load_q = [&] {
    const Row row = row_of();
    const uint16_t *src = p.a.q + row.at * p.a.q_row + row.head * p.a.q_head + 8 * (lane_here() >> 5);
#pragma unroll
    for (int s = 0; s < kDSteps; ++s) {
      qf[s] = *reinterpret_cast<const u32x4 *>(src + 16 * s);
    }
  };
  /* The first two blocks of K and the first of V are on their way before anything
   * else is looked at. */
  issue(0, 0);
  issue(0, 1);
  if (turns > 1) {
    issue(1, 0);
  }
  load_q();

  /* The last key that each of the wave's rows sees, and all or any of them. */
  const int wave_row = row0 + 32 * wq;
  const int lim_lo =
      p.a.causal ? __builtin_amdgcn_readfirstlane(wave_row / p.group) : keys_all - 1;
  const int lim_hi =
      wave_row >= rows_all ? -1
      : p.a.causal
          ? __builtin_amdgcn_readfirstlane(min(wave_row + 31, rows_all - 1) / p.group)
          : keys_all - 1;
  const int limit = p.a.causal ? row_of().pos : keys_all - 1;

  /* Where the lane reads in a slot's K plane (row lq, chunk g: chunk 2 ds + g
   * of a place that is an XOR lies at the address XOR 32 ds) and, transposing,
   * in its V plane: key 4 g + i / 4 of a 16-key step, d 16 j + 4 (i % 4) of a
   * 32-wide tile, i = lane % 16, j = lane / 16 % 2, which hands it the 8 keys
   * of its k-slots at d = lane % 32; tile i lies at XOR 64 i. */
  auto keys_at = [&](int j) {
    const int l = lane;
    return ring_base + (uint32_t)((j & 1) * 2 * kUnits * 16 + (l & 31) * kRowBytes +
                                  place_k<kChunks>(l & 31, l >> 5) * 16);
  };
  auto values_at = [&](int j) {
    const int l = lane_for();
    const int key = 4 * (l >> 5) + ((l & 15) >> 2);
    const int d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
    return ring_base + (uint32_t)(((j & 1) * 2 + 1) * kUnits * 16 + key * kRowBytes +
                                  place_v<kChunks>(key, d >> 3) * 16 + (d & 7) * 2);
  };

  f32x16 o[kDTiles];
  float m_run, l_run;

  typedef f32x16 Scores[kKT];
  auto scores = [&](int j, Scores &st) {
    const uint32_t at = keys_at(j);
#pragma unroll
    for (int ds = 0; ds < kDSteps; ++ds) {
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt) {
        const u32x4 a = *(const VX_LDS u32x4 *)(uintptr_t)((at ^ (uint32_t)(ds << 5)) +
                                                           (uint32_t)(kt * 32 * kRowBytes));
        st[kt] = mfma32(a, qf[ds], ds == 0 ? f32x16{} : st[kt]);
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

  /* What a block hides of a wave's rows: keys past the sequence's last, or past
   * those that a row sees. */
  struct Block {
    int key0, keys; /* from the block's first on */
    bool hidden, mask;
  };
  auto block_of = [&](int j) {
    const int key0 = key_of(j), keys = keys_all - key0;
    const bool hidden = key0 + min(keys, kTileKeys) - 1 > lim_lo;
    return Block{key0, keys, hidden, keys < kTileKeys || hidden};
  };
  auto hide = [&](const Block &b, Scores &st) {
    /* the last key of the block it sees, against constants: keys that are
     * registers would be kept through the loop, and spilled */
    const int seen = min(limit - b.key0, b.keys - 1) - 4 * (lane_here() >> 5);
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[kt][r] = 32 * kt + 8 * (r >> 2) + (r & 3) <= seen ? st[kt][r] : -INFINITY;
      }
    }
  };
  auto rescale = [&](bool bump, float alpha) {
    if (__builtin_amdgcn_ballot_w64(bump) != 0) {
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          o[i][r] *= alpha;
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
    const Block b = block_of(j);
    if (b.key0 > lim_hi) {
      return;
    }
    const bool ahead = j + 1 < turns && key_of(j + 1) <= lim_hi;
    u32x4 pt[kKS];
    float alpha;
    bool bump;
    if (!b.mask && ahead) {
      scores(j + 1, sn);
      bump = softmax(st, pt, alpha);
      constexpr int kProducts = kDSteps * kKT, kLead = kProducts >= 16 ? 8 : 4;
      __builtin_amdgcn_sched_group_barrier(0x100, kLead, 0); /* DS read */
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); /* MFMA */
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0); /* VALU */
        if (i < kProducts - kLead) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
      }
    } else {
      if (ahead) {
        scores(j + 1, sn);
      }
      if (b.mask) {
        hide(b, st);
      }
      bump = softmax(st, pt, alpha);
    }
    rescale(bump, alpha);
    accumulate(j, pt);
  };
  /* The tile's queries, loaded, as scores() takes them; and nothing seen yet. */
  auto start = [&] {
#pragma unroll
    for (int s = 0; s < kDSteps; ++s) {
      /* the scale's sign goes into the query, so that a hidden key's score is -inf
       * whatever the scale */
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        qf[s][e] = (qf[s][e] & p.q_and) ^ p.q_xor;
      }
    }
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) {
      o[i] = f32x16{};
    }
    m_run = -INFINITY;
    l_run = 0.0f;
  };
  /* The tile over again, a block at a time. */
  auto carefully = [&] {
    load_q();
    start();
#pragma unroll 1
    for (int j = 0; j < turns; ++j) {
      lds_barrier();
      issue(j, 0);
      issue(j, 1);
      wait_vm<0>();
      lds_barrier();
      const Block b = block_of(j);
      if (b.key0 > lim_hi) {
        continue;
      }
      Scores st;
      scores(j, st);
      if (b.mask) {
        hide(b, st);
      }
      u32x4 pt[kKS];
      float alpha;
      const bool bump = softmax(st, pt, alpha);
      rescale(bump, alpha);
      if (b.hidden) {
        accumulate_apart(j, pt, min(limit - b.key0, b.keys - 1));
      } else {
        accumulate(j, pt);
      }
    }
  };

  start();
  Scores sa, sb;
  wait_vm<0>();
  lds_barrier();
  if (key_of(0) <= lim_hi) {
    scores(0, sa);
  }
  for (int j = 0; j < turns; j += 2) {
    step(j, sa, sb);
    if (j + 1 < turns) {
      step(j + 1, sb, sa);
    }
  }
  if (p.a.causal) {
    /* x 0 is NaN of what is not finite */
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        zero = __builtin_fmaf(o[i][r], 0.0f, zero);
      }
    }
    if (__syncthreads_or(zero != zero)) {
      carefully();
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
  const Row row = row_of();
  if (row.real) {
    const bool seen = m_run > -INFINITY || l_run != 0.0f;
    const float inv = seen ? 1.0f / l_run : 0.0f;
    uint16_t *dst = p.a.o + row.at * p.a.o_row + row.head * p.a.o_head;
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
      p.a.lse[(int64_t)row.head * p.a.total + row.at] =
          seen ? (m_run + log2f(l_run)) * kLn2 : -INFINITY;
    }
  }
}

template <int kD, int kGroups> void launch(KernelArgs p, hipStream_t stream) {
  constexpr int kTileRows = 128 / kGroups;
  const int64_t workgroups =
      ((int64_t)p.a.total * p.group / kTileRows + p.a.sequences) * p.a.kv_heads;
  /* Two fit on a CU. Heaviest first ends evenly where they come in a few rounds: 30
   * sequences of up to 500, 8 heads on 1, 500 workgroups, 19.6 us, in the sequences'
   * order 22.5; 64 of up to 300, 12 heads, 1670, 40.5 and 43.6; 64 of up to 1024, 32
   * on 8, 3000, 89.9 and 92.7. In one round the search costs more than it gains (8 of
   * up to 260, 32 on 8, tiles of 64 rows, 16.2 and 14.7), in many the keys of other
   * sequences in between (64 of up to 1024, 12 heads, 3830, 146 and 137; 32 on 8,
   * 8760, 309 and 284). */
  p.sorted = kGroups == 1 && p.a.sequences <= 64 && workgroups <= 12 * (int64_t)device_cu_count();
  hipLaunchKernelGGL((flash_packed<kD, kGroups>), dim3((unsigned)workgroups), dim3(kThreads), 0,
                     stream, p);
}

} // namespace

void flash_packed_launch(const PackedAttnArgs &a, int head_dim, hipStream_t stream) {
  KernelArgs p{};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  /* a scale of 0 is a query of 0 */
  p.scale_log2 = a.scale != 0.0f ? std::fabs(a.scale) * 1.4426950408889634f : 1.0f;
  p.q_and = a.scale != 0.0f ? 0xffffffffu : 0u;
  p.q_xor = a.scale < 0.0f ? 0x80008000u : 0u;
  /* Tiles of 64 rows, whose keys two halves of the workgroup divide, where those of
   * 128 would be few: 1 sequence of 1000, 12 heads (108 workgroups) 18.8 us, in tiles
   * of 128 25.9; 1 of 4000 (384) 67.6 and 80.7; 20 of up to 1000 (444) 21.5 and 27.6;
   * but 1 of 1800, 32 heads on 8 (456), 47.3 and 44.4, and 1 of 2500 (632) 77.5 and
   * 68.6. Half of the tiles of one row that many sequences may need are counted. */
  const int64_t wide = ((int64_t)a.total * p.group / 128 + (a.sequences + 1) / 2) * a.kv_heads;
  const bool two = 4 * wide < 7 * (int64_t)device_cu_count();
  if (head_dim == 64) {
    two ? launch<64, 2>(p, stream) : launch<64, 1>(p, stream);
  } else {
    two ? launch<128, 2>(p, stream) : launch<128, 1>(p, stream);
  }
}

} // namespace vxk
