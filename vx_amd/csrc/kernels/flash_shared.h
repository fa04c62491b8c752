/*
 * flash_shared.h -- how attention over a shared prefix (flash_shared.hip) is
 * divided. Plain C++, so g++ builds the CPU check of the plans that the GPU
 * tests run (tests/native/shared_plan.cpp).
 */
#ifndef VX_AMD_FLASH_SHARED_H
#define VX_AMD_FLASH_SHARED_H

#include <algorithm>
#include <cstdint>

namespace vxk {

/* How a call is divided: `shared_groups` workgroups over the shared keys of
 * all sequences' queries, `own_groups` over own keys (`together`: over shared
 * and own ones), parts merged from `ws_bytes` of workspace. */
struct SharedPlan {
  int rows;        /* queries of all heads */
  int parts;       /* partial results of each (1: none, the result itself) */
  int shared_splits, own_splits; /* workgroups that divide a tile's keys */
  int shared_groups, own_groups;
  int own_tiles;   /* tiles of a sequence's queries of a KV head */
  int tile;        /* rows of a wide tile: 64 or 128 */
  bool together;
  bool shared_rows, own_rows; /* 16-row tiles */
  int64_t ws_bytes;
};

namespace shared {

constexpr int kBK = 64; /* keys per block of a wide tile */

/* Floats of a part of the workspace. Parts begin on 16 bytes, as their loads
 * and stores do. */
constexpr int64_t part_floats(int64_t rows, int head_dim) {
  return (rows * (head_dim + 2) + 3) & ~int64_t(3);
}

/* Workgroups that divide the keys of each of `items` tiles: one a CU of at
 * least 8 blocks of 64 keys, or half as many of at least 4. A workgroup costs 5
 * us besides its blocks, and its partial results as much traffic as 130 keys:
 * 64 sequences of 32 heads on 4 over 8192 keys (16 tiles) 30 us in 16 splits,
 * 39 in 8 or 32; 128 sequences, 32 heads on 8, over 2048 31 in 4, 38 in 8; 16
 * over 4096 (8 tiles) 15 in 16, 19 in 8. 64 at most, and 256 instead, for one tile:
 * 4 sequences of 4 queries, 8 heads on 1, over 32768, 50000 and 131072 keys 23, 28
 * and 50 us, and 26, 29 and 38; 4 of single queries 21, 26 and 47, and 20, 23 and
 * 32; 2 of them, 4 heads on 1 (16 rows), 16.6, 19.5 and 30, and 17.8, 19.3 and 31. */
inline int shared_splits(int64_t items, int64_t blocks, int cus) {
  int64_t s = std::min(cus / items, blocks / 8);
  if (items * s < cus / 2) {
    s = std::min(cus / 2 / items, blocks / 4);
  }
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, 64));
}

/* Whether tiles of one sequence's queries walk the shared keys too, each for
 * itself: with many queries a sequence no key is read less often otherwise,
 * and over few shared keys reading them again costs less than the merge. In
 * us, together and apart, 16, 64 and 256 sequences of 32 heads on 8: 250 keys
 * 8.4 and 13, 12.5 and 17, 41 and 29.5; 500 keys 10.6 and 13, 17 and 17.6, 59
 * and 32; 1000 keys 15 and 13.7, 26 and 19; with 8 queries each, 500 keys and
 * 4, 16 and 64 sequences 16.3 and 13.7, 16.5 and 16.5, 18 and 29. */
inline bool together(int64_t items, int rows_seq, int shared_len, int cus) {
  if (rows_seq > 64 || shared_len == 0) {
    return true;
  }
  const int64_t rounds = std::max<int64_t>(1, (items + 2 * cus - 1) / (2 * cus));
  return rounds * shared_len <= (rows_seq <= 16 || items >= cus / 2 ? 512 : 256);
}

} // namespace shared

/* `may_split` false: a plan without a workspace. */
inline SharedPlan flash_shared_plan(int64_t batch, int heads, int kv_heads, int seq_q,
                                    int shared_len, int capacity, int head_dim, int cus,
                                    bool may_split) {
  using namespace shared;
  SharedPlan p{};
  const int rows_seq = heads / kv_heads * seq_q;
  p.rows = (int)(batch * heads * seq_q);
  p.own_splits = 1;
  p.own_rows = rows_seq <= 16;
  p.tile = rows_seq <= 64 ? 64 : 128;
  p.together = !may_split || batch == 1 || together(batch * kv_heads, rows_seq, shared_len, cus);
  if (!p.together) {
    /* the shared keys once for rows of many sequences */
    const int64_t rows_kv = batch * rows_seq;
    p.shared_rows = p.own_rows && rows_kv <= 16;
    const int64_t blocks = (shared_len + kBK - 1) / kBK;
    /* 128 rows where there are as many and their workgroups half fill the CUs:
     * 33 sequences of 5 queries, 21 heads on 3, over 2047 keys 17 us in tiles
     * of 64 and 19 of 128, 64 of 8, 32 heads on 8, over 4000 87 and 69 */
    const int64_t wide = kv_heads * ((rows_kv + 127) / 128);
    p.tile = rows_kv <= 64 || (!p.own_rows && wide * shared_splits(wide, blocks, cus) < cus / 2)
                 ? 64
                 : 128;
    const int tile = p.shared_rows ? 16 : p.tile;
    const int64_t items = kv_heads * ((rows_kv + tile - 1) / tile);
    p.shared_splits = shared_splits(items, blocks, cus);
    p.shared_groups = (int)(items * p.shared_splits);
    p.own_splits = capacity > 0 ? 1 : 0;
  }
  const int own_tile = p.own_rows ? 16 : p.tile;
  p.own_tiles = (rows_seq + own_tile - 1) / own_tile;
  const int64_t items = batch * kv_heads * p.own_tiles;
  if (may_split && p.own_splits) {
    /* up to one workgroup a CU, where it makes up for the merge (16 sequences
     * of 32 heads on 8, 1024 own keys each: 65 us in 2 splits, 66 in 1, 68 in 4),
     * and 16: the lengths are not known here, and the parts of an emptier cache
     * are merged for nothing. One sequence, 8 heads on 1 of 128, a cache of 131072
     * with 500, 16000 and all keys in it: 8.7, 17 and 81 us in 16, 9.7, 14 and 46
     * in 32, 11, 13.5 and 30 in 64, 15, 16 and 25 in 128; with 8 queries 11, 28 and
     * 157, and in 64 14, 17 and 50; 32 heads on 8: 9.1, 19 and 109, and in 32 9.9,
     * 19 and 97 */
    const int64_t keys = p.together ? shared_len + (int64_t)capacity : capacity;
    p.own_splits = (int)std::max<int64_t>(
        1, std::min<int64_t>({cus / items, keys / (p.together && p.own_rows ? 1024 : 512), 16}));
  }
  p.own_groups = (int)(items * p.own_splits);
  p.parts = p.shared_splits + p.own_splits;
  p.ws_bytes = p.parts > 1 ? p.parts * part_floats(p.rows, head_dim) * 4 : 0;
  return p;
}

} // namespace vxk

#endif /* VX_AMD_FLASH_SHARED_H */
