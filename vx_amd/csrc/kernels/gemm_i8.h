/*
 * gemm_i8.h -- the choice of kernel, tile and splits of an int8 product
 * (gemm_i8.hip). Plain host arithmetic.
 */
#ifndef VX_AMD_GEMM_I8_H
#define VX_AMD_GEMM_I8_H

#include <algorithm>
#include <cstdint>

namespace vxk {

/* Most columns: 128 x 128 x this stays below 2^31. */
constexpr int64_t kGemmI8MaxCols = 131056;

struct GemmI8Plan {
  enum Kind { kRow, kFew, kTiles } kind;
  int tile;   /* kTiles: of i8::kTile */
  int splits; /* kTiles: workgroups that divide a tile's columns */
  int64_t ws_bytes;
};

namespace i8 {

constexpr int kLine = 128; /* columns of a stage: a cache line of each row */

/* Tiles of bm tokens x bn rows, per_cu of them to a CU, and what a round of them
 * takes on a 256-CU MI355X: `fixed` us to start and store, and a stage `full` us
 * where all CUs have their per_cu, `some` where few have one (two to a CU: where
 * all have one). At 32 stages (4096 columns), rounds of 256 and of fewer tiles:
 * 64x64 13 us, and two to a CU 19.6; 128x128 24.5 (86: 20), 128x192 28.3 (176:
 * 27.3), 256x128 36.6 (128: 32), 256x256 59 (96: 49), two of 128x128 37 (256:
 * 28.5); at 2 stages 128x128 4.1, two of them 5.5, 128x192 5.2, 256x128 6.2, 256x256
 * 12.4. Two of 128x128 have a ring of two slots each, one alone of four. */
struct Tile {
  int bm, bn, per_cu;
  double fixed, full, some;
};
constexpr Tile kTile[] = {{64, 64, 2, 2.1, 0.42, 0.25},   {128, 128, 1, 2.9, 0.60, 0.42},
                          {128, 128, 2, 3.4, 1.05, 0.70}, {128, 192, 1, 3.65, 0.78, 0.45},
                          {256, 128, 1, 4.2, 0.98, 0.65}, {256, 256, 1, 7.4, 1.55, 1.00}};
constexpr int kTiles = sizeof(kTile) / sizeof(kTile[0]);
constexpr int kSplitTiles = 2; /* the first of them, which may be split */
constexpr int kMaxSplits = 16;

inline int64_t count(const Tile &t, int64_t tokens, int64_t rows) {
  return ((tokens + t.bm - 1) / t.bm) * ((rows + t.bn - 1) / t.bn);
}

/* Splits leave 4 bytes a sum in a workspace, which a second launch reads. They are
 * no more than fit the CUs at once, 64 KiB a CU: one tile of 128x128 or two of 64x64. */
inline int64_t ws_bytes(const Tile &t, int64_t tokens, int64_t rows, int splits) {
  return splits > 1 ? count(t, tokens, rows) * splits * t.bm * t.bn * 4 : 0;
}

inline double us(const Tile &t, int64_t tokens, int64_t rows, int64_t cols, int splits, int cus) {
  const int64_t units = count(t, tokens, rows) * splits, slots = (int64_t)t.per_cu * cus;
  const int64_t full = units / slots, rest = units % slots;
  const int64_t stages = ((cols + kLine - 1) / kLine + splits - 1) / splits;
  double v = 2.5 + (double)full * (t.fixed + t.full * (double)stages);
  if (rest > 0) {
    const int64_t from = t.per_cu > 1 ? cus : 0; /* `some` up to here */
    const double more = (double)std::max<int64_t>(rest - from, 0) / (double)(slots - from);
    v += t.fixed + (t.some + (t.full - t.some) * more) * (double)stages;
  }
  return splits > 1 ? v + 3.0 + (double)ws_bytes(t, tokens, rows, splits) / 2e6 : v;
}

} // namespace i8

inline GemmI8Plan gemm_i8_plan(int64_t tokens, int64_t rows, int64_t cols, int cus,
                               bool may_split) {
  GemmI8Plan p{GemmI8Plan::kTiles, 0, 1, 0};
  if (tokens == 1) {
    /* 32000 x 768 6.2 us, and 6.7 as few; 11008 x 4096 8.9 and 11.3 */
    p.kind = GemmI8Plan::kRow;
    return p;
  }
  if (tokens <= 16 || (tokens <= 32 && rows * cols <= (int64_t(1) << 24))) {
    /* In us, by this kernel and by tiles, weights from HBM: 2 x 11008 x 4096 10.9 and
     * 13.2, 16 x 4096 x 4096 6.7 and 9.2, 24 x 4096 x 4096 7.6 and 9.3, 32 x 4096 x 4096
     * 8.3 and 9.5, 24 x 768 x 2048 5.0 and 7.4; past the border 32 x 11008 x 4096 21 and
     * 13.7, 32 x 32000 x 768 12.8 and 7.7. It is drawn by tokens and weights alone, and
     * near it gives some away where rows are many: 16 x 11008 x 4096 14.0 and 13.4, 16 x
     * 32000 x 768 8.3 and 7.5, 16 x 32000 x 1024 10.2 and 8.8, 24 x 16000 x 1024 7.9 and
     * 6.2. */
    p.kind = GemmI8Plan::kFew;
    return p;
  }
  double best = 1e30;
  for (int i = 0; i < i8::kTiles; ++i) {
    const i8::Tile &t = i8::kTile[i];
    const int64_t units = i8::count(t, tokens, rows), lines = (cols + i8::kLine - 1) / i8::kLine;
    for (int s = 1; s <= (may_split && i < i8::kSplitTiles ? i8::kMaxSplits : 1); ++s) {
      if (s > 1 && (units * s > (int64_t)t.per_cu * cus || lines < 4 * s)) {
        break;
      }
      const double v = i8::us(t, tokens, rows, cols, s, cus);
      if (v < best) {
        best = v;
        p.tile = i;
        p.splits = s;
      }
    }
  }
  p.ws_bytes = i8::ws_bytes(i8::kTile[p.tile], tokens, rows, p.splits);
  return p;
}

} // namespace vxk

#endif /* VX_AMD_GEMM_I8_H */
