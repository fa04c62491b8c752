/*
 * gemm_i8.h -- how an int8 product (gemm_i8.hip) is divided. Plain host
 * arithmetic.
 */
#ifndef VX_AMD_GEMM_I8_H
#define VX_AMD_GEMM_I8_H

#include <algorithm>
#include <cstdint>

namespace vxk {

/* Most columns: 128 x 128 x this stays below 2^31. */
constexpr int64_t kGemmI8MaxCols = 131056;

struct GemmI8Plan {
  enum Kind { kFew, kTiles } kind;
  int waves; /* kFew: waves that divide the columns of 16 rows */
  int splits; /* kTiles: workgroups that divide a tile's columns */
  int64_t ws_bytes;
};

inline GemmI8Plan gemm_i8_plan(int64_t tokens, int64_t rows, int64_t cols, int cus,
                               bool may_split) {
  (void)may_split;
  GemmI8Plan p{};
  p.splits = 1;
  if (tokens <= 64) {
    p.kind = GemmI8Plan::kFew;
    const int64_t groups = (rows + 15) / 16, stages = (cols + 63) / 64;
    p.waves = 4;
    while (p.waves < 16 && groups * p.waves < 8 * (int64_t)cus && stages > p.waves) {
      p.waves *= 2;
    }
  } else {
    p.kind = GemmI8Plan::kTiles;
  }
  return p;
}

} // namespace vxk

#endif /* VX_AMD_GEMM_I8_H */
