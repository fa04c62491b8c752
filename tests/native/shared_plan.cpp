// Prints how attention over a shared prefix is divided on 256 CUs: a line of
// numbers for each seven extents among the arguments.

#include "../../vx_amd/csrc/kernels/flash_shared.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char **argv) {
  for (int i = 1; i + 6 < argc; i += 7) {
    int x[7];
    for (int j = 0; j < 7; ++j) {
      x[j] = atoi(argv[i + j]);
    }
    const vxk::SharedPlan p =
        vxk::flash_shared_plan(x[0], x[1], x[2], x[3], x[4], x[5], x[6], 256, true);
    printf("%d %d %d %d %d %d %d\n", p.together, p.shared_rows, p.own_rows, p.tile,
           p.shared_splits, p.own_splits, p.parts);
  }
}
