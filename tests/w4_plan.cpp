// The form that a product with 4-bit weights takes (sb::w4_plan of semblend_amd/csrc/sb_w4_plan.h), for
// lines of "rows features inputs group bf16" from the standard input, a line each:
//   rows R J groups-of-a-tile waves once
//   tiles groups-of-a-tile splits steps-of-a-slice sum-steps
#include <cstdio>

#include "../semblend_amd/csrc/sb_w4_plan.h"

int main() {
  long long m, n, k, group;
  int bf16;
  while (std::scanf("%lld %lld %lld %lld %d", &m, &n, &k, &group, &bf16) == 5) {
    const sb::W4Plan p = sb::w4_plan(m, n, k, group, bf16 != 0);
    const int gpt = static_cast<int>(sb::kTileK / sb::table_step(group));
    if (p.tiled) std::printf("tiles %d %d %d %d\n", gpt, p.splits, p.split_steps, p.sum_blocks);
    else std::printf("rows %d %d %d %d %d\n", p.r, p.j, gpt, p.waves, p.once ? 1 : 0);
  }
  return 0;
}
