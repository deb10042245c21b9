// How a product with 4-bit weights runs (sb_w4.hip): the form and its sizes, by the sizes of the call.
//
// Compiled for the host as well, so that a CPU test can say which form a size takes: the tests of every
// form then keep reaching it.
#pragma once

#include <cstdint>

namespace sb {
namespace {

constexpr int kTileN = 16;    // features of a tile
constexpr int kTileK = 128;   // inputs of a tile
constexpr int kBM = 128, kBN = 128;  // rows and features of a workgroup of many rows

constexpr int64_t tiles(int64_t x, int64_t by) { return (x + by - 1) / by; }

// Inputs that share a table word: the group, or the largest of 32, 64 and 128 that divides it.
inline int64_t table_step(int64_t group) { return group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32; }

inline int64_t sum_blocks(int64_t k, int64_t group) {
  return tiles(tiles(k, kTileK) * (kTileK / table_step(group)), 32);
}

// Few rows (workgroups of R rows and 16 J features), or 128 x 128 tiles with the steps (tiles of inputs, and
// of sums) in `splits` slices.
struct W4Plan {
  bool tiled;
  int r, j;
  int waves;   // few rows: of a workgroup
  bool once;   // few rows: codes past the caches
  int splits, split_steps, sum_blocks;
};

// The few-rows kernel: a workgroup reads its rows once for all of its features and its codes once for all
// of its rows, so that more of either mean fewer reads and fewer, longer workgroups. R (no larger than holds
// the rows) and J are those of the least time by this model, in us for K inputs on 256 CUs: 2.5 + rounds (0.5
// + kRound K / 1024), a round a workgroup per CU (32 and 64 rows: its second part a fifth more from five
// rounds on). Measured, J = 1 to 4: 64 rows, R = 64, of 3584 -> 4608 13.7, 9.0, 11.0, 13.4 us; 4096 -> 12288
// 25.8, 19.0, 14.7, 14.6; 3584 -> 37888 59.0, 38.8, 38.8, 36.2; 18944 -> 3584 29.8, 39.0, 45.0, 59.0; 32
// rows, R = 32, of 4096 -> 131072 (fp16) 146, 106, 88, 80; 16 of 4096 -> 12288 9.2, 8.4, 7.5, 7.9. The
// largest R and the one taken: 64 rows of 3584 -> 4608 8.9 and 7.7 (R = 32, J = 3), of 18944 -> 3584 29.5 and
// 22.4 (32, 2); 32 rows of 18944 -> 3584 18.1 and 16.5 (16, 2). (Up to 4 rows J = 1 or 2: what is left is
// the codes.)
// More than 64 rows take tiles where their model is less: 3, the sums' launch 4 (bf16), a step 1.08 with one
// workgroup a CU and 0.85 each with more; slices: the merge's launch 4 and their traffic. Measured, few rows
// against tiles in their best split: 3584 -> 4608, 128 rows 11.4 and 22.9 us, 256 rows 20.5 and 26.0, 614 rows
// 38.3 and 37.2; 18944 -> 3584 (groups of 64), 192 rows 50.7 and 55.2, 320 rows 94.1 and 72.6; 3584 -> 37888,
// 96 rows 61.9 and 53.8; 896 -> 1152, 256 rows 5.1 and 14.7. (Of 60 sizes drawn at random, up to 630 rows, 30000
// features and 16384 inputs, the form taken is within 6% of the fastest one, but for six of under 10 us that
// are 8 to 22% behind. Tiles of 32 and 64 rows that four waves share were no faster: 64 rows of 3584 ->
// 37888 42 us.)
inline W4Plan w4_plan(int64_t m, int64_t n, int64_t k, int64_t group, bool bf16) {
  W4Plan p = {};
  const int64_t nt = tiles(n, kTileN), kt = tiles(k, kTileK);
  const auto rounds = [](int64_t wgs) { return tiles(wgs, 256); };
  constexpr int kRows[4] = {4, 16, 32, 64};
  constexpr double kNever = 1e30;
  constexpr double kRound[4][4] = {{0.6, 0.7, kNever, kNever},
                                   {0.6, 0.75, 1.1, 1.38},
                                   {0.83, 1.1, 1.5, 1.75},
                                   {1.47, 1.84, 2.35, 2.87}};
  const int first = m <= 4 ? 0 : 1, last = m <= 4 ? 0 : m <= 16 ? 1 : m <= 32 ? 2 : 3;
  double best = kNever;
  for (int r = first; r <= last; ++r)
    for (int j = 1; j <= 4; ++j) {
      const int64_t gy = tiles(m, kRows[r]), turns = rounds(tiles(nt, j) * gy);
      const double more = r > 1 && turns > 4 ? 1.2 : 1.0;
      const double t = 2.5 + static_cast<double>(turns) *
                                 (0.5 + kRound[r][j - 1] * more * static_cast<double>(k) / 1024);
      if (gy > 65535 || t >= best) continue;  // (a grid's second axis ends there)
      best = t;
      p.r = kRows[r], p.j = j;
    }
  p.splits = 1;
  p.split_steps = static_cast<int>(kt);
  const int64_t blocks = bf16 ? sum_blocks(k, group) : 0;
  const int64_t steps = kt + blocks, grid = tiles(m, kBM) * tiles(n, kBN);
  for (int64_t s = 1; m > 64 && s <= 32 && (s == 1 || 2 * s <= steps); ++s) {
    const int64_t per = tiles(steps, s), slices = tiles(steps, per);
    if (slices != s) continue;
    const double load = static_cast<double>(rounds(grid * s));
    double t = 3.0 + (blocks ? 4.0 : 0.0) + static_cast<double>(per) * (load <= 1.0 ? 1.08 : 0.85 * load);
    if (s > 1) t += 4.0 + static_cast<double>(s * m) * static_cast<double>(n) * 8.0 / 6e6;
    if (t >= best) continue;
    best = t;
    p.tiled = true;
    p.splits = static_cast<int>(s);
    p.split_steps = static_cast<int>(per);
    p.sum_blocks = static_cast<int>(blocks);
  }
  // Up to 16 rows: 16 waves where a workgroup has 16 features (a CU has one or two of them then) and a
  // tile of inputs for each wave (one row of 18944 -> 3584 9.8 -> 9.1 us, 16 rows 12.9 -> 11.8; of 896 ->
  // 1152 2.9 and 3.0). (64 rows and features: LDS holds seven waves' steps)
  p.waves = p.r <= 16 && p.j == 1 && kt > 16 ? 16 : p.r == 64 && p.j == 4 ? 7 : 8;
  // Codes read past the caches (nontemporal) where the 256 MB last one cannot hold them until the next call
  // with these weights, whatever runs between: from 192 MB on. Measured, plain and nontemporal reads: weights
  // that are in no cache (a ring of 1.5 GB of them), one row of 4096 -> 131072, 285 MB, 45.6 and 44.1 us, 16
  // rows 56.5 and 52.6; 16 rows of 3584 -> 37888, 72 MB, 20.3 and 19.0, one of 4096 -> 28672, 62 MB, 13.2 and
  // 12.7. Weights called again while the cache holds them (three of these in turn): 14.4 and 19.1, 12.6 and
  // 12.4. Below 192 MB a call cannot know which it is; plain reads lose up to 8% of the one and save a
  // quarter of the other.
  p.once = p.r <= 16 && p.j > 1 && tiles(m, p.r) == 1 && nt * kt * 1024 >= (int64_t{192} << 20);
  return p;
}

}  // namespace
}  // namespace sb
