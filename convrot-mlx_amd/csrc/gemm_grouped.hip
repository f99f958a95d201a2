// Products of rows grouped by expert in 16 bits (gemm_grouped_tile.h): the choice of tile.
#include <algorithm>

#include "convrot_launch.h"
#include "gemm_groups.h"

namespace convrot {
namespace {

// Time of a tile's block of 64 (few tiles, and with every CU busy), and what its prologue and epilogue add, in
// microseconds, fitted to measurements on weights from memory: over 145 forward products (1 to 6000 rows, 1 to 64
// experts, 256 to 8100 features) the tile taken is 2 % slower than the best of the six on average, 32 % at worst.
struct Cost {
  int bm, bn, per_cu;
  float lone, full, fixed;
};
constexpr Cost kCosts[] = {{256, 256, 1, 1.15f, 1.45f, 11.4f}, {128, 128, 2, 0.71f, 1.28f, 4.0f},
                           {64, 128, 2, 0.29f, 0.69f, 3.7f},  {64, 64, 2, 0.23f, 0.43f, 3.9f},
                           {32, 128, 2, 0.20f, 0.48f, 4.4f},  {32, 64, 2, 0.18f, 0.20f, 3.2f}};

float time_of(const Cost& c, int64_t groups, float blocks) {
  const int64_t slots = 256 * c.per_cu, rounds = groups / slots;
  const float part = (float)(groups - rounds * slots) / (float)slots;
  float t = (float)rounds * (blocks * c.full + c.fixed);
  if (part > 0.0f && part <= 0.5f && c.bm == 256)  // in quarters or halves
    t += part <= 0.25f ? blocks * 0.58f + 4.0f : blocks * 1.03f + 5.0f;
  else if (part > 0.0f) {
    // few workgroups run at a higher clock, and of two a CU the first ones alone
    const float crowd = c.per_cu == 1 ? part : std::max(0.0f, 2.0f * part - 1.0f);
    t += blocks * (c.lone + (c.full - c.lone) * crowd) + c.fixed;
  }
  return t;
}

// Tiles of `bm` rows that `rows` rows of `experts` experts make.  How they spread is known on the device alone: taken
// as half to one and a half times the mean.
float tile_rows(int64_t rows, int64_t experts, int bm) {
  if (experts == 1) return (float)((rows + bm - 1) / bm);
  const int64_t met = std::max<int64_t>(1, std::min(experts, rows));
  int64_t tiles = 0;
  for (int q = 2; q <= 6; ++q) tiles += std::max<int64_t>(1, (rows * q / 4 / met + bm - 1) / bm);
  return (float)tiles / 5.0f * (float)met;
}

int choose(int kind, const GroupedOperands& p) {
  const int forced = tuning(kTuneGroupedTile);
  if (forced > 0 && (kind < 3 || grouped_weight_tile_known(forced & 1023, forced >> 10))) return forced;
  const int64_t met = std::max<int64_t>(1, std::min<int64_t>(p.g.experts, p.R));
  const float weights = (float)(met * p.N) * (float)p.C * 2.0f / 5.5e6f;  // from or to memory, at 5.5 TB/s
  // rows that do not begin on 128 bytes take two requests a block (1384 and 1408 features, 2060 rows of 16 experts ->
  // 2688: 49.8 and 42.6 us on 256 x 256, 74 and 56 on 128 x 128)
  const bool apart = p.ld_rows % 64 != 0 || p.ld_other % 64 != 0;
  const auto over = [](int64_t n, int b) { return (n + b - 1) / b; };
  int best = 0;
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (kind >= 3 && !grouped_weight_tile_known(c.bm, c.bn)) continue;
    const int64_t most = kind >= 3 ? over(p.N, c.bm) * p.g.experts * over(p.C, c.bn)
                                   : most_tile_rows(p.R, p.g.experts, c.bm) * over(p.N, c.bn);
    if (most > max_groups(256) - 1024) continue;  // no launch so large
    const float rows = kind >= 3 ? (float)(over(p.N, c.bm) * p.g.experts) : tile_rows(p.R, p.g.experts, c.bm);
    const float blocks = kind >= 3 ? (float)p.R / (float)met / 64.0f + 0.5f : (float)over(p.C, 64);
    const int64_t groups = (int64_t)(rows * (float)over(kind >= 3 ? p.C : p.N, c.bn));
    float t = time_of(c, groups, blocks), read = weights;
    if (kind < 3) {
      // every tile row of an expert reads its weights, and few workgroups do not keep the memory busy (16 choices of 8
      // experts, 5424 -> 5376: 336 of 32 x 128 110 us, 672 of 32 x 64 86)
      read *= 1.0f + 0.57f * (std::min(8.0f, rows / (float)met) - 1.0f);
      read *= 1.0f + 0.46f * std::max(0.0f, 1.0f - (float)groups / 512.0f);
      if (apart) t *= c.bm == 256 ? 1.09f : 1.15f, read *= c.bm == 256 ? 1.09f : 1.15f;
    }
    t = std::max(t, read) + 0.04f * t;
    if (best == 0 || t < best_time) best_time = t, best = tile_code(c.bm, c.bn);
  }
  return best;
}

}  // namespace

bool grouped_tile_known(int bm, int bn) {
#define GROUPED_KNOWN(BM, BN, STAGES, PER_CU) \
  if (bm == BM && bn == BN) return true;
  GROUPED_TILES(GROUPED_KNOWN)
  return false;
}
bool grouped_weight_tile_known(int bm, int bn) {
  GROUPED_WEIGHT_TILES(GROUPED_KNOWN)
  return false;
}

hipError_t launch_grouped(int kind, const GroupedOperands& p, int dtype, hipStream_t stream) {
  const int tile = choose(kind, p);
  if (dtype == kF16) return launch_grouped_tile<kF16>(tile, kind, p, stream);
  return launch_grouped_tile<kBF16>(tile, kind, p, stream);
}

}  // namespace convrot
