// Products of rows grouped by expert in 16 bits (gemm_grouped_tile.h): the choice of tile.
#include <algorithm>

#include "convrot_launch.h"
#include "gemm_groups.h"

namespace convrot {
namespace {

// Time of a tile's block of 64 (few tiles, and with every CU busy), and what its prologue and epilogue add, in
// microseconds, fitted to measurements on weights from memory.
struct Cost {
  int bm, bn, per_cu;
  float lone, full, fixed;
};
constexpr Cost kCosts[] = {{256, 256, 1, 1.30f, 1.62f, 8.0f}, {128, 128, 2, 0.70f, 1.15f, 3.0f},
                           {64, 128, 2, 0.36f, 0.72f, 3.0f},  {64, 64, 2, 0.25f, 0.46f, 3.0f},
                           {32, 128, 2, 0.26f, 0.42f, 3.0f},  {32, 64, 2, 0.19f, 0.31f, 3.0f}};

float time_of(const Cost& c, int64_t groups, float blocks) {
  const int64_t slots = 256 * c.per_cu, rounds = groups / slots;
  const float part = (float)(groups - rounds * slots) / (float)slots;
  float t = (float)rounds * (blocks * c.full + c.fixed);
  if (part > 0.0f && part <= 0.5f && c.bm == 256)  // in quarters or halves
    t += part <= 0.25f ? blocks * 0.55f + 4.0f : blocks * 0.85f + 5.0f;
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
  if (forced > 0 && (kind != 3 || grouped_weight_tile_known(forced & 1023, forced >> 10))) return forced;
  const int64_t met = std::max<int64_t>(1, std::min<int64_t>(p.g.experts, p.R));
  const float weights = (float)(met * p.N) * (float)p.C * 2.0f / 5.0e6f;  // from or to memory, at 5 TB/s
  const auto over = [](int64_t n, int b) { return (n + b - 1) / b; };
  int best = 0;
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (kind == 3 && !grouped_weight_tile_known(c.bm, c.bn)) continue;
    const float rows = kind == 3 ? (float)(over(p.N, c.bm) * p.g.experts) : tile_rows(p.R, p.g.experts, c.bm);
    const float blocks = kind == 3 ? (float)p.R / (float)met / 64.0f + 0.5f : (float)over(p.C, 64);
    float t = time_of(c, (int64_t)(rows * (float)over(kind == 3 ? p.C : p.N, c.bn)), blocks);
    t = std::max(t, weights) + 0.1f * t;
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
  return dtype == kF16 ? launch_grouped_tile<kF16>(tile, kind, p, stream) : launch_grouped_tile<kBF16>(tile, kind, p, stream);
}

}  // namespace convrot
