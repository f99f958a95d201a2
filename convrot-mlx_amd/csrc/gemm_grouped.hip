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
constexpr Cost kCosts[] = {{256, 256, 1, 1.25f, 1.56f, 8.0f}, {128, 128, 2, 0.62f, 0.92f, 3.0f},
                           {64, 128, 2, 0.33f, 0.60f, 3.0f},  {64, 64, 2, 0.24f, 0.38f, 3.0f},
                           {32, 128, 2, 0.24f, 0.36f, 3.0f},  {32, 64, 2, 0.19f, 0.27f, 3.0f}};

float time_of(const Cost& c, int64_t groups, float blocks) {
  const int64_t slots = 256 * c.per_cu, rounds = groups / slots;
  const float part = (float)(groups - rounds * slots) / (float)slots;
  float t = (float)rounds * (blocks * c.full + c.fixed);
  if (part > 0.0f && part <= 0.5f && c.bm == 256)  // in quarters or halves
    t += part <= 0.25f ? blocks * 0.55f + 4.0f : blocks * 0.85f + 5.0f;
  else if (part > 0.0f)
    t += blocks * (c.lone + (c.full - c.lone) * part) + c.fixed;
  return t;
}

// How the rows spread over the experts is known on the device alone: taken as even, each expert's last tile half
// full.
int choose(int kind, const GroupedOperands& p) {
  const int forced = tuning(kTuneGroupedTile);
  if (forced > 0 && (kind != 3 || grouped_weight_tile_known(forced & 1023, forced >> 10))) return forced;
  const int64_t met = std::max<int64_t>(1, std::min<int64_t>(p.g.experts, p.R));
  const float each = (float)p.R / (float)met;
  const auto over = [](int64_t n, int b) { return (n + b - 1) / b; };
  int best = 0;
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (kind == 3 && !grouped_weight_tile_known(c.bm, c.bn)) continue;
    const float rows = kind == 3 ? (float)(over(p.N, c.bm) * p.g.experts)
                                 : std::max(1.0f, each / (float)c.bm + (met > 1 ? 0.5f : 0.0f)) * (float)met;
    const float blocks = kind == 3 ? each / 64.0f + 0.5f : (float)over(p.C, 64);
    const float t = time_of(c, (int64_t)(rows * (float)over(kind == 3 ? p.C : p.N, c.bn)), blocks);
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
