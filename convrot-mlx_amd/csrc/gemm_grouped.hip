// Products of rows grouped by expert in 16 bits (gemm_grouped_tile.h): the choice of tile.
#include "convrot_launch.h"
#include "gemm_groups.h"

namespace convrot {
namespace {

int choose(int kind, const GroupedOperands& p) {
  const int forced = tuning(kTuneGroupedTile);
  if (forced > 0 && (kind != 3 || grouped_weight_tile_known(forced & 1023, forced >> 10))) return forced;
  const auto tiles = [](int64_t n, int b) { return (n + b - 1) / b; };
  if (kind == 3)
    return p.g.experts * tiles(p.N, 256) * tiles(p.C, 256) >= 128 ? tile_code(256, 256) : tile_code(128, 128);
  const int64_t each = (p.R + p.g.experts - 1) / p.g.experts;  // rows of an expert, were they all alike
  if (each <= 32) return tile_code(32, 64);
  if (each <= 64) return tile_code(64, 128);
  if (each <= 256) return tile_code(128, 128);
  return tile_code(256, 256);
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
