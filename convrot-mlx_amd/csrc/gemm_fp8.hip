// Products in 8-bit floating point for gfx950 (the product and its numerics are stated
// in gemm_fp8_tile.h): the choice of tile.
#include <algorithm>

#include "convrot_launch.h"
#include "fp8_device.h"

namespace convrot {
namespace {

// Time of a tile's block of 128 features (few tiles, and with every CU busy), and what its prologue and
// epilogue add, in microseconds, fitted to 16-bit products without a residual on weights from memory.
struct Cost {
  int bm, bn, per_cu;
  float lone, full, fixed;
};
constexpr Cost kCosts[] = {{256, 256, 1, 1.31f, 1.74f, 7.0f},
                           {128, 128, 2, 0.575f, 1.11f, 3.7f},
                           {64, 128, 2, 0.39f, 0.71f, 3.7f},
                           {64, 64, 2, 0.27f, 0.44f, 3.6f},
                           {32, 64, 2, 0.25f, 0.29f, 3.4f}};

// The most workgroups that may share the K of one of `tiles` tiles.
int most_splits(int64_t tiles, int kblocks, int64_t tile_bytes, const Workspace& work) {
  const int64_t bytes = work.ptr ? (int64_t)work.bytes - (int64_t)kW8a8PartialOffset : 0;
  if (bytes <= 0 || tiles > kW8a8Counters) return 1;
  return (int)std::max<int64_t>(1, std::min({(int64_t)kblocks, bytes / (tiles * tile_bytes), (int64_t)64}));
}

W8a8Split make_split(int splits, int kblocks, const Workspace& work) {
  W8a8Split s;
  s.kblocks = (kblocks + splits - 1) / splits;
  s.splits = (kblocks + s.kblocks - 1) / s.kblocks;  // no workgroup without a block
  if (s.splits > 1) {
    s.counters = (int*)(work.ptr + kW8a8CounterOffset);
    s.partials = work.ptr + kW8a8PartialOffset;
  }
  return s;
}

// Microseconds of `groups` workgroups of a tile, each of `blocks` blocks.
float time_of(const Cost& c, int64_t groups, float blocks) {
  const int64_t slots = 256 * c.per_cu, rounds = groups / slots;
  const float part = (float)(groups - rounds * slots) / (float)slots;
  float t = (float)rounds * (blocks * c.full + c.fixed);
  if (part > 0.0f && part <= 0.5f && c.bm == 256)  // in quarters or halves
    t += part <= 0.25f ? blocks * 0.65f + 5.0f : blocks * 0.95f + 6.0f;
  else if (part > 0.0f) {
    // few workgroups run at a higher clock, and of two a CU the first ones alone
    const float crowd = c.per_cu == 1 ? part : std::max(0.0f, 2.0f * part - 1.0f);
    t += blocks * (c.lone + (c.full - c.lone) * crowd) + c.fixed * (0.65f + 0.35f * part);
  }
  return t;
}

struct Choice {
  int tile, splits;
};

// The tile, and the workgroups that share its K, that the costs make fastest.  What sharing adds is the exchange
// of partial sums, written once and read once; more than a workgroup a CU loses.
Choice choose(int64_t M, int64_t N, int64_t K, const Workspace& work) {
  const int forced_tile = tuning(kTuneFp8Tile), forced_splits = tuning(kTuneFp8Split);
  const int kblocks = (int)((K + 127) / 128);
  Choice best{0, 1};
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (forced_tile > 0 && forced_tile != tile_code(c.bm, c.bn)) continue;
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const int64_t bytes = (int64_t)c.bm * c.bn * 4;
    const int most = c.bm * c.bn <= kMaxFp8SplitTile ? most_splits(tiles, kblocks, bytes, work) : 1;
    for (int s = 1; s <= most; ++s) {
      if (forced_splits > 0 ? s != std::min(forced_splits, most) : s > 1 && (kblocks < 8 * s || tiles * s > 256)) continue;
      const int64_t groups = tiles * s;
      if (groups > max_groups(512) || groups > 0x7fff0000) continue;
      float t = time_of(c, groups, (float)((kblocks + s - 1) / s));
      if (s > 1) t += 2.0f + (float)(groups * bytes) * 2.0f / 3.0e6f;
      if (best.tile == 0 || t < best_time) best_time = t, best = {tile_code(c.bm, c.bn), s};
    }
  }
  return best;
}

// The tile of grouped rows.  How they spread over the experts is known on the device alone: taken as even, each
// expert's last tile half full.
int grouped_tile(const Fp8Operands& p) {
  const int forced = tuning(kTuneFp8Tile);
  if (forced > 0) return forced;
  const int64_t met = std::min<int64_t>(p.g.experts, p.M), kblocks = (p.K + 127) / 128;
  const float each = (float)p.M / (float)met;
  int best = 0;
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    const float rows = std::max(1.0f, each / (float)c.bm + 0.5f) * (float)met;
    const float t = time_of(c, (int64_t)(rows * (float)((p.N + c.bn - 1) / c.bn)), (float)kblocks);
    if (best == 0 || t < best_time) best_time = t, best = tile_code(c.bm, c.bn);
  }
  return best;
}

template <int DT>
hipError_t launch_t(const Fp8Operands& p, const Workspace& work, hipStream_t s) {
  const int kblocks = (p.K + 127) / 128;
  if (p.g.offsets) return launch_fp8_tile<DT>(grouped_tile(p), p, make_split(1, kblocks, work), s);
  const Choice c = choose(p.M, p.N, p.K, work);
  return launch_fp8_tile<DT>(c.tile, p, make_split(c.splits, kblocks, work), s);
}

}  // namespace

bool fp8_tile_known(int bm, int bn) {
#define FP8_KNOWN(BM, BN, WM, WN, STAGES, PER_CU, SLOTS) \
  if (bm == BM && bn == BN) return true;
  FP8_TILES(FP8_KNOWN)
#undef FP8_KNOWN
  return false;
}

hipError_t launch_fp8_gemm(const Fp8Operands& p, int out_dtype, hipStream_t stream, const Workspace& work) {
  switch (out_dtype) {
    case kF32: return launch_t<kF32>(p, work, stream);
    case kF16: return launch_t<kF16>(p, work, stream);
    default: return launch_t<kBF16>(p, work, stream);
  }
}

int64_t fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  const Workspace all{(uint8_t*)256, kSkWorkspaceBytes};  // never read here
  const Choice c = choose(M, N, K, all);
  if (c.tile == 0 || c.splits <= 1) return 0;
  const int64_t bm = c.tile & 1023, bn = c.tile >> 10, tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
  return (int64_t)kW8a8PartialOffset + tiles * c.splits * bm * bn * 4;
}

}  // namespace convrot
