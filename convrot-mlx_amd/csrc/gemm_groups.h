// Output tiles of products whose rows are grouped by expert, shared by the grouped kernels.
#pragma once

#include "fp8_device.h"

namespace convrot {

// offsets[i], within 0 .. rows whatever the caller's array holds; the first group begins at row 0.
__device__ __forceinline__ int group_start(const Groups& g, int i, int rows) {
  return i == 0 ? 0 : min(max(g.offsets[i], 0), rows);
}

struct GroupTile {
  int expert;        // -1: no such tile; g.experts: rows of no expert
  int row0, row_end; // the tile's first row, and where its group ends
};

// Rows of tiles of BM rows: the experts' in order, then those of the rows behind the last one.  Every
// wave finds its own: 64 experts a step, their tiles summed over the lanes.
template <int BM>
__device__ __forceinline__ int group_tile_rows(const Groups& g, int rows) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int e0 = 0; e0 <= g.experts; e0 += 64) {
    const int e = e0 + lane;
    int n = 0;
    if (e <= g.experts) {
      const int a = group_start(g, e, rows), b = e < g.experts ? group_start(g, e + 1, rows) : rows;
      n = b > a ? (b - a + BM - 1) / BM : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d);
    total += n;
  }
  return __builtin_amdgcn_readfirstlane(total);
}

template <int BM>
__device__ __forceinline__ GroupTile group_tile(const Groups& g, int rows, int tile_row) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 <= g.experts; e0 += 64) {
    const int e = e0 + lane;
    int a = 0, b = 0;
    if (e <= g.experts) {
      a = group_start(g, e, rows);
      b = e < g.experts ? group_start(g, e + 1, rows) : rows;
    }
    const int n = b > a ? (b - a + BM - 1) / BM : 0;
    int upto = n;  // tiles of this lane's expert and those before it
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    const int first = before + upto - n;
    const uint64_t hit = __ballot(tile_row >= first && tile_row < first + n);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      const int r0 = __builtin_amdgcn_readlane(a, src) + (tile_row - __builtin_amdgcn_readlane(first, src)) * BM;
      return {e0 + src, r0, __builtin_amdgcn_readlane(b, src)};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0};
}

// How `tiles` large tiles run on `slots` CUs: whole ones in whole rounds, and those of the last round as 4 or 2
// parts each while that gives a CU at most one workgroup.
struct LastRound {
  int whole, parts;
};
__host__ __device__ __forceinline__ LastRound last_round(int tiles, int slots) {
  const int rest = tiles % slots;
  const int parts = rest == 0 ? 1 : rest * 4 <= slots ? 4 : rest * 2 <= slots ? 2 : 1;
  return {parts == 1 ? tiles : tiles - rest, parts};
}

// A wave's TM x TN corner of a 16-bit [.., N] array between memory and its LDS rows (TN * 2 + 16 bytes apart), 16
// bytes a lane and step; rows below row_end.  A row of any N begins anywhere: the hardware takes 16 bytes at any
// address, which for odd N costs less than shifting the rows in LDS to whole aligned chunks with part chunks at both
// ends of every corner's row (2060 rows of 16 experts, 1384 -> 2685, on 256 x 256: 52.2 and 61.5 us).  BATCH loads of
// a lane are in flight at a time.
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
template <int TM, int TN, bool STORE, int BATCH = 16>
__device__ __forceinline__ void move_rows(uint8_t* region, uint16_t* base, int lane, int mw, int nw, int row_end, int N) {
  constexpr int RS = TN * 2 + 16, CPR = TN / 8, NIT = TM * CPR / 64;
  static_assert(TM * CPR % 64 == 0, "whole steps");
  const int cols = min(TN, N - nw), rows = min(TM, row_end - mw);
  if constexpr (!STORE) {
    for (int b0 = 0; b0 < NIT; b0 += BATCH) {
      u32x4 v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int c = (b0 + i) * 64 + lane, row = c / CPR, first = c % CPR * 8;
        v[i] = (u32x4){0, 0, 0, 0};
        if (row < rows && first + 8 <= cols)
          v[i] = *(const u32x4_at2*)(base + (int64_t)(mw + row) * N + nw + first);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int c = (b0 + i) * 64 + lane;
        if (c < TM * CPR) *(u32x4*)(region + c / CPR * RS + c % CPR * 16) = v[i];
      }
    }
  } else {
#pragma unroll 4
    for (int it = 0; it < NIT; ++it) {
      const int c = it * 64 + lane, row = c / CPR, first = c % CPR * 8;
      if (row < rows && first + 8 <= cols)
        *(u32x4_at2*)(base + (int64_t)(mw + row) * N + nw + first) = *(const u32x4*)(region + row * RS + first * 2);
    }
  }
  // the last columns where N is no multiple of 8, 8 lanes a row
  const int last = cols & ~7;
  if (last < cols && last >= 0) {
    for (int row = lane >> 3; row < rows; row += 8) {
      const int col = last + (lane & 7);
      if (col >= cols) continue;
      uint16_t* at = (uint16_t*)(region + row * RS) + col;
      uint16_t* g = base + (int64_t)(mw + row) * N + nw + col;
      if constexpr (STORE) *g = *at;
      else *at = *g;
    }
  }
}

// Most rows of tiles that any split of `rows` over the experts (and none) makes.
inline int64_t most_tile_rows(int64_t rows, int64_t experts, int bm) {
  const int64_t bound = rows / bm + experts + 1;
  return rows < bound ? rows : bound;
}

// n / d for 0 <= n < 2^31 by a product: d in 1 .. 2^31 - 1.
struct Divisor {
  uint32_t factor = 1;
  int shift = 0;
  Divisor() = default;
  explicit Divisor(uint32_t d) {
    while ((uint64_t(1) << shift) < d) ++shift;
    factor = (uint32_t)((((uint64_t(1) << shift) - d) << 32) / d) + 1;
  }
  __device__ __forceinline__ uint32_t divide(uint32_t n) const { return (__umulhi(factor, n) + n) >> shift; }
};

// What a launch computes: KIND 0 forward on sorted rows, 1 on rows read through the index, 2 the rows' gradient,
// 3 the weights' on sorted rows, 4 on rows of x read through the index.
struct GroupedOperands {
  const uint16_t *rows, *other;  // x (or dy); the weights, or (KIND 3, 4) x beside dy
  int64_t ld_rows, ld_other;     // elements between rows
  int64_t expert;                // elements between experts' weights
  uint16_t* out;
  int R;                         // sorted rows
  int N, C;                      // columns of the output, length contracted (KIND 3, 4: rows and columns of a weight, N x C)
  Groups g;
  Divisor choices;               // KIND 4: g.choices
};

// The tiled product of one type (gemm_grouped_tile.h, one source a type).
template <int DT>
hipError_t launch_grouped_tile(int tile, int kind, const GroupedOperands& p, hipStream_t stream);

// The tiles built: BM, BN, ring stages, workgroups a CU; for rows, and for the weights' gradient.
#define GROUPED_TILES(X) \
  X(256, 256, 2, 1) X(128, 128, 2, 2) X(64, 128, 3, 2) X(64, 64, 5, 2) X(32, 128, 4, 2) X(32, 64, 6, 2)
#define GROUPED_WEIGHT_TILES(X) X(256, 256, 2, 1) X(128, 128, 2, 2)

}  // namespace convrot
