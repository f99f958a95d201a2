// What the W8A8 kernels share: their operands, and the gated residual and store
// of a lane's 4 outputs.
#pragma once

#include "convrot_device.h"

namespace convrot {

constexpr uint32_t kOutOfRange = 0x80000000u;  // buffer offset past every operand: reads zero

struct W8a8Operands {
  const int8_t* act;
  const int8_t* weight;
  int64_t lda, ldw;
  const float *xscales, *wscales, *bias;
  void* out;
  int M, N, K;
  GatedResidual gr;
};

// Gate of outputs n .. n + 3 of row m (1 without a gate; columns past N: any).
template <int ODT>
__device__ __forceinline__ void load_gate4(const GatedResidual& gr, int m, int n, int N, float (&g)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = 1.0f;
  if (!gr.gate) return;
  const int64_t at = (int64_t)(m / gr.rows_per_gate) * gr.gate_stride + n;
  if ((gr.gate_stride & 3) == 0 && n + 3 < N) {
    load_elem4<ODT>(gr.gate, at, g);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < N) g[j] = load_elem<ODT>(gr.gate, at + j);
  }
}

// Outputs n .. n + 3 of row m < M (those below N), with the gated residual; vec: N % 4 == 0.
template <int ODT>
__device__ __forceinline__ void store4(const W8a8Operands& p, int m, int n, bool vec, float (&o)[4]) {
  const int64_t at = (int64_t)m * p.N + n;
  if (p.gr.residual) {
    float g[4], res[4];
    load_gate4<ODT>(p.gr, m, n, p.N, g);
    if (vec) {
      load_elem4<ODT>(p.gr.residual, at, res);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) res[j] = n + j < p.N ? load_elem<ODT>(p.gr.residual, at + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = res[j] + g[j] * o[j];
  }
  if (vec) {
    store_out4<ODT>(p.out, at, o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) store_out<ODT>(p.out, at + j, o[j]);
  }
}

// The tiled product of one output type (gemm_w8a8_tile.h, one source a type);
// `tile` is one of W8A8_TILES.
template <int ODT>
hipError_t launch_w8a8_tile(int tile, const W8a8Operands& p, hipStream_t stream);

constexpr int tile_code(int bm, int bn) { return bm | bn << 10; }

// The tiles built: BM, BN, ring stages, workgroups a CU.
#define W8A8_TILES(X) \
  X(256, 256, 2, 1) X(256, 224, 2, 1) X(224, 256, 2, 1) X(256, 192, 2, 1) X(192, 256, 2, 1) X(256, 128, 3, 1) \
  X(128, 256, 3, 1) X(192, 192, 3, 1) X(192, 128, 3, 1) X(128, 192, 3, 1) X(160, 128, 4, 1) X(128, 160, 4, 1) \
  X(128, 128, 2, 2) X(128, 64, 3, 2) X(64, 128, 3, 2) X(64, 64, 4, 2)

}  // namespace convrot
