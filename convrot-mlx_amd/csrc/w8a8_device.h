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

// LDS position of a 16-byte chunk of a 128-byte row: 16 rows of one fragment read meet no bank twice.
__device__ __forceinline__ int chunk_swizzle(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Partial sums of workgroups that share a tile's K travel through the caller's
// workspace with device scope (sc1): coherent across the XCDs' L2s without
// writing one back.  Both are ordinary buffer accesses to the compiler, which
// waits for them.
constexpr int kDeviceScope = 16;  // sc1
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t partial_rsrc(void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(base, (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void store_partial(__amdgpu_buffer_rsrc_t r, uint32_t off, const i32x4& v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, (int)off, 0, kDeviceScope);
}
__device__ __forceinline__ i32x4 load_partial(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, kDeviceScope));
}

// Called by every thread of a workgroup after its store_partials: whether it is
// the last of the `splits` workgroups of its tile to arrive, whose partials are
// then all in memory.  The counter is back at zero when the launch ends.
__device__ __forceinline__ bool last_to_arrive(int* counter, int splits, int* shared) {
  __builtin_amdgcn_s_waitcnt(0);  // this wave's partials are at the coherence point
  asm volatile("" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = n == splits - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = last;
  }
  __syncthreads();
  return *shared != 0;
}

constexpr int kMaxSplitTile = 160 * 128;  // tiles up to this size may share their K between workgroups

// How a launch shares K: `splits` workgroups a tile, each `kblocks` blocks of 128.
struct W8a8Split {
  int splits = 1, kblocks = 0;
  int* counters = nullptr;
  uint8_t* partials = nullptr;
};

// The tiled product of one output type (gemm_w8a8_tile.h, one source a type);
// `tile` is one of W8A8_TILES.
template <int ODT>
hipError_t launch_w8a8_tile(int tile, const W8a8Operands& p, const W8a8Split& split, hipStream_t stream);

constexpr int tile_code(int bm, int bn) { return bm | bn << 10; }

// The tiles built: BM, BN, ring stages, workgroups a CU.
#define W8A8_TILES(X) \
  X(256, 256, 2, 1) X(256, 224, 2, 1) X(224, 256, 2, 1) X(256, 192, 2, 1) X(192, 256, 2, 1) X(256, 128, 3, 1) \
  X(128, 256, 3, 1) X(192, 192, 3, 1) X(192, 128, 2, 2) X(128, 192, 2, 2) X(160, 128, 4, 1) X(128, 160, 4, 1) \
  X(128, 128, 2, 2) X(128, 64, 3, 2) X(64, 128, 3, 2) X(64, 64, 4, 2)

}  // namespace convrot
