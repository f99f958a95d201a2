// Rows of features held in the registers of a team of threads: loads, stores
// and reductions shared by the row kernels (norm.hip, rotary.hip).
#pragma once

#include "convrot_device.h"

namespace convrot {

// A team of T threads holds a row as C chunks of 8 features a thread.  VEC:
// chunk c of thread t is features 8 (c T + t) .. +7, moved as 16-byte accesses
// (rows 16-byte aligned, features % 8 == 0).  Otherwise value j of the chunk
// is feature (8 c + j) T + t: any alignment, one element an access, whole
// lines a wave.
template <int T, int C, bool VEC>
__device__ __forceinline__ int feature_of(int t, int c, int j) {
  return VEC ? (c * T + t) * 8 + j : (c * 8 + j) * T + t;
}

// Eight consecutive values at p (16-byte aligned) as floats.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, float (&v)[8]) {
  if constexpr (DT == kF32) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 w = *(const uint4*)p;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kBF16) {
        v[2 * i] = bf16_lo(u[i]), v[2 * i + 1] = bf16_hi(u[i]);
      } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 h = __builtin_bit_cast(f16x2, u[i]);
        v[2 * i] = (float)h.x, v[2 * i + 1] = (float)h.y;
      }
    }
  }
}

// The same values rounded once to DT.
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&v)[8]) {
  if constexpr (DT == kF32) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (DT == kBF16) {
    *(uint4*)p = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                            pack_bf16x2(v[6], v[7]));
  } else {
    *(uint4*)p = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]),
                            pack_f16x2(v[6], v[7]));
  }
}

// Chunk c of a row of K features; features past the row read as `pad`.
template <int DT, int T, int C, bool VEC>
__device__ __forceinline__ void load_chunk(const typename Elem<DT>::T* row, int K, int t, int c, float (&v)[8],
                                           float pad = 0.0f) {
  if constexpr (VEC) {
    const int f = feature_of<T, C, VEC>(t, c, 0);
    if (f < K) {
      load8<DT>(row + f, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = pad;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = feature_of<T, C, VEC>(t, c, j);
      v[j] = f < K ? (float)row[f] : pad;
    }
  }
}

template <int DT, int T, int C, bool VEC>
__device__ __forceinline__ void store_chunk(typename Elem<DT>::T* row, int K, int t, int c, const float (&v)[8]) {
  if constexpr (VEC) {
    const int f = feature_of<T, C, VEC>(t, c, 0);
    if (f < K) store8<DT>(row + f, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = feature_of<T, C, VEC>(t, c, j);
      if (f < K) row[f] = (typename Elem<DT>::T)v[j];
    }
  }
}

// The same of a parameter row, whose type is known at run time only (the
// activations' or float32).
template <int DT, int T, int C, bool VEC>
__device__ __forceinline__ void load_param(const void* row, int dtype, int K, int t, int c, float (&v)[8]) {
  if (DT != kF32 && dtype == kF32) load_chunk<kF32, T, C, VEC>((const float*)row, K, t, c, v);
  else load_chunk<DT, T, C, VEC>((const typename Elem<DT>::T*)row, K, t, c, v);
}

// Sum (or maximum of unsigned words) over a wave of 64, in every lane.  The
// order of the additions is fixed, so results repeat bit for bit.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

}  // namespace convrot
