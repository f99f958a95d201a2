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

// Eight values of a row as they were loaded (widened to floats only when used).
template <int DT, int T, int C, bool VEC>
struct RawChunk {
  static constexpr int W = DT == kF32 ? 8 : 4;  // 32-bit words
  uint32_t w[W];
  __device__ __forceinline__ void load(const typename Elem<DT>::T* row, int K, int t, int c) {
    if constexpr (VEC) {
      const int f = feature_of<T, C, VEC>(t, c, 0);
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (f < K) v = ((const uint4*)(row + f))[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (DT == kF32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int f = feature_of<T, C, VEC>(t, c, j);
        w[j] = f < K ? ((const uint32_t*)row)[f] : 0;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const int f = feature_of<T, C, VEC>(t, c, j), g = feature_of<T, C, VEC>(t, c, j + 1);
        const uint32_t lo = f < K ? ((const uint16_t*)row)[f] : 0, hi = g < K ? ((const uint16_t*)row)[g] : 0;
        w[j / 2] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (W == 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_bit_cast(float, w[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kBF16) {
          v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
        } else {
          typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
          const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
          v[2 * i] = (float)h.x, v[2 * i + 1] = (float)h.y;
        }
      }
    }
  }
};

// The same of a parameter row, whose type is known at run time only (the
// activations' or float32).
template <int DT, int T, int C, bool VEC>
__device__ __forceinline__ void load_param(const void* row, int dtype, int K, int t, int c, float (&v)[8]) {
  if (DT != kF32 && dtype == kF32) load_chunk<kF32, T, C, VEC>((const float*)row, K, t, c, v);
  else load_chunk<DT, T, C, VEC>((const typename Elem<DT>::T*)row, K, t, c, v);
}

template <int V>
struct Const {
  static constexpr int value = V;
};

// v of the lane that DPP control CTRL pairs this one with.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e;                // quad_perm
constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;      // lane i <-> 7 - i of 8, 15 - i of 16

// Sum over aligned groups of G <= 64 lanes (a power of two), in every lane, in a fixed order.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp<kDppXor1>(v);
  if constexpr (G >= 4) v += dpp<kDppXor2>(v);
  if constexpr (G >= 8) v += dpp<kDppHalfMirror>(v);
  if constexpr (G >= 16) v += dpp<kDppMirror>(v);
  if constexpr (G == 32) v += __shfl_xor(v, 16);
  if constexpr (G == 64) {
    const int w = __builtin_bit_cast(int, v);
    v = (__builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 0)) +
         __builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 16))) +
        (__builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 32)) +
         __builtin_bit_cast(float, __builtin_amdgcn_readlane(w, 48)));
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) { return group_sum<64>(v); }

// The bits of the largest magnitude of 8 values, and over 16 neighbouring lanes.
__device__ __forceinline__ uint32_t most_of(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t max_of_16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor1, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor2, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppHalfMirror, 0xf, 0xf, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppMirror, 0xf, 0xf, true));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto other = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  v = max(v, other(v, Const<kDppXor1>{}));
  v = max(v, other(v, Const<kDppXor2>{}));
  v = max(v, other(v, Const<kDppHalfMirror>{}));
  v = max(v, other(v, Const<kDppMirror>{}));
  const int w = (int)v;
  return max(max((uint32_t)__builtin_amdgcn_readlane(w, 0), (uint32_t)__builtin_amdgcn_readlane(w, 16)),
             max((uint32_t)__builtin_amdgcn_readlane(w, 32), (uint32_t)__builtin_amdgcn_readlane(w, 48)));
}

// ---- 8-bit codes of a row whose largest |x| has the bits `most` (as an unsigned
// word, infinity lies above every number and NaN above infinity).
struct Int8Row {
  float inv, scale;
  bool finite;
};
__device__ __forceinline__ Int8Row int8_row(uint32_t most) {
  const float a = __builtin_bit_cast(float, most);
  const bool finite = most < 0x7f800000u, zero = a < 0x1p-100f;
  return {finite && !zero ? 127.0f / a : 0.0f, !finite ? __builtin_nanf("") : zero ? 0.0f : a * (1.0f / 127.0f),
          finite};
}
// |x inv| <= 127 up to its last bit, which the rounding drops; a row that is not finite gets zeros.
__device__ __forceinline__ int int8_code(float v, const Int8Row& q) { return q.finite ? (int)rintf(v * q.inv) : 0; }

__device__ __forceinline__ uint2 int8_codes(const float (&v)[8], const Int8Row& q) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j / 4] |= (uint32_t)(int8_code(v[j], q) & 0xff) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}

}  // namespace convrot
