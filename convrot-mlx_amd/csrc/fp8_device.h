// What the kernels of 8-bit floating point share: e4m3 codes with a float32 scale
// for each block of 128, and the operands of their products.
//
// A block whose largest magnitude is a has the scale s = 2^p, the smallest power of
// two with a / s <= 448, the type's largest value.  Dividing by a power of two is
// exact, so the code is x / s rounded once (to the nearest, ties to even), whatever
// order or precision the scale is applied in; against s = a / 448 the codes lose at
// most a bit of range at the low end (values below 2^-6 s lose mantissa bits), none
// of their precision.
#pragma once

#include "w8a8_device.h"

namespace convrot {

constexpr int kBlock = 128;                      // features (and of a weight, outputs) under one scale
constexpr uint32_t kPastEnd = 0xffffff00u;       // buffer offset past every operand: reads zero
constexpr int64_t kMaxExtent = 0xfffff000ll;     // bytes of an operand that is addressed as one buffer

struct Fp8Scale {
  float inverse, scale;
};
// From the bits of a block's largest magnitude (infinity lies above every number, NaN above
// infinity).  Below 2^-100: a block of zeros; not finite: the scale NaN (every product of the block
// is NaN).
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t most) {
  if (most >= 0x7f800000u) return {0.0f, __builtin_nanf("")};
  if (most < (27u << 23)) return {0.0f, 0.0f};
  // a = m 2^e with m in [1, 2): 448 = 1.75 * 2^8
  const uint32_t p = (most >> 23) - 8u + ((most & 0x7fffffu) > 0x600000u ? 1u : 0u);  // biased
  return {__builtin_bit_cast(float, (254u - p) << 23), __builtin_bit_cast(float, p << 23)};
}
// Four codes of values over the scale; in a block that is not finite any value is 0 (the scale is NaN).
__device__ __forceinline__ uint32_t fp8_codes4(const float* v, float inverse) {
  float t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = inverse == 0.0f ? 0.0f : v[j] * inverse;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
}

// The 32 codes of a lane's part of a fragment as bf16 (exact).
typedef int i32x8 __attribute__((ext_vector_type(8)));
struct WideCodes {
  bf16x8 v[4];
};
__device__ __forceinline__ WideCodes widen_codes(const i32x8& c) {
  WideCodes w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    i32x4 t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      t[2 * h] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i + h], 1.0f, false));
      t[2 * h + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i + h], 1.0f, true));
    }
    w.v[i] = __builtin_bit_cast(bf16x8, t);
  }
  return w;
}

// Rows grouped by expert: expert e has rows offsets[e] .. offsets[e + 1] - 1 of `rows`; those from
// offsets[experts] on have none and give zeros.  With `index`, sorted row s is row index[s] / choices
// of the activations.
struct Groups {
  const int* offsets = nullptr;
  const int* index = nullptr;
  int experts = 0, choices = 1;
  int64_t act_rows = 0;
};

struct Fp8Operands {
  const uint8_t* act;
  const uint8_t* weight;
  int64_t lda, ldw;
  const float *xscales, *wscales, *bias;
  int64_t xs_row, xs_block;  // floats between the scales of rows, of blocks
  int64_t ws_row;            // floats between the scales of blocks of outputs
  void* out;
  int M, N, K;
  GatedResidual gr;
  Groups g;
  int64_t weight_expert, ws_expert;  // bytes and floats between experts
};

// The tiled product of one output type (gemm_fp8_tile.h, one source a type); `tile` is one of FP8_TILES.
template <int ODT>
hipError_t launch_fp8_tile(int tile, const Fp8Operands& p, const W8a8Split& split, hipStream_t stream);

constexpr int kMaxFp8SplitTile = 128 * 128;  // tiles up to this size may share their K between workgroups

// The tiles built: BM, BN, waves along each, ring stages, workgroups a CU, and whether the MFMAs run in slots
// (run_slots of gemm_fp8_tile.h).  In slots and not, in us: 256 x 256 (8192 x 8192 -> 8192) 468 and 540, 32 x 64 (1 row
// 4096 -> 12288) 11.8 and 12.5, 64 x 64 (128 rows 4096 -> 4096) 12.8 and 13.3; 128 x 128 and 64 x 128, whose LDS traffic
// bounds them, 640 and 573 (8192 x 8192 -> 8192), 29.0 and 27.0 (1024 x 4096 -> 4096).  With 8 waves 128 x 128 takes
// 26 us there, with 4 29.9.
#define FP8_TILES(X) \
  X(256, 256, 4, 2, 2, 1, true) X(128, 128, 2, 4, 2, 2, false) X(64, 128, 2, 4, 3, 2, false) X(64, 64, 2, 2, 4, 2, true) \
  X(32, 64, 1, 4, 5, 2, true)

}  // namespace convrot
