// W8A8 GEMM for gfx950 (8-bit integer activations and weights; the product and its
// numerics are stated in gemm_w8a8_tile.h): the kernel for a few token rows, and
// the choice of kernel.
#include <stdlib.h>

#include <algorithm>

#include "convrot_launch.h"
#include "w8a8_device.h"

namespace convrot {
namespace {

// ---- few rows
//
// The weights' bytes bound it: each is read once, straight into registers.  A
// workgroup owns NB tiles of 16 output channels and 16 FM tokens; its SPLIT
// waves share K, a block of 128 in turn, and add their integer sums through LDS.
template <int FM, int NB, int SPLIT, int UNROLL, int ODT>
__global__ __launch_bounds__(SPLIT * 64) void w8a8_rows_kernel(W8a8Operands p) {
  __shared__ __attribute__((aligned(16))) i32x4 red[SPLIT][NB * FM][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, r = lane & 15;
  const int n0 = blockIdx.x * (16 * NB), m0 = blockIdx.y * (16 * FM);
  const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u;
  const int mrows = min(16 * FM, p.M - m0), nrows = min(16 * NB, p.N - n0);
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.act + (int64_t)m0 * p.lda), (short)0, (int)((uint32_t)(mrows - 1) * (uint32_t)p.lda + k16), 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.weight + (int64_t)n0 * p.ldw), (short)0, (int)((uint32_t)(nrows - 1) * (uint32_t)p.ldw + k16),
      0x00020000);
  i32x4 acc[NB][FM];
#pragma unroll
  for (int a = 0; a < NB; ++a)
#pragma unroll
    for (int b = 0; b < FM; ++b) acc[a][b] = (i32x4){0, 0, 0, 0};

  const uint32_t steps = (k16 + 63) / 64;  // of 64 features
  for (uint32_t s0 = wave * UNROLL; s0 < steps; s0 += SPLIT * UNROLL) {
    u32x4 w[UNROLL][NB], a[UNROLL][FM];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const uint32_t k = (s0 + i) * 64u + (uint32_t)q * 16u;  // the lane's 16 features
      const uint32_t wo = k < k16 ? (uint32_t)r * (uint32_t)p.ldw + k : kOutOfRange;
#pragma unroll
      for (int t = 0; t < NB; ++t)
        w[i][t] = __builtin_amdgcn_raw_buffer_load_b128(rw, (int)(wo + (uint32_t)t * 16u * (uint32_t)p.ldw), 0, 0);
#pragma unroll
      for (int f = 0; f < FM; ++f)
        a[i][f] = __builtin_amdgcn_raw_buffer_load_b128(ra, (int)((uint32_t)(16 * f + r) * (uint32_t)p.lda + k), 0, 0);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
#pragma unroll
      for (int t = 0; t < NB; ++t)
#pragma unroll
        for (int f = 0; f < FM; ++f)
          acc[t][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w[i][t]),
                                                            __builtin_bit_cast(i32x4, a[i][f]), acc[t][f], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < NB; ++t)
#pragma unroll
    for (int f = 0; f < FM; ++f) red[wave][t * FM + f][lane] = acc[t][f];
  __syncthreads();
  // wave w finishes the output tiles w, w + SPLIT, ..
  const bool vec = (p.N & 3) == 0;
  for (int i = wave; i < NB * FM; i += SPLIT) {
    const int t = i / FM, f = i % FM;
    i32x4 s = red[0][i][lane];
#pragma unroll
    for (int w2 = 1; w2 < SPLIT; ++w2) s += red[w2][i][lane];
    const int m = m0 + f * 16 + r, n = n0 + t * 16 + 4 * q;
    if (m >= p.M || n >= p.N) continue;
    const float xs = p.xscales[m];
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int nn = min(n + j, p.N - 1);
      o[j] = (((float)s[j] * xs) * p.wscales[nn]) + (p.bias ? p.bias[nn] : 0.0f);
    }
    store4<ODT>(p, m, n, vec, o);
  }
}

template <int FM, int NB, int SPLIT, int UNROLL, int ODT>
hipError_t launch_rows(const W8a8Operands& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 16 * NB - 1) / (16 * NB)), (unsigned)((p.M + 16 * FM - 1) / (16 * FM)));
  w8a8_rows_kernel<FM, NB, SPLIT, UNROLL, ODT><<<grid, dim3(SPLIT * 64), 0, s>>>(p);
  return hipGetLastError();
}

// Kernel of a product: 0 few rows, else tile_code of a tile.
int plan(int64_t M, int64_t N, int64_t K) {
  const int forced = tuning(kTuneW8a8Tile);
  if (forced >= 0) return forced;
  if (M <= 64) return 0;
  return N >= 512 && M >= 512 ? tile_code(256, 256) : tile_code(128, 128);
}

template <int ODT>
hipError_t launch_t(const W8a8Operands& p, hipStream_t s) {
  const int tile = plan(p.M, p.N, p.K);
  switch (tile) {
    case 0:
      if (p.M <= 16) {
        if (p.N <= 8192) return launch_rows<1, 1, 16, 4, ODT>(p, s);
        return launch_rows<1, 1, 4, 6, ODT>(p, s);
      }
      if (p.M <= 32) return launch_rows<2, 1, 8, 4, ODT>(p, s);
      return launch_rows<4, 1, 8, 2, ODT>(p, s);
    default: return launch_w8a8_tile<ODT>(tile, p, s);
  }
}

}  // namespace

bool w8a8_tile_known(int bm, int bn) {
  if (bm == 0 && bn == 0) return true;
#define W8A8_KNOWN(BM, BN, STAGES, PER_CU) \
  if (bm == BM && bn == BN) return true;
  W8A8_TILES(W8A8_KNOWN)
#undef W8A8_KNOWN
  return false;
}

hipError_t launch_w8a8_gemm(const int8_t* act, int64_t lda, const float* xscales, const int8_t* weight, int64_t ldw,
                            const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K, void* out,
                            int out_dtype, hipStream_t stream, const GatedResidual& gr) {
  const W8a8Operands p{act, weight, lda, ldw, xscales, wscales, bias, out, (int)M, (int)N, (int)K, gr};
  switch (out_dtype) {
    case kF32: return launch_t<kF32>(p, stream);
    case kF16: return launch_t<kF16>(p, stream);
    default: return launch_t<kBF16>(p, stream);
  }
}

}  // namespace convrot
