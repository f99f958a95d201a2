// Quantizers to 8-bit floating point: rows in blocks of 128 features, weights in
// blocks of 128 x 128 (fp8_device.h).
#include "convrot_launch.h"
#include "fp8_device.h"
#include "row_device.h"

namespace convrot {
namespace {

// Eight features from k on of a row of K (zeros past its end).
template <int DT, bool VEC>
__device__ __forceinline__ void load_features(const typename Elem<DT>::T* row, int64_t k, int64_t K, float (&v)[8]) {
  if (VEC && k + 8 <= K) {
    load8<DT>(row + k, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? (float)row[k + j] : 0.0f;
  }
}

// 16 lanes a block, 8 features a lane: one pass, bound by reading the rows.  A workgroup takes 16
// rows and `per` blocks of them behind each other, so that the scales of 16 rows, which lie beside
// each other, go out as one line.  Codes from K to the end of the last block are zeros.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t rows,
                                                       int64_t K, int64_t x_stride, uint8_t* __restrict__ codes,
                                                       int64_t codes_stride, float* __restrict__ scales,
                                                       int64_t xs_row, int64_t xs_block, int blocks, int per) {
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane = threadIdx.x & 15;
  const int b1 = min(blocks, (int)(blockIdx.y + 1) * per);
  if (row >= rows) return;  // whole groups of 16 lanes
  const typename Elem<DT>::T* xr = x + row * x_stride;
  for (int b = (int)blockIdx.y * per; b < b1; ++b) {
    const int64_t k = (int64_t)b * kBlock + lane * 8;
    float v[8];
    load_features<DT, VEC>(xr, k, K, v);
    const Fp8Scale s = fp8_scale(max_of_16(most_of(v)));
    const uint2 w = {fp8_codes4(v, s.inverse), fp8_codes4(v + 4, s.inverse)};
    if (k + 8 <= codes_stride) *(uint2*)(codes + row * codes_stride + k) = w;
    if (lane == 0) scales[row * xs_row + b * xs_block] = s.scale;
  }
}

// A workgroup a block of 128 x 128: each thread holds 8 rows' 8 features, so the weight is read once: 8192 x 8192 in
// bfloat16 40 us (5.0 TB/s), 2048 x 2048 of one expert 9.2.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const typename Elem<DT>::T* __restrict__ w, int64_t N,
                                                         int64_t K, int64_t w_stride, uint8_t* __restrict__ codes,
                                                         int64_t codes_stride, float* __restrict__ scales, int blocks) {
  __shared__ uint32_t part[4];
  const int64_t nb = blockIdx.x / blocks, kb = blockIdx.x % blocks;
  const int lane = threadIdx.x & 15;
  const int64_t k = kb * kBlock + lane * 8, n0 = nb * kBlock + (threadIdx.x >> 4);
  float v[8][8];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + 16 * i;
    if (n < N) {
      load_features<DT, VEC>(w + n * w_stride, k, K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
    most = max(most, most_of(v[i]));
  }
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
  const Fp8Scale s = fp8_scale(max(max(part[0], part[1]), max(part[2], part[3])));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + 16 * i;
    const uint2 c = {fp8_codes4(v[i], s.inverse), fp8_codes4(v[i] + 4, s.inverse)};
    if (n < N && k + 8 <= codes_stride) *(uint2*)(codes + n * codes_stride + k) = c;
  }
  if (threadIdx.x == 0) scales[nb * blocks + kb] = s.scale;
}

template <int DT>
bool vectors(const void* x, int64_t rows, int64_t stride) {
  constexpr int64_t ES = DT == kF32 ? 4 : 2;
  return ((uintptr_t)x & 15) == 0 && (rows == 1 || stride * ES % 16 == 0);
}

template <int DT>
hipError_t rows_t(const void* x, int64_t rows, int64_t K, int64_t stride, uint8_t* codes, int64_t codes_stride,
                  float* scales, int64_t xs_row, int64_t xs_block, hipStream_t s) {
  typedef typename Elem<DT>::T T;
  const int blocks = (int)((K + kBlock - 1) / kBlock);
  const int64_t groups = (rows + 15) / 16;
  // up to 8 blocks a workgroup while there are 2048 workgroups
  int per = 1;
  while (per < 8 && per < blocks && groups * ((blocks + 2 * per - 1) / (2 * per)) >= 2048) per *= 2;
  const unsigned split = (unsigned)((blocks + per - 1) / per);
  const int64_t most = max_groups(256);
  for (int64_t g0 = 0; g0 < groups; g0 += most) {
    const dim3 grid((unsigned)(groups - g0 < most ? groups - g0 : most), split);
    const T* xg = (const T*)x + g0 * 16 * stride;
    uint8_t* cg = codes + g0 * 16 * codes_stride;
    if (vectors<DT>(x, rows, stride))
      fp8_rows_kernel<DT, true><<<grid, dim3(256), 0, s>>>(xg, rows - g0 * 16, K, stride, cg, codes_stride,
                                                           scales + g0 * 16 * xs_row, xs_row, xs_block, blocks, per);
    else
      fp8_rows_kernel<DT, false><<<grid, dim3(256), 0, s>>>(xg, rows - g0 * 16, K, stride, cg, codes_stride,
                                                            scales + g0 * 16 * xs_row, xs_row, xs_block, blocks, per);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

template <int DT>
hipError_t weight_t(const void* w, int64_t N, int64_t K, int64_t stride, uint8_t* codes, int64_t codes_stride,
                    float* scales, hipStream_t s) {
  typedef typename Elem<DT>::T T;
  const int64_t blocks = (K + kBlock - 1) / kBlock, nblocks = (N + kBlock - 1) / kBlock;
  const int64_t most = max_groups(256) / blocks;  // blocks of outputs a launch takes
  for (int64_t n0 = 0; n0 < nblocks; n0 += most) {
    const int64_t some = nblocks - n0 < most ? nblocks - n0 : most, n = n0 * kBlock;
    const dim3 grid((unsigned)(some * blocks));
    if (vectors<DT>(w, N, stride))
      fp8_weight_kernel<DT, true><<<grid, dim3(256), 0, s>>>((const T*)w + n * stride, N - n, K, stride,
                                                             codes + n * codes_stride, codes_stride,
                                                             scales + n0 * blocks, (int)blocks);
    else
      fp8_weight_kernel<DT, false><<<grid, dim3(256), 0, s>>>((const T*)w + n * stride, N - n, K, stride,
                                                              codes + n * codes_stride, codes_stride,
                                                              scales + n0 * blocks, (int)blocks);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_quantize_fp8(const void* x, int dtype, int64_t rows, int64_t K, int64_t x_stride, uint8_t* codes,
                               int64_t codes_stride, float* scales, int64_t xs_row, int64_t xs_block,
                               hipStream_t stream) {
  switch (dtype) {
    case kF32: return rows_t<kF32>(x, rows, K, x_stride, codes, codes_stride, scales, xs_row, xs_block, stream);
    case kF16: return rows_t<kF16>(x, rows, K, x_stride, codes, codes_stride, scales, xs_row, xs_block, stream);
    default: return rows_t<kBF16>(x, rows, K, x_stride, codes, codes_stride, scales, xs_row, xs_block, stream);
  }
}

hipError_t launch_quantize_fp8_weight(const void* w, int dtype, int64_t N, int64_t K, int64_t w_stride, uint8_t* codes,
                                      int64_t codes_stride, float* scales, hipStream_t stream) {
  switch (dtype) {
    case kF32: return weight_t<kF32>(w, N, K, w_stride, codes, codes_stride, scales, stream);
    case kF16: return weight_t<kF16>(w, N, K, w_stride, codes, codes_stride, scales, stream);
    default: return weight_t<kBF16>(w, N, K, w_stride, codes, codes_stride, scales, stream);
  }
}

}  // namespace convrot
