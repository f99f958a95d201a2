// What lies around the linears of a mixture of experts: the order of the tokens'
// choices by expert, rows gathered in that order, and the experts' rows summed back to
// tokens with its gradient.
#include <algorithm>

#include "convrot_launch.h"
#include "row_device.h"

namespace convrot {
namespace {

// ---- order by expert
//
// A stable counting sort of `count` choices by their expert (those of none last, as if of
// expert E).  A workgroup of 16 waves takes `each` of them, each wave a run of them 64 at a
// time: first it counts its experts' choices in LDS, then, after sums over waves and experts, it
// places them: a choice's rank among its 64 is the number of lower lanes with the same expert, found
// bit by bit with ballots.  So the order never depends on which wave was first.  With several
// workgroups a launch before counts for each, and a workgroup adds the counts of those before it.
// Bound by latency: in a graph 1024 choices of 64 experts 6.1 us, 4096 in two launches 9.6, 36864 11.2 (with 8192 a
// workgroup 29), a million of 256 experts 37.
constexpr int kPlanWaves = 16, kPlanAlone = 2048, kPlanEach = 1024, kPlanGroups = 64;

// Workgroups and the choices of each: one up to kPlanAlone choices, then at most kPlanGroups.
struct PlanSplit {
  int64_t each, groups;
};
PlanSplit plan_split(int64_t count) {
  if (count <= kPlanAlone) return {kPlanAlone, 1};
  const int64_t runs = (count + kPlanEach - 1) / kPlanEach, each = (runs + kPlanGroups - 1) / kPlanGroups * kPlanEach;
  return {each, (count + each - 1) / each};
}

template <typename I>
__device__ __forceinline__ int expert_of(const I* ids, int64_t i, int experts) {
  const int64_t e = (int64_t)ids[i];
  return e >= 0 && e < experts ? (int)e : experts;
}

template <typename I>
__global__ __launch_bounds__(256) void plan_count_kernel(const I* __restrict__ ids, int64_t count, int64_t each,
                                                         int experts, int* __restrict__ counts) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= experts; e += 256) hist[e] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * each, i1 = min(count, i0 + each);
#pragma unroll 4
  for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) atomicAdd(&hist[expert_of(ids, i, experts)], 1);
  __syncthreads();
  int* mine = counts + (int64_t)blockIdx.x * (experts + 1);
  for (int e = threadIdx.x; e <= experts; e += 256) mine[e] = hist[e];
}

template <typename I>
__global__ __launch_bounds__(kPlanWaves * 64) void plan_place_kernel(const I* __restrict__ ids, int64_t count,
                                                                     int64_t choices, int experts,
                                                                     const int* __restrict__ counts,
                                                                     int* __restrict__ offsets, int* __restrict__ order,
                                                                     int* __restrict__ slots) {
  extern __shared__ int hist[];  // [waves][experts + 1]: counts, then places of the next choice
  __shared__ int wave_total[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, stride = experts + 1;
  for (int i = tid; i < kPlanWaves * stride; i += kPlanWaves * 64) hist[i] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * choices;
  const int n = (int)min(choices, count - i0);
  const int each = ((n + kPlanWaves - 1) / kPlanWaves + 63) / 64 * 64;  // a wave's run
  const int a = min(n, wave * each), b = min(n, a + each);
  int* mine = hist + wave * stride;
  for (int i = a + lane; i < b; i += 64) atomicAdd(&mine[expert_of(ids, i0 + i, experts)], 1);
  __syncthreads();

  // thread e: expert e's choices in this workgroup, before it and in all
  int total = 0, before = 0;
  if (tid < experts) {
    int here = 0;
    for (int w = 0; w < kPlanWaves; ++w) here += hist[w * stride + tid];
    total = here;
    if (counts) {
      total = 0;
#pragma unroll 8
      for (unsigned g = 0; g < gridDim.x; ++g) {
        const int c = counts[(int64_t)g * stride + tid];
        total += c;
        if (g < blockIdx.x) before += c;
      }
    }
  }
  int upto = total;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) wave_total[wave] = upto;
  __syncthreads();
  int sum = 0, all = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) sum += wave_total[w];
    all += wave_total[w];
  }
  if (tid < experts) {
    const int first = sum + upto - total;
    if (blockIdx.x == 0) offsets[tid] = first;
    int at = first + before;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = hist[w * stride + tid];
      hist[w * stride + tid] = at;
      at += c;
    }
  }
  int none = 0;  // choices of no expert before this workgroup
  if (counts && wave == 0) {
    none = (unsigned)lane < blockIdx.x ? counts[(int64_t)lane * stride + experts] : 0;  // at most 64 workgroups
#pragma unroll
    for (int d = 1; d < 64; d *= 2) none += __shfl_xor(none, d);
  }
  if (tid == 0) {
    if (blockIdx.x == 0) offsets[experts] = all;
    int at = all + none;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = hist[w * stride + experts];
      hist[w * stride + experts] = at;
      at += c;
    }
  }
  __syncthreads();

  const int bits = 32 - __builtin_clz((unsigned)experts);  // of 0 .. experts
  volatile int* next = mine;
  for (int i = a; i < b; i += 64) {  // uniform over the wave
    const bool on = i + lane < b;
    const int e = on ? expert_of(ids, i0 + i + lane, experts) : 0;
    uint64_t alike = __ballot(on);
    for (int k = 0; k < bits; ++k) {
      const uint64_t set = __ballot((e >> k) & 1);
      alike &= (e >> k) & 1 ? set : ~set;
    }
    const int rank = __popcll(alike & ((1ull << lane) - 1));
    const int base = on ? next[e] : 0;
    __builtin_amdgcn_wave_barrier();  // every lane has read before one writes
    if (on && rank == __popcll(alike) - 1) next[e] = base + rank + 1;
    __builtin_amdgcn_wave_barrier();
    if (on) {
      order[base + rank] = (int)(i0 + i + lane);
      slots[i0 + i + lane] = base + rank;
    }
  }
}

template <typename I>
hipError_t plan_t(const void* ids, int64_t count, int experts, int* offsets, int* order, int* slots, int* work,
                  hipStream_t s) {
  const PlanSplit p = plan_split(count);
  const size_t lds = (size_t)(experts + 1) * sizeof(int);
  const bool alone = p.groups == 1;
  if (!alone) {
    plan_count_kernel<I><<<dim3((unsigned)p.groups), dim3(256), lds, s>>>((const I*)ids, count, p.each, experts, work);
    if (hipError_t e = hipGetLastError()) return e;
  }
  plan_place_kernel<I><<<dim3((unsigned)p.groups), dim3(kPlanWaves * 64), kPlanWaves * lds, s>>>(
      (const I*)ids, count, p.each, experts, alone ? nullptr : work, offsets, order, slots);
  return hipGetLastError();
}

// ---- rows
//
// A row is the work of `threads` threads (a power of two, 32 .. 256), 8 features a thread and step
// where rows are 16-byte aligned, else one.  All are bound by the rows' bytes: 36864 rows of 4096 in 16 bits summed to
// 9216 tokens 75 to 92 us (4.1 TB/s and more), the gradient 129 to 151 (4.5 TB/s and more); 9216 rows of 4096 gathered
// 23 to 25 us (5.9 TB/s, most of what is read from the last-level cache).  One by one (4095 features) the sum takes 295
// us and its gradient 284.

template <int DT, bool VEC>
struct Piece {
  static constexpr int W = VEC ? 8 : 1;
  float v[W];
  __device__ __forceinline__ void load(const typename Elem<DT>::T* p) {
    if constexpr (VEC) load8<DT>(p, v);
    else v[0] = (float)*p;
  }
  __device__ __forceinline__ void store(typename Elem<DT>::T* p) const {
    if constexpr (VEC) store8<DT>(p, v);
    else *p = (typename Elem<DT>::T)v[0];
  }
};

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void gather_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_rows,
                                                     int64_t x_stride, const int* __restrict__ index, int choices,
                                                     int64_t row0, int64_t rows, int features, int threads,
                                                     typename Elem<DT>::T* __restrict__ out) {
  const int each = 256 / threads, at = threadIdx.x & (threads - 1);
  const int64_t s = row0 + (int64_t)blockIdx.x * each + threadIdx.x / threads;
  if (s >= rows) return;
  const int i = index[s];
  const int64_t t = i < 0 ? x_rows : (int64_t)((uint32_t)i / (uint32_t)choices);
  constexpr int W = Piece<DT, VEC>::W;
  for (int f = at * W; f < features; f += threads * W) {
    Piece<DT, VEC> p{};
    if (t < x_rows) p.load(x + t * x_stride + f);
    p.store(out + s * features + f);
  }
}

// out[t] = sum over c of weights[t][c] * y[slots[t][c]], in float32, the choices in order.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const typename Elem<DT>::T* __restrict__ y, int64_t y_rows,
                                                      int64_t y_stride, const int* __restrict__ slots,
                                                      const float* __restrict__ weights, int64_t token0,
                                                      int64_t tokens, int choices, int features, int threads,
                                                      typename Elem<DT>::T* __restrict__ out) {
  const int each = 256 / threads, at = threadIdx.x & (threads - 1);
  const int64_t t = token0 + (int64_t)blockIdx.x * each + threadIdx.x / threads;
  if (t >= tokens) return;
  constexpr int W = Piece<DT, VEC>::W, BATCH = 4;  // rows whose loads are in flight together
  const int* sl = slots + t * choices;
  const float* wt = weights ? weights + t * choices : nullptr;
  for (int f = at * W; f < features; f += threads * W) {
    Piece<DT, VEC> sum{};
    for (int c0 = 0; c0 < choices; c0 += BATCH) {
      Piece<DT, VEC> p[BATCH];
      float w[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int64_t r = c0 + j < choices ? (int64_t)sl[c0 + j] : -1;
        p[j] = {};
        w[j] = r >= 0 && wt ? wt[c0 + j] : 1.0f;
        if (r >= 0 && r < y_rows) p[j].load(y + r * y_stride + f);
        else w[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j)
        if (c0 + j < choices) {
#pragma unroll
          for (int k = 0; k < W; ++k) sum.v[k] = __builtin_fmaf(w[j], p[j].v[k], sum.v[k]);
        }
    }
    sum.store(out + t * features + f);
  }
}

// Zeros in the rows of dy from row0 to row_end that no choice has: order names none for them, or one whose place is
// another row (in a caller's own plan).  A wave looks at 64 rows at a time.
template <int DT, bool VEC>
__device__ __forceinline__ void clear_rows_of_none(const int* __restrict__ order, const int* __restrict__ slots,
                                                   int64_t row0, int64_t row_end, int64_t rows, int features, int wave,
                                                   int waves, typename Elem<DT>::T* __restrict__ dy) {
  const int lane = threadIdx.x & 63;
  constexpr int W = Piece<DT, VEC>::W;
  for (int64_t s0 = row0 + (int64_t)wave * 64; s0 < row_end; s0 += (int64_t)waves * 64) {
    const int64_t s = s0 + lane;
    const int i = s < row_end ? order[s] : -1;
    uint64_t none = __ballot(s < row_end && !(i >= 0 && i < rows && slots[i] == (int)s));
    for (; none; none &= none - 1) {
      typename Elem<DT>::T* row = dy + (s0 + __builtin_ctzll(none)) * features;
      const Piece<DT, VEC> zero{};
      for (int f = lane * W; f < features; f += 64 * W) zero.store(row + f);
    }
  }
}

// dy[s] = weights[t][c] * dout[t] and dweights[t][c] = <dout[t], y[s]>, s = slots[t][c], a token's
// threads together: dout is read once, y once, dy written once.  A row is written by the choice that
// `order` names for it alone, so none is written twice; the last `clearing` workgroups clear those of no choice, among
// the rows whose numbers are the launch's choices (36864 rows of 4096: 134 to 137 us with them and without; looked
// for by the tokens' own threads, whose loads then wait for two more, 175).
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void combine_backward_kernel(
    const typename Elem<DT>::T* __restrict__ dout, int64_t dout_stride, const typename Elem<DT>::T* __restrict__ y,
    int64_t y_rows, int64_t y_stride, const int* __restrict__ order, const int* __restrict__ slots,
    const float* __restrict__ weights, int64_t token0, int64_t tokens, int choices, int features, int threads,
    unsigned clearing, typename Elem<DT>::T* __restrict__ dy, float* __restrict__ dweights) {
  __shared__ float part[4][4];  // [choice of the batch][wave]
  const int each = 256 / threads, at = threadIdx.x & (threads - 1), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= gridDim.x - clearing) {
    const unsigned mine = blockIdx.x - (gridDim.x - clearing);
    const int64_t end = min(tokens, token0 + (int64_t)(gridDim.x - clearing) * each) * choices;
    clear_rows_of_none<DT, VEC>(order, slots, token0 * choices, end, y_rows, features, (int)mine * 4 + wave,
                                (int)clearing * 4, dy);
    return;
  }
  const int64_t t = token0 + (int64_t)blockIdx.x * each + threadIdx.x / threads;
  constexpr int W = Piece<DT, VEC>::W, BATCH = 4;
  const bool on = t < tokens;
  for (int c0 = 0; c0 < choices; c0 += BATCH) {
    int64_t r[BATCH];
    float w[BATCH], dot[BATCH];
    bool write[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const bool any = on && c0 + j < choices;
      const int64_t i = any ? t * choices + c0 + j : 0;
      r[j] = any ? (int64_t)slots[i] : -1;
      if (r[j] >= y_rows) r[j] = -1;
      w[j] = any && weights ? weights[i] : 1.0f;
      write[j] = dy && r[j] >= 0 && order[r[j]] == (int)i;
      dot[j] = 0.0f;
    }
    if (on) {
      for (int f = at * W; f < features; f += threads * W) {
        Piece<DT, VEC> g, p[BATCH];
        g.load(dout + t * dout_stride + f);
        if (dweights) {
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            p[j] = {};
            if (r[j] >= 0) p[j].load(y + r[j] * y_stride + f);
          }
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          if (dweights) {
#pragma unroll
            for (int k = 0; k < W; ++k) dot[j] = __builtin_fmaf(g.v[k], p[j].v[k], dot[j]);
          }
          if (write[j]) {
            Piece<DT, VEC> d;
#pragma unroll
            for (int k = 0; k < W; ++k) d.v[k] = w[j] * g.v[k];
            d.store(dy + r[j] * features + f);
          }
        }
      }
    }
    if (dweights) {  // uniform
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        dot[j] = group_sum<32>(dot[j]);
        if (threads >= 64) dot[j] += __shfl_xor(dot[j], 32);
      }
      if (threads > 64) {
        __syncthreads();
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < BATCH; ++j) part[j][wave] = dot[j];
        }
        __syncthreads();
        const int w0 = wave & ~(threads / 64 - 1);  // the first wave of the token's threads
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          dot[j] = part[j][w0] + part[j][w0 + 1];
          if (threads == 256) dot[j] += part[j][2] + part[j][3];
        }
      }
      if (on && at == 0) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
          if (c0 + j < choices) dweights[t * choices + c0 + j] = dot[j];
      }
    }
  }
}

// Threads a row: as many as it has steps for, up to a workgroup.
int threads_of(int64_t features, bool vec) {
  const int64_t steps = vec ? (features + 7) / 8 : features;
  int n = 32;
  while (n < 256 && n < steps) n *= 2;
  return n;
}

template <int DT>
bool in_pieces(int64_t features, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
  constexpr int64_t ES = DT == kF32 ? 4 : 2;
  bool good = features % 8 == 0;
  for (const void* p : bases) good &= ((uintptr_t)p & 15) == 0;
  for (int64_t s : strides) good &= s * ES % 16 == 0;
  return good;
}

// Launches of at most as many workgroups as one takes, `more` beside the rows': run(first row, the rows' workgroups).
template <class F>
hipError_t in_launches(int64_t rows, int threads, F&& run, unsigned more = 0) {
  const int64_t each = 256 / threads, most = (max_groups(256) - more) * each;
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t some = rows - r0 < most ? rows - r0 : most;
    run(r0, dim3((unsigned)((some + each - 1) / each)));
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

template <int DT>
hipError_t gather_t(const void* x, int64_t x_rows, int64_t x_stride, const int* index, int choices, int64_t rows,
                    int64_t features, void* out, hipStream_t s) {
  typedef typename Elem<DT>::T T;
  const bool vec = in_pieces<DT>(features, {x, out}, {x_stride});
  const int threads = threads_of(features, vec);
  return in_launches(rows, threads, [&](int64_t r0, dim3 grid) {
    if (vec)
      gather_kernel<DT, true><<<grid, dim3(256), 0, s>>>((const T*)x, x_rows, x_stride, index, choices, r0, rows,
                                                         (int)features, threads, (T*)out);
    else
      gather_kernel<DT, false><<<grid, dim3(256), 0, s>>>((const T*)x, x_rows, x_stride, index, choices, r0, rows,
                                                          (int)features, threads, (T*)out);
  });
}

template <int DT>
hipError_t combine_t(const void* y, int64_t y_rows, int64_t y_stride, const int* slots, const float* weights,
                     int64_t tokens, int choices, int64_t features, void* out, hipStream_t s) {
  typedef typename Elem<DT>::T T;
  const bool vec = in_pieces<DT>(features, {y, out}, {y_stride});
  const int threads = threads_of(features, vec);
  return in_launches(tokens, threads, [&](int64_t t0, dim3 grid) {
    if (vec)
      combine_kernel<DT, true><<<grid, dim3(256), 0, s>>>((const T*)y, y_rows, y_stride, slots, weights, t0, tokens,
                                                          choices, (int)features, threads, (T*)out);
    else
      combine_kernel<DT, false><<<grid, dim3(256), 0, s>>>((const T*)y, y_rows, y_stride, slots, weights, t0, tokens,
                                                           choices, (int)features, threads, (T*)out);
  });
}

template <int DT>
hipError_t combine_backward_t(const void* dout, int64_t dout_stride, const void* y, int64_t y_rows, int64_t y_stride,
                              const int* order, const int* slots, const float* weights, int64_t tokens, int choices,
                              int64_t features, void* dy, float* dweights, hipStream_t s) {
  typedef typename Elem<DT>::T T;
  const bool vec = in_pieces<DT>(features, {dout, y, dy}, {dout_stride, y_stride});
  const int threads = threads_of(features, vec);
  // a workgroup for 1024 rows, up to one a CU
  const unsigned clearing = dy ? (unsigned)std::min<int64_t>((y_rows + 1023) / 1024, 256) : 0;
  return in_launches(tokens, threads, [&](int64_t t0, dim3 grid) {
    grid.x += clearing;
    if (vec)
      combine_backward_kernel<DT, true><<<grid, dim3(256), 0, s>>>(
          (const T*)dout, dout_stride, (const T*)y, y_rows, y_stride, order, slots, weights, t0, tokens, choices,
          (int)features, threads, clearing, (T*)dy, dweights);
    else
      combine_backward_kernel<DT, false><<<grid, dim3(256), 0, s>>>(
          (const T*)dout, dout_stride, (const T*)y, y_rows, y_stride, order, slots, weights, t0, tokens, choices,
          (int)features, threads, clearing, (T*)dy, dweights);
  }, clearing);
}

}  // namespace

int64_t expert_plan_workspace_bytes(int64_t count, int experts) {
  const int64_t groups = plan_split(count).groups;
  return groups > 1 ? groups * (experts + 1) * (int64_t)sizeof(int) : 0;
}

hipError_t launch_expert_plan(const void* ids, bool ids64, int64_t count, int experts, int* offsets, int* order,
                              int* slots, int* workspace, hipStream_t stream) {
  if (ids64) return plan_t<int64_t>(ids, count, experts, offsets, order, slots, workspace, stream);
  return plan_t<int32_t>(ids, count, experts, offsets, order, slots, workspace, stream);
}

hipError_t launch_gather_rows(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const int* index, int choices,
                              int64_t rows, int64_t features, void* out, hipStream_t stream) {
  switch (dtype) {
    case kF32: return gather_t<kF32>(x, x_rows, x_stride, index, choices, rows, features, out, stream);
    case kF16: return gather_t<kF16>(x, x_rows, x_stride, index, choices, rows, features, out, stream);
    default: return gather_t<kBF16>(x, x_rows, x_stride, index, choices, rows, features, out, stream);
  }
}

hipError_t launch_combine_rows(const void* y, int dtype, int64_t y_rows, int64_t y_stride, const int* slots,
                               const float* weights, int64_t tokens, int choices, int64_t features, void* out,
                               hipStream_t stream) {
  switch (dtype) {
    case kF32: return combine_t<kF32>(y, y_rows, y_stride, slots, weights, tokens, choices, features, out, stream);
    case kF16: return combine_t<kF16>(y, y_rows, y_stride, slots, weights, tokens, choices, features, out, stream);
    default: return combine_t<kBF16>(y, y_rows, y_stride, slots, weights, tokens, choices, features, out, stream);
  }
}

hipError_t launch_combine_rows_backward(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride,
                                        int dtype, int64_t y_rows, const int* order, const int* slots,
                                        const float* weights, int64_t tokens, int choices, int64_t features, void* dy,
                                        float* dweights, hipStream_t stream) {
  switch (dtype) {
    case kF32:
      return combine_backward_t<kF32>(dout, dout_stride, y, y_rows, y_stride, order, slots, weights, tokens, choices,
                                      features, dy, dweights, stream);
    case kF16:
      return combine_backward_t<kF16>(dout, dout_stride, y, y_rows, y_stride, order, slots, weights, tokens, choices,
                                      features, dy, dweights, stream);
    default:
      return combine_backward_t<kBF16>(dout, dout_stride, y, y_rows, y_stride, order, slots, weights, tokens, choices,
                                       features, dy, dweights, stream);
  }
}

}  // namespace convrot
