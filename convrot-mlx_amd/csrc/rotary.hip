// Per-head RMS norm and rotary positions of queries and keys, and their
// gradients, for positions of several axes.
//
// A head's D features x of token l, in float32:
//   n = x rsqrt(sum(x^2) / D + eps) w          (w: one weight a feature; left out without weights)
//   the first 2 P features in P pairs (a, b), turned by the pair's angle:
//   (a cos - b sin, a sin + b cos); the features from 2 P on stay as n has them,
// rounded once.  Pairs are features (2 p, 2 p + 1) or, split in halves,
// (p, P + p).  The angle of a pair belongs to one axis of the position (time,
// height, width): its cosine and sine come from a table [B or 1][L][P][2] that
// is made once for all heads and layers (axes_table_kernel).
//
// Backward: with g the output's gradient turned back by the angle,
// u = x rsqrt(..) and h = g w:
//   dx = rsqrt(..) (h - u sum(h u) / D),   dw = sum over tokens and heads of g u.
//
// The work is moving q and k once each way.  One wave owns one token: a lane
// holds 16 features of a head (8 pairs), 64 / G heads at a time in groups of
// G lanes, so the token's cosines and sines are read into registers once and
// serve all its heads, and a head's sum is log2(G) lane exchanges.  Measured,
// bf16, heads of 128: 4608 tokens of 24 q and 24 k heads 21.3 us (113 MB at 5.3
// TB/s, partly from the Infinity Cache), 7800 of 40 and 40 86 us forward (320 MB
// at 3.7 TB/s; 1 to 5 rounds of heads a wave make no difference of 5 %) and 104
// backward (480 MB at 4.6).
#include "convrot_launch.h"
#include "row_device.h"

namespace convrot {
namespace {

struct HeadTensor {
  const void* x;
  int64_t sb, sh, sl;  // strides in elements; features are adjacent
};

struct RotaryArgs {
  HeadTensor in[2], out[2];    // q, k
  HeadTensor grad[2];          // backward: gradients of the outputs
  const void* weight[2];       // null: no norm
  int heads[2];
  int weight_dtype;
  int batch, D, P;
  int64_t length;
  const float* table;
  int64_t table_sb;            // elements from one batch entry's table to the next, 0: shared
  float eps;
  int splits;                  // waves that share a token's heads (forward)
  int64_t first;               // first unit (token and split) of a launch (forward)
  int64_t tokens;              // batch * length
  float* partial;              // backward: [workgroups][2][D]
};

// Where lane c of a head's group finds its two chunks of 8 features: those of
// pairs 8 c .. 8 c + 7, or behind them 16 features that are not turned.
template <bool PAIRS>
__device__ __forceinline__ void chunk_at(int c, int P, int& a, int& b) {
  if (PAIRS || 8 * c >= P) {
    a = 16 * c, b = a + 8;
  } else {
    a = 8 * c, b = P + 8 * c;
  }
}

// (a, b) of pair j in a lane's 16 values.
template <bool PAIRS>
__device__ __forceinline__ int first_of(int j) { return PAIRS ? 2 * j : j; }
template <bool PAIRS>
__device__ __forceinline__ int second_of(int j) { return PAIRS ? 2 * j + 1 : j + 8; }

__device__ __forceinline__ void load_angles(const float* t, float (&cs)[8], float (&sn)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = *(const float4*)(t + 4 * i);
    cs[2 * i] = v.x, sn[2 * i] = v.y, cs[2 * i + 1] = v.z, sn[2 * i + 1] = v.w;
  }
}

template <int DT>
__device__ __forceinline__ void load16(const void* base, int64_t at, int a, int b, float (&v)[16]) {
  const typename Elem<DT>::T* p = (const typename Elem<DT>::T*)base + at;
  load8<DT>(p + a, *(float(*)[8]) & v[0]);
  load8<DT>(p + b, *(float(*)[8]) & v[8]);
}

template <int DT>
__device__ __forceinline__ void store16(const void* base, int64_t at, int a, int b, const float (&v)[16]) {
  typename Elem<DT>::T* p = (typename Elem<DT>::T*)base + at;
  store8<DT>(p + a, *(const float(*)[8]) & v[0]);
  store8<DT>(p + b, *(const float(*)[8]) & v[8]);
}

template <int DT>
__device__ __forceinline__ void load_weight16(const void* w, int wdt, int a, int b, float (&v)[16]) {
  if (DT != kF32 && wdt == kF32) load16<kF32>(w, 0, a, b, v);
  else load16<DT>(w, 0, a, b, v);
}

// Forward.  D % 16 == 0, P % 8 == 0, 16-byte aligned heads.
template <int DT, int G, bool PAIRS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs r) {
  constexpr int HPW = 64 / G;  // heads a wave holds at a time
  const int lane = threadIdx.x & 63, c = lane % G, slot = lane / G;
  const int64_t unit = r.first + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t token = (uint32_t)(unit / (uint32_t)r.splits), split = (uint32_t)(unit % (uint32_t)r.splits);
  if (token >= r.tokens) return;
  const uint32_t b = token / (uint32_t)r.length, l = token % (uint32_t)r.length;
  const bool has = 16 * c < r.D, turned = 8 * c < r.P;
  int ca, cb;
  chunk_at<PAIRS>(c, r.P, ca, cb);
  float cs[8], sn[8];
  if (turned) load_angles(r.table + b * r.table_sb + ((int64_t)l * r.P + 8 * c) * 2, cs, sn);
  const int qsteps = (r.heads[0] + HPW - 1) / HPW, ksteps = (r.heads[1] + HPW - 1) / HPW;
  for (int i = split; i < qsteps + ksteps; i += r.splits) {
    const int which = i >= qsteps;
    const int head = (which ? i - qsteps : i) * HPW + slot;
    const bool live = has && head < (which ? r.heads[1] : r.heads[0]);
    const HeadTensor& in = which ? r.in[1] : r.in[0];
    const HeadTensor& out = which ? r.out[1] : r.out[0];
    const void* w = which ? r.weight[1] : r.weight[0];
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.0f;
    if (live) load16<DT>(in.x, b * in.sb + head * in.sh + (int64_t)l * in.sl, ca, cb, v);
    if (w) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) s += v[j] * v[j];
      s = group_sum<G>(s);
      const float rs = 1.0f / sqrtf(s / (float)r.D + r.eps);
      float wv[16];
      if (live) {
        load_weight16<DT>(w, r.weight_dtype, ca, cb, wv);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = v[j] * rs * wv[j];
      }
    }
    if (!live) continue;
    if (turned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = v[first_of<PAIRS>(j)], y = v[second_of<PAIRS>(j)];
        v[first_of<PAIRS>(j)] = x * cs[j] - y * sn[j];
        v[second_of<PAIRS>(j)] = x * sn[j] + y * cs[j];
      }
    }
    store16<DT>(out.x, b * out.sb + head * out.sh + (int64_t)l * out.sl, ca, cb, v);
  }
}

// Backward.  Each wave walks tokens and keeps the sums of dw for its lanes'
// features; the lanes of one feature, then the waves of the workgroup, are
// added in order.
template <int DT, int G, bool PAIRS>
__global__ __launch_bounds__(256) void rotary_backward_kernel(RotaryArgs r) {
  constexpr int HPW = 64 / G;
  __shared__ float sums[4][2][G * 16];
  const int lane = threadIdx.x & 63, c = lane % G, slot = lane / G, wave = threadIdx.x >> 6;
  const bool has = 16 * c < r.D, turned = 8 * c < r.P;
  int ca, cb;
  chunk_at<PAIRS>(c, r.P, ca, cb);
  const int qsteps = (r.heads[0] + HPW - 1) / HPW, ksteps = (r.heads[1] + HPW - 1) / HPW;
  float dw[2][16];
#pragma unroll
  for (int j = 0; j < 16; ++j) dw[0][j] = dw[1][j] = 0.0f;

  for (int64_t token = (int64_t)blockIdx.x * 4 + wave; token < r.tokens; token += (int64_t)gridDim.x * 4) {
    const uint32_t b = (uint32_t)token / (uint32_t)r.length, l = (uint32_t)token % (uint32_t)r.length;
    float cs[8], sn[8];
    if (turned) load_angles(r.table + b * r.table_sb + ((int64_t)l * r.P + 8 * c) * 2, cs, sn);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const HeadTensor &in = r.in[which], &grad = r.grad[which], &out = r.out[which];
      const void* w = r.weight[which];
      float wv[16];
      if (w && has) load_weight16<DT>(w, r.weight_dtype, ca, cb, wv);
      const int steps = which ? ksteps : qsteps;
      for (int i = 0; i < steps; ++i) {
        const int head = i * HPW + slot;
        const bool live = has && head < r.heads[which];
        float g[16], u[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) g[j] = u[j] = 0.0f;
        if (live) {
          load16<DT>(grad.x, b * grad.sb + head * grad.sh + (int64_t)l * grad.sl, ca, cb, g);
          if (w) load16<DT>(in.x, b * in.sb + head * in.sh + (int64_t)l * in.sl, ca, cb, u);
        }
        if (turned) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = g[first_of<PAIRS>(j)], y = g[second_of<PAIRS>(j)];
            g[first_of<PAIRS>(j)] = x * cs[j] + y * sn[j];
            g[second_of<PAIRS>(j)] = y * cs[j] - x * sn[j];
          }
        }
        if (w) {
          float s = 0.0f;
#pragma unroll
          for (int j = 0; j < 16; ++j) s += u[j] * u[j];
          s = group_sum<G>(s);
          const float rs = 1.0f / sqrtf(s / (float)r.D + r.eps);
          float along = 0.0f;
          if (live) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              u[j] *= rs;
              dw[which][j] += g[j] * u[j];
              g[j] *= wv[j];
              along += g[j] * u[j];
            }
          }
          along = group_sum<G>(along) / (float)r.D;
#pragma unroll
          for (int j = 0; j < 16; ++j) g[j] = rs * (g[j] - u[j] * along);
        }
        if (live) store16<DT>(out.x, b * out.sb + head * out.sh + (int64_t)l * out.sl, ca, cb, g);
      }
    }
  }

  if (!r.partial) return;
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
#pragma unroll
      for (int d = G; d < 64; d <<= 1) dw[which][j] += __shfl_xor(dw[which][j], d);
    }
  if (slot == 0 && has) {
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[wave][which][j < 8 ? ca + j : cb + j - 8] = dw[which][j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * r.D; i += 256) {
    const int which = i >= r.D, f = which ? i - r.D : i;
    r.partial[(size_t)blockIdx.x * 2 * r.D + i] =
        sums[0][which][f] + sums[1][which][f] + sums[2][which][f] + sums[3][which][f];
  }
}

// Any D up to 512, any P and alignment: a wave a (token, head), lane s holds
// pairs s, s + 64, .. (behind the P pairs, two features each that are not
// turned).  dw is added over the heads and tokens that a wave walks.
constexpr int kMaxDim = 512;
constexpr int kSlots = kMaxDim / 128;

template <int DT, bool PAIRS, bool BACKWARD>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryArgs r) {
  typedef typename Elem<DT>::T E;
  __shared__ float sums[BACKWARD ? 4 : 1][2][BACKWARD ? kMaxDim : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int heads = r.heads[0] + r.heads[1];
  int fa[kSlots], fb[kSlots];
  bool turned[kSlots];
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    const int s = lane + 64 * j;
    turned[j] = s < r.P;
    if (turned[j] && !PAIRS) fa[j] = s, fb[j] = r.P + s;
    else fa[j] = 2 * s, fb[j] = 2 * s + 1;
  }
  float dw[2][kSlots][2];
#pragma unroll
  for (int j = 0; j < kSlots; ++j) dw[0][j][0] = dw[0][j][1] = dw[1][j][0] = dw[1][j][1] = 0.0f;

  for (int64_t unit = (int64_t)blockIdx.x * 4 + wave; unit < r.tokens * heads; unit += (int64_t)gridDim.x * 4) {
    const uint32_t token = (uint32_t)(unit / (uint32_t)heads), hh = (uint32_t)(unit % (uint32_t)heads);
    const uint32_t b = token / (uint32_t)r.length, l = token % (uint32_t)r.length;
    const bool which = hh >= (uint32_t)r.heads[0];
    const int head = which ? hh - r.heads[0] : hh;
    const HeadTensor& in = which ? r.in[1] : r.in[0];
    const HeadTensor& out = which ? r.out[1] : r.out[0];
    const HeadTensor& grad = which ? r.grad[1] : r.grad[0];
    const void* w = which ? r.weight[1] : r.weight[0];
    const E* x = (const E*)in.x + b * in.sb + head * in.sh + (int64_t)l * in.sl;
    const E* dy = BACKWARD ? (const E*)grad.x + b * grad.sb + head * grad.sh + (int64_t)l * grad.sl : nullptr;
    E* o = (E*)out.x + b * out.sb + head * out.sh + (int64_t)l * out.sl;
    const float* ang = r.table + b * r.table_sb + (int64_t)l * r.P * 2;
    float u[kSlots][2], g[kSlots][2], wv[kSlots][2], cs[kSlots], sn[kSlots];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const bool ina = fa[j] < r.D, inb = fb[j] < r.D;
      const bool need = !BACKWARD || w;
      u[j][0] = need && ina ? (float)x[fa[j]] : 0.0f;
      u[j][1] = need && inb ? (float)x[fb[j]] : 0.0f;
      g[j][0] = BACKWARD && ina ? (float)dy[fa[j]] : 0.0f;
      g[j][1] = BACKWARD && inb ? (float)dy[fb[j]] : 0.0f;
      cs[j] = turned[j] ? ang[2 * (lane + 64 * j)] : 1.0f;
      sn[j] = turned[j] ? ang[2 * (lane + 64 * j) + 1] : 0.0f;
      wv[j][0] = wv[j][1] = 1.0f;
      if (w && ina) wv[j][0] = r.weight_dtype == kF32 ? ((const float*)w)[fa[j]] : (float)((const E*)w)[fa[j]];
      if (w && inb) wv[j][1] = r.weight_dtype == kF32 ? ((const float*)w)[fb[j]] : (float)((const E*)w)[fb[j]];
      s += u[j][0] * u[j][0] + u[j][1] * u[j][1];
    }
    float rs = 1.0f;
    if (w) rs = 1.0f / sqrtf(wave_sum(s) / (float)r.D + r.eps);
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        float a = u[j][0], bb = u[j][1];
        if (w) a = a * rs * wv[j][0], bb = bb * rs * wv[j][1];
        const float ya = turned[j] ? a * cs[j] - bb * sn[j] : a, yb = turned[j] ? a * sn[j] + bb * cs[j] : bb;
        if (fa[j] < r.D) o[fa[j]] = (E)ya;
        if (fb[j] < r.D) o[fb[j]] = (E)yb;
      }
    } else {
      float along = 0.0f;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const float a = g[j][0], bb = g[j][1];
        if (turned[j]) g[j][0] = a * cs[j] + bb * sn[j], g[j][1] = bb * cs[j] - a * sn[j];
        if (w) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u[j][e] *= rs;
            dw[0][j][e] += which ? 0.0f : g[j][e] * u[j][e];
            dw[1][j][e] += which ? g[j][e] * u[j][e] : 0.0f;
            g[j][e] *= wv[j][e];
            along += g[j][e] * u[j][e];
          }
        }
      }
      if (w) along = wave_sum(along) / (float)r.D;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (w) {
          g[j][0] = rs * (g[j][0] - u[j][0] * along);
          g[j][1] = rs * (g[j][1] - u[j][1] * along);
        }
        if (fa[j] < r.D) o[fa[j]] = (E)g[j][0];
        if (fb[j] < r.D) o[fb[j]] = (E)g[j][1];
      }
    }
  }

  if constexpr (BACKWARD) {
    if (!r.partial) return;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (fa[j] < r.D) sums[wave][which][fa[j]] = dw[which][j][0];
        if (fb[j] < r.D) sums[wave][which][fb[j]] = dw[which][j][1];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * r.D; i += 256) {
      const int which = i >= r.D, f = which ? i - r.D : i;
      r.partial[(size_t)blockIdx.x * 2 * r.D + i] =
          sums[0][which][f] + sums[1][which][f] + sums[2][which][f] + sums[3][which][f];
    }
  }
}

// dw[which][f]: the workgroups' partials, 64 threads a feature each adding
// every 64th, then their sums in order.
__global__ __launch_bounds__(1024) void sum_heads_kernel(const float* __restrict__ partial, int parts, int D,
                                                         void* __restrict__ dqw, void* __restrict__ dkw, int dtype) {
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, lot = threadIdx.x >> 4;
  const int i = blockIdx.x * 16 + col;  // of 2 D
  float s = 0.0f;
  if (i < 2 * D) {
#pragma unroll 4
    for (int p = lot; p < parts; p += 64) s += partial[(size_t)p * 2 * D + i];
  }
  red[lot][col] = s;
  __syncthreads();
  if (lot != 0 || i >= 2 * D) return;
  for (int p = 1; p < 64; ++p) s += red[p][col];
  void* o = i < D ? dqw : dkw;
  if (!o) return;
  const int f = i < D ? i : i - D;
  if (dtype == kF32) store_out<kF32>(o, f, s);
  else if (dtype == kF16) store_out<kF16>(o, f, s);
  else store_out<kBF16>(o, f, s);
}

// [rows][A] positions -> [rows][P][2]: pair p of axis a, the i-th of its d_a / 2,
// turns by position theta^(-2 i / d_a).  Angles in float64 (a float32 angle of
// a position in the thousands is off by its last bits, 1e-4 and more).
struct AxesArgs {
  int axes, half[8];
};
template <class PT>
__global__ __launch_bounds__(256) void axes_table_kernel(const PT* __restrict__ pos, int64_t rows, AxesArgs ax, int P,
                                                         double log_theta, float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * P) return;
  const int64_t row = i / P;
  int p = (int)(i % P), a = 0;
  while (p >= ax.half[a]) p -= ax.half[a++];
  const double angle = (double)pos[row * ax.axes + a] * exp(-log_theta * (double)p / (double)ax.half[a]);
  out[2 * i] = (float)cos(angle);
  out[2 * i + 1] = (float)sin(angle);
}

// Workgroups of the backward kernels: each leaves a partial of dw (512 against 1024: 41.0 -> 37.8 us
// at 4608 tokens of 24 heads, 24.4 -> 19.6 at 4000 of 16 heads of 64).
constexpr int kBackwardGroups = 512;

int64_t backward_groups(int64_t units) {
  const int64_t g = (units + 3) / 4;
  return g < kBackwardGroups ? g : kBackwardGroups;
}

template <int DT, int G>
void run_vec(const RotaryArgs& r, bool interleaved, bool backward, unsigned grid, hipStream_t s) {
  if (backward) {
    if (interleaved) rotary_backward_kernel<DT, G, true><<<grid, 256, 0, s>>>(r);
    else rotary_backward_kernel<DT, G, false><<<grid, 256, 0, s>>>(r);
  } else {
    if (interleaved) rotary_kernel<DT, G, true><<<grid, 256, 0, s>>>(r);
    else rotary_kernel<DT, G, false><<<grid, 256, 0, s>>>(r);
  }
}

template <int DT>
void run_any(const RotaryArgs& r, bool interleaved, bool backward, unsigned grid, hipStream_t s) {
  if (backward) {
    if (interleaved) rotary_any_kernel<DT, true, true><<<grid, 256, 0, s>>>(r);
    else rotary_any_kernel<DT, false, true><<<grid, 256, 0, s>>>(r);
  } else {
    if (interleaved) rotary_any_kernel<DT, true, false><<<grid, 256, 0, s>>>(r);
    else rotary_any_kernel<DT, false, false><<<grid, 256, 0, s>>>(r);
  }
}

int group_lanes(int D) {
  int g = 1;
  while (16 * g < D) g *= 2;
  return g;
}

bool vector_form(const RotaryArgs& r, size_t es, bool backward) {
  auto al = [&](const HeadTensor& t, int heads) {
    return heads == 0 || (((uintptr_t)t.x & 15) == 0 && (t.sb * es) % 16 == 0 && (t.sh * es) % 16 == 0 &&
                          (t.sl * es) % 16 == 0);
  };
  bool ok = r.D % 16 == 0 && r.P % 8 == 0 && r.D <= kMaxDim && ((uintptr_t)r.table & 15) == 0;
  for (int i = 0; i < 2; ++i) {
    ok = ok && al(r.in[i], r.heads[i]) && al(r.out[i], r.heads[i]) && (!backward || al(r.grad[i], r.heads[i]));
    ok = ok && ((uintptr_t)r.weight[i] & 15) == 0;
  }
  return ok;
}

template <int DT>
hipError_t run_rotary(RotaryArgs r, bool interleaved, bool backward, hipStream_t s) {
  const bool vec = vector_form(r, sizeof(typename Elem<DT>::T), backward);
  if (!vec) {
    const int64_t units = r.tokens * (r.heads[0] + r.heads[1]);
    const int64_t g = backward ? backward_groups(units) : std::min<int64_t>((units + 3) / 4, 65536);
    run_any<DT>(r, interleaved, backward, (unsigned)g, s);
    return hipGetLastError();
  }
  const int G = group_lanes(r.D), hpw = 64 / G;
  const int steps = (r.heads[0] + hpw - 1) / hpw + (r.heads[1] + hpw - 1) / hpw;
  int64_t waves = r.tokens;
  if (!backward) {
    // few tokens: several waves share a token's heads, until the chip holds 8 a CU
    r.splits = (int)std::min<int64_t>(steps, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, r.tokens)));
    waves *= r.splits;
  }
  const int64_t blocks = backward ? backward_groups(r.tokens) : (waves + 3) / 4;
  for (int64_t b = 0; b < blocks; b += max_groups(256)) {
    r.first = 4 * b;
    const unsigned grid = (unsigned)std::min(blocks - b, max_groups(256));
    switch (G) {
      case 1: run_vec<DT, 1>(r, interleaved, backward, grid, s); break;
      case 2: run_vec<DT, 2>(r, interleaved, backward, grid, s); break;
      case 4: run_vec<DT, 4>(r, interleaved, backward, grid, s); break;
      case 8: run_vec<DT, 8>(r, interleaved, backward, grid, s); break;
      case 16: run_vec<DT, 16>(r, interleaved, backward, grid, s); break;
      default: run_vec<DT, 32>(r, interleaved, backward, grid, s); break;
    }
  }
  return hipGetLastError();
}

RotaryArgs rotary_args(const RotaryShape& sh) {
  RotaryArgs r{};
  r.heads[0] = sh.q_heads, r.heads[1] = sh.k_heads;
  r.batch = sh.batch, r.length = sh.length, r.D = sh.dim, r.P = sh.pairs;
  r.tokens = (int64_t)sh.batch * sh.length;
  r.table = sh.table, r.table_sb = sh.table_batch_stride;
  r.weight[0] = sh.q_weight, r.weight[1] = sh.k_weight, r.weight_dtype = sh.weight_dtype;
  r.eps = sh.eps;
  r.splits = 1;
  return r;
}

// The stride of an axis of one entry says nothing (and need not be aligned).
HeadTensor head_tensor(const RotaryArgs& r, int which, const void* p, const int64_t* st) {
  return HeadTensor{p, r.batch > 1 ? st[0] : 0, r.heads[which] > 1 ? st[1] : 0, r.length > 1 ? st[2] : 0};
}

hipError_t dispatch(const RotaryArgs& r, int dtype, bool interleaved, bool backward, hipStream_t s) {
  switch (dtype) {
    case kF32: return run_rotary<kF32>(r, interleaved, backward, s);
    case kF16: return run_rotary<kF16>(r, interleaved, backward, s);
    default: return run_rotary<kBF16>(r, interleaved, backward, s);
  }
}

}  // namespace

hipError_t launch_qk_rotary(const RotaryShape& sh, const void* q, const void* k, void* q_out, void* k_out,
                            const int64_t* strides, hipStream_t stream) {
  RotaryArgs r = rotary_args(sh);
  r.in[0] = head_tensor(r, 0, q, strides), r.in[1] = head_tensor(r, 1, k, strides + 3);
  r.out[0] = head_tensor(r, 0, q_out, strides + 6), r.out[1] = head_tensor(r, 1, k_out, strides + 9);
  return dispatch(r, sh.dtype, sh.interleaved, false, stream);
}

int64_t qk_rotary_workspace_bytes(int dim) { return (int64_t)kBackwardGroups * 2 * dim * 4; }

hipError_t launch_qk_rotary_backward(const RotaryShape& sh, const void* dq, const void* dk, const void* q,
                                     const void* k, void* q_grad, void* k_grad, void* q_weight_grad,
                                     void* k_weight_grad, const int64_t* strides, float* workspace,
                                     hipStream_t stream) {
  RotaryArgs r = rotary_args(sh);
  r.grad[0] = head_tensor(r, 0, dq, strides), r.grad[1] = head_tensor(r, 1, dk, strides + 3);
  r.in[0] = head_tensor(r, 0, q, strides + 6), r.in[1] = head_tensor(r, 1, k, strides + 9);
  r.out[0] = head_tensor(r, 0, q_grad, strides + 12), r.out[1] = head_tensor(r, 1, k_grad, strides + 15);
  r.partial = q_weight_grad || k_weight_grad ? workspace : nullptr;
  const hipError_t e = dispatch(r, sh.dtype, sh.interleaved, true, stream);
  if (e != hipSuccess || !r.partial) return e;
  const size_t es = sh.dtype == kF32 ? 4 : 2;
  const int64_t units = vector_form(r, es, true) ? r.tokens : r.tokens * (r.heads[0] + r.heads[1]);
  sum_heads_kernel<<<dim3((unsigned)((2 * sh.dim + 15) / 16)), dim3(1024), 0, stream>>>(
      r.partial, (int)backward_groups(units), sh.dim, q_weight_grad, k_weight_grad, sh.weight_dtype);
  return hipGetLastError();
}

hipError_t launch_axes_table(const void* positions, int kind, int64_t rows, int axes, const int* dims, double theta,
                             float* out, hipStream_t stream) {
  AxesArgs ax{};
  ax.axes = axes;
  int P = 0;
  for (int a = 0; a < axes; ++a) ax.half[a] = dims[a] / 2, P += dims[a] / 2;
  const int64_t n = rows * P;
  if (n == 0) return hipSuccess;
  const double lt = log(theta);
  const int64_t most = max_groups(256) * 256 / P;  // rows of a launch
  for (int64_t row = 0; row < rows; row += most) {
    const int64_t count = std::min(most, rows - row), at = row * axes;
    float* o = out + row * P * 2;
    const dim3 grid((unsigned)((count * P + 255) / 256)), block(256);
    switch (kind) {
      case CONVROT_POS_F32: axes_table_kernel<float><<<grid, block, 0, stream>>>((const float*)positions + at, count, ax, P, lt, o); break;
      case CONVROT_POS_F64: axes_table_kernel<double><<<grid, block, 0, stream>>>((const double*)positions + at, count, ax, P, lt, o); break;
      case CONVROT_POS_I32: axes_table_kernel<int><<<grid, block, 0, stream>>>((const int*)positions + at, count, ax, P, lt, o); break;
      default: axes_table_kernel<int64_t><<<grid, block, 0, stream>>>((const int64_t*)positions + at, count, ax, P, lt, o); break;
    }
  }
  return hipGetLastError();
}

}  // namespace convrot
