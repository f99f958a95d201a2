// Layer norm, its gradient, and the quantizer of activation rows to 8 bits.
//
// Forward, row by row, in float32:
//   mean = sum(x) / K,  rstd = 1 / sqrt(sum((x - mean)^2) / K + eps),
//   y = (x - mean) rstd g + b,
// with g, b a weight and bias of all rows, or g = 1 + scale[v], b = shift[v] of
// the row's group v (the adaptive norm of a diffusion transformer); y is
// rounded once.  The row stays in registers between the sums, so it is read
// once; the second sum takes differences from the mean (no cancellation).  Memory
// bounds it: 8800 x 5120 bf16 38 us, 180 MB at 4.7 TB/s (a large copy: 5.0).
//
// Backward, with u = (x - mean) rstd and h = dy g:
//   dx = rstd (h - sum(h) / K - u sum(h u) / K),  dg = sum_rows dy u,  db = sum_rows dy.
//
// Quantizer: a = max |x|, codes = round(x (127 / a)) to nearest even,
// scale = a (1 / 127) (10017 x 2688 f16 16.6 us, 81 MB at 4.9 TB/s).  With the norm in front, the normalized row goes to
// codes from registers.  A row that holds a NaN or an infinity gets the scale
// NaN and codes 0, so every product of it is NaN; a row below 2^-100 counts as
// zero (codes 0, scale 0), where 127 / a would overflow.
#include <algorithm>

#include "convrot_launch.h"
#include "row_device.h"

namespace convrot {
namespace {

enum RowOp : int { kNormOut = 0, kNormCodes = 1, kCodes = 2 };

// Sum over a team of T threads (T / 64 waves, `red` its own floats), in every
// thread.  Every thread of the workgroup calls it.
template <int T, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[T / 64], int team_wave) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[i][team_wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[i][0];
#pragma unroll
      for (int w = 1; w < T / 64; ++w) v[i] += red[i][w];
    }
  }
}

// One row a team; a workgroup is one team, or four one-wave teams.
template <int DT, int T, int C, bool VEC, int OP>
__global__ __launch_bounds__(T == 64 ? 256 : T) void row_kernel(
    const void* __restrict__ x, int64_t rows, int K, int64_t x_stride, const void* __restrict__ gain,
    const void* __restrict__ shift, int param_dtype, int plus_one, int64_t rows_per_vector, float eps,
    void* __restrict__ out, int64_t out_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out,
    float* __restrict__ scales) {
  typedef typename Elem<DT>::T E;
  constexpr int TEAMS = T == 64 ? 4 : 1, W = T / 64;
  __shared__ float red[3][1][W];
  __shared__ uint32_t redmax[W];
  const int t = threadIdx.x % T, wave = t >> 6;
  const int64_t row = (int64_t)blockIdx.x * TEAMS + (TEAMS > 1 ? threadIdx.x / T : 0);
  if (TEAMS > 1 && row >= rows) return;  // one-wave teams: no barrier below

  float v[C][8];
  const E* xr = (const E*)x + row * x_stride;
#pragma unroll
  for (int c = 0; c < C; ++c) load_chunk<DT, T, C, VEC>(xr, K, t, c, v[c]);

  if constexpr (OP != kCodes) {
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += v[c][j];
    team_sum<T>(s, red[0], wave);
    const float mean = s[0] / (float)K;
    float q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[c][j] -= mean;
        const float sq = v[c][j] * v[c][j];
        q[0] += feature_of<T, C, VEC>(t, c, j) < K ? sq : 0.0f;
      }
    team_sum<T>(q, red[1], wave);
    const float rstd = 1.0f / sqrtf(q[0] / (float)K + eps);
    if (t == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
    const uint32_t param_row = rows_per_vector > 0 ? (uint32_t)row / (uint32_t)rows_per_vector : 0;
    const size_t psize = param_dtype == kF32 ? 4 : 2;
    const char* gr = gain ? (const char*)gain + (size_t)param_row * K * psize : nullptr;
    const char* br = shift ? (const char*)shift + (size_t)param_row * K * psize : nullptr;
    const float one = plus_one ? 1.0f : 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float g[8], b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = 1.0f, b[j] = 0.0f;
      if (gr) {
        load_param<DT, T, C, VEC>(gr, param_dtype, K, t, c, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] += one;
      }
      if (br) load_param<DT, T, C, VEC>(br, param_dtype, K, t, c, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * rstd * g[j] + b[j];
    }
  }

  if constexpr (OP == kNormOut) {
    E* o = (E*)out + row * out_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) store_chunk<DT, T, C, VEC>(o, K, t, c, v[c]);
  } else {
    // As unsigned words, |x| orders infinity above every number and NaN above infinity.
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = __builtin_bit_cast(uint32_t, v[c][j]) & 0x7fffffffu;
        most = max(most, feature_of<T, C, VEC>(t, c, j) < K ? a : 0u);
      }
    most = wave_max(most);
    if constexpr (T > 64) {
      if ((t & 63) == 0) redmax[wave] = most;
      __syncthreads();
      most = redmax[0];
#pragma unroll
      for (int w = 1; w < W; ++w) most = max(most, redmax[w]);
    }
    const Int8Row q = int8_row(most);
    if (t == 0) scales[row] = q.scale;
    int8_t* o = (int8_t*)out + row * out_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j)  // columns K .. stride - 1 are zero
        v[c][j] = feature_of<T, C, VEC>(t, c, j) < K ? v[c][j] : 0.0f;
      if constexpr (VEC) {
        const int f = feature_of<T, C, VEC>(t, c, 0);
        if (f < out_stride) *(uint2*)(o + f) = int8_codes(v[c], q);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int f = feature_of<T, C, VEC>(t, c, j);
          if (f < out_stride) o[f] = (int8_t)int8_code(v[c][j], q);
        }
      }
    }
  }
}

struct RowArgs {
  const void* x;
  int64_t rows, K, x_stride;
  const void *gain, *shift;
  int param_dtype, plus_one;
  int64_t rows_per_vector;
  float eps;
  void* out;
  int64_t out_stride;
  float *mean, *rstd, *scales;
};

template <int DT, int OP, int T, int C, bool VEC>
void run_rows(const RowArgs& a, hipStream_t stream) {
  constexpr int TEAMS = T == 64 ? 4 : 1;
  constexpr int64_t MOST = max_groups(T * TEAMS) * TEAMS;
  const int64_t es = DT == kF32 ? 4 : 2, out_row = a.out_stride * (OP == kNormOut ? es : 1);
  const int64_t param_row = a.K * (a.param_dtype == kF32 ? 4 : 2), each = a.rows_per_vector;
  for (int64_t row = 0; row < a.rows;) {
    // whole vectors, or rows inside one that is longer than a launch
    const int64_t vector = each > 0 ? row / each : 0, in_vector = each > 0 ? row % each : 0;
    int64_t n = std::min(a.rows - row, MOST), rows_per_vector = each;
    if (each > MOST) n = rows_per_vector = std::min(n, each - in_vector);
    else if (each > 0 && n < a.rows - row) n = n / each * each;
    auto params = [&](const void* p) { return p ? (const char*)p + vector * param_row : nullptr; };
    row_kernel<DT, T, C, VEC, OP><<<dim3((unsigned)((n + TEAMS - 1) / TEAMS)), dim3(T * TEAMS), 0, stream>>>(
        (const char*)a.x + row * a.x_stride * es, n, (int)a.K, a.x_stride, params(a.gain), params(a.shift),
        a.param_dtype, a.plus_one, rows_per_vector, a.eps, (char*)a.out + row * out_row, a.out_stride,
        a.mean ? a.mean + row : nullptr, a.rstd ? a.rstd + row : nullptr, a.scales ? a.scales + row : nullptr);
    row += n;
  }
}

template <int DT, int OP>
hipError_t pick_rows(const RowArgs& a, bool vec, hipStream_t stream) {
  const int64_t k = OP == kNormOut ? a.K : a.out_stride;  // codes are written up to their stride
  if (vec) {
    if (k <= 512) run_rows<DT, OP, 64, 1, true>(a, stream);
    else if (k <= 1024) run_rows<DT, OP, 64, 2, true>(a, stream);
    else if (k <= 2048) run_rows<DT, OP, 256, 1, true>(a, stream);
    else if (k <= 4096) run_rows<DT, OP, 256, 2, true>(a, stream);
    else if (k <= 6144) run_rows<DT, OP, 256, 3, true>(a, stream);
    else if (k <= 8192) run_rows<DT, OP, 256, 4, true>(a, stream);
    else if (k <= 16384) run_rows<DT, OP, 1024, 2, true>(a, stream);
    else if (k <= 32768) run_rows<DT, OP, 1024, 4, true>(a, stream);
    else run_rows<DT, OP, 1024, 8, true>(a, stream);
  } else {
    if (k <= 2048) run_rows<DT, OP, 256, 1, false>(a, stream);
    else if (k <= 8192) run_rows<DT, OP, 1024, 1, false>(a, stream);
    else if (k <= 16384) run_rows<DT, OP, 1024, 2, false>(a, stream);
    else if (k <= 32768) run_rows<DT, OP, 1024, 4, false>(a, stream);
    else run_rows<DT, OP, 1024, 8, false>(a, stream);
  }
  return hipGetLastError();
}

template <int OP>
hipError_t launch_rows(const RowArgs& a, int dtype, hipStream_t stream) {
  const size_t es = dtype == kF32 ? 4 : 2;
  auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  // the stride of a single row says nothing
  bool vec = a.K % 8 == 0 && al(a.x) && (a.rows == 1 || (a.x_stride * es) % 16 == 0) && al(a.out) && al(a.gain) &&
             al(a.shift);
  if (OP == kNormOut) vec = vec && (a.out_stride * es) % 16 == 0;
  else vec = vec && a.out_stride % 8 == 0;
  switch (dtype) {
    case kF32: return pick_rows<kF32, OP>(a, vec, stream);
    case kF16: return pick_rows<kF16, OP>(a, vec, stream);
    default: return pick_rows<kBF16, OP>(a, vec, stream);
  }
}

// ---- backward
//
// A workgroup is TEAMS teams that walk the rows of one group (vector) of the
// norm's parameters, R rows a step; each thread keeps the sums of dg and db of
// its features in registers, the teams' sums are added through LDS at the end
// and stored as one partial of the workgroup.  A second kernel adds the
// partials in order, so gradients repeat bit for bit.  The next step's rows are
// loaded before this step's sums meet (PREFETCH), and rows are kept as they were
// loaded: what the second half of a step needs is computed again from them (held
// as floats in teams of 256 it spilled: 8800 x 5120 bf16 141 us, so 59, 270 MB at
// 4.6 TB/s, the partials' 21 MB not counted).

template <int DT, int T, int C, bool VEC, int TEAMS>
__global__ __launch_bounds__(T* TEAMS) void norm_backward_kernel(
    const void* __restrict__ dy, int64_t dy_stride, const void* __restrict__ x, int64_t x_stride,
    const float* __restrict__ mean, const float* __restrict__ rstd, int K, const void* __restrict__ gain,
    int param_dtype, int plus_one, int64_t rows_per_vector, int parts, void* __restrict__ dx,
    float* __restrict__ partial) {
  typedef typename Elem<DT>::T E;
  constexpr int W = T / 64, R = C == 1 && T < 1024 ? 2 : 1;  // teams of 1024 have 128 registers a thread
  constexpr bool PREFETCH = C == 1;
  __shared__ float red[2][TEAMS][2 * R][W];
  extern __shared__ float sums[];  // [2][K] of the teams' sums, where TEAMS > 1
  const int team = TEAMS > 1 ? threadIdx.x / T : 0, t = TEAMS > 1 ? threadIdx.x % T : threadIdx.x, wave = t >> 6;
  const int64_t vector = blockIdx.x / parts, part = blockIdx.x % parts;
  const int64_t r0 = vector * rows_per_vector, r1 = r0 + rows_per_vector, step = (int64_t)parts * TEAMS * R;
  const size_t psize = param_dtype == kF32 ? 4 : 2;
  const char* gr = gain ? (const char*)gain + (size_t)vector * K * psize : nullptr;
  const float one = plus_one ? 1.0f : 0.0f, inv_k = 1.0f / (float)K;
  auto gains = [&](int c, float (&g)[8]) {
    if (gr) {
      load_param<DT, T, C, VEC>(gr, param_dtype, K, t, c, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += one;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = 1.0f;
    }
  };

  // The mean, but zero past the row: of a constant row of large values (0 - mean) rstd is infinite,
  // and zero (d there) times it no number.  (float16 has no such values: 65504 / sqrt(eps) is finite.)
  auto centre = [&](float mu, int c, int j) {
    return DT == kF16 || feature_of<T, C, VEC>(t, c, VEC ? 0 : j) < K ? mu : 0.0f;
  };

  struct Rows {
    RawChunk<DT, T, C, VEC> x[R][C], d[R][C];
    float mu[R], rs[R];
  };
  // rows past the end count as zeros (every team makes as many steps: the barriers below)
  auto load = [&](Rows& q, int64_t base) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = base + team * R + i;
      const bool live = row < r1;
      q.mu[i] = live ? mean[row] : 0.0f;
      q.rs[i] = live ? rstd[row] : 0.0f;
      const int k = live ? K : 0;
      const E* xr = (const E*)x + (live ? row : r0) * x_stride;
      const E* dr = (const E*)dy + (live ? row : r0) * dy_stride;
#pragma unroll
      for (int c = 0; c < C; ++c) q.x[i][c].load(xr, k, t, c), q.d[i][c].load(dr, k, t, c);
    }
  };

  float dg[C][8], db[C][8], g1[8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[c][j] = db[c][j] = 0.0f;
  if constexpr (C == 1) gains(0, g1);
  Rows cur, next;
  load(cur, r0 + part * TEAMS * R);
  int flip = 0;
  for (int64_t base = r0 + part * TEAMS * R; base < r1; base += step) {
    if constexpr (PREFETCH) load(next, base + step);
    float s[2 * R];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) s[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float g[8];
      if constexpr (C > 1) gains(c, g);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float u[8], d[8];
        cur.x[i][c].get(u), cur.d[i][c].get(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // features past the row: d is zero
          u[j] = (u[j] - centre(cur.mu[i], c, j)) * cur.rs[i];
          db[c][j] += d[j];
          dg[c][j] += d[j] * u[j];
          const float h = d[j] * (C == 1 ? g1[j] : g[j]);
          s[2 * i] += h;
          s[2 * i + 1] += h * u[j];
        }
      }
    }
    team_sum<T>(s, red[flip][team], wave);
    flip ^= 1;  // the next step's sums go elsewhere: one barrier a step is enough
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float g[8];
      if constexpr (C > 1) gains(c, g);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int64_t row = base + team * R + i;
        if (row >= r1) continue;
        const float m0 = s[2 * i] * inv_k, m1 = s[2 * i + 1] * inv_k;
        float u[8], d[8];
        cur.x[i][c].get(u), cur.d[i][c].get(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] = (u[j] - centre(cur.mu[i], c, j)) * cur.rs[i];
          d[j] = cur.rs[i] * (d[j] * (C == 1 ? g1[j] : g[j]) - m0 - u[j] * m1);
        }
        store_chunk<DT, T, C, VEC>((E*)dx + row * (int64_t)K, K, t, c, d);
      }
    }
    if constexpr (PREFETCH) cur = next;
    else load(cur, base + step);
  }

  if (!partial) return;
  if constexpr (TEAMS > 1) {
    // team by team, in order
    for (int i = TEAMS - 1; i > 0; --i) {
      __syncthreads();
      if (team == i) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int f = feature_of<T, C, VEC>(t, c, j);
            if (f < K) {
              sums[f] = i == TEAMS - 1 ? dg[c][j] : sums[f] + dg[c][j];
              sums[K + f] = i == TEAMS - 1 ? db[c][j] : sums[K + f] + db[c][j];
            }
          }
      }
    }
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int f = feature_of<T, C, VEC>(t, c, j);
        if (f < K) dg[c][j] += sums[f], db[c][j] += sums[K + f];
      }
  }
  float* p = partial + (size_t)blockIdx.x * 2 * K;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    store_chunk<kF32, T, C, VEC>(p, K, t, c, dg[c]);
    store_chunk<kF32, T, C, VEC>(p + K, K, t, c, db[c]);
  }
}

// out[v][f] = sum over the parts of partial[v][part][which][f], f < K: 16
// threads a feature each add every 16th part, then their sums in order.
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ partial, int parts, int K,
                                                         void* __restrict__ dgain, void* __restrict__ dshift,
                                                         int dtype) {
  __shared__ float red[16][64];
  const int col = threadIdx.x & 63, lot = threadIdx.x >> 6;
  const int blocks = (2 * K + 63) / 64;  // of one vector
  const int64_t vector = blockIdx.x / blocks;
  const int f = (blockIdx.x % blocks) * 64 + col;  // of 2 K: dg then db
  float s = 0.0f;
  if (f < 2 * K) {
    const float* p = partial + (size_t)vector * parts * 2 * K + f;
#pragma unroll 4
    for (int i = lot; i < parts; i += 16) s += p[(size_t)i * 2 * K];
  }
  red[lot][col] = s;
  __syncthreads();
  if (lot != 0 || f >= 2 * K) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += red[i][col];
  void* o = f < K ? dgain : dshift;
  if (!o) return;
  const int64_t at = vector * K + (f < K ? f : f - K);
  if (dtype == kF32) store_out<kF32>(o, at, s);
  else if (dtype == kF16) store_out<kF16>(o, at, s);
  else store_out<kBF16>(o, at, s);
}

struct BackwardArgs {
  const void* dy;
  int64_t dy_stride;
  const void* x;
  int64_t x_stride;
  const float *mean, *rstd;
  int64_t rows, K;
  const void* gain;
  int param_dtype, plus_one;
  int64_t rows_per_vector;
  int parts;
  void* dx;
  float* partial;
};

// Threads a row takes in the backward kernel, 8 features each (16 or 32 past
// 8192 features), and the teams of a workgroup.
constexpr int kTeamThreads[] = {64, 128, 256, 384, 512, 640, 768, 1024};
int backward_team(int64_t K) {
  for (int t : kTeamThreads)
    if (K <= 8 * t) return t;
  return 1024;
}
constexpr int backward_teams(int T) { return T <= 256 ? 512 / T : 1; }

template <int DT, int T, int C, bool VEC>
hipError_t run_backward(const BackwardArgs& a, hipStream_t stream) {
  constexpr int TEAMS = backward_teams(T);
  const size_t lds = TEAMS > 1 && a.partial ? (size_t)a.K * 8 : 0;  // at most 16 KB
  const int64_t vectors = a.rows / a.rows_per_vector, most = std::max<int64_t>(1, max_groups(T * TEAMS) / a.parts);
  const int64_t es = DT == kF32 ? 4 : 2, param_row = a.K * (a.param_dtype == kF32 ? 4 : 2);
  for (int64_t v = 0; v < vectors; v += most) {
    const int64_t n = std::min(most, vectors - v), row = v * a.rows_per_vector;
    norm_backward_kernel<DT, T, C, VEC, TEAMS><<<dim3((unsigned)(n * a.parts)), dim3(T * TEAMS), lds, stream>>>(
        (const char*)a.dy + row * a.dy_stride * es, a.dy_stride, (const char*)a.x + row * a.x_stride * es, a.x_stride,
        a.mean + row, a.rstd + row, (int)a.K, a.gain ? (const char*)a.gain + v * param_row : nullptr, a.param_dtype,
        a.plus_one, a.rows_per_vector, a.parts, (char*)a.dx + row * a.K * es,
        a.partial ? a.partial + v * a.parts * 2 * a.K : nullptr);
  }
  return hipGetLastError();
}

template <int DT, bool VEC>
hipError_t pick_backward(const BackwardArgs& a, hipStream_t s) {
  if (a.K > 16384) return run_backward<DT, 1024, 4, VEC>(a, s);
  if (a.K > 8192) return run_backward<DT, 1024, 2, VEC>(a, s);
  switch (backward_team(a.K)) {
    case 64: return run_backward<DT, 64, 1, VEC>(a, s);
    case 128: return run_backward<DT, 128, 1, VEC>(a, s);
    case 256: return run_backward<DT, 256, 1, VEC>(a, s);
    case 384: return run_backward<DT, 384, 1, VEC>(a, s);
    case 512: return run_backward<DT, 512, 1, VEC>(a, s);
    case 640: return run_backward<DT, 640, 1, VEC>(a, s);
    case 768: return run_backward<DT, 768, 1, VEC>(a, s);
    default: return run_backward<DT, 1024, 1, VEC>(a, s);
  }
}

}  // namespace

hipError_t launch_quantize_int8(const void* x, int dtype, int64_t rows, int64_t K, int64_t x_stride, int8_t* codes,
                                int64_t codes_stride, float* scales, hipStream_t stream) {
  RowArgs a{x, rows, K, x_stride, nullptr, nullptr, kF32, 0, 0, 0.0f, codes, codes_stride, nullptr, nullptr, scales};
  return launch_rows<kCodes>(a, dtype, stream);
}

hipError_t launch_layer_norm(const void* x, int dtype, int64_t rows, int64_t K, int64_t x_stride, const void* gain,
                             const void* shift, int param_dtype, int plus_one, int64_t rows_per_vector, float eps,
                             void* out, float* mean, float* rstd, hipStream_t stream) {
  RowArgs a{x, rows, K, x_stride, gain, shift, param_dtype, plus_one, rows_per_vector, eps, out, K, mean, rstd, nullptr};
  return launch_rows<kNormOut>(a, dtype, stream);
}

hipError_t launch_layer_norm_int8(const void* x, int dtype, int64_t rows, int64_t K, int64_t x_stride,
                                  const void* gain, const void* shift, int param_dtype, int plus_one,
                                  int64_t rows_per_vector, float eps, int8_t* codes, int64_t codes_stride,
                                  float* scales, hipStream_t stream) {
  RowArgs a{x,   rows,  K,            x_stride, gain,    shift,  param_dtype, plus_one, rows_per_vector,
            eps, codes, codes_stride, nullptr,  nullptr, scales};
  return launch_rows<kNormCodes>(a, dtype, stream);
}

// Workgroups that share the rows of one vector: up to 16 waves a CU in all (each
// workgroup costs a partial of 2 K floats), and no more than the rows feed.
int layer_norm_parts(int64_t rows, int64_t K, int64_t rows_per_vector) {
  const int64_t team = backward_team(K), teams = backward_teams((int)team), vectors = rows / rows_per_vector;
  const int64_t step = teams * (team < 1024 ? 2 : 1), steps = (rows_per_vector + step - 1) / step;
  const int64_t groups = 256 * std::max<int64_t>(1, 1024 / (team * teams));
  const int64_t parts = std::min((groups + vectors - 1) / vectors, steps);
  return (int)std::max<int64_t>(1, parts);
}

hipError_t launch_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                      const float* mean, const float* rstd, int dtype, int64_t rows, int64_t K,
                                      const void* gain, int param_dtype, int plus_one, int64_t rows_per_vector,
                                      void* dx, void* dgain, void* dshift, float* workspace, hipStream_t stream) {
  BackwardArgs a{dy, dy_stride, x, x_stride, mean, rstd, rows, K, gain, param_dtype, plus_one, rows_per_vector,
                 layer_norm_parts(rows, K, rows_per_vector), dx, (dgain || dshift) ? workspace : nullptr};
  const size_t es = dtype == kF32 ? 4 : 2;
  auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const bool vec = K % 8 == 0 && al(dy) && al(x) && al(dx) && al(gain) &&
                   (rows == 1 || ((dy_stride * es) % 16 == 0 && (x_stride * es) % 16 == 0));
  hipError_t e;
  if (dtype == kF32) e = vec ? pick_backward<kF32, true>(a, stream) : pick_backward<kF32, false>(a, stream);
  else if (dtype == kF16) e = vec ? pick_backward<kF16, true>(a, stream) : pick_backward<kF16, false>(a, stream);
  else e = vec ? pick_backward<kBF16, true>(a, stream) : pick_backward<kBF16, false>(a, stream);
  if (e != hipSuccess || !a.partial) return e;
  const int64_t vectors = rows / rows_per_vector, groups = (2 * K + 63) / 64, most = max_groups(1024) / groups;
  const int64_t param_row = K * (param_dtype == kF32 ? 4 : 2);
  for (int64_t v = 0; v < vectors; v += most) {
    auto params = [&](void* p) { return p ? (char*)p + v * param_row : nullptr; };
    sum_parts_kernel<<<dim3((unsigned)(std::min(most, vectors - v) * groups)), dim3(1024), 0, stream>>>(
        a.partial + v * a.parts * 2 * K, a.parts, (int)K, params(dgain), params(dshift), param_dtype);
  }
  return hipGetLastError();
}

}  // namespace convrot
