// W8A8 GEMM for gfx950 (8-bit integer activations and weights; the product and its
// numerics are stated in gemm_w8a8_tile.h): the kernel for a few token rows, and
// the choice of kernel.
#include <algorithm>

#include "convrot_launch.h"
#include "row_device.h"
#include "w8a8_device.h"

namespace convrot {
namespace {

// ---- few rows
//
// Up to 16 token rows: the weights' bytes bound it, each read once.  A workgroup
// owns 64 output channels, each of its 4 waves 16 of them and, for itself (no
// barrier in the loop), a ring of STAGES blocks of 128 features in LDS that it
// keeps full by direct-to-LDS loads; the rows' codes lie in LDS from the start.
// Where the channels make too few workgroups for the chip, several share K and
// the last to arrive adds their integer sums.  With FUSED the rows come as they
// are and each workgroup quantizes them itself (as convrot_quantize_int8 does):
// one launch instead of two.  Rows or codes are the first loads, the ring's fill
// the next: the quantization runs while the first weights are on their way (with
// the rows behind the ring, 1 row of 3072 -> 18432 took 18.2 us, so 12.9).
// Measured: 1 row 3072 -> 18432 12.3 us without the quantization, 56.6 MB of
// weights at 4.6 TB/s; 8 rows 8192 -> 8192 14.3 us, 4.7 TB/s.  Against the 64 x 64
// tile: 12.3 and 13.4 us, 7.5 and 8.8 (16 rows, 4096 -> 4096).
constexpr int kRowsMax = 16, kRowsN = 64;
// Rows of a fused call, which lie in LDS beside their codes.  One launch and two, in a graph, weights
// cold: 1 row 3072 -> 18432 15.4 and 18.0 us, 2 rows of 4096 -> 4096 9.5 and 10.6, at the limit 1 row
// 8192 -> 2048 9.7 and 11.9, 8192 -> 8192 19.0 and 20.9, 8 rows of 1024 -> 4096 6.06 and 6.15, 16 rows of
// 512 -> 4096 5.7 and 5.8; an eager call saves 4 us of host time besides.  Rows past the limit (one of
// 12288 in 16 bits) take two launches; one has not been tried there.
constexpr int kFusedBytes = 16384;
constexpr size_t kTwoPerCu = 79 * 1024;  // dynamic LDS of two workgroups a CU

__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor1, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor2, 0xf, 0xf, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppHalfMirror, 0xf, 0xf, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppMirror, 0xf, 0xf, true));
}

template <int DT, bool FUSED, int STAGES>
__global__ __launch_bounds__(256) void w8a8_rows_kernel(W8a8Operands p, const void* __restrict__ x, int64_t x_stride,
                                                        W8a8Split split, int tiles) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  __shared__ uint32_t row_max[kRowsMax];
  __shared__ float row_scale[kRowsMax];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
  const int kblocks = (p.K + 127) / 128, kb0 = part * split.kblocks, n = min(split.kblocks, kblocks - kb0);
  const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u, k0 = (uint32_t)kb0 * 128u, kn = (uint32_t)n * 128u;
  uint8_t* ring = smem + wave * (STAGES * 2048);
  uint8_t* codes = smem + 4 * STAGES * 2048;      // [M][kn], chunks swizzled
  uint8_t* raw = codes + (uint32_t)p.M * kn;      // FUSED: the rows as they are
  const uint32_t ring_addr = (uint32_t)(uintptr_t)ring;

  if constexpr (FUSED) {
    // 16-byte chunk i of the rows behind each other, a wave 64 of them at a time
    constexpr uint32_t ES = DT == kF32 ? 4 : 2;
    const uint32_t per_row = (uint32_t)p.K * ES / 16u, chunks = (uint32_t)p.M * per_row;
    const i32x4_sgpr rx = buffer_rsrc(x, (uint32_t)(((int64_t)(p.M - 1) * x_stride + p.K) * ES));
    for (uint32_t i0 = wave * 64u; i0 < chunks; i0 += 256u) {
      const uint32_t i = i0 + (uint32_t)lane, r = p.M == 1 ? 0u : i / per_row;
      const uint32_t off = i < chunks ? (uint32_t)(r * (uint32_t)x_stride * ES) + (i - r * per_row) * 16u : kOutOfRange;
      dma16(rx, off, (uint32_t)(uintptr_t)raw + i0 * 16u);
    }
  } else {
    const uint32_t per_row = kn / 16u, chunks = (uint32_t)p.M * per_row;
    const i32x4_sgpr ra = buffer_rsrc(p.act, (uint32_t)(p.M - 1) * (uint32_t)p.lda + k16);
    for (uint32_t i0 = wave * 64u; i0 < chunks; i0 += 256u) {
      const uint32_t i = i0 + (uint32_t)lane, r = p.M == 1 ? 0u : i / per_row, at = i - r * per_row;
      const uint32_t k = k0 + (at >> 3) * 128u + (((at & 7u) ^ (uint32_t)chunk_swizzle((int)r)) << 4);
      dma16(ra, i < chunks && k < k16 ? r * (uint32_t)p.lda + k : kOutOfRange, (uint32_t)(uintptr_t)codes + i0 * 16u);
    }
  }

  // the wave's 16 weight rows (none past N)
  const int nw = tile * kRowsN + wave * 16, nrows = min(16, p.N - nw);
  const i32x4_sgpr rw =
      buffer_rsrc(p.weight + (int64_t)(nrows > 0 ? nw : 0) * p.ldw, nrows > 0 ? (uint32_t)(nrows - 1) * (uint32_t)p.ldw + k16 : 0u);
  const int rl = lane >> 3, c = lane & 7;
  const uint32_t rest = k16 & 127u, tail_kb = rest ? k16 >> 7 : ~0u, lastkb = (uint32_t)(kb0 + n - 1);
  uint32_t vw[2];
  bool past[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t cw = 16u * (uint32_t)(c ^ rl ^ j);
    vw[j] = (uint32_t)(8 * j + rl) * (uint32_t)p.ldw + cw;
    past[j] = cw >= rest;
  }
  auto issue = [&](uint32_t kb, int stage) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t off = vw[j] + kb * 128u;
      if (kb == tail_kb) off = past[j] ? kOutOfRange : off;
      dma16(rw, off, ring_addr + (uint32_t)(stage * 2048 + j * 1024));
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) issue(min((uint32_t)(kb0 + s), lastkb), s);

  if (FUSED && tid < kRowsMax) row_max[tid] = 0;
  wait_vmcnt<2 * STAGES>();  // the rows, but not the ring
  __syncthreads();
  // place of the codes at feature k of row r
  auto code_at = [&](int r, uint32_t k) {
    const uint32_t b = (k - k0) >> 7, ch = (k >> 4) & 7;
    return codes + (uint32_t)r * kn + b * 128u + ((ch ^ (uint32_t)chunk_swizzle(r)) << 4) + (k & 15u);
  };
  if constexpr (FUSED) {
    typedef typename Elem<DT>::T E;
    const uint32_t total = (uint32_t)p.M * (uint32_t)p.K;
    // 8 values a thread, 16 lanes' 128 in one row where K % 128 == 0 (past the end: zeros)
    for (uint32_t i0 = 0; i0 < total; i0 += 2048u) {
      const uint32_t at = i0 + (uint32_t)tid * 8u, r = p.M == 1 ? 0u : at / (uint32_t)p.K;
      uint32_t most = 0;
      if (at < total) {
        float v[8];
        load8<DT>((const E*)raw + at, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
      }
      if ((p.K & 127) == 0) {
        most = max16(most);
        if ((lane & 15) == 0 && at < total) atomicMax(&row_max[r], most);
      } else if (at < total) {
        atomicMax(&row_max[r], most);
      }
    }
    __syncthreads();
    for (uint32_t at = (uint32_t)tid * 8u; at < total; at += 2048u) {
      const uint32_t r = p.M == 1 ? 0u : at / (uint32_t)p.K, k = at - r * (uint32_t)p.K;
      if (k < k0 || k >= k0 + kn) continue;
      float v[8];
      load8<DT>((const E*)raw + at, v);
      *(uint2*)code_at((int)r, k) = int8_codes(v, int8_row(row_max[r]));
    }
    if (tid < p.M) row_scale[tid] = int8_row(row_max[tid]).scale;
    __syncthreads();
  }

  const int q = lane >> 4, r = lane & 15, ra = min(r, p.M - 1);  // columns past M: some row's, never stored
  i32x4 acc = {0, 0, 0, 0};
  int st = 0;
  for (int i = 0; i < n; ++i) {
    wait_vmcnt<2 * (STAGES - 1)>();
    i32x4 w[2], a[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      w[ks] = *(const i32x4*)(ring + st * 2048 + r * 128 + (((2 * q + ks) ^ chunk_swizzle(r)) << 4));
      a[ks] = *(const i32x4*)(codes + (uint32_t)ra * kn + (uint32_t)i * 128u +
                              (((2 * q + ks) ^ chunk_swizzle(ra)) << 4));
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[ks], a[ks], acc, 0, 0, 0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the stage has been read
    asm volatile("" ::: "memory");
    issue(min((uint32_t)(kb0 + i + STAGES), lastkb), st);
    st = st + 1 == STAGES ? 0 : st + 1;
  }
  wait_vmcnt<0>();

  if (split.splits > 1) {
    const __amdgpu_buffer_rsrc_t rp =
        partial_rsrc(split.partials + (size_t)tile * split.splits * 4096, (uint32_t)split.splits * 4096u);
    store_partial(rp, (uint32_t)(part * 4096 + tid * 16), acc);
    if (!last_to_arrive(split.counters + tile, split.splits, &last)) return;
    acc = (i32x4){0, 0, 0, 0};
    for (int s = 0; s < split.splits; ++s) acc += load_partial(rp, (uint32_t)(s * 4096 + tid * 16));
  }
  const int nn = nw + 4 * q;
  if (r >= p.M || nn >= p.N) return;
  const float xs = FUSED ? row_scale[r] : p.xscales[r];
  float o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = min(nn + j, p.N - 1);
    o[j] = (((float)acc[j] * xs) * p.wscales[at]) + (p.bias ? p.bias[at] : 0.0f);
  }
  store4<DT>(p, r, nn, (p.N & 3) == 0, o);
}

// ---- choice of kernel

// Time of a tile's k-block (alone on its CU, and with every CU busy, where the
// clock drops) and what its prologue, epilogue and stores add, in microseconds,
// fitted to measurements of 16-bit outputs without a residual, and used for all.  Of 15
// shapes x 16 tiles (16-bit) the tile that the model picks is within 4 % of the fastest on 12
// (4608 x 3072 -> 12288: 256 x 224 160 us, the others 159 to 287; 1536 x 15360 -> 3072:
// 160 x 128 72 us, 256 x 256 153); it loses 8 % at 77 x 3072 -> 9216 (12.1 us, 128 x 64
// 11.2), 11 % at 512 x 3072 -> 12288 (31.1, 256 x 128 28.1) and 18 % at 512 x 3072 -> 3072
// (13.6, 128 x 64 11.5).
struct Cost {
  int bm, bn, per_cu;
  float lone, full, fixed;
};
constexpr Cost kCosts[] = {
    {256, 256, 1, 1.07f, 1.24f, 16.0f}, {256, 224, 1, 0.95f, 1.10f, 14.5f}, {224, 256, 1, 0.95f, 1.10f, 14.5f},
    {256, 192, 1, 0.84f, 1.00f, 13.0f}, {192, 256, 1, 0.84f, 1.05f, 13.0f}, {256, 128, 1, 0.63f, 0.77f, 9.0f},
    {128, 256, 1, 0.63f, 0.77f, 9.0f},  {192, 192, 1, 0.67f, 0.80f, 10.0f}, {192, 128, 1, 0.49f, 0.58f, 7.5f},
    {128, 192, 1, 0.49f, 0.58f, 7.5f},  {160, 128, 1, 0.42f, 0.52f, 7.0f},  {128, 160, 1, 0.42f, 0.52f, 7.0f},
    {128, 128, 2, 0.62f, 0.85f, 7.0f},  {128, 64, 2, 0.265f, 0.50f, 6.0f},  {64, 128, 2, 0.265f, 0.50f, 6.0f},
    {64, 64, 2, 0.18f, 0.32f, 4.5f}};

// The most workgroups that may share the K of one of `tiles` tiles.
int most_splits(int64_t tiles, int kblocks, int64_t tile_bytes, const Workspace& work) {
  const int64_t bytes = work.ptr ? (int64_t)work.bytes - (int64_t)kW8a8PartialOffset : 0;
  if (bytes <= 0 || tiles > kW8a8Counters) return 1;
  return (int)std::max<int64_t>(1, std::min({(int64_t)kblocks, bytes / (tiles * tile_bytes), (int64_t)64}));
}

// Splits of K of the few-row kernel: while the chip is not full and a part keeps 8
// blocks.  The exchange of partial sums costs 2 to 4 us: 4 rows 12288 -> 3072 (48
// tiles) 20.5 us with one, 14.1 with two, 12.4 with three, 11.9 with four (the rule's),
// 14.5 with six; 8 rows 8192 -> 4096 (64 tiles) 14.8 with one, 10.7 with three (the
// rule's), 12.9 with eight.  Few tiles of long rows: 4 rows 16384 -> 1024 (16 tiles) 21.6
// with one, 9.5 with six or eight, 10.9 with the rule's twelve.
int rows_splits(int64_t tiles, int kblocks, const Workspace& work) {
  const int forced = tuning(kTuneW8a8Split);
  const int64_t s = forced > 0 ? forced : std::min<int64_t>(192 / tiles, kblocks / 8);
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, most_splits(tiles, kblocks, 4096, work)));
}

W8a8Split make_split(int splits, int kblocks, const Workspace& work) {
  W8a8Split s;
  s.kblocks = (kblocks + splits - 1) / splits;
  s.splits = (kblocks + s.kblocks - 1) / s.kblocks;  // no workgroup without a block
  if (s.splits > 1) {
    s.counters = (int*)(work.ptr + kW8a8CounterOffset);
    s.partials = work.ptr + kW8a8PartialOffset;
  }
  return s;
}

struct Choice {
  int tile, splits;
};

// The tile, and the workgroups that share its K, that the costs make fastest.  What
// sharing adds is the exchange of partial sums, written once and read once; more than
// a workgroup a CU loses: 24 rows
// 12288 -> 3072 (48 tiles of 64 x 64) 21.2 us with one, 14.6 with two, 12.7 with
// four, 14.7 with six; 77 rows 3072 -> 9216 (288 tiles) 10.3 with one, 15.9 with two.
Choice choose(int64_t M, int64_t N, int64_t K, const Workspace& work) {
  const int forced_tile = tuning(kTuneW8a8Tile), forced_splits = tuning(kTuneW8a8Split);
  const int kblocks = (int)((K + 127) / 128);
  Choice best{0, 1};
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (forced_tile > 0 && forced_tile != tile_code(c.bm, c.bn)) continue;
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn), slots = 256 * c.per_cu;
    const int64_t bytes = (int64_t)c.bm * c.bn * 4;
    const int most = c.bm * c.bn <= kMaxSplitTile ? most_splits(tiles, kblocks, bytes, work) : 1;
    for (int s = 1; s <= most; ++s) {
      if (forced_splits > 0 ? s != std::min(forced_splits, most) : s > 1 && (kblocks < 8 * s || tiles * s > 256)) continue;
      const int64_t groups = tiles * s, rounds = groups / slots;
      if (groups > max_groups(256)) continue;
      const float part = (float)(groups - rounds * slots) / (float)slots, blocks = (float)((kblocks + s - 1) / s);
      float t = (float)rounds * (blocks * c.full + c.fixed);
      if (part > 0.0f)  // few workgroups run at a higher clock, and alone on their CUs
        t += blocks * (c.lone + (c.full - c.lone) * part) + c.fixed * (0.65f + 0.35f * part);
      if (s > 1) t += 2.0f + (float)(groups * bytes) * 2.0f / 3.0e6f;
      if (best.tile == 0 || t < best_time) best_time = t, best = {tile_code(c.bm, c.bn), s};
    }
  }
  return best;
}

bool rows_kernel(int64_t M) {
  const int forced = tuning(kTuneW8a8Tile);
  return forced > 0 ? false : M <= kRowsMax;
}

// LDS of the few-row kernel: ring, codes and (fused) the rows as they are, in whole DMAs of 1 KB.
size_t rows_lds(int64_t M, int stages, int kblocks, int64_t raw_bytes) {
  return (size_t)stages * 8192 + ((size_t)M * kblocks * 128 + 1023) / 1024 * 1024 + (size_t)(raw_bytes + 1023) / 1024 * 1024;
}

template <int DT, bool FUSED, int STAGES>
hipError_t launch_rows_s(const W8a8Operands& p, const void* x, int64_t x_stride, const W8a8Split& split, int tiles,
                         hipStream_t s) {
  const size_t lds = rows_lds(p.M, STAGES, split.kblocks, FUSED ? (int64_t)p.M * p.K * (DT == kF32 ? 4 : 2) : 0);
  w8a8_rows_kernel<DT, FUSED, STAGES><<<dim3((unsigned)(tiles * split.splits)), dim3(256), lds, s>>>(p, x, x_stride,
                                                                                                    split, tiles);
  return hipGetLastError();
}

template <int DT, bool FUSED>
hipError_t launch_rows(const W8a8Operands& p, const void* x, int64_t x_stride, const Workspace& work, hipStream_t s) {
  const int64_t tiles = (p.N + kRowsN - 1) / kRowsN;
  const int kblocks = (p.K + 127) / 128;
  W8a8Split split = make_split(rows_splits(tiles, kblocks, work), kblocks, work);
  // two workgroups a CU where the codes leave room beside the deep ring, else beside the short one
  const int64_t raw = FUSED ? (int64_t)p.M * p.K * (DT == kF32 ? 4 : 2) : 0;
  const bool deep =
      rows_lds(p.M, 8, split.kblocks, raw) <= kTwoPerCu || rows_lds(p.M, 4, split.kblocks, raw) > kTwoPerCu;
  if (deep) return launch_rows_s<DT, FUSED, 8>(p, x, x_stride, split, (int)tiles, s);
  return launch_rows_s<DT, FUSED, 4>(p, x, x_stride, split, (int)tiles, s);
}

// Whether the few-row kernel has room for the codes of a product's rows, whatever the split, and
// room for two workgroups a CU where there are more of them than CUs (16 rows 3072 -> 18432, one a
// CU: 15.8 us, on tiles 14.0).
bool rows_fit(int64_t M, int64_t N, int64_t K) {
  const int kblocks = (int)((K + 127) / 128);
  return rows_lds(M, 8, kblocks, 0) + 1024 <= 160 * 1024 &&
         ((N + kRowsN - 1) / kRowsN <= 256 || rows_lds(M, 4, kblocks, 0) <= kTwoPerCu);
}

template <int DT>
hipError_t launch_t(const W8a8Operands& p, const Workspace& work, hipStream_t s) {
  if (rows_kernel(p.M) && rows_fit(p.M, p.N, p.K)) return launch_rows<DT, false>(p, nullptr, 0, work, s);
  const Choice c = choose(p.M, p.N, p.K, work);
  return launch_w8a8_tile<DT>(c.tile, p, make_split(c.splits, (p.K + 127) / 128, work), s);
}

}  // namespace

bool w8a8_tile_known(int bm, int bn) {
#define W8A8_KNOWN(BM, BN, STAGES, PER_CU) \
  if (bm == BM && bn == BN) return true;
  W8A8_TILES(W8A8_KNOWN)
#undef W8A8_KNOWN
  return false;
}

hipError_t launch_w8a8_gemm(const int8_t* act, int64_t lda, const float* xscales, const int8_t* weight, int64_t ldw,
                            const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K, void* out,
                            int out_dtype, hipStream_t stream, const GatedResidual& gr, const Workspace& work) {
  const W8a8Operands p{act, weight, lda, ldw, xscales, wscales, bias, out, (int)M, (int)N, (int)K, gr};
  switch (out_dtype) {
    case kF32: return launch_t<kF32>(p, work, stream);
    case kF16: return launch_t<kF16>(p, work, stream);
    default: return launch_t<kBF16>(p, work, stream);
  }
}

// What a product asks of a workspace as large as the W4A4 GEMM's: with these bytes the choices above
// come out the same.
int64_t w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  const Workspace all{(uint8_t*)256, kSkWorkspaceBytes};  // never read here
  const int kblocks = (int)((K + 127) / 128);
  int64_t tiles, splits, bytes;
  if (rows_kernel(M) && rows_fit(M, N, K)) {
    tiles = (N + kRowsN - 1) / kRowsN, bytes = 4096;
    splits = rows_splits(tiles, kblocks, all);
  } else {
    const Choice c = choose(M, N, K, all);
    if (c.tile == 0) return 0;  // more tiles than a launch takes, whichever it is
    const int64_t bm = c.tile & 1023, bn = c.tile >> 10;
    tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn), bytes = bm * bn * 4;
    splits = c.splits;
  }
  return splits > 1 ? (int64_t)kW8a8PartialOffset + tiles * splits * bytes : 0;
}

bool w8a8_fused(const void* x, int dtype, int64_t M, int64_t K, int64_t x_stride) {
  const size_t es = dtype == kF32 ? 4 : 2;
  return rows_kernel(M) && M * K * (int64_t)es <= kFusedBytes && K % 16 == 0 && ((uintptr_t)x & 15) == 0 &&
         (M == 1 || ((x_stride * es) % 16 == 0 && x_stride < (int64_t(1) << 24)));
}

hipError_t launch_w8a8_fused(const void* x, int64_t x_stride, int dtype, const int8_t* weight, int64_t ldw,
                             const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K, void* out,
                             hipStream_t stream, const GatedResidual& gr, const Workspace& work) {
  const W8a8Operands p{nullptr, weight, 0, ldw, nullptr, wscales, bias, out, (int)M, (int)N, (int)K, gr};
  switch (dtype) {
    case kF32: return launch_rows<kF32, true>(p, x, x_stride, work, stream);
    case kF16: return launch_rows<kF16, true>(p, x, x_stride, work, stream);
    default: return launch_rows<kBF16, true>(p, x, x_stride, work, stream);
  }
}

}  // namespace convrot
