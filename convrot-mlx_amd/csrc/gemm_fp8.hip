// Products in 8-bit floating point for gfx950 (the product and its numerics are stated
// in gemm_fp8_tile.h): the kernel for a few token rows, and the choice of kernel.
#include <algorithm>

#include "convrot_launch.h"
#include "fp8_device.h"
#include "gemm_groups.h"
#include "row_device.h"

namespace convrot {
namespace {

// ---- few rows
//
// Up to 16 token rows: the weights' bytes bound it, each read once.  A workgroup owns 64 output channels, each of
// its 4 waves 16 of them and, for itself (no barrier in the loop), a ring of STAGES blocks of 128 features in LDS
// that it keeps full by loads straight to LDS; the rows' codes and scales of its part of K lie in LDS from the
// start.  Where the channels make too few workgroups for the chip, several share K, and the last to arrive adds
// their sums in the parts' order.  With FUSED the rows come as they are and each workgroup quantizes its part of
// them itself (as convrot_quantize_fp8 does, block by block): one launch instead of two, while the first weights
// are on their way.  Here and on the 32 x 64 tile in us, from
// codes: 1 row 4096 -> 12288 10.1 (5.0 TB/s) and 12.0, 8 rows 10.4 and 12.1, 16 rows 1024 -> 4096 4.2 and 5.3, 1 row
// 15360 -> 5120 17.8 and 21.0; from 16-bit rows: 10.0 and 14.4 (1 row 4096 -> 12288), 4.2 and 7.6 (1 row 1024 -> 4096).
constexpr int kRowsMax = 16, kRowsN = 64;
// Bytes of a fused call's rows, which lie in LDS beside their codes, and which every workgroup quantizes: of one row,
// and of several.  Fused and not, in us: 2 x 4096 -> 12288 10.6 and 13.1, 4 x 4096 -> 12288 12.7 and 12.7, 8 x 2048 ->
// 24576 16.8 and 13.1, 1 x 15360 -> 5120 17.8 and 20.4.
constexpr int64_t kFusedRowBytes = 32768, kFusedBytes = 16384;
constexpr size_t kTwoPerCu = 79 * 1024;    // dynamic LDS of two workgroups a CU

// LDS of the few-row kernel, in bytes from its start: the rings, the codes [block][row][128], the scales of
// rows [block][row] and of the weights [block], and (fused) the rows as they are.
struct RowsLds {
  uint32_t codes, xs, ws, raw, end;
};
__host__ __device__ __forceinline__ RowsLds rows_lds(int stages, int rows, int blocks, int raw_size) {
  const auto whole = [](uint32_t n) { return (n + 1023u) & ~1023u; };  // whole wave loads
  RowsLds l;
  l.codes = (uint32_t)stages * 8192u;
  l.xs = l.codes + whole((uint32_t)(rows * blocks) * 128u);
  l.ws = l.xs + whole((uint32_t)(rows * blocks) * 4u);
  l.raw = l.ws + whole((uint32_t)blocks * 4u);
  l.end = l.raw + whole((uint32_t)(rows * blocks) * 128u * (uint32_t)raw_size);
  return l;
}

template <int DT, bool FUSED, int STAGES>
__global__ __launch_bounds__(256) void fp8_few_rows_kernel(Fp8Operands p, const void* __restrict__ x, int64_t x_stride,
                                                           W8a8Split split, int tiles) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  __shared__ int last;
  constexpr uint32_t ES = DT == kF32 ? 4 : 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
  const int kblocks = (p.K + kBlock - 1) / kBlock, kb0 = part * split.kblocks, n = min(split.kblocks, kblocks - kb0);
  const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u, k0 = (uint32_t)kb0 * 128u, M = (uint32_t)p.M;
  const RowsLds at = rows_lds(STAGES, p.M, n, FUSED ? (int)ES : 0);
  const uint32_t base = (uint32_t)(uintptr_t)smem;

  // the weights' scales, and the rows: as they are, 16-byte chunks of [row][n 128], or their codes and scales
  const i32x4_sgpr rs = dma_rsrc(p.wscales + (int64_t)(tile * kRowsN / kBlock) * p.ws_row + kb0, (uint32_t)n * 4u);
  for (uint32_t i0 = wave * 64u; i0 < (uint32_t)n; i0 += 256u) dma4(rs, (i0 + lane) * 4u, base + at.ws + i0 * 4u);
  if constexpr (FUSED) {
    const uint32_t per_row = (uint32_t)n * 8u * ES, chunks = M * per_row;
    const i32x4_sgpr rx = dma_rsrc(x, (uint32_t)(((int64_t)(p.M - 1) * x_stride + p.K) * ES));
    for (uint32_t i0 = wave * 64u; i0 < chunks; i0 += 256u) {
      const uint32_t i = i0 + (uint32_t)lane, r = M == 1 ? 0u : i / per_row, b = k0 * ES + (i - r * per_row) * 16u;
      dma16(rx, i < chunks && b < (uint32_t)p.K * ES ? r * (uint32_t)x_stride * ES + b : kPastEnd,
                 base + at.raw + i0 * 16u);
    }
  } else {
    const uint32_t per_block = M * 8u, chunks = (uint32_t)n * per_block;
    const i32x4_sgpr ra = dma_rsrc(p.act, (uint32_t)(p.M - 1) * (uint32_t)p.lda + k16);
    for (uint32_t i0 = wave * 64u; i0 < chunks; i0 += 256u) {
      const uint32_t i = i0 + (uint32_t)lane, b = i / per_block, r = (i - b * per_block) >> 3;
      const uint32_t k = k0 + b * 128u + (((i & 7u) ^ (uint32_t)chunk_swizzle((int)r)) << 4);
      dma16(ra, i < chunks && k < k16 ? r * (uint32_t)p.lda + k : kPastEnd, base + at.codes + i0 * 16u);
    }
    const i32x4_sgpr rx = dma_rsrc(p.xscales, (uint32_t)((p.M - 1) * p.xs_row + (kblocks - 1) * p.xs_block) * 4u + 4u);
    for (uint32_t i0 = wave * 64u; i0 < M * (uint32_t)n; i0 += 256u) {
      const uint32_t i = i0 + (uint32_t)lane, b = i / M, r = i - b * M;
      dma4(rx, i < M * (uint32_t)n ? (r * (uint32_t)p.xs_row + (kb0 + b) * (uint32_t)p.xs_block) * 4u : kPastEnd,
                base + at.xs + i0 * 4u);
    }
  }

  // the wave's 16 weight rows (none past N)
  const int nw = tile * kRowsN + wave * 16, nrows = min(16, p.N - nw);
  const i32x4_sgpr rw = dma_rsrc(p.weight + (int64_t)(nrows > 0 ? nw : 0) * p.ldw,
                                 nrows > 0 ? (uint32_t)(nrows - 1) * (uint32_t)p.ldw + k16 : 0u);
  const int rl = lane >> 3, c = lane & 7;
  const uint32_t rest = k16 & 127u, tail_kb = rest ? k16 >> 7 : ~0u, lastkb = (uint32_t)(kb0 + n - 1);
  const uint32_t ring = base + (uint32_t)wave * (STAGES * 2048u);
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
      if (kb == tail_kb) off = past[j] ? kPastEnd : off;
      dma16(rw, off, ring + (uint32_t)(stage * 2048 + j * 1024));
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) issue(min((uint32_t)(kb0 + s), lastkb), s);
  wait_vmcnt<2 * STAGES>();  // the rows, but not the ring
  __syncthreads();
  if constexpr (FUSED) {
    typedef typename Elem<DT>::T T;
    // 16 lanes a block of a row, 8 features a lane
    const uint32_t sub = (uint32_t)tid & 15u, total = M * (uint32_t)n;
    for (uint32_t i = (uint32_t)tid >> 4; i < total; i += 16u) {  // uniform over the 16 lanes
      const uint32_t r = M == 1 ? 0u : i / (uint32_t)n, b = i - r * (uint32_t)n;
      float v[8];
      load8<DT>((const T*)(smem + at.raw) + (i * 128u + sub * 8u), v);
      const Fp8Scale sc = fp8_scale(max_of_16(most_of(v)));
      const uint2 w = {fp8_codes4(v, sc.inverse), fp8_codes4(v + 4, sc.inverse)};
      const uint32_t row = b * M + r, chunk = (sub >> 1) ^ (uint32_t)chunk_swizzle((int)r);
      *(uint2*)(smem + at.codes + row * 128u + (chunk << 4) + (sub & 1u) * 8u) = w;
      if (sub == 0) ((float*)(smem + at.xs))[row] = sc.scale;
    }
    __syncthreads();
  }

  const int q = lane >> 4, r = lane & 15, ra = min(r, p.M - 1);  // columns past M: some row's, never stored
  const auto fragment = [&](const uint8_t* row, int swizzle) {
    const i32x4 lo = *(const i32x4*)(row + ((2 * q) ^ swizzle) * 16);
    const i32x4 hi = *(const i32x4*)(row + ((2 * q + 1) ^ swizzle) * 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const uint8_t* wr = smem + wave * (STAGES * 2048) + r * 128;
  const uint8_t* ar = smem + at.codes + ra * 128;
  const float *xs = (const float*)(smem + at.xs) + ra, *ws = (const float*)(smem + at.ws);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  int st = 0;
  for (int i = 0; i < n; ++i) {
    wait_vmcnt<2 * (STAGES - 1)>();
    const auto w = fragment(wr + st * 2048, chunk_swizzle(r));
    const auto a = fragment(ar + (uint32_t)i * M * 128u, chunk_swizzle(ra));
    const float s = xs[(uint32_t)i * M] * ws[i];
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (DT == kF32) {
      const WideCodes wide = widen_codes(w), act = widen_codes(a);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide.v[j], act.v[j], sum, 0, 0, 0);
    } else {
      sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, sum, 0, 0, 0, 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
    issue(min((uint32_t)(kb0 + i + STAGES), lastkb), st);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(sum[j], s, acc[j]);
    st = st + 1 == STAGES ? 0 : st + 1;
  }
  wait_vmcnt<0>();

  if (split.splits > 1) {
    const __amdgpu_buffer_rsrc_t rp =
        partial_rsrc(split.partials + (size_t)tile * split.splits * 4096, (uint32_t)split.splits * 4096u);
    store_partial(rp, (uint32_t)(part * 4096 + tid * 16), __builtin_bit_cast(i32x4, acc));
    if (!last_to_arrive(split.counters + tile, split.splits, &last)) return;
    acc = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < split.splits; ++s)
      acc += __builtin_bit_cast(f32x4, load_partial(rp, (uint32_t)(s * 4096 + tid * 16)));
  }
  const int nn = nw + 4 * q;
  if (r >= p.M || nn >= p.N) return;
  float o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = acc[j] + (p.bias ? p.bias[min(nn + j, p.N - 1)] : 0.0f);
  const W8a8Operands out{nullptr, nullptr, 0, 0, nullptr, nullptr, nullptr, p.out, p.M, p.N, p.K, p.gr};
  store4<DT>(out, r, nn, (p.N & 3) == 0, o);
}

// ---- choice of kernel

// Time of a tile's block of 128 features (few tiles, and with every CU busy), and what its prologue and
// epilogue add, in microseconds, fitted to 16-bit products without a residual on weights from memory.
struct Cost {
  int bm, bn, per_cu;
  float lone, full, fixed;
};
constexpr Cost kCosts[] = {{256, 256, 1, 1.31f, 1.74f, 7.0f},
                           {128, 128, 2, 0.575f, 1.11f, 3.7f},
                           {64, 128, 2, 0.39f, 0.71f, 3.7f},
                           {64, 64, 2, 0.27f, 0.44f, 3.6f},
                           {32, 64, 2, 0.25f, 0.29f, 3.4f}};

// The most workgroups that may share the K of one of `tiles` tiles.
int most_splits(int64_t tiles, int kblocks, int64_t tile_bytes, const Workspace& work) {
  const int64_t bytes = work.ptr ? (int64_t)work.bytes - (int64_t)kW8a8PartialOffset : 0;
  if (bytes <= 0 || tiles > kW8a8Counters) return 1;
  return (int)std::max<int64_t>(1, std::min({(int64_t)kblocks, bytes / (tiles * tile_bytes), (int64_t)64}));
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

// Microseconds of `groups` workgroups of a tile, each of `blocks` blocks.
float time_of(const Cost& c, int64_t groups, float blocks) {
  const int64_t slots = 256 * c.per_cu, rounds = groups / slots;
  const float part = (float)(groups - rounds * slots) / (float)slots;
  float t = (float)rounds * (blocks * c.full + c.fixed);
  if (part > 0.0f && part <= 0.5f && c.bm == 256)  // in quarters or halves
    t += part <= 0.25f ? blocks * 0.59f + 5.0f : blocks * 0.87f + 6.0f;
  else if (part > 0.0f) {
    // few workgroups run at a higher clock, and of two a CU the first ones alone
    const float crowd = c.per_cu == 1 ? part : std::max(0.0f, 2.0f * part - 1.0f);
    t += blocks * (c.lone + (c.full - c.lone) * crowd) + c.fixed * (0.65f + 0.35f * part);
  }
  return t;
}

struct Choice {
  int tile, splits;
};

// The tile, and the workgroups that share its K, that the costs make fastest.  What sharing adds is the exchange
// of partial sums, written once and read once; more than a workgroup a CU loses.
Choice choose(int64_t M, int64_t N, int64_t K, const Workspace& work) {
  const int forced_tile = tuning(kTuneFp8Tile), forced_splits = tuning(kTuneFp8Split);
  const int kblocks = (int)((K + 127) / 128);
  Choice best{0, 1};
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (forced_tile > 0 && forced_tile != tile_code(c.bm, c.bn)) continue;
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const int64_t bytes = (int64_t)c.bm * c.bn * 4;
    const int most = c.bm * c.bn <= kMaxFp8SplitTile ? most_splits(tiles, kblocks, bytes, work) : 1;
    for (int s = 1; s <= most; ++s) {
      if (forced_splits > 0 ? s != std::min(forced_splits, most) : s > 1 && (kblocks < 8 * s || tiles * s > 256)) continue;
      const int64_t groups = tiles * s;
      if (groups > max_groups(512) || groups > 0x7fff0000) continue;
      float t = time_of(c, groups, (float)((kblocks + s - 1) / s));
      if (s > 1) t += 2.0f + (float)(groups * bytes) * 2.0f / 3.0e6f;
      if (best.tile == 0 || t < best_time) best_time = t, best = {tile_code(c.bm, c.bn), s};
    }
  }
  return best;
}

// The tile of grouped rows.  How they spread over the experts is known on the device alone: taken as even, each
// expert's last tile half full: over 89 sizes (1 to 14000 rows, 1 to 64 experts) the tile taken is 1 % slower than the
// best of the five on average, 21 % at worst.
int grouped_tile(const Fp8Operands& p) {
  const int forced = tuning(kTuneFp8Tile);
  if (forced > 0) return forced;
  const int64_t met = std::min<int64_t>(p.g.experts, p.M), kblocks = (p.K + 127) / 128;
  const float each = (float)p.M / (float)met;
  int best = 0;
  float best_time = 0.0f;
  for (const Cost& c : kCosts) {
    if (most_tile_rows(p.M, p.g.experts, c.bm) * ((p.N + c.bn - 1) / c.bn) > max_groups(512) - 1024) continue;
    const float rows = std::max(1.0f, each / (float)c.bm + 0.5f) * (float)met;
    const float t = time_of(c, (int64_t)(rows * (float)((p.N + c.bn - 1) / c.bn)), (float)kblocks);
    if (best == 0 || t < best_time) best_time = t, best = tile_code(c.bm, c.bn);
  }
  return best;
}

// Workgroups that share the K of the few-row kernel's tiles: while the chip is not full, up to 8, and a part keeps 12
// blocks.  1 row 15360 -> 5120 (80 tiles) 19.8 us with one, 17.7 with three (the rule's), 20.3 with eight; 16384 ->
// 1024 (16 tiles) 20.0 with one, 10.5 with eight (the rule's), 13.8 with sixteen; 4096 -> 1024 7.1 with one, 8.1 with
// two (the rule's), but for 16 rows, on the short ring, 11.2 and 10.6.
int rows_splits(int64_t tiles, int kblocks, const Workspace& work) {
  const int forced = tuning(kTuneFp8Split);
  const int64_t s = forced > 0 ? forced : std::min<int64_t>({256 / tiles, kblocks / 12, 8});
  return (int)std::max<int64_t>(1, std::min<int64_t>(s, most_splits(tiles, kblocks, 4096, work)));
}

// Whether the few-row kernel takes a product: its workgroups in one launch, its rows' codes beside the ring, two
// workgroups a CU.
bool few_rows_shape(int64_t M, int64_t N) {
  return tuning(kTuneFp8Tile) <= 0 && M <= kRowsMax && (N + kRowsN - 1) / kRowsN <= max_groups(256);
}
bool few_rows(const Fp8Operands& p) {
  return few_rows_shape(p.M, p.N) &&
         rows_lds(4, p.M, (p.K + kBlock - 1) / kBlock, 0).end <= kTwoPerCu;
}

template <int DT, bool FUSED>
hipError_t launch_few_rows(const Fp8Operands& p, const void* x, int64_t x_stride, const Workspace& work,
                           hipStream_t s) {
  const int64_t tiles = ((int64_t)p.N + kRowsN - 1) / kRowsN;
  const int kblocks = (p.K + kBlock - 1) / kBlock;
  const W8a8Split split = make_split(rows_splits(tiles, kblocks, work), kblocks, work);
  const int raw = FUSED ? (DT == kF32 ? 4 : 2) : 0;
  const dim3 grid((unsigned)(tiles * split.splits));
  // two workgroups a CU where the rows leave room beside the deep ring, else beside the short one
  const uint32_t deep = rows_lds(8, p.M, split.kblocks, raw).end, flat = rows_lds(4, p.M, split.kblocks, raw).end;
  if (deep <= kTwoPerCu || flat > kTwoPerCu)
    fp8_few_rows_kernel<DT, FUSED, 8><<<grid, dim3(256), deep, s>>>(p, x, x_stride, split, (int)tiles);
  else
    fp8_few_rows_kernel<DT, FUSED, 4><<<grid, dim3(256), flat, s>>>(p, x, x_stride, split, (int)tiles);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_t(const Fp8Operands& p, const Workspace& work, hipStream_t s) {
  const int kblocks = (p.K + 127) / 128;
  // (scales far apart: the tiles walk to them block by block)
  if (!p.g.offsets && few_rows(p) && (p.M - 1) * p.xs_row + (int64_t)kblocks * p.xs_block < (int64_t(1) << 29))
    return launch_few_rows<DT, false>(p, nullptr, 0, work, s);
  if (p.g.offsets) return launch_fp8_tile<DT>(grouped_tile(p), p, make_split(1, kblocks, work), s);
  const Choice c = choose(p.M, p.N, p.K, work);
  return launch_fp8_tile<DT>(c.tile, p, make_split(c.splits, kblocks, work), s);
}

}  // namespace

bool fp8_tile_known(int bm, int bn) {
#define FP8_KNOWN(BM, BN, WM, WN, STAGES, PER_CU, SLOTS) \
  if (bm == BM && bn == BN) return true;
  FP8_TILES(FP8_KNOWN)
#undef FP8_KNOWN
  return false;
}

hipError_t launch_fp8_gemm(const Fp8Operands& p, int out_dtype, hipStream_t stream, const Workspace& work) {
  switch (out_dtype) {
    case kF32: return launch_t<kF32>(p, work, stream);
    case kF16: return launch_t<kF16>(p, work, stream);
    default: return launch_t<kBF16>(p, work, stream);
  }
}

bool fp8_fused(const void* x, int dtype, int64_t M, int64_t N, int64_t K, int64_t x_stride) {
  const int64_t es = dtype == kF32 ? 4 : 2;
  return few_rows_shape(M, N) && M * K * es <= (M == 1 ? kFusedRowBytes : kFusedBytes) &&
         K * es % 16 == 0 && ((uintptr_t)x & 15) == 0 &&
         (M == 1 || (x_stride * es % 16 == 0 && x_stride < (int64_t(1) << 24)));
}

hipError_t launch_fp8_fused(const Fp8Operands& p, const void* x, int64_t x_stride, int dtype, hipStream_t stream,
                            const Workspace& work) {
  switch (dtype) {
    case kF32: return launch_few_rows<kF32, true>(p, x, x_stride, work, stream);
    case kF16: return launch_few_rows<kF16, true>(p, x, x_stride, work, stream);
    default: return launch_few_rows<kBF16, true>(p, x, x_stride, work, stream);
  }
}

static int64_t fp8_tile_workspace_bytes(int64_t M, int64_t N, int64_t K, const Workspace& all) {
  const Choice c = choose(M, N, K, all);
  if (c.tile == 0 || c.splits <= 1) return 0;
  const int64_t bm = c.tile & 1023, bn = c.tile >> 10, tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
  return (int64_t)kW8a8PartialOffset + tiles * c.splits * bm * bn * 4;
}

int64_t fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  const Workspace all{(uint8_t*)256, kSkWorkspaceBytes};  // never read here
  if (few_rows_shape(M, N)) {
    // the few-row kernel, if it takes the product (the tiles may need more: the larger of both)
    const int64_t tiles = (N + kRowsN - 1) / kRowsN, splits = rows_splits(tiles, (int)((K + 127) / 128), all);
    const int64_t rows = splits > 1 ? (int64_t)kW8a8PartialOffset + tiles * splits * 4096 : 0;
    return std::max(rows, fp8_tile_workspace_bytes(M, N, K, all));
  }
  return fp8_tile_workspace_bytes(M, N, K, all);
}

}  // namespace convrot
