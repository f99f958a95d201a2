// Products of e4m3 codes with a float32 scale for each block of 128, for gfx950:
//
//   out[m][n] = dt( sum_b (xs[m][b] ws[n / 128][b]) * (sum_{k in block b} act[m][k] w[n][k]) + bias[n] )
//
// with an optional gated residual in float32 before the one rounding, for rows of one
// weight, and for rows grouped by expert (fp8_device.h), sorted or read through an index.
//
// The codes of one block go through one MFMA of K = 128 (v_mfma_f32_16x16x128_f8f6f4,
// from zero); its 4 results a lane are multiplied by their scales and added in float32
// by the vector unit (4 FMAs of 4 cycles beside 32 cycles of the MFMA: hidden while two
// waves share a SIMD).  So the sums of different blocks are added at float32, and the
// scales may be any numbers.
//
// What the FP8 form keeps of a sum: the 16 products of features 16 i .. 16 i + 15 are
// aligned to the largest of them and lose what lies more than 13 bits below its leading
// one (measured with single products; sums of different sixteens are float32's own), up
// to 15 * 2^-13 of the largest product, 1.5e-5 of a sum of normal values: a sixteenth of
// float16's own rounding.  Float32 outputs get their products added at float32 instead,
// on bf16 MFMAs (codes are exact in bf16), at half the rate: 8800 x 8192 -> 4096 from codes
// 604 us, bfloat16 outputs 291.
//
// Operands: codes row-major, rows of 16-byte aligned strides that cover K rounded up to
// 16, zeros from K on.  Each 1 KB piece of a block (8 rows x 128 bytes: whole cache
// lines) goes by one wave instruction straight into an LDS ring of STAGES blocks; the
// 16-byte chunks of a row are permuted by its row number, so that the fragment reads (16
// rows x 16 bytes) meet no bank twice.  Beside the codes of a block lie the scales of its
// rows; the weights' scales of all blocks lie in LDS from the start.
#pragma once

#include <type_traits>

#include "convrot_launch.h"
#include "gemm_groups.h"
#include "gemm_w8a8_tile.h"

namespace convrot {
namespace {

constexpr int kMaxBlocks = 512;  // K up to 65536

template <int BM, int BN, int WM, int WN, int STAGES, int PER_CU, bool IN_SLOTS>
struct Fp8Engine {
  static constexpr int NW = WM * WN, THREADS = NW * 64;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr int APW = BM / 8 / NW, BPW = BN / 8 / NW, LPW = APW + BPW + 1;  // DMAs a wave and block
  static constexpr int XS_OFF = (BM + BN) * 128, STAGE_BYTES = XS_OFF + NW * 256;
  static constexpr int RING = STAGES * STAGE_BYTES, STAGING = NW * TM * (TN * 2 + 16);  // 16-bit epilogue
  // weights' scales of the tile's blocks of outputs (WS of them: the tile lies in one, or covers two)
  static constexpr int WS = BN > kBlock ? BN / kBlock : 1;
  static constexpr int WS_OFF = RING > STAGING ? RING : STAGING;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM <= NW * 64, "whole pieces a wave");
  static_assert(kBlock % TN == 0 && (BN % kBlock == 0 || kBlock % BN == 0), "a wave's corner under one scale");
  static_assert((STAGES - 1) * LPW <= 63, "vmcnt counts at most 63 DMAs");
  static constexpr int smem_bytes(int blocks) { return WS_OFF + WS * ((blocks * 4 + 255) / 256 * 256); }

  uint8_t* smem;
  uint32_t smem_addr;
  int lane, wave, wm, wn;
  i32x4_sgpr ra, rw;
  uint32_t va[APW], vw[BPW], vx;
  bool past_a[2], past_w[2];  // lane's chunk of the last block lies past the row's end, in even and odd pieces
  uint32_t tail;              // the block that rows end in, ~0 where they fill it
  const float* xs_base;
  int64_t xs_block;
  uint32_t xs_bytes;

  __device__ __forceinline__ explicit Fp8Engine(uint8_t* s) : smem(s) {
    smem_addr = (uint32_t)(uintptr_t)s;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / WN;
    wn = wave % WN;
  }

  // Sorted row m's row of the activations, -1 for none.
  __device__ __forceinline__ static int64_t source(const Fp8Operands& p, int m, int row_end) {
    if (m >= row_end) return -1;
    const int i = p.g.index[m];
    const uint32_t t = (uint32_t)i / (uint32_t)p.g.choices;
    return i < 0 || t >= p.g.act_rows ? -1 : (int64_t)t;
  }

  template <bool GATHER>
  __device__ __forceinline__ void set_tile(const Fp8Operands& p, int expert, int m0, int row_end, int n0) {
    const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u, rest = k16 & 127u;
    tail = rest ? k16 >> 7 : ~0u;
    const int mrows = min(BM, row_end - m0), nrows = min(BN, p.N - n0);
    const int rl = lane >> 3, c = lane & 7;
    rw = dma_rsrc(p.weight + (int64_t)expert * p.weight_expert + (int64_t)n0 * p.ldw,
                     (uint32_t)(nrows - 1) * (uint32_t)p.ldw + k16);
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const int piece = wave * BPW + i;
      vw[i] = (uint32_t)(8 * piece + rl) * (uint32_t)p.ldw + 16u * (uint32_t)(c ^ rl ^ (piece & 1));
    }
    xs_block = p.xs_block;
    const int xr = wave * 64 + lane;  // the row whose scale this lane moves
    if constexpr (GATHER) {
      ra = dma_rsrc(p.act, (uint32_t)((p.g.act_rows - 1) * p.lda) + k16);
#pragma unroll
      for (int i = 0; i < APW; ++i) {
        const int piece = wave * APW + i;
        const int64_t t = source(p, m0 + 8 * piece + rl, row_end);
        va[i] = t < 0 ? kPastEnd : (uint32_t)(t * p.lda) + 16u * (uint32_t)(c ^ rl ^ (piece & 1));
      }
      const int64_t t = xr < BM ? source(p, m0 + xr, row_end) : -1;
      vx = t < 0 ? kPastEnd : (uint32_t)(t * p.xs_row) * 4u;
      xs_base = p.xscales;
      xs_bytes = (uint32_t)((p.g.act_rows - 1) * p.xs_row) * 4u + 4u;
    } else {
      ra = dma_rsrc(p.act + (int64_t)m0 * p.lda, (uint32_t)(mrows - 1) * (uint32_t)p.lda + k16);
#pragma unroll
      for (int i = 0; i < APW; ++i) {
        const int piece = wave * APW + i;
        va[i] = 8 * piece + rl < mrows
                    ? (uint32_t)(8 * piece + rl) * (uint32_t)p.lda + 16u * (uint32_t)(c ^ rl ^ (piece & 1))
                    : kPastEnd;
      }
      vx = xr < mrows ? (uint32_t)xr * (uint32_t)p.xs_row * 4u : kPastEnd;
      xs_base = p.xscales + (int64_t)m0 * p.xs_row;
      xs_bytes = (uint32_t)(mrows - 1) * (uint32_t)p.xs_row * 4u + 4u;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      past_a[e] = 16u * (uint32_t)(c ^ rl ^ ((wave * APW + e) & 1)) >= rest;
      past_w[e] = 16u * (uint32_t)(c ^ rl ^ ((wave * BPW + e) & 1)) >= rest;
    }
  }

  // The weights' scales of the tile into LDS, block b of output block j at float j * stride + b.
  __device__ __forceinline__ void issue_ws(const Fp8Operands& p, int expert, int n0) const {
    const int blocks = (p.K + kBlock - 1) / kBlock, pieces = (blocks + 63) / 64;
    const int nb = min(WS, (p.N + kBlock - 1) / kBlock - n0 / kBlock);
    const float* base = p.wscales + (int64_t)expert * p.ws_expert + (int64_t)(n0 / kBlock) * p.ws_row;
    for (int d = wave; d < nb * pieces; d += NW) {
      const int j = d / pieces, at = d - j * pieces;
      dma4(dma_rsrc(base + j * p.ws_row, (uint32_t)blocks * 4u), (uint32_t)(at * 256 + lane * 4),
           smem_addr + (uint32_t)(WS_OFF + d * 256));
    }
  }

  __device__ __forceinline__ void issue(uint32_t kb, int stage) const {
    const uint32_t base = smem_addr + (uint32_t)(stage * STAGE_BYTES), k = kb * 128u;
    const bool last = kb == tail;
#pragma unroll
    for (int i = 0; i < APW; ++i) {
      uint32_t off = va[i] == kPastEnd ? kPastEnd : va[i] + k;
      if (last) off = past_a[i & 1] ? kPastEnd : off;
      dma16(ra, off, base + (uint32_t)(wave * APW + i) * 1024u);
    }
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      uint32_t off = vw[i] + k;
      if (last) off = past_w[i & 1] ? kPastEnd : off;
      dma16(rw, off, base + (uint32_t)BM * 128u + (uint32_t)(wave * BPW + i) * 1024u);
    }
    dma4(dma_rsrc(xs_base + (int64_t)kb * xs_block, xs_bytes), vx, base + (uint32_t)XS_OFF + (uint32_t)wave * 256u);
  }

  __device__ __forceinline__ i32x8 fragment(const uint8_t* row) const {
    const int r = lane & 15, q = lane >> 4, sw = chunk_swizzle(r);
    const i32x4 lo = *(const i32x4*)(row + ((2 * q) ^ sw) * 16), hi = *(const i32x4*)(row + ((2 * q + 1) ^ sw) * 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  __device__ __forceinline__ i32x8 a_fragment(int stage, int fm) const {
    return fragment(smem + stage * STAGE_BYTES + (wm * TM + fm * 16 + (lane & 15)) * 128);
  }
  __device__ __forceinline__ i32x8 w_fragment(int stage, int fn) const {
    return fragment(smem + stage * STAGE_BYTES + BM * 128 + (wn * TN + fn * 16 + (lane & 15)) * 128);
  }
  // The scale of the lane's row of fragment fm.
  __device__ __forceinline__ float xscale(int stage, int fm) const {
    return *(const float*)(smem + stage * STAGE_BYTES + XS_OFF + (wm * TM + fm * 16 + (lane & 15)) * 4);
  }

  // acc += the scaled products of one block.  WIDE (float32 outputs): on bf16 MFMAs, whose sums are float32's own.
  template <bool WIDE>
  __device__ __forceinline__ void block(int stage, float ws, f32x4 (&acc)[FN][FM]) const {
    using Frag = std::conditional_t<WIDE, WideCodes, i32x8>;
    const auto as = [](const i32x8& c) __attribute__((always_inline)) {
      if constexpr (WIDE) return widen_codes(c);
      else return c;
    };
    Frag a[FM];
    float s[FM];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      a[fm] = as(a_fragment(stage, fm));
      s[fm] = xscale(stage, fm) * ws;
    }
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) {
      const Frag w = as(w_fragment(stage, fn));
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        f32x4 part = zero;
        if constexpr (WIDE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a[fm].v[i], part, 0, 0, 0);
        } else {
          part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a[fm], zero, 0, 0, 0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[fn][fm][j] = __builtin_fmaf(part[j], s[fm], acc[fn][fm][j]);
      }
    }
  }

  template <bool WIDE>
  __device__ __forceinline__ void run_blocks(uint32_t kb0, int n, const float* ws, f32x4 (&acc)[FN][FM]) const {
    const uint32_t last = kb0 + (uint32_t)n - 1;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(min(kb0 + s, last), s);
    int st = 0;
    for (uint32_t kb = kb0; kb <= last; ++kb) {
      wait_vmcnt<(STAGES - 2) * LPW>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave is done with the stage before
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      // into the stage that every wave is done with (past the last block: the last one again)
      issue(min(kb + STAGES - 1, last), st == 0 ? STAGES - 1 : st - 1);
      block<WIDE>(st, ws[kb], acc);
      st = st + 1 == STAGES ? 0 : st + 1;
    }
  }

  // The same for 16-bit outputs, with the instructions in an order of their own.  Slot (fn, fm) of a block is an MFMA, and beside it the FMAs of the MFMA LAG slots
  // before, whose results are there by then, and a fragment read: of the next fn's weights, and in the last
  // fn of the next block's activations, each into the registers that its slot has just used.  Before that
  // last fn the wave has read all of its block: a barrier there frees the block's stage, which the DMA of
  // block kb + STAGES fills, and publishes block kb + 1.  (Left to the compiler's order, every MFMA is waited for by
  // its FMAs, and the other waves of the SIMD have to fill the gap: with two of them, of 256 x 256 tiles, they
  // do not.)
  __device__ __forceinline__ void run_slots(uint32_t kb0, int n, const float* ws, f32x4 (&acc)[FN][FM]) const {
    constexpr int LAG = FM - 1, SLOTS = FN * FM;
    static_assert(LAG > 0, "an MFMA is not followed by its own FMAs");
    const uint32_t last = kb0 + (uint32_t)n - 1;
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(min(kb0 + s, last), s);
    wait_vmcnt<(STAGES - 1) * LPW>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    i32x8 a[FM], w[2];
    float xs[FM], s[FM], wsv = ws[kb0];
    f32x4 part[FM];
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    w[0] = w_fragment(0, 0);
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      a[fm] = a_fragment(0, fm);
      xs[fm] = xscale(0, fm);
      s[fm] = 0.0f;
      part[fm] = zero;
    }
    int st = 0;
    for (uint32_t kb = kb0; kb <= last; ++kb) {
      const int nst = st + 1 == STAGES ? 0 : st + 1;
      // weights of fn = 0 lie in w[0] at the start of a block, so an odd FN would need them to change places
      static_assert(FN == 1 || FN % 2 == 0, "fragments in turn");
      static_for<SLOTS>([&](auto slot) __attribute__((always_inline)) {
        constexpr int t = slot.value, fn = t / FM, fm = t % FM;
        if constexpr (fn == FN - 1 && fm == 0) {
          wait_vmcnt<(STAGES - 2) * LPW>();
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          // past the last block: the last one again, into stages nothing reads
          issue(min(kb + STAGES, last), st);
        }
        if constexpr (fm == 0 && FN > 1) w[(fn + 1) & 1] = fn + 1 < FN ? w_fragment(st, fn + 1) : w_fragment(nst, 0);
        const f32x4 now = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[FN > 1 ? fn & 1 : 0], a[fm], zero, 0, 0, 0, 0, 0, 0);
        // the MFMA of LAG slots before (of the block before, in the first ones)
        constexpr int of = (fm + FM - LAG) % FM, on = t >= LAG ? (t - LAG) / FM : FN - 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[on][of][j] = __builtin_fmaf(part[of][j], s[of], acc[on][of][j]);
        if constexpr (fn == 0) {
          if constexpr (fm < LAG) s[of] = xs[of] * wsv;
          if constexpr (fm == 0) s[0] = xs[0] * wsv;
        }
        part[fm] = now;
        if constexpr (fn == FN - 1) {
          if constexpr (fm == 0) wsv = ws[min(kb + 1, last)];
          a[fm] = a_fragment(nst, fm);
          xs[fm] = xscale(nst, fm);
          if constexpr (FN == 1 && fm == FM - 1) w[0] = w_fragment(nst, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      st = nst;
    }
#pragma unroll
    for (int i = 0; i < LAG; ++i) {
      const int of = FM - LAG + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[FN - 1][of][j] = __builtin_fmaf(part[of][j], s[of], acc[FN - 1][of][j]);
    }
  }

  // acc += the products of blocks kb0 .. kb0 + n - 1, n >= 1.
  template <bool WIDE>
  __device__ __forceinline__ void run(uint32_t kb0, int n, int ws_stride, f32x4 (&acc)[FN][FM]) const {
    const float* ws = (const float*)(smem + WS_OFF) + (WS > 1 ? wn * TN / kBlock * ws_stride : 0);
    if constexpr (IN_SLOTS && !WIDE) run_slots(kb0, n, ws, acc);
    else run_blocks<WIDE>(kb0, n, ws, acc);
    wait_vmcnt<0>();  // the DMAs past the last block have landed before the ring is reused
  }
};

// Bias of outputs n .. n + 3 (0 without one, or past N).
__device__ __forceinline__ void load_bias4(const Fp8Operands& p, int n, float (&b)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = p.bias && n + j < p.N ? p.bias[n + j] : 0.0f;
}

// The wave's corner of the tile: bias, gated residual, rounding, store; rows m0 .. row_end - 1.  16-bit
// outputs (and residuals) go through the wave's part of LDS in chunks of 16 bytes.
template <class E, int ODT>
__device__ __forceinline__ void fp8_epilogue16(const E& e, const f32x4 (&acc)[E::FN][E::FM], const Fp8Operands& p, int m0,
                                               int row_end, int n0) {
  constexpr int FM = E::FM, FN = E::FN, TM = E::TM, TN = E::TN, RS = TN * 2 + 16;
  const int lane = e.lane, mw = m0 + e.wm * TM, nw = n0 + e.wn * TN;
  uint8_t* region = e.smem + e.wave * (TM * RS);
  const bool residual = p.gr.residual != nullptr;
  const bool one_gate = residual && mw / p.gr.rows_per_gate == (min(mw + TM, row_end) - 1) / p.gr.rows_per_gate;
  if (residual) {
    move_rows<TM, TN, false, (FM * FN > 16 ? 4 : 16)>(region, (uint16_t*)p.gr.residual, lane, mw, nw, row_end, p.N);
    wave_lds_fence();
  }
  static_for<FN>([&](auto frag) __attribute__((always_inline)) {
    constexpr int fn = frag.value;
    const int nl = fn * 16 + 4 * (lane >> 4);
    float b[4], g[4];
    load_bias4(p, nw + nl, b);
    if (one_gate && mw < row_end) load_gate4<ODT>(p.gr, mw, nw + nl, p.N, g);
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = acc[fn][fm][r] + b[r];
      uint16_t* q = (uint16_t*)(region + (fm * 16 + (lane & 15)) * RS + nl * 2);
      if (residual) {
        const int m = mw + fm * 16 + (lane & 15);
        if (!one_gate && m < row_end) load_gate4<ODT>(p.gr, m, nw + nl, p.N, g);
        float res[4];
        load_elem4<ODT>(q, 0, res);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = res[r] + g[r] * o[r];
      }
      store_out4<ODT>(q, 0, o[0], o[1], o[2], o[3]);
    }
  });
  wave_lds_fence();
  move_rows<TM, TN, true>(region, (uint16_t*)p.out, lane, mw, nw, row_end, p.N);
}

template <class E>
__device__ __forceinline__ void fp8_epilogue32(const E& e, const f32x4 (&acc)[E::FN][E::FM], const Fp8Operands& p, int m0,
                                               int row_end, int n0) {
  const int lane = e.lane, mw = m0 + e.wm * E::TM, nw = n0 + e.wn * E::TN;
  const W8a8Operands q{nullptr, nullptr, 0, 0, nullptr, nullptr, nullptr, p.out, row_end, p.N, p.K, p.gr};
  static_for<E::FN>([&](auto frag) __attribute__((always_inline)) {
    constexpr int fn = frag.value;
    const int n = nw + fn * 16 + 4 * (lane >> 4);
    if (n >= p.N) return;
    float b[4];
    load_bias4(p, n, b);
#pragma unroll
    for (int fm = 0; fm < E::FM; ++fm) {
      const int m = mw + fm * 16 + (lane & 15);
      if (m >= row_end) continue;
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = acc[fn][fm][r] + b[r];
      store4<kF32>(q, m, n, (p.N & 3) == 0, o);
    }
  });
}

// Where a launch's t-th tile lies: tiles that one XCD (one L2) runs are neighbours, in groups of kGroupM tile rows.
struct TilePlace {
  int row, column;
};
__device__ __forceinline__ TilePlace place_of(int t, int tiles, int tiles_m, int tiles_n) {
  const int per_xcd = tiles / kXcds;
  if (t < per_xcd * kXcds) t = (t % kXcds) * per_xcd + t / kXcds;
  const int group = t / (kGroupM * tiles_n), first_m = group * kGroupM;
  const int group_rows = min(kGroupM, tiles_m - first_m), in_group = t - group * kGroupM * tiles_n;
  return {first_m + in_group % group_rows, in_group / group_rows};
}

// What the rows of a launch are. KIND 0: rows of one weight (their K may be shared between workgroups), 1: sorted rows of
// experts, 2: rows of experts read through the index.
template <int BM, int KIND>
__device__ __forceinline__ int tile_rows_of(const Fp8Operands& p, int tiles_m) {
  return KIND == 0 ? tiles_m : group_tile_rows<BM>(p.g, p.M);
}
template <int BM, int KIND>
__device__ __forceinline__ GroupTile rows_at(const Fp8Operands& p, int row) {
  return KIND == 0 ? GroupTile{0, row * BM, p.M} : group_tile<BM>(p.g, p.M, row);
}

template <class E, int ODT>
__device__ __forceinline__ void fp8_epilogue(const E& e, const f32x4 (&acc)[E::FN][E::FM], const Fp8Operands& p, int m0,
                                             int row_end, int n0) {
  __syncthreads();  // every wave is done with the ring before it stages outputs
  if constexpr (ODT == kF32) fp8_epilogue32<E>(e, acc, p, m0, row_end, n0);
  else fp8_epilogue16<E, ODT>(e, acc, p, m0, row_end, n0);
}

template <class E>
__device__ __forceinline__ void clear(f32x4 (&acc)[E::FN][E::FM]) {
#pragma unroll
  for (int a = 0; a < E::FN; ++a)
#pragma unroll
    for (int b = 0; b < E::FM; ++b) acc[a][b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
}

// A whole tile: rows m0 .. (m0 + BM or) row_end - 1 of an expert, outputs n0 ..
template <class E, int ODT, int KIND>
__device__ __forceinline__ void fp8_tile(uint8_t* smem, const Fp8Operands& p, int expert, int m0, int row_end, int n0) {
  E e(smem);
  f32x4 acc[E::FN][E::FM];
  clear<E>(acc);
  const int kblocks = (p.K + kBlock - 1) / kBlock;
  if (KIND == 0 || expert < p.g.experts) {
    e.issue_ws(p, expert, n0);
    e.template set_tile<KIND == 2>(p, expert, m0, row_end, n0);
    e.template run<ODT == kF32>(0, kblocks, (kblocks + 63) / 64 * 64, acc);
  }
  fp8_epilogue<E, ODT>(e, acc, p, m0, row_end, n0);
}

// Tiles of 256 x 256.  The last round of them, of `slots` workgroups, runs as halves or quarters while that
// gives each CU at most one: 8800 x 8192 -> 4096 (560 tiles, 48 past two rounds) 272 us, with whole ones 313 to 318.
// Alone on their CUs the parts take deeper rings, and their MFMAs run in slots: 1536 x 15360 -> 5120 (120 tiles, as
// halves) 130 us (1860 TFLOP/s), with rings of 2 and no slots 148, with either 146 and 141; 1536 x 4096 -> 2560 (60,
// as quarters) 23.8 and 25.5.
struct LargeTiles {
  using Whole = Fp8Engine<256, 256, 4, 2, 2, 1, true>;
  using Half = Fp8Engine<256, 128, 4, 2, 3, 1, true>;
  using Quarter = Fp8Engine<128, 128, 2, 4, 4, 1, true>;
  static constexpr int smem_bytes(int blocks) {
    const int w = Whole::smem_bytes(blocks), h = Half::smem_bytes(blocks), q = Quarter::smem_bytes(blocks);
    return w > h ? (w > q ? w : q) : (h > q ? h : q);
  }
  static_assert(Half::THREADS == Whole::THREADS && Quarter::THREADS == Whole::THREADS, "one launch");
};

template <int ODT, int KIND>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_large_kernel(Fp8Operands p,
                                                                                                 int tiles_m,
                                                                                                 int tiles_n, int slots) {
  using E = LargeTiles::Whole;
  using Half = LargeTiles::Half;
  using Quarter = LargeTiles::Quarter;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  tiles_m = tile_rows_of<256, KIND>(p, tiles_m);
  const int tiles = tiles_m * tiles_n;
  const LastRound last = last_round(tiles, slots);
  const int t = blockIdx.x;
  if (t < last.whole) {
    const TilePlace at = place_of(t, last.whole, tiles_m, tiles_n);
    const GroupTile r = rows_at<256, KIND>(p, at.row);
    if (r.expert < 0) return;
    fp8_tile<E, ODT, KIND>(smem, p, r.expert, r.row0, r.row_end, at.column * 256);
    return;
  }
  const int u = t - last.whole, tile = last.whole + u / last.parts, part = u % last.parts;
  if (tile >= tiles) return;
  // in the order of the whole ones, without the XCDs' turns
  const int group = tile / (kGroupM * tiles_n), first_m = group * kGroupM;
  const int group_rows = min(kGroupM, tiles_m - first_m), in_group = tile - group * kGroupM * tiles_n;
  const GroupTile r = rows_at<256, KIND>(p, first_m + in_group % group_rows);
  if (r.expert < 0) return;
  const int n0 = in_group / group_rows * 256 + (part & 1) * 128, m0 = r.row0 + (part >> 1) * 128;
  if (n0 >= p.N || m0 >= r.row_end) return;
  if (last.parts == 2) fp8_tile<Half, ODT, KIND>(smem, p, r.expert, m0, r.row_end, n0);
  else fp8_tile<Quarter, ODT, KIND>(smem, p, r.expert, m0, r.row_end, n0);
}

template <int BM, int BN, int WM, int WN, int STAGES, int PER_CU, bool IN_SLOTS, int ODT, int KIND>
__global__ __launch_bounds__(WM* WN * 64) __attribute__((amdgpu_waves_per_eu(PER_CU* WM* WN / 4, PER_CU* WM* WN / 4)))
void fp8_tile_kernel(Fp8Operands p, int tiles_m, int tiles_n, W8a8Split split) {
  using E = Fp8Engine<BM, BN, WM, WN, STAGES, PER_CU, IN_SLOTS>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  tiles_m = tile_rows_of<BM, KIND>(p, tiles_m);
  const int tiles = tiles_m * tiles_n;
  const int part = KIND == 0 && split.splits > 1 ? blockIdx.x / tiles : 0, t = blockIdx.x - part * tiles;
  if (KIND != 0 && t >= tiles) return;
  const TilePlace at = place_of(t, tiles, tiles_m, tiles_n);
  const GroupTile r = rows_at<BM, KIND>(p, at.row);
  if (r.expert < 0) return;
  const int n0 = at.column * BN;
  if constexpr (KIND != 0) {
    fp8_tile<E, ODT, KIND>(smem, p, r.expert, r.row0, r.row_end, n0);
  } else {
    E e(smem);
    f32x4 acc[E::FN][E::FM];
    clear<E>(acc);
    const int kblocks = (p.K + kBlock - 1) / kBlock, kb0 = part * split.kblocks;
    e.issue_ws(p, 0, n0);
    e.template set_tile<false>(p, 0, r.row0, r.row_end, n0);
    e.template run<ODT == kF32>((uint32_t)kb0, min(split.kblocks, kblocks - kb0), (kblocks + 63) / 64 * 64, acc);
    if (split.splits > 1) {
      // partials [tile][part][fragment][thread], added in the parts' order by the last workgroup to arrive
      __shared__ int last;
      constexpr uint32_t BYTES = BM * BN * 4, STEP = E::THREADS * 16u;
      const int slot = at.row * tiles_n + at.column;
      const __amdgpu_buffer_rsrc_t rp =
          partial_rsrc(split.partials + (size_t)slot * split.splits * BYTES, (uint32_t)split.splits * BYTES);
      const uint32_t mine = threadIdx.x * 16u;
      static_for<E::FN>([&](auto fn) __attribute__((always_inline)) {
#pragma unroll
        for (int fm = 0; fm < E::FM; ++fm)
          store_partial(rp, (uint32_t)part * BYTES + (uint32_t)(fn.value * E::FM + fm) * STEP + mine,
                        __builtin_bit_cast(i32x4, acc[fn.value][fm]));
      });
      if (!last_to_arrive(split.counters + slot, split.splits, &last)) return;
      clear<E>(acc);
      for (int q = 0; q < split.splits; ++q)
        static_for<E::FN>([&](auto fn) __attribute__((always_inline)) {
#pragma unroll
          for (int fm = 0; fm < E::FM; ++fm)
            acc[fn.value][fm] += __builtin_bit_cast(
                f32x4, load_partial(rp, (uint32_t)q * BYTES + (uint32_t)(fn.value * E::FM + fm) * STEP + mine));
        });
    }
    fp8_epilogue<E, ODT>(e, acc, p, r.row0, r.row_end, n0);
  }
}

template <int BM, int BN, int WM, int WN, int STAGES, int PER_CU, bool IN_SLOTS, int ODT, int KIND>
hipError_t launch_fp8_tile_k(const Fp8Operands& p, const W8a8Split& split, hipStream_t s) {
  using E = Fp8Engine<BM, BN, WM, WN, STAGES, PER_CU, IN_SLOTS>;
  static_assert(E::smem_bytes(kMaxBlocks) <= 160 * 1024 - 64, "LDS of one CU");
  const int64_t tm = KIND == 0 ? ((int64_t)p.M + BM - 1) / BM : most_tile_rows(p.M, p.g.experts, BM);
  const int64_t tn = ((int64_t)p.N + BN - 1) / BN;
  const size_t lds = (size_t)E::smem_bytes((p.K + kBlock - 1) / kBlock);
  if constexpr (BM == 256) {
    static_assert(LargeTiles::smem_bytes(kMaxBlocks) <= 160 * 1024 - 64, "LDS of one CU");
    const size_t most = (size_t)LargeTiles::smem_bytes((p.K + kBlock - 1) / kBlock);
    const int slots = device_cus();
    // (what experts make of the bound's tiles is known on the device alone)
    if (tm * tn > 0x7fff0000 || slots < 1) return hipErrorInvalidValue;
    const LastRound last = last_round((int)(tm * tn), slots);
    const int64_t groups = KIND == 0 ? last.whole + (tm * tn - last.whole) * last.parts : tm * tn + slots;
    if (groups > max_groups(E::THREADS)) return hipErrorInvalidValue;
    fp8_large_kernel<ODT, KIND><<<dim3((unsigned)groups), dim3(E::THREADS), most, s>>>(p, (int)tm, (int)tn, slots);
  } else {
    const int64_t groups = tm * tn * split.splits;
    if (groups > max_groups(E::THREADS) || groups > 0x7fffffff) return hipErrorInvalidValue;
    fp8_tile_kernel<BM, BN, WM, WN, STAGES, PER_CU, IN_SLOTS, ODT, KIND>
        <<<dim3((unsigned)groups), dim3(E::THREADS), lds, s>>>(p, (int)tm, (int)tn, split);
  }
  return hipGetLastError();
}

}  // namespace

template <int ODT>
hipError_t launch_fp8_tile(int tile, const Fp8Operands& p, const W8a8Split& split, hipStream_t stream) {
  switch (tile) {
#define FP8_CASE(BM, BN, WM, WN, STAGES, PER_CU, SLOTS)                                                         \
  case tile_code(BM, BN):                                                                                       \
    if (!p.g.offsets) return launch_fp8_tile_k<BM, BN, WM, WN, STAGES, PER_CU, SLOTS, ODT, 0>(p, split, stream);       \
    if (!p.g.index) return launch_fp8_tile_k<BM, BN, WM, WN, STAGES, PER_CU, SLOTS, ODT, 1>(p, split, stream);         \
    return launch_fp8_tile_k<BM, BN, WM, WN, STAGES, PER_CU, SLOTS, ODT, 2>(p, split, stream);
    FP8_TILES(FP8_CASE)
#undef FP8_CASE
    default: return hipErrorInvalidValue;
  }
}

}  // namespace convrot
