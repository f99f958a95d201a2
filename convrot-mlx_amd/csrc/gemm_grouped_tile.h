// Products of rows grouped by expert in 16 bits, for gfx950, and their gradients:
//
//   forward   out[s][n] = sum_k x[row(s)][k] w[e(s)][n][k]
//   rows      dx[s][k]  = sum_n dy[s][n] w[e(s)][n][k]
//   weights   dw[e][n][k] = sum over the rows s of expert e of dy[s][n] x[row(s)][k]
//
// on 16-bit MFMAs (float32 sums, one rounding).  All three are one tiled product
// C[i][j] = sum_c A[i][c] B[j][c]; what differs is which operand has its contracted index c
// along its rows in memory and which across them:
//
//   forward   A = x (along)    B = w (along)
//   rows      A = dy (along)   B = w (across: c is its row)
//   weights   A = dy (across)  B = x (across), c runs over the expert's rows
//
// Rows of x through the index: forward by the offsets of a tile's rows, in the weights' gradient by scalar loads of 16
// numbers a wave and block, a block ahead (4608 tokens of 2 choices, 8 experts, 4096 -> 2048, in a graph: 177 us, on
// gathered rows 160 and 25 for the gather, which also holds them in memory; eager calls 190 to 201, and 182 and 23).
//
// An operand "across" is loaded as it lies, 64 rows of c, and transposed on the way from LDS to
// the registers (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block and get its columns), so
// nothing is transposed in memory.
//
// A workgroup of 2 x 2 waves owns a BM x BN tile and walks c in blocks of 64 (128 bytes).  Each
// 1 KB piece of a block goes by one wave instruction straight into an LDS ring of STAGES blocks.
// In an operand along, the 16-byte chunks of a row are permuted by its row number (no bank
// twice among the 16 rows of a fragment read); in one across, the 32-byte units of a row of c
// are, by bits of c (no bank twice among the 4 rows of a transposing read).  Per block, two
// k-steps of 32: the MFMAs of the first run beside the fragment reads of the second, those
// of the second beside the reads of the next block's first and the DMA of the block after.
#pragma once

#include "convrot_launch.h"
#include "gemm_groups.h"
#include "gemm_w8a8_tile.h"

namespace convrot {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ void mfma_16(f32x4& c, const i32x4& b, const i32x4& a) {
  if constexpr (DT == kBF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a) : "memory");
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a) : "memory");
}

template <int FN, int FM>
__device__ __forceinline__ void mfma_drain(f32x4 (&acc)[FN][FM]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int fn = 0; fn < FN; ++fn)
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) asm volatile("" : "+a"(acc[fn][fm]));
}

struct RowNumbers {
  int v[16];
};

// One operand of a tile of T rows (or, across, columns) by the workgroup's 4 waves.  GATHER: across, its rows of c
// read through an index.
template <int T, bool ACROSS, bool GATHER = false>
struct Side {
  static_assert(ACROSS || !GATHER, "rows along are gathered by their offsets");
  typedef const __attribute__((address_space(4))) int* Index;  // scalar loads
  static constexpr int PW = T / 32;             // 1 KB pieces a wave and block
  static constexpr int ROW = ACROSS ? T * 2 : 128;  // bytes of an LDS row
  static constexpr int RPP = 1024 / ROW, CPR = ROW / 16;  // rows a piece, chunks a row
  static_assert(!GATHER || PW * RPP == 16, "16 rows of c a wave");
  static_assert(T % 32 == 0 && (!ACROSS || (T & (T - 1)) == 0), "tile");

  const uint16_t* base;
  int64_t step;      // elements to the next block
  uint32_t bytes;    // of the buffer from base (along), of a row's columns (across)
  uint32_t row_bytes;
  uint32_t off[PW];
  bool past[2];      // along: the lane's chunk of the last block lies past the row's end
  uint32_t tail;     // along: the block that rows end in, ~0 where they fill it
  int count;         // length of c
  Index index;       // GATHER: of row 0 of c
  Divisor choices;
  uint32_t numbers;  // those below it name a row

  // Which unit of 32 bytes of a row of c lies at unit u.
  __device__ __forceinline__ static int unit_swizzle(int row) {
    return T >= 128 ? (row & 3) ^ (((row >> 4) & 1) << 2) : T == 64 ? row & 3 : row & 1;
  }

  // along: `rows` rows of `length` elements at p, ld apart
  __device__ __forceinline__ void set_along(const uint16_t* p, int64_t ld, int rows, int length, int lane, int wave) {
    base = p;
    step = 64;
    count = length;
    bytes = (uint32_t)(rows - 1) * (uint32_t)ld * 2u + whole(length);
    set_tail(length, lane, wave);
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int row = 8 * (wave * PW + i) + (lane >> 3);
      off[i] = row < rows ? (uint32_t)row * (uint32_t)ld * 2u + chunk(lane, wave * PW + i) : kPastEnd;
    }
  }
  // along, row r read from row source(r) of p (-1: none); `total` rows in all
  template <class F>
  __device__ __forceinline__ void set_gather(const uint16_t* p, int64_t ld, int64_t total, int length, int lane, int wave,
                                             F&& source) {
    base = p;
    step = 64;
    count = length;
    bytes = (uint32_t)((total - 1) * ld * 2) + whole(length);
    set_tail(length, lane, wave);
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int64_t t = source(8 * (wave * PW + i) + (lane >> 3));
      off[i] = t < 0 ? kPastEnd : (uint32_t)(t * ld * 2) + chunk(lane, wave * PW + i);
    }
  }
  // across: `length` rows of c at p, ld apart, `columns` of them
  __device__ __forceinline__ void set_across(const uint16_t* p, int64_t ld, int columns, int length, int lane, int wave) {
    base = p;
    step = 64 * ld;
    count = length;
    bytes = whole(min(columns, T));
    row_bytes = (uint32_t)ld * 2u;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int row = (wave * PW + i) * RPP + lane / CPR, c = lane % CPR;
      const uint32_t at = (uint32_t)((((c >> 1) ^ unit_swizzle(row)) * 2 + (c & 1)) * 16);
      off[i] = at < bytes ? (uint32_t)row * row_bytes + at : kPastEnd;
    }
  }

  // the same, row c of it row index[c] / choices of the `total` rows at p
  __device__ __forceinline__ void set_gather_across(const uint16_t* p, int64_t ld, int columns, int length, int lane,
                                                    int wave, const int* rows, const Divisor& d, int each, int64_t total) {
    base = p;
    count = length;
    index = (Index)(uintptr_t)rows;
    choices = d;
    numbers = (uint32_t)min(total * each, (int64_t)1 << 31);
    row_bytes = (uint32_t)ld * 2u;
    const uint32_t width = whole(min(columns, T));
    bytes = (uint32_t)(total - 1) * row_bytes + width;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int row = (wave * PW + i) * RPP + lane / CPR, c = lane % CPR;
      const uint32_t at = (uint32_t)((((c >> 1) ^ unit_swizzle(row)) * 2 + (c & 1)) * 16);
      off[i] = at < width ? at : kPastEnd;
    }
  }
  // GATHER: the index of the wave's 16 rows of block kb, -1 past the last one.
  __device__ __forceinline__ RowNumbers fetch(uint32_t kb, int wave) const {
    RowNumbers o{};
    if constexpr (GATHER) {
      const int c0 = (int)kb * 64 + wave * 16;
      if (c0 + 16 <= count) {
#pragma unroll
        for (int j = 0; j < 16; ++j) o.v[j] = index[c0 + j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) o.v[j] = c0 + j < count ? index[min(c0 + j, count - 1)] : -1;
      }
    }
    return o;
  }
  // The offset of a row from its number in the index.
  __device__ __forceinline__ uint32_t row_offset(int n) const {
    const uint32_t o = choices.divide((uint32_t)n) * row_bytes;
    return __builtin_amdgcn_readfirstlane((uint32_t)n < numbers ? o : kNoRow);
  }
  static constexpr uint32_t kNoRow = 0xfffff000u;  // with a column's offset still past every operand

  // bytes of `n` elements in whole chunks (rows are padded to them: a chunk cut by the range check would
  // lose elements of its last word)
  __device__ __forceinline__ static uint32_t whole(int n) { return ((uint32_t)n * 2u + 15u) & ~15u; }
  __device__ __forceinline__ static uint32_t chunk(int lane, int piece) {
    return 16u * (uint32_t)((lane & 7) ^ (lane >> 3) ^ (piece & 1));
  }
  __device__ __forceinline__ void set_tail(int length, int lane, int wave) {
    const uint32_t rest = (uint32_t)(length & 63) * 2u;
    tail = rest ? (uint32_t)(length >> 6) : ~0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) past[e] = chunk(lane, wave * PW + e) >= rest;
  }

  __device__ __forceinline__ i32x4_sgpr rsrc(uint32_t kb) const {
    if constexpr (GATHER) {
      return dma_rsrc(base, bytes);
    } else if constexpr (ACROSS) {
      const int left = min(64, count - (int)kb * 64);
      return dma_rsrc(base + (int64_t)kb * step, (uint32_t)(left - 1) * row_bytes + bytes);
    } else {
      return dma_rsrc(base, bytes);
    }
  }
  __device__ __forceinline__ void issue(i32x4_sgpr r, uint32_t kb, int i, int wave, uint32_t lds,
                                        const RowNumbers& rows) const {
    uint32_t o = off[i];
    if constexpr (GATHER) {
      const int mine = (threadIdx.x & 63) / CPR;
      uint32_t row = row_offset(rows.v[i * RPP]);
#pragma unroll
      for (int j = 1; j < RPP; ++j) {
        const uint32_t other = row_offset(rows.v[i * RPP + j]);
        row = mine == j ? other : row;
      }
      o = o == kPastEnd ? kPastEnd : row + o;
    } else if constexpr (!ACROSS) {
      o = o == kPastEnd ? kPastEnd : o + kb * 128u;
      if (kb == tail) o = past[i & 1] ? kPastEnd : o;
    }
    dma16(r, o, lds + (uint32_t)(wave * PW + i) * 1024u);
  }

  // The address of this lane's part of fragment 0 of the wave's corner at `first`, k-step 0; of
  // fragment f and k-step ks: see fragment().
  __device__ __forceinline__ static uint32_t lane_address(int lane, int first) {
    if constexpr (ACROSS) {
      const int j = lane & 15, q = lane >> 4, row = 16 * q + (j >> 2);
      return (uint32_t)(row * ROW + ((first >> 4) ^ unit_swizzle(row)) * 32 + (j & 3) * 8);
    } else {
      const int r = lane & 15;
      return (uint32_t)((first + r) * 128 + (((2 * (lane >> 4)) ^ chunk_swizzle(r)) * 16));
    }
  }
  // Fragment f (16 rows or columns from the corner's 16 f on) of k-step ks: lane l has its row or column
  // l % 16 and the contracted 16 (l / 16) + 8 ks .. + 7.
  template <int F, int KS>
  __device__ __forceinline__ static i32x4 fragment(uint32_t at) {
    if constexpr (ACROSS) {
      // the corner begins at a multiple of its size, so f and the swizzle's bits lie apart from it
      const uint32_t a = (at ^ (uint32_t)(F * 32)) + (uint32_t)(KS * 8 * ROW);
      typedef __attribute__((address_space(3))) s16x4* P;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)(a + 4 * ROW));
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      typedef __attribute__((address_space(3))) i32x4* P;
      return *(P)(uintptr_t)((at ^ (uint32_t)(KS * 16)) + (uint32_t)(F * 2048));
    }
  }
};

template <int BM_, int BN_, int STAGES, int DT, bool ACROSS_A, bool ACROSS_B, bool GATHER_B = false>
struct Engine16 {
  static constexpr int BM = BM_, BN = BN_;
  using A = Side<BM, ACROSS_A>;
  using B = Side<BN, ACROSS_B, GATHER_B>;
  static constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16, LPW = A::PW + B::PW;
  static constexpr int STAGE_BYTES = (BM + BN) * 128, RING = STAGES * STAGE_BYTES;
  static constexpr int STAGING = 4 * TM * (TN * 2 + 16);  // the epilogue's
  static constexpr int SMEM_BYTES = RING > STAGING ? RING : STAGING;
  static constexpr int SLOTS = FM * FN, READS = FM + FN;
  static_assert(SMEM_BYTES <= 160 * 1024, "LDS of one CU");
  static_assert(STAGES >= 2 && (STAGES - 1) * LPW <= 63, "vmcnt counts at most 63 DMAs");
  static constexpr int SPAN0 = SLOTS * 3 / 4, SPAN1 = SLOTS * 7 / 8, SPAN_DMA = SLOTS / 2;
  static_assert(SPAN_DMA >= 1, "slots");

  uint8_t* smem;
  uint32_t smem_addr;
  int lane, wave, wm, wn;
  A a;
  B b;

  __device__ __forceinline__ explicit Engine16(uint8_t* s) : smem(s) {
    smem_addr = (uint32_t)(uintptr_t)s;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave >> 1;
    wn = wave & 1;
  }

  struct Rsrc {
    i32x4_sgpr a, b;
  };
  __device__ __forceinline__ Rsrc rsrc(uint32_t kb) const { return {a.rsrc(kb), b.rsrc(kb)}; }
  __device__ __forceinline__ void issue(const Rsrc& r, uint32_t kb, int stage, int idx, const RowNumbers& rows) const {
    const uint32_t base = smem_addr + (uint32_t)(stage * STAGE_BYTES);
    if (idx < A::PW) a.issue(r.a, kb, idx, wave, base, rows);
    else b.issue(r.b, kb, idx - A::PW, wave, base + (uint32_t)BM * 128u, rows);
  }

  // n fillers spread over the first `span` MFMA slots: those after slot t are filler(t) .. filler(t + 1) - 1.
  static constexpr int filler(int t, int n, int span) {
    return t >= span ? n : (t * n + span - 1) / span;
  }

  // acc += the products of blocks 0 .. n - 1, n >= 1.
  __device__ __forceinline__ void run(int n, f32x4 (&acc)[FN][FM]) {
    i32x4 b0[FN], a0[FM], b1[FN], a1[FM];
    const uint32_t last = (uint32_t)n - 1;
    const uint32_t la = A::lane_address(lane, wm * TM), lb = (uint32_t)BM * 128u + B::lane_address(lane, wn * TN);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      const uint32_t kb = min((uint32_t)s, last);
      const Rsrc r = rsrc(kb);
      const RowNumbers rows = b.fetch(kb, wave);
#pragma unroll
      for (int i = 0; i < LPW; ++i) issue(r, kb, s, i, rows);
    }
    // fragment i of a k-step, B's first (every MFMA of the first row needs them)
    auto read = [&](auto i, auto ks, uint32_t stage, i32x4(&bf)[FN], i32x4(&af)[FM]) __attribute__((always_inline)) {
      constexpr int I = decltype(i)::value, KS = decltype(ks)::value;
      if constexpr (I < FN) bf[I] = B::template fragment<I, KS>(stage + lb);
      else af[I - FN] = A::template fragment<I - FN, KS>(stage + la);
    };
    constexpr std::integral_constant<int, 0> K0{};
    constexpr std::integral_constant<int, 1> K1{};
    wait_vmcnt<(STAGES - 1) * LPW>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_for<READS>([&](auto i) __attribute__((always_inline)) { read(i, K0, smem_addr, b0, a0); });
    int st = 0;
    for (uint32_t kb = 0; kb <= last; ++kb) {
      const int nst = st + 1 == STAGES ? 0 : st + 1;
      RowNumbers rows = b.fetch(min(kb + STAGES, last), wave);  // arrives beside the first k-step
      const uint32_t here = smem_addr + (uint32_t)(st * STAGE_BYTES), next = smem_addr + (uint32_t)(nst * STAGE_BYTES);
      static_for<SLOTS>([&](auto slot) __attribute__((always_inline)) {
        constexpr int t = slot.value, lo = filler(t, READS, SPAN0), hi = filler(t + 1, READS, SPAN0);
        mfma_16<DT>(acc[t % FN][t / FN], b0[t % FN], a0[t / FN]);
        static_for<hi - lo>([&](auto f) __attribute__((always_inline)) {
          read(std::integral_constant<int, lo + f.value>{}, K1, here, b1, a1);
        });
      });
      wait_vmcnt<(STAGES - 2) * LPW>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      if constexpr (GATHER_B) {
#pragma unroll
        for (int j = 0; j < 16; ++j) asm volatile("" : "+s"(rows.v[j]));
      }
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      // past the last block: the last one again, into stages nothing reads
      const uint32_t nkb = min(kb + STAGES, last);
      const Rsrc r = rsrc(nkb);
      static_for<SLOTS>([&](auto slot) __attribute__((always_inline)) {
        constexpr int t = slot.value, lo = filler(t, READS, SPAN1), hi = filler(t + 1, READS, SPAN1);
        constexpr int dlo = filler(t, LPW, SPAN_DMA), dhi = filler(t + 1, LPW, SPAN_DMA);
        mfma_16<DT>(acc[t % FN][t / FN], b1[t % FN], a1[t / FN]);
        static_for<dhi - dlo>([&](auto f) __attribute__((always_inline)) { issue(r, nkb, st, dlo + f.value, rows); });
        static_for<hi - lo>([&](auto f) __attribute__((always_inline)) {
          read(std::integral_constant<int, lo + f.value>{}, K0, next, b0, a0);
        });
      });
      st = nst;
    }
    mfma_drain(acc);
    wait_vmcnt<0>();  // the DMAs past the last block have landed before the ring is reused
  }
};

// The wave's corner of the tile of a [.., N] array: rounded, then by its part of LDS in chunks of 16 bytes; rows
// below row_end.
template <class E, int DT>
__device__ __forceinline__ void store_tile(const E& e, const f32x4 (&acc)[E::FN][E::FM], void* out, int m0, int row_end,
                                           int n0, int N) {
  constexpr int FM = E::FM, FN = E::FN, TM = E::TM, TN = E::TN, RS = TN * 2 + 16;
  const int lane = e.lane, mw = m0 + e.wm * TM, nw = n0 + e.wn * TN;
  uint8_t* region = e.smem + e.wave * (TM * RS);
  static_for<FN>([&](auto frag) __attribute__((always_inline)) {
    constexpr int fn = frag.value;
    const int nl = fn * 16 + 4 * (lane >> 4);
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const f32x4 v = acc[fn][fm];
      store_out4<DT>((uint16_t*)(region + (fm * 16 + (lane & 15)) * RS + nl * 2), 0, v[0], v[1], v[2], v[3]);
    }
  });
  wave_lds_fence();
  move_rows<TM, TN, true>(region, (uint16_t*)out, lane, mw, nw, row_end, N);
}

// One tile: output rows m0 .. (m0 + BM or) row_end - 1, columns n0 .., of an expert (whose rows, with KIND 3 and 4, are
// the contracted ones).
template <class E, int DT, int KIND>
__device__ __forceinline__ void grouped_tile(uint8_t* smem, const GroupedOperands& p, int expert, int m0, int row_end,
                                             int n0) {
  E e(smem);
  f32x4 acc[E::FN][E::FM];
#pragma unroll
  for (int i = 0; i < E::FN; ++i)
#pragma unroll
    for (int j = 0; j < E::FM; ++j) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  int columns = p.N;
  uint16_t* out = p.out;
  if constexpr (KIND >= 3) {
    columns = p.C;
    out += (int64_t)expert * p.N * p.C;
    const int a = __builtin_amdgcn_readfirstlane(group_start(p.g, expert, p.R));
    const int b = __builtin_amdgcn_readfirstlane(group_start(p.g, expert + 1, p.R));
    if (b > a) {
      e.a.set_across(p.rows + (int64_t)a * p.ld_rows + m0, p.ld_rows, p.N - m0, b - a, e.lane, e.wave);
      if constexpr (KIND == 4)
        e.b.set_gather_across(p.other + n0, p.ld_other, p.C - n0, b - a, e.lane, e.wave, p.g.index + a, p.choices,
                              p.g.choices, p.g.act_rows);
      else
        e.b.set_across(p.other + (int64_t)a * p.ld_other + n0, p.ld_other, p.C - n0, b - a, e.lane, e.wave);
      e.run((b - a + 63) / 64, acc);
    }
  } else if (expert < p.g.experts) {
    const int rows = min(E::BM, row_end - m0);
    if constexpr (KIND == 1) {
      e.a.set_gather(p.rows, p.ld_rows, p.g.act_rows, p.C, e.lane, e.wave, [&](int r) __attribute__((always_inline)) {
        if (r >= rows) return (int64_t)-1;
        const int i = p.g.index[m0 + r];
        const uint32_t token = (uint32_t)i / (uint32_t)p.g.choices;
        return i < 0 || token >= p.g.act_rows ? (int64_t)-1 : (int64_t)token;
      });
    } else {
      e.a.set_along(p.rows + (int64_t)m0 * p.ld_rows, p.ld_rows, rows, p.C, e.lane, e.wave);
    }
    const uint16_t* w = p.other + expert * p.expert;
    if constexpr (KIND == 2) e.b.set_across(w + n0, p.ld_other, p.N - n0, p.C, e.lane, e.wave);
    else e.b.set_along(w + (int64_t)n0 * p.ld_other, p.ld_other, min(E::BN, p.N - n0), p.C, e.lane, e.wave);
    e.run((p.C + 63) / 64, acc);
  }
  __syncthreads();  // every wave is done with the ring before it stages outputs
  store_tile<E, DT>(e, acc, out, m0, row_end, n0, columns);
}

// Where the t-th tile of a launch lies.  The first `turns` of them go to the XCDs (and their L2s) in runs of
// neighbours.  Of rows: in groups of kGroupM tile rows; of the weights' gradient: one expert behind the other, each
// on all XCDs, as experts of many rows take longer.
template <int BM, int KIND>
__device__ __forceinline__ GroupTile grouped_place(const GroupedOperands& p, int t, int turns, int tiles_i, int tiles_j,
                                                   int* column) {
  if constexpr (KIND >= 3) {
    const int tiles = tiles_i * tiles_j, per_xcd = tiles / kXcds, expert = t / tiles;
    t -= expert * tiles;
    if (t < per_xcd * kXcds && (expert + 1) * tiles <= turns) t = (t % kXcds) * per_xcd + t / kXcds;
    *column = t % tiles_j;
    return {expert, t / tiles_j * BM, p.N};
  } else {
    const int per_xcd = turns / kXcds;
    if (t < per_xcd * kXcds) t = (t % kXcds) * per_xcd + t / kXcds;
    const int group = t / (kGroupM * tiles_j), first = group * kGroupM;
    const int group_rows = min(kGroupM, tiles_i - first), in_group = t - group * kGroupM * tiles_j;
    *column = in_group / group_rows;
    return group_tile<BM>(p.g, p.R, first + in_group % group_rows);
  }
}

template <int BM, int BN, int STAGES, int PER_CU, int DT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_CU, PER_CU))) void grouped_kernel(
    GroupedOperands p, int tiles_i, int tiles_j) {
  using E = Engine16<BM, BN, STAGES, DT, KIND >= 3, KIND >= 2, KIND == 4>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[E::SMEM_BYTES];
  if constexpr (KIND < 3) tiles_i = group_tile_rows<BM>(p.g, p.R);
  const int tiles = tiles_i * tiles_j * (KIND >= 3 ? p.g.experts : 1), t = blockIdx.x;
  if (t >= tiles) return;
  int column;
  const GroupTile at = grouped_place<BM, KIND>(p, t, tiles, tiles_i, tiles_j, &column);
  if (at.expert < 0) return;
  grouped_tile<E, DT, KIND>(smem, p, at.expert, at.row0, at.row_end, column * BN);
}

// Tiles of 256 x 256, the last round of them in halves or quarters (last_round of gemm_groups.h).
template <int DT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void grouped_large_kernel(GroupedOperands p,
                                                                                                     int tiles_i,
                                                                                                     int tiles_j,
                                                                                                     int slots) {
  constexpr bool AA = KIND >= 3, AB = KIND >= 2, GB = KIND == 4;
  using E = Engine16<256, 256, 2, DT, AA, AB, GB>;
  using Half = Engine16<256, 128, 3, DT, AA, AB, GB>;
  using Quarter = Engine16<128, 128, 4, DT, AA, AB, GB>;
  constexpr int PARTS = Half::SMEM_BYTES > Quarter::SMEM_BYTES ? Half::SMEM_BYTES : Quarter::SMEM_BYTES;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[E::SMEM_BYTES > PARTS ? E::SMEM_BYTES : PARTS];
  if constexpr (KIND < 3) tiles_i = group_tile_rows<256>(p.g, p.R);
  const int tiles = tiles_i * tiles_j * (KIND >= 3 ? p.g.experts : 1), t = blockIdx.x;
  const LastRound last = last_round(tiles, slots);
  int column;
  if (t < last.whole) {
    const GroupTile at = grouped_place<256, KIND>(p, t, last.whole, tiles_i, tiles_j, &column);
    if (at.expert < 0) return;
    grouped_tile<E, DT, KIND>(smem, p, at.expert, at.row0, at.row_end, column * 256);
    return;
  }
  const int u = t - last.whole, tile = last.whole + u / last.parts, part = u % last.parts;
  if (tile >= tiles) return;
  const GroupTile at = grouped_place<256, KIND>(p, tile, 0, tiles_i, tiles_j, &column);
  if (at.expert < 0) return;
  const int m0 = at.row0 + (part >> 1) * 128, n0 = column * 256 + (part & 1) * 128;
  if (m0 >= at.row_end || n0 >= (KIND >= 3 ? p.C : p.N)) return;
  if (last.parts == 2) grouped_tile<Half, DT, KIND>(smem, p, at.expert, m0, at.row_end, n0);
  else grouped_tile<Quarter, DT, KIND>(smem, p, at.expert, m0, at.row_end, n0);
}

template <int BM, int BN, int STAGES, int PER_CU, int DT, int KIND>
hipError_t launch_grouped_k(const GroupedOperands& p, hipStream_t s) {
  const int64_t ti = KIND >= 3 ? ((int64_t)p.N + BM - 1) / BM : most_tile_rows(p.R, p.g.experts, BM);
  const int64_t tj = ((int64_t)(KIND >= 3 ? p.C : p.N) + BN - 1) / BN;
  const int64_t tiles = ti * tj * (KIND >= 3 ? p.g.experts : 1), slots = device_cus();
  if (tiles > max_groups(256) - slots || tiles > 0x7fff0000 || slots < 1) return hipErrorInvalidValue;
  if constexpr (BM == 256) {
    // (what experts make of the bound's tiles is known on the device alone)
    const LastRound last = last_round((int)tiles, (int)slots);
    const int64_t groups = KIND >= 3 ? last.whole + (tiles - last.whole) * last.parts : tiles + slots;
    grouped_large_kernel<DT, KIND><<<dim3((unsigned)groups), dim3(256), 0, s>>>(p, (int)ti, (int)tj, (int)slots);
  } else {
    grouped_kernel<BM, BN, STAGES, PER_CU, DT, KIND><<<dim3((unsigned)tiles), dim3(256), 0, s>>>(p, (int)ti, (int)tj);
  }
  return hipGetLastError();
}

}  // namespace

template <int DT>
hipError_t launch_grouped_tile(int tile, int kind, const GroupedOperands& p, hipStream_t stream) {
  switch (tile << 3 | kind) {
#define GROUPED_CASE(BM, BN, STAGES, PER_CU, KIND) \
  case tile_code(BM, BN) << 3 | KIND: return launch_grouped_k<BM, BN, STAGES, PER_CU, DT, KIND>(p, stream);
#define GROUPED_ROWS(BM, BN, STAGES, PER_CU)                                              \
  GROUPED_CASE(BM, BN, STAGES, PER_CU, 0) GROUPED_CASE(BM, BN, STAGES, PER_CU, 1) \
  GROUPED_CASE(BM, BN, STAGES, PER_CU, 2)
#define GROUPED_WEIGHTS(BM, BN, STAGES, PER_CU) \
  GROUPED_CASE(BM, BN, STAGES, PER_CU, 3) GROUPED_CASE(BM, BN, STAGES, PER_CU, 4)
    GROUPED_TILES(GROUPED_ROWS)
    GROUPED_WEIGHT_TILES(GROUPED_WEIGHTS)
    default: return hipErrorInvalidValue;
  }
}

}  // namespace convrot
