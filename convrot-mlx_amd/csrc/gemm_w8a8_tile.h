// W8A8 GEMM for gfx950: 8-bit integer activations and weights, one scale a
// token and one an output channel, on INT8 MFMA with the epilogue fused.
//
//   out[m][n] = dt( (float(sum_k act[m][k] w[n][k]) * xs[m]) * ws[n] + bias[n] )
//
// The integer sum is exact (K <= 65536: |sum| <= 2^14 K = 2^30), so the order in
// which K is walked or split cannot change a bit.  An optional gated residual
// follows in float32 and is rounded once, dt(res[m][n] + gate[n] * that): the
// 4-bit linears round each of its operations, to give the bits of the array
// operations that they stand for.
//
// Operands: activations [M, K] and weights [N, K] as they are, row-major with
// row strides of a multiple of 16 bytes, so 8-bit checkpoints need no layout of
// their own.  Bytes of a weight row from K to the next multiple of 16 are zero;
// those of an activation row may be anything.
#pragma once

#include <utility>

#include "convrot_launch.h"
#include "w8a8_device.h"

namespace convrot {
namespace {

constexpr int kXcds = 8;  // workgroups are dispatched over 8 XCDs in turn
constexpr int kGroupM = 4;
// f(0), f(1), .. f(N - 1) with constants, straight-line whatever N is.
template <class F, int... I>
__device__ __forceinline__ void static_each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  static_each(f, std::make_integer_sequence<int, N>{});
}

// acc += w . a on the accumulator c, which stays in the AGPRs (as builtins the
// compiler copies accumulators around every MFMA of the loop).  The compiler
// does not see an MFMA here: operands come from LDS reads, which it waits for,
// and mfma_drain stands between the last MFMA and the first accumulator read.
__device__ __forceinline__ void mfma_i8(i32x4& c, const i32x4& w, const i32x4& a) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(w), "v"(a) : "memory");
}

template <int FN, int FM>
__device__ __forceinline__ void mfma_drain(i32x4 (&acc)[FN][FM]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int fn = 0; fn < FN; ++fn)
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) asm volatile("" : "+a"(acc[fn][fm]));
}

// ---- tiles
//
// A workgroup of 2 x 2 waves owns a BM x BN tile of the output and walks K in
// blocks of 128 bytes.  Each 1 KB piece of a block (8 rows x 128 bytes: whole
// cache lines) goes by one wave instruction straight into an LDS ring of STAGES
// blocks; the 16-byte chunks of a row are permuted by its row number, so that
// the fragment reads (16 rows x 16 bytes) meet no bank twice.
//
// Per block i (two k-steps of 64), the wave overlaps everything with its MFMAs:
//   k-step 0: MFMAs on (w0, a0); reads of the fragments w1, a1 of k-step 1;
//   middle:   block i+1 has landed, this wave's reads of block i are done; a
//             barrier publishes the one and frees the other's ring stage;
//   k-step 1: MFMAs on (w1, a1); DMA of block i+STAGES into the freed stage,
//             reads of block i+1's w0, a0.
// Both operands take a byte a value in LDS, so a wave's corner has to be large:
// of the LDS port's 128 bytes a clock, 128 x 128 corners (256 x 256 tile) take
// 64 for reads and 32 for the DMA's writes, 64 x 64 corners 128 and 64.
// Measured: 2048 x 8192 -> 8192 (256 tiles of 256 x 256) 104 us, 2.64 POPS; a
// k-block takes 1.2 to 1.4 us there with every CU busy, 3.0 to 3.4 POPS, which is
// what the chip's power sustains of this MFMA.  A tile adds 10 to 16 us to its
// k-blocks: first loads, scaling, and the outputs' write-back, which dominates
// short K (4608 x 128 -> 12288: 38 us for 113 MB).  With 192 x 128 tiles two
// workgroups share a CU and one's stores run beside the other's k-blocks, for
// more operand traffic: 4608 x 3072 -> 12288 165 us, with 256 x 224 165, 128 x 128 178.

template <int BM, int BN, int STAGES, bool LATE_EPI>
struct Engine {
  static constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16;
  static constexpr int APW = BM / 32, BPW = BN / 32, LPW = APW + BPW;  // 1 KB pieces a wave moves
  static constexpr int STAGE_BYTES = (BM + BN) * 128;
  static constexpr int STAGING = 4 * TM * (TN * 2 + 16);  // 16-bit epilogue
  // The epilogue's operands come with the first k-blocks, or (LATE_EPI, where two workgroups
  // fill the CU's LDS) after the last, behind the staged outputs in the ring.
  static constexpr int BASE = LATE_EPI ? STAGING : STAGES * STAGE_BYTES > STAGING ? STAGES * STAGE_BYTES : STAGING;
  // xs, ws, bias of the tile, in 256-byte DMAs
  static constexpr int XS_DMAS = (BM * 4 + 255) / 256, WS_DMAS = (BN * 4 + 255) / 256;
  static constexpr int XS_OFF = BASE, WS_OFF = XS_OFF + XS_DMAS * 256, BIAS_OFF = WS_OFF + WS_DMAS * 256;
  static constexpr int EPI_END = BIAS_OFF + WS_DMAS * 256;
  static constexpr int SMEM_BYTES = EPI_END > STAGES * STAGE_BYTES ? EPI_END : STAGES * STAGE_BYTES;
  static constexpr int SLOTS = FM * FN, READS = FM + FN;
  static_assert(SMEM_BYTES <= 160 * 1024, "LDS of one CU");
  static_assert(STAGES >= 2 && (STAGES - 1) * LPW <= 63, "vmcnt counts at most 63 DMAs");
  static constexpr int SPAN0 = SLOTS * 3 / 4, SPAN1 = SLOTS * 7 / 8, SPAN_DMA = SLOTS / 2;

  uint8_t* smem;
  uint32_t smem_addr;
  int lane, wave, wm, wn;
  i32x4_sgpr ra, rw;
  uint32_t va[2], vw[2];  // per-lane offsets of even and odd pieces
  uint32_t tail_kb;       // the k-block that the weight rows end in, ~0 where they fill it
  bool past[2];           // lane's chunk of that block lies past the row's end
  uint32_t a_rows8, w_rows8;

  __device__ __forceinline__ explicit Engine(uint8_t* s) : smem(s) {
    smem_addr = (uint32_t)(uintptr_t)s;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave >> 1;
    wn = wave & 1;
  }

  __device__ __forceinline__ void set_tile(const W8a8Operands& p, int m0, int n0) {
    const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u;
    const int mrows = min(BM, p.M - m0), nrows = min(BN, p.N - n0);
    ra = buffer_rsrc(p.act + (int64_t)m0 * p.lda, (uint32_t)(mrows - 1) * (uint32_t)p.lda + k16);
    rw = buffer_rsrc(p.weight + (int64_t)n0 * p.ldw, (uint32_t)(nrows - 1) * (uint32_t)p.ldw + k16);
    // Piece j: lane L reads row 8 j + L / 8, chunk (L % 8) ^ swizzle(row)
    const int rl = lane >> 3, c = lane & 7;
    const uint32_t rest = k16 & 127u;
    tail_kb = rest ? k16 >> 7 : ~0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int fa = (APW & 1) ? (wave & 1) ^ e : e, fw = (BPW & 1) ? (wave & 1) ^ e : e;  // parity of the piece
      const uint32_t ca = 16u * (uint32_t)(c ^ rl ^ fa), cw = 16u * (uint32_t)(c ^ rl ^ fw);
      va[e] = (uint32_t)rl * (uint32_t)p.lda + ca;
      vw[e] = (uint32_t)rl * (uint32_t)p.ldw + cw;
      past[e] = cw >= rest;
    }
    a_rows8 = 8u * (uint32_t)p.lda;
    w_rows8 = 8u * (uint32_t)p.ldw;
  }

  __device__ __forceinline__ void issue_epi(const W8a8Operands& p, int m0, int n0) {
    for (int d = wave; d < XS_DMAS + 2 * WS_DMAS; d += 4) {
      const int arr = d < XS_DMAS ? 0 : d < XS_DMAS + WS_DMAS ? 1 : 2;
      const int q = d - (arr == 0 ? 0 : arr == 1 ? XS_DMAS : XS_DMAS + WS_DMAS);
      const int off = arr == 0 ? XS_OFF : arr == 1 ? WS_OFF : BIAS_OFF;
      const float* base = arr == 0 ? p.xscales + m0 : arr == 1 ? p.wscales + n0 : (p.bias ? p.bias + n0 : p.wscales);
      // at most the tile's: four bytes times all that follow may pass 32 bits
      const int count = arr == 0 ? min(BM, p.M - m0) : (arr == 1 || p.bias) ? min(BN, p.N - n0) : 0;
      dma4(dma_rsrc(base, (uint32_t)count * 4u), (uint32_t)(q * 256 + lane * 4), smem_addr + (uint32_t)(off + q * 256));
    }
  }

  // DMA piece idx (activations first) of k-block kb into ring stage `stage`.
  __device__ __forceinline__ void issue_piece(uint32_t kb, int stage, int idx) {
    const uint32_t base = smem_addr + (uint32_t)(stage * STAGE_BYTES);
    if (idx < APW) {
      const uint32_t j = (uint32_t)(wave * APW + idx);
      uint32_t so = j * a_rows8 + kb * 128u;
      asm volatile("" : "+s"(so));  // one scalar a piece, not a register a piece for the whole loop
      dma16(ra, va[idx & 1] + so, base + j * 1024u);
    } else {
      const int i = idx - APW;
      const uint32_t j = (uint32_t)(wave * BPW + i);
      uint32_t so = j * w_rows8 + kb * 128u;
      asm volatile("" : "+s"(so));
      uint32_t off = vw[i & 1] + so;
      if (kb == tail_kb) off = past[i & 1] ? kOutOfRange : off;
      dma16(rw, off, base + (uint32_t)BM * 128u + j * 1024u);
    }
  }

  __device__ __forceinline__ const uint8_t* a_frag(int stage, int ks) const {
    const int r = lane & 15;
    return smem + stage * STAGE_BYTES + (wm * TM + r) * 128 + (((2 * (lane >> 4) + ks) ^ chunk_swizzle(r)) * 16);
  }
  __device__ __forceinline__ const uint8_t* w_frag(int stage, int ks) const {
    const int r = lane & 15;
    return smem + stage * STAGE_BYTES + BM * 128 + (wn * TN + r) * 128 +
           (((2 * (lane >> 4) + ks) ^ chunk_swizzle(r)) * 16);
  }

  // Fragment i of a k-step: the weights' first (every MFMA of the first row needs them).
  template <int I>
  __device__ __forceinline__ static void read(const uint8_t* sw, const uint8_t* sa, i32x4 (&w)[FN], i32x4 (&a)[FM]) {
    if constexpr (I < FN) w[I] = *(const i32x4*)(sw + I * 2048);
    else a[I - FN] = *(const i32x4*)(sa + (I - FN) * 2048);
  }

  // n fillers spread over the first `span` MFMA slots: those after slot t are
  // filler(t) .. filler(t + 1) - 1.
  static constexpr int filler(int t, int n, int span) { return t >= span ? n : (t * n + span - 1) / span; }
  // acc += the products of k-blocks kb0 .. kb0 + n - 1, n >= 1.
  __device__ __forceinline__ void run(uint32_t kb0, int n, i32x4 (&acc)[FN][FM]) {
    i32x4 w0[FN], a0[FM], w1[FN], a1[FM];
    const uint32_t last = kb0 + (uint32_t)n - 1;
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
      for (int i = 0; i < LPW; ++i) issue_piece(min(kb0 + s, last), s, i);
    wait_vmcnt<(STAGES - 1) * LPW>();  // block 0 and the epilogue's operands
    __builtin_amdgcn_s_barrier();
    {
      const uint8_t *sw = w_frag(0, 0), *sa = a_frag(0, 0);
      static_for<READS>([&](auto i) __attribute__((always_inline)) { read<i.value>(sw, sa, w0, a0); });
    }
    int st = 0;
    for (uint32_t kb = kb0; kb <= last; ++kb) {
      const int nst = st + 1 == STAGES ? 0 : st + 1;
      {
        const uint8_t *sw = w_frag(st, 1), *sa = a_frag(st, 1);
        static_for<SLOTS>([&](auto slot) __attribute__((always_inline)) {
          constexpr int t = slot.value, lo = filler(t, READS, SPAN0), hi = filler(t + 1, READS, SPAN0);
          mfma_i8(acc[t % FN][t / FN], w0[t % FN], a0[t / FN]);
          static_for<hi - lo>([&](auto f) __attribute__((always_inline)) { read<lo + f.value>(sw, sa, w1, a1); });
        });
      }
      wait_vmcnt<(STAGES - 2) * LPW>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      // past the last block: the last one again, into stages nothing reads
      const uint32_t next = min(kb + STAGES, last);
      {
        const uint8_t *sw = w_frag(nst, 0), *sa = a_frag(nst, 0);
        static_for<SLOTS>([&](auto slot) __attribute__((always_inline)) {
          constexpr int t = slot.value, lo = filler(t, READS, SPAN1), hi = filler(t + 1, READS, SPAN1);
          constexpr int dlo = filler(t, LPW, SPAN_DMA), dhi = filler(t + 1, LPW, SPAN_DMA);
          mfma_i8(acc[t % FN][t / FN], w1[t % FN], a1[t / FN]);
          static_for<dhi - dlo>([&](auto f) __attribute__((always_inline)) { issue_piece(next, st, dlo + f.value); });
          static_for<hi - lo>([&](auto f) __attribute__((always_inline)) { read<lo + f.value>(sw, sa, w0, a0); });
        });
      }
      st = nst;
    }
    mfma_drain(acc);
    wait_vmcnt<0>();  // the DMAs past the last block have landed before the ring is reused
  }
};

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Moves a wave's TM x TN corner of a 16-bit [M, N] array between memory and its
// LDS rows, 16 aligned bytes a lane: row r's first column sits at element
// (m N + nw) % 8 of its LDS row, so that aligned chunks of the array are aligned
// in LDS whatever N is.  ALIGNED: N % 8 == 0 (that element is 0, no part chunks).
template <int TM, int TN, bool ALIGNED, bool STORE>
__device__ __forceinline__ void move_corner(uint8_t* region, uint16_t* base, int lane, int mw, int nw, int M, int N) {
  constexpr int RS = TN * 2 + 16, CPR = ALIGNED ? TN / 8 : TN / 8 + 1, NIT = (TM * CPR + 63) / 64;
  const int cols = min(TN, N - nw), rows = min(TM, M - mw);
  if constexpr (!STORE) {
    // 16 loads in flight at a time
    constexpr int BATCH = 16;
    for (int b0 = 0; b0 < NIT; b0 += BATCH) {
      u32x4 v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int c = (b0 + i) * 64 + lane, row = c / CPR, ch = c % CPR;
        const int64_t start = (int64_t)(mw + row) * N + nw;
        const int first = ALIGNED ? ch * 8 : ch * 8 - (int)(start & 7);
        v[i] = (u32x4){0, 0, 0, 0};
        if (row < rows && first >= 0 && first + 8 <= cols) v[i] = *(const u32x4*)(base + start + first);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int c = (b0 + i) * 64 + lane;
        if (c < TM * CPR) *(u32x4*)(region + c / CPR * RS + c % CPR * 16) = v[i];
      }
    }
  } else {
#pragma unroll 4
    for (int it = 0; it < NIT; ++it) {
      const int c = it * 64 + lane, row = c / CPR, ch = c % CPR;
      const int64_t start = (int64_t)(mw + row) * N + nw;
      const int first = ALIGNED ? ch * 8 : ch * 8 - (int)(start & 7);  // the chunk's first column
      if (row >= rows || first < 0 || first + 8 > cols) continue;
      uint8_t* at = region + row * RS + ch * 16;
      uint16_t* g = base + start + first;
      *(uint4*)g = *(const uint4*)at;
    }
  }
  if constexpr (!ALIGNED) {
    // the part chunks: up to 7 elements at either end of a row, 16 lanes a row
#pragma unroll 4
    for (int it = 0; it < TM / 4; ++it) {
      const int row = it * 4 + (lane >> 4), e = lane & 7;
      const int64_t start = (int64_t)(mw + row) * N + nw;
      const int s = (int)(start & 7), head = min((8 - s) & 7, cols), body = (cols - head) / 8 * 8;
      const int col = lane & 8 ? head + body + e : e;  // the tail's or the head's e-th
      if (row >= rows || col >= (lane & 8 ? cols : head)) continue;
      uint16_t* at = (uint16_t*)(region + row * RS) + s + col;
      if constexpr (STORE) base[start + col] = *at;
      else *at = base[start + col];
    }
  }
}

// The wave's corner of the tile: scale, bias, gated residual, rounding, store.
// 16-bit outputs go through the wave's part of LDS, so that lanes store whole
// aligned chunks; the accumulators hold 4 consecutive n of one m a lane.  The
// residual takes the same way in the other direction: no load or store is
// narrower than 16 bytes but at the corner's edges.
template <class E, int ODT, bool ALIGNED>
__device__ __forceinline__ void epilogue16(const E& e, const i32x4 (&acc)[E::FN][E::FM], const W8a8Operands& p, int m0,
                                           int n0) {
  constexpr int FM = E::FM, FN = E::FN, TM = E::TM, TN = E::TN, RS = TN * 2 + 16;
  const int lane = e.lane, mw = m0 + e.wm * TM, nw = n0 + e.wn * TN;
  const float* xs_lds = (const float*)(e.smem + E::XS_OFF) + e.wm * TM;
  const float* ws_lds = (const float*)(e.smem + E::WS_OFF) + e.wn * TN;
  const float* bias_lds = (const float*)(e.smem + E::BIAS_OFF) + e.wn * TN;
  uint8_t* region = e.smem + e.wave * (TM * RS);
  const bool residual = p.gr.residual != nullptr;
  // rows of the corner under one gate row: its values are loaded once, ahead of the residual
  const bool one_gate = residual && mw / p.gr.rows_per_gate == (min(mw + TM, p.M) - 1) / p.gr.rows_per_gate;
  float gates[FN][4];
  if (one_gate) {
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) load_gate4<ODT>(p.gr, mw, nw + fn * 16 + 4 * (lane >> 4), p.N, gates[fn]);
  }
  if (residual) {
    move_corner<TM, TN, ALIGNED, false>(region, (uint16_t*)p.gr.residual, lane, mw, nw, p.M, p.N);
    wave_lds_fence();
  }
  float xs[FM];
  uint8_t* at[FM];  // the lane's row of each fragment, at the corner's first column
#pragma unroll
  for (int fm = 0; fm < FM; ++fm) {
    const int row = fm * 16 + (lane & 15);
    xs[fm] = xs_lds[row];
    at[fm] = region + row * RS + (ALIGNED ? 0 : 2 * (int)(((int64_t)(mw + row) * p.N + nw) & 7));
  }
  static_for<FN>([&](auto frag) __attribute__((always_inline)) {
    constexpr int fn = frag.value;
    const int nl = fn * 16 + 4 * (lane >> 4);
    const float4 w4 = *(const float4*)(ws_lds + nl), b4 = *(const float4*)(bias_lds + nl);
    const float wsv[4] = {w4.x, w4.y, w4.z, w4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
    float g[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) g[r] = gates[fn][r];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (((float)acc[fn][fm][r] * xs[fm]) * wsv[r]) + bv[r];
      uint16_t* q = (uint16_t*)(at[fm] + nl * 2);
      if (residual) {
        const int m = mw + fm * 16 + (lane & 15);
        if (!one_gate && m < p.M) load_gate4<ODT>(p.gr, m, nw + nl, p.N, g);
        float res[4];
        if constexpr (ALIGNED) {
          load_elem4<ODT>(q, 0, res);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) res[r] = load_elem<ODT>(q, r);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = res[r] + g[r] * o[r];
      }
      if constexpr (ALIGNED) {
        store_out4<ODT>(q, 0, o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) store_out<ODT>(q, r, o[r]);
      }
    }
  });
  wave_lds_fence();
  move_corner<TM, TN, ALIGNED, true>(region, (uint16_t*)p.out, lane, mw, nw, p.M, p.N);
}

template <class E>
__device__ __forceinline__ void epilogue32(const E& e, const i32x4 (&acc)[E::FN][E::FM], const W8a8Operands& p, int m0,
                                           int n0) {
  constexpr int FM = E::FM, FN = E::FN, TM = E::TM, TN = E::TN;
  const int lane = e.lane, mw = m0 + e.wm * TM, nw = n0 + e.wn * TN;
  const float* xs_lds = (const float*)(e.smem + E::XS_OFF) + e.wm * TM;
  const float* ws_lds = (const float*)(e.smem + E::WS_OFF) + e.wn * TN;
  const float* bias_lds = (const float*)(e.smem + E::BIAS_OFF) + e.wn * TN;
  const bool vec = (p.N & 3) == 0;
  static_for<FN>([&](auto frag) __attribute__((always_inline)) {
    constexpr int fn = frag.value;
    const int nl = fn * 16 + 4 * (lane >> 4), n = nw + nl;
    if (n >= p.N) return;
    const float4 w4 = *(const float4*)(ws_lds + nl), b4 = *(const float4*)(bias_lds + nl);
    const float wsv[4] = {w4.x, w4.y, w4.z, w4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int row = fm * 16 + (lane & 15), m = mw + row;
      if (m >= p.M) continue;
      const float xs = xs_lds[row];
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (((float)acc[fn][fm][r] * xs) * wsv[r]) + bv[r];
      store4<kF32>(p, m, n, vec, o);
    }
  });
}

template <class E, int ODT>
__device__ __forceinline__ void epilogue(const E& e, const i32x4 (&acc)[E::FN][E::FM], const W8a8Operands& p, int m0,
                                         int n0) {
  if constexpr (ODT == kF32) epilogue32<E>(e, acc, p, m0, n0);
  else if ((p.N & 7) == 0) epilogue16<E, ODT, true>(e, acc, p, m0, n0);
  else epilogue16<E, ODT, false>(e, acc, p, m0, n0);
}

template <int BM, int BN, int STAGES, int PER_CU, int ODT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_CU, PER_CU))) void w8a8_tile_kernel(
    W8a8Operands p, int tiles_m, int tiles_n, W8a8Split split) {
  constexpr bool LATE_EPI = PER_CU == 2 && BM * BN > 128 * 128;
  using E = Engine<BM, BN, STAGES, LATE_EPI>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[E::SMEM_BYTES];
  E e(smem);
  // tiles that one XCD (one L2) runs are neighbours, in groups of kGroupM tile rows
  const int tiles = tiles_m * tiles_n, per_xcd = tiles / kXcds;
  const int part = BM * BN <= kMaxSplitTile && split.splits > 1 ? blockIdx.x / tiles : 0;
  int t = blockIdx.x - part * tiles;
  if (t < per_xcd * kXcds) t = (t % kXcds) * per_xcd + t / kXcds;
  const int group = t / (kGroupM * tiles_n), first_m = group * kGroupM;
  const int group_rows = min(kGroupM, tiles_m - first_m), in_group = t - group * kGroupM * tiles_n;
  const int m0 = (first_m + in_group % group_rows) * BM, n0 = (in_group / group_rows) * BN;

  e.set_tile(p, m0, n0);
  if constexpr (!LATE_EPI) e.issue_epi(p, m0, n0);
  i32x4 acc[E::FN][E::FM];
#pragma unroll
  for (int a = 0; a < E::FN; ++a)
#pragma unroll
    for (int b = 0; b < E::FM; ++b) acc[a][b] = (i32x4){0, 0, 0, 0};
  const int kblocks = (p.K + 127) / 128;
  if (BM * BN > kMaxSplitTile || split.splits == 1) {
    e.run(0, kblocks, acc);
  } else if constexpr (BM * BN <= kMaxSplitTile) {
    e.run((uint32_t)(part * split.kblocks), min(split.kblocks, kblocks - part * split.kblocks), acc);
    // partials [tile][part][fragment][thread], added by the last workgroup of the tile to arrive
    __shared__ int last;
    constexpr uint32_t BYTES = BM * BN * 4;
    const __amdgpu_buffer_rsrc_t r =
        partial_rsrc(split.partials + (size_t)t * split.splits * BYTES, (uint32_t)split.splits * BYTES);
    const uint32_t at = threadIdx.x * 16u;
    static_for<E::FN>([&](auto fn) __attribute__((always_inline)) {
#pragma unroll
      for (int fm = 0; fm < E::FM; ++fm)
        store_partial(r, (uint32_t)part * BYTES + (uint32_t)(fn.value * E::FM + fm) * 4096u + at, acc[fn.value][fm]);
    });
    if (!last_to_arrive(split.counters + t, split.splits, &last)) return;
    static_for<E::FN>([&](auto fn) __attribute__((always_inline)) {
#pragma unroll
      for (int fm = 0; fm < E::FM; ++fm) acc[fn.value][fm] = (i32x4){0, 0, 0, 0};
    });
    for (int q = 0; q < split.splits; ++q)  // sums of integers: any order gives the same
      static_for<E::FN>([&](auto fn) __attribute__((always_inline)) {
#pragma unroll
        for (int fm = 0; fm < E::FM; ++fm)
          acc[fn.value][fm] += load_partial(r, (uint32_t)q * BYTES + (uint32_t)(fn.value * E::FM + fm) * 4096u + at);
      });
  }
  __syncthreads();  // every wave is done with the ring before it stages outputs
  if constexpr (LATE_EPI) {
    e.issue_epi(p, m0, n0);
    wait_vmcnt<0>();
    __syncthreads();
  }
  epilogue<E, ODT>(e, acc, p, m0, n0);
}

template <int BM, int BN, int STAGES, int PER_CU, int ODT>
hipError_t launch_tile(const W8a8Operands& p, const W8a8Split& split, hipStream_t s) {
  const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  if (tm * tn * split.splits > max_groups(256)) return hipErrorInvalidValue;
  w8a8_tile_kernel<BM, BN, STAGES, PER_CU, ODT><<<dim3((unsigned)(tm * tn * split.splits)), dim3(256), 0, s>>>(
      p, (int)tm, (int)tn, split);
  return hipGetLastError();
}

}  // namespace

template <int ODT>
hipError_t launch_w8a8_tile(int tile, const W8a8Operands& p, const W8a8Split& split, hipStream_t stream) {
  switch (tile) {
#define W8A8_CASE(BM, BN, STAGES, PER_CU) \
  case tile_code(BM, BN): return launch_tile<BM, BN, STAGES, PER_CU, ODT>(p, split, stream);
    W8A8_TILES(W8A8_CASE)
#undef W8A8_CASE
    default: return hipErrorInvalidValue;
  }
}

}  // namespace convrot
