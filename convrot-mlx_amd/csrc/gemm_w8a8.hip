// W8A8 GEMM for gfx950: 8-bit integer activations and weights, one scale a
// token and one an output channel, on INT8 MFMA with the epilogue fused.
//
//   out[m][n] = dt( (float(sum_k act[m][k] w[n][k]) * xs[m]) * ws[n] + bias[n] )
//
// The integer sum is exact (K <= 65536: |sum| <= 2^14 K = 2^30), so the order in
// which K is walked or split cannot change a bit.  An optional gated residual
// follows with the rounding of each of its operations, as for the 4-bit linears
// (convrot_device.h).
//
// Operands: activations [M, K] and weights [N, K] as they are, row-major with
// row strides of a multiple of 16 bytes, so 8-bit checkpoints need no layout of
// their own.  Bytes of a weight row from K to the next multiple of 16 are zero;
// those of an activation row may be anything.
#include <stdlib.h>

#include <algorithm>

#include "convrot_device.h"
#include "convrot_launch.h"

namespace convrot {
namespace {

constexpr int kXcds = 8;  // workgroups are dispatched over 8 XCDs in turn
constexpr int kGroupM = 4;
constexpr uint32_t kOutOfRange = 0x80000000u;  // buffer offset past every operand: reads zero

struct Operands {
  const int8_t* act;
  const int8_t* weight;
  int64_t lda, ldw;
  const float *xscales, *wscales, *bias;
  void* out;
  int M, N, K;
  GatedResidual gr;
};

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
__device__ __forceinline__ int chunk_swizzle(int row) { return (row & 7) ^ ((row >> 3) & 1); }

template <int BM, int BN, int STAGES>
struct Engine {
  static constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16;
  static constexpr int APW = BM / 32, BPW = BN / 32, LPW = APW + BPW;  // 1 KB pieces a wave moves
  static constexpr int STAGE_BYTES = (BM + BN) * 128;
  static constexpr int STAGING = 4 * TM * (TN * 2 + 16);  // 16-bit epilogue
  static constexpr int RING = STAGES * STAGE_BYTES > STAGING ? STAGES * STAGE_BYTES : STAGING;
  // xs, ws, bias of the tile, in 256-byte DMAs
  static constexpr int XS_DMAS = (BM * 4 + 255) / 256, WS_DMAS = (BN * 4 + 255) / 256;
  static constexpr int XS_OFF = RING, WS_OFF = XS_OFF + XS_DMAS * 256, BIAS_OFF = WS_OFF + WS_DMAS * 256;
  static constexpr int SMEM_BYTES = BIAS_OFF + WS_DMAS * 256;
  static constexpr int SLOTS = FM * FN, READS = FM + FN;
  static_assert(SMEM_BYTES <= 160 * 1024, "LDS of one CU");
  static_assert(STAGES >= 2 && (STAGES - 1) * LPW <= 63, "vmcnt counts at most 63 DMAs");
  static_assert(READS <= SLOTS * 3 / 4 && LPW <= SLOTS / 2, "fillers between the MFMAs");

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

  __device__ __forceinline__ void set_tile(const Operands& p, int m0, int n0) {
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

  __device__ __forceinline__ void issue_epi(const Operands& p, int m0, int n0) {
    for (int d = wave; d < XS_DMAS + 2 * WS_DMAS; d += 4) {
      const int arr = d < XS_DMAS ? 0 : d < XS_DMAS + WS_DMAS ? 1 : 2;
      const int q = d - (arr == 0 ? 0 : arr == 1 ? XS_DMAS : XS_DMAS + WS_DMAS);
      const int off = arr == 0 ? XS_OFF : arr == 1 ? WS_OFF : BIAS_OFF;
      const float* base = arr == 0 ? p.xscales + m0 : arr == 1 ? p.wscales + n0 : (p.bias ? p.bias + n0 : p.wscales);
      const int count = arr == 0 ? p.M - m0 : (arr == 1 || p.bias) ? p.N - n0 : 0;
      dma4(buffer_rsrc(base, (uint32_t)count * 4u), (uint32_t)(q * 256 + lane * 4), smem_addr + (uint32_t)(off + q * 256));
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
  __device__ __forceinline__ static void read(const uint8_t* sw, const uint8_t* sa, int i, i32x4 (&w)[FN],
                                              i32x4 (&a)[FM]) {
    if (i < FN) w[i] = *(const i32x4*)(sw + i * 2048);
    else a[i - FN] = *(const i32x4*)(sa + (i - FN) * 2048);
  }

  // n fillers spread over the first `span` >= n MFMA slots: the filler after slot t, or -1.
  static constexpr int filler(int t, int n, int span) {
    const int i = (t * n + span - 1) / span;
    return i < n && i * span / n == t ? i : -1;
  }

  __device__ __forceinline__ void run(int kblocks, i32x4 (&acc)[FN][FM]) {
    i32x4 w0[FN], a0[FM], w1[FN], a1[FM];
    const uint32_t last = (uint32_t)kblocks - 1;
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
      for (int i = 0; i < LPW; ++i) issue_piece(min((uint32_t)s, last), s, i);
    wait_vmcnt<(STAGES - 1) * LPW>();  // block 0 and the epilogue's operands
    __builtin_amdgcn_s_barrier();
    {
      const uint8_t *sw = w_frag(0, 0), *sa = a_frag(0, 0);
#pragma unroll
      for (int i = 0; i < READS; ++i) read(sw, sa, i, w0, a0);
    }
    int st = 0;
    for (uint32_t kb = 0; kb <= last; ++kb) {
      const int nst = st + 1 == STAGES ? 0 : st + 1;
      {
        const uint8_t *sw = w_frag(st, 1), *sa = a_frag(st, 1);
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
          mfma_i8(acc[t % FN][t / FN], w0[t % FN], a0[t / FN]);
          const int i = filler(t, READS, SLOTS * 3 / 4);
          if (i >= 0) read(sw, sa, i, w1, a1);
        }
      }
      wait_vmcnt<(STAGES - 2) * LPW>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      // past the last block: the last one again, into stages nothing reads
      const uint32_t next = min(kb + STAGES, last);
      {
        const uint8_t *sw = w_frag(nst, 0), *sa = a_frag(nst, 0);
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
          mfma_i8(acc[t % FN][t / FN], w1[t % FN], a1[t / FN]);
          const int d = filler(t, LPW, SLOTS / 2), i = filler(t, READS, SLOTS * 7 / 8);
          if (d >= 0) issue_piece(next, st, d);
          if (i >= 0) read(sw, sa, i, w0, a0);
        }
      }
      st = nst;
    }
    mfma_drain(acc);
    wait_vmcnt<0>();  // the DMAs past the last block have landed before the ring is reused
  }
};

// The wave's corner of the tile: scale, bias, rounding, gated residual, store.
// 16-bit outputs go through the wave's part of LDS, so that lanes store whole
// row segments (16 bytes a lane, or where N % 8 != 0 two neighbouring lanes'
// elements); the accumulators hold 4 consecutive n of one m a lane.
template <class E, int ODT>
__device__ __forceinline__ void epilogue(const E& e, const i32x4 (&acc)[E::FN][E::FM], const Operands& p, int m0,
                                         int n0) {
  constexpr int FM = E::FM, FN = E::FN, TM = E::TM, TN = E::TN;
  const int lane = e.lane;
  const float* xs_lds = (const float*)(e.smem + E::XS_OFF) + e.wm * TM;
  const float* ws_lds = (const float*)(e.smem + E::WS_OFF) + e.wn * TN;
  const float* bias_lds = (const float*)(e.smem + E::BIAS_OFF) + e.wn * TN;
  const int mw = m0 + e.wm * TM, nw = n0 + e.wn * TN;
  float xs[FM];
#pragma unroll
  for (int fm = 0; fm < FM; ++fm) xs[fm] = xs_lds[fm * 16 + (lane & 15)];
  auto values = [&](int fn, int fm, const float4& w4, const float4& b4, float (&o)[4]) {
    const float wsv[4] = {w4.x, w4.y, w4.z, w4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (((float)acc[fn][fm][r] * xs[fm]) * wsv[r]) + bv[r];
  };
  if constexpr (ODT == kF32) {
    const bool vec = (p.N & 3) == 0;
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) {
      const int nl = fn * 16 + 4 * (lane >> 4), n = nw + nl;
      if (n >= p.N) continue;
      const float4 w4 = *(const float4*)(ws_lds + nl), b4 = *(const float4*)(bias_lds + nl);
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        const int m = mw + fm * 16 + (lane & 15);
        if (m >= p.M) continue;
        float o[4];
        values(fn, fm, w4, b4, o);
        if (p.gr.residual) gate_residual4<ODT>(p.gr, m, n, p.N, vec, o);
        const int64_t idx = (int64_t)m * p.N + n;
        if (vec) {
          store_out4<ODT>(p.out, idx, o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < p.N) store_out<ODT>(p.out, idx + r, o[r]);
        }
      }
    }
  } else {
    constexpr int RS = TN * 2 + 16;
    uint8_t* region = e.smem + e.wave * (TM * RS);
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) {
      const int nl = fn * 16 + 4 * (lane >> 4);
      const float4 w4 = *(const float4*)(ws_lds + nl), b4 = *(const float4*)(bias_lds + nl);
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        float o[4];
        values(fn, fm, w4, b4, o);
        *(uint2*)(region + (fm * 16 + (lane & 15)) * RS + nl * 2) =
            ODT == kBF16 ? make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]))
                         : make_uint2(pack_f16x2(o[0], o[1]), pack_f16x2(o[2], o[3]));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if ((p.N & 7) == 0) {
      constexpr int CPR = TN / 8, NIT = TM * CPR / 64, BATCH = 4;
      static_assert(TM * CPR % 64 == 0 && NIT % BATCH == 0, "whole batches of stores");
#pragma unroll
      for (int b0 = 0; b0 < NIT; b0 += BATCH) {
        Gated8 ops[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int c = (b0 + i) * 64 + lane, m = mw + c / CPR, n = nw + (c % CPR) * 8;
          if (p.gr.residual && m < p.M && n < p.N) gate_load8<ODT>(p.gr, m, n, p.N, true, ops[i]);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int c = (b0 + i) * 64 + lane, row = c / CPR, cc = c % CPR, m = mw + row, n = nw + cc * 8;
          if (m >= p.M || n >= p.N) continue;
          uint4 v = *(const uint4*)(region + row * RS + cc * 16);
          if (p.gr.residual) v = gate_apply8<ODT>(ops[i], v);
          *(uint4*)((uint16_t*)p.out + (int64_t)m * p.N + n) = v;
        }
      }
    } else {
      typedef typename Elem<ODT>::T T;
      for (int i = lane; i < TM * TN; i += 64) {
        const int row = i / TN, col = i % TN, m = mw + row, n = nw + col;
        if (m >= p.M || n >= p.N) continue;
        float v = (float)*(const T*)(region + row * RS + col * 2);
        const int64_t idx = (int64_t)m * p.N + n;
        if (p.gr.residual) {
          const float g =
              p.gr.gate ? load_elem<ODT>(p.gr.gate, (int64_t)(m / p.gr.rows_per_gate) * p.gr.gate_stride + n) : 1.0f;
          v = gated_sum<ODT>(v, load_elem<ODT>(p.gr.residual, idx), g);
        }
        store_out<ODT>(p.out, idx, v);
      }
    }
  }
}

template <int BM, int BN, int STAGES, int PER_CU, int ODT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_CU, PER_CU))) void w8a8_tile_kernel(
    Operands p, int tiles_m, int tiles_n) {
  using E = Engine<BM, BN, STAGES>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[E::SMEM_BYTES];
  E e(smem);
  // tiles that one XCD (one L2) runs are neighbours, in groups of kGroupM tile rows
  const int tiles = tiles_m * tiles_n, per_xcd = tiles / kXcds;
  int t = blockIdx.x;
  if (t < per_xcd * kXcds) t = (t % kXcds) * per_xcd + t / kXcds;
  const int group = t / (kGroupM * tiles_n), first_m = group * kGroupM;
  const int group_rows = min(kGroupM, tiles_m - first_m), in_group = t - group * kGroupM * tiles_n;
  const int m0 = (first_m + in_group % group_rows) * BM, n0 = (in_group / group_rows) * BN;

  e.set_tile(p, m0, n0);
  e.issue_epi(p, m0, n0);
  i32x4 acc[E::FN][E::FM];
#pragma unroll
  for (int a = 0; a < E::FN; ++a)
#pragma unroll
    for (int b = 0; b < E::FM; ++b) acc[a][b] = (i32x4){0, 0, 0, 0};
  e.run((p.K + 127) / 128, acc);
  __syncthreads();  // every wave is done with the ring before it stages outputs
  epilogue<E, ODT>(e, acc, p, m0, n0);
}

// ---- few rows
//
// The weights' bytes bound it: each is read once, straight into registers.  A
// workgroup owns NB tiles of 16 output channels and 16 FM tokens; its SPLIT
// waves share K, a block of 128 in turn, and add their integer sums through LDS.
template <int FM, int NB, int SPLIT, int UNROLL, int ODT>
__global__ __launch_bounds__(SPLIT * 64) void w8a8_rows_kernel(Operands p) {
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
    if (p.gr.residual) gate_residual4<ODT>(p.gr, m, n, p.N, vec, o);
    const int64_t idx = (int64_t)m * p.N + n;
    if (vec) {
      store_out4<ODT>(p.out, idx, o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < p.N) store_out<ODT>(p.out, idx + j, o[j]);
    }
  }
}

template <int BM, int BN, int STAGES, int PER_CU, int ODT>
hipError_t launch_tile(const Operands& p, hipStream_t s) {
  const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
  if (tm * tn > 0x7fffffff) return hipErrorInvalidValue;
  w8a8_tile_kernel<BM, BN, STAGES, PER_CU, ODT><<<dim3((unsigned)(tm * tn)), dim3(256), 0, s>>>(p, (int)tm, (int)tn);
  return hipGetLastError();
}

template <int FM, int NB, int SPLIT, int UNROLL, int ODT>
hipError_t launch_rows(const Operands& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 16 * NB - 1) / (16 * NB)), (unsigned)((p.M + 16 * FM - 1) / (16 * FM)));
  w8a8_rows_kernel<FM, NB, SPLIT, UNROLL, ODT><<<grid, dim3(SPLIT * 64), 0, s>>>(p);
  return hipGetLastError();
}

// Kernel of a product: 0 few rows, else BM | BN << 10 of a tile.
int plan(int64_t M, int64_t N, int64_t K) {
  const int forced = tuning(kTuneW8a8Tile);
  if (forced >= 0) return forced;
  if (M <= 64) return 0;
  return N >= 512 && M >= 512 ? (256 | 256 << 10) : (128 | 128 << 10);
}

template <int ODT>
hipError_t launch_t(const Operands& p, hipStream_t s) {
  switch (plan(p.M, p.N, p.K)) {
    case 0:
      if (p.M <= 16) {
        if (p.N <= 8192) return launch_rows<1, 1, 16, 4, ODT>(p, s);
        return launch_rows<1, 1, 4, 6, ODT>(p, s);
      }
      if (p.M <= 32) return launch_rows<2, 1, 8, 4, ODT>(p, s);
      return launch_rows<4, 1, 8, 2, ODT>(p, s);
    case 256 | 256 << 10: return launch_tile<256, 256, 2, 1, ODT>(p, s);
    default: return launch_tile<128, 128, 2, 2, ODT>(p, s);
  }
}

}  // namespace

bool w8a8_tile_known(int bm, int bn) { return (bm == 0 && bn == 0) || (bm == 256 && bn == 256) || (bm == 128 && bn == 128); }

hipError_t launch_w8a8_gemm(const int8_t* act, int64_t lda, const float* xscales, const int8_t* weight, int64_t ldw,
                            const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K, void* out,
                            int out_dtype, hipStream_t stream, const GatedResidual& gr) {
  const Operands p{act, weight, lda, ldw, xscales, wscales, bias, out, (int)M, (int)N, (int)K, gr};
  switch (out_dtype) {
    case kF32: return launch_t<kF32>(p, stream);
    case kF16: return launch_t<kF16>(p, stream);
    default: return launch_t<kBF16>(p, stream);
  }
}

}  // namespace convrot
