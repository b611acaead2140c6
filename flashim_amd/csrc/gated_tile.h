// The matrix products of the gated feed-forward operator on large tiles: BF16 or FP16, FP32 sums.
//
// A workgroup of four wavefronts (2 x 2) computes 64 MB x 64 NB products on 32 x 32 x 16 MFMAs, each wavefront MB x NB
// blocks. The contraction is walked in steps of 64: both operands of a step lie in one of two LDS stages, filled by
// 16-byte loads straight into LDS. An operand whose rows run along the contraction is staged as rows of 128 bytes and read
// in 16-byte pieces; one whose rows run across it (the weights for dx, both operands for the weights' gradients) is staged
// as it lies, 64 rows of the tile's width, and read transposed by the LDS itself (ds_read_tr16_b64: each 16 lanes read a 4 x
// 16 block and lane i gets its column i; layout measured), so nothing is transposed in memory. Both layouts are swizzled in
// 16-byte or 64-byte units against bank conflicts.
//
// The loop's order: while the MFMAs of one 16-wide sub-step run, the operands of the next are read, one read between two
// MFMAs; the next step's stage is waited for before the last sub-step, whose MFMAs cover the first reads from it, and from
// then on the consumed stage is refilled. One barrier per step.
//
// The matrix cores bound it, and below them the loop's LDS reads and the epilogue (the activation's vector work, nothing left to
// overlap it on a CU's only tile). Measured (device time after a hundred calls, MI355X, BF16; a large library product reaches 1400
// to 1440 TFLOP/s): 16384 x 1024 -> 2 x 4096 with SiLU, 255 us (1080 TFLOP/s), its backward's products 210 us (dx, 1310) and 208 us
// (weights, 1320), dg and du 315 us on 128 x 128 tiles (870: the epilogue has no registers left beside 256 x 256 accumulators);
// 20000 x 512 -> 2 x 2048 forward with GELU and biases 113 us (740). FP16 dx on 256 x 256 tiles spills 64 of its 256 registers
// around its conversions, and is still ahead of 128 x 128: 237 against 292 us.
#pragma once

#include "activation.h"

namespace fim {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int DT>
__device__ __forceinline__ v16f mfma16(s16x8 a, s16x8 b, v16f c) {
  typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (DT == FIM_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint16_t to16(float v) {
  return DT == FIM_BF16 ? (uint16_t)(pack_bf16x2(v, 0.0f) & 0xffff) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ uint32_t to16x2(float a, float b) {
  if constexpr (DT == FIM_BF16) return pack_bf16x2(a, b);
  return (uint32_t)to16<DT>(a) | (uint32_t)to16<DT>(b) << 16;
}
template <int DT>
__device__ __forceinline__ float from16(uint16_t h) {
  return DT == FIM_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// A buffer access's bit for lines that are not read again soon (non-temporal): out and dx, written past the operands that the
// other tiles still read (16384 x 1024 -> 2 x 4096 with its backward 1012 -> 1000 us, a product that reads `out` next takes as
// long as before). dg and du are read next.
constexpr int STREAM_BIT = 2;

// FORWARD: out = act(g) u.  GRAD: the same products, out dg and du.  DX: dg Wg + du Wu.  DW: dg^T x and du^T x.
enum { GATED_FORWARD, GATED_GRAD, GATED_DX, GATED_DW };

// What a product's operands are: x supplies the output rows (the MFMA's columns, one per lane), w the output columns (its
// rows, four neighbours per lane and register group). 16-byte aligned, row strides and widths multiples of 8, row strides
// not below the width.
struct TileArgs {
  const uint16_t* x[2];  // FORWARD, GRAD: x[0]. DX: dg, du. DW: x[0], whose columns are the output rows
  const uint16_t* w[2];  // FORWARD, GRAD, DX: gate, up. DW: dg, du, whose columns are the output columns
  int64_t ldx, ldw;
  int64_t M, N, K;       // output rows, columns (of one half), contraction (DX: of one half)
  int64_t xw, ww;        // columns of x and w that may be read where they run across the contraction
  const void* bias[2];
  int bias_dtype;
  const uint16_t* dout;
  int64_t ldd;
  uint16_t* out[2];
  int64_t ldo, out_cols;  // columns written: N, or more (GRAD: with zeros)
  int wide_out, wide_dout;  // rows of out and dout are 16-byte aligned
  float* col_sums;        // GRAD: [2 m tiles][2][N] sums of dg and du over 32 MB rows, or null
  float* part;            // DW: [splits][2][N][M]; DX: [splits][M][N], or null
  int mt, nt, group;      // tiles; m tiles of a group that share the columns' operands in L2
  int64_t k_split;        // contraction of one split: DW rows (a multiple of 64), DX steps over both halves
};

constexpr int TILE_K = 64;
constexpr uint32_t TILE_OOB = 0x80000000u;  // past every buffer: reads as zero

constexpr int tile_wait(int vm) { return (vm & 0xF) | (0x7 << 4) | (((vm >> 4) & 0x3) << 14); }  // and lgkmcnt(0)

// Orders this wavefront's LDS writes before its reads of what other lanes wrote
__device__ __forceinline__ void wave_lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// v[i] summed over the 32 lanes of this half wavefront; lane l ends with the sum of v[l % 32] in v[0]. Each step halves the
// values: a lane keeps one half and adds the other lane's (31 exchanges for 32 sums).
template <int S>
__device__ __forceinline__ void sum_lanes(float (&v)[32], int lane) {
  const bool up = lane & S;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const float keep = up ? v[i + S] : v[i], send = up ? v[i] : v[i + S];
    v[i] = keep + __shfl_xor(send, S);
  }
  if constexpr (S > 1) sum_lanes<S / 2>(v, lane);
}

// Sixteen bytes of a row whose width or address is not a multiple of 16 bytes: global loads and stores take any alignment of
// the element.
typedef v4i v4i_any __attribute__((aligned(2)));

template <int DT, int MODE, int ACT, int MB, int NB>
__global__ __launch_bounds__(256, MB * NB > 8 ? 1 : 2) void gated_tile_kernel(const TileArgs a) {
  constexpr bool PAIR = MODE == GATED_FORWARD || MODE == GATED_GRAD;
  constexpr bool XT = MODE == GATED_DW, WT = MODE == GATED_DX || MODE == GATED_DW;  // rows run across the contraction
  constexpr int BM = 64 * MB, BN = 64 * NB;
  constexpr int CX = BM / 32, CW = BN / 32;  // 1 KB loads of a stage per wavefront
  constexpr int STAGE = (BM + BN) * 2 * TILE_K;
  static_assert(!PAIR || NB % 2 == 0, "gate and up blocks");
  __shared__ __attribute__((aligned(16))) uint8_t st0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t st1[STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, h = lane >> 5;

  // workgroups go round the 8 XCDs: each takes a contiguous run of tiles, group by group of m tiles, n slowest in a group
  const int tiles = a.mt * a.nt;
  const int per_xcd = (int)(gridDim.x >> 3);
  int t = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  const int half_steps = (int)((a.K + TILE_K - 1) / TILE_K);
  const int splits = MODE == GATED_DW   ? (int)((a.K + a.k_split - 1) / a.k_split)
                     : MODE == GATED_DX ? (int)((2 * half_steps + a.k_split - 1) / a.k_split)
                                        : 1;
  if (t >= tiles * splits) return;
  const int split = WT ? __builtin_amdgcn_readfirstlane(t / tiles) : 0;
  t -= split * tiles;
  const int grp = t / (a.group * a.nt), in_grp = t - grp * a.group * a.nt;
  const int gm = a.mt - grp * a.group < a.group ? a.mt - grp * a.group : a.group;
  // (quotients come from the vector unit: back to scalars, or every buffer descriptor becomes a loop over lanes)
  const int tn = __builtin_amdgcn_readfirstlane(in_grp / gm);
  const int tm = __builtin_amdgcn_readfirstlane(grp * a.group + in_grp - tn * gm);
  const int half = MODE == GATED_DW ? tn & 1 : 0;
  const int64_t m0 = (int64_t)tm * BM;
  const int64_t n0 = PAIR ? (int64_t)tn * (BN / 2) : MODE == GATED_DW ? (int64_t)(tn >> 1) * BN : (int64_t)tn * BN;

  const int64_t kb = MODE == GATED_DW ? split * a.k_split : 0;
  const int64_t klen = MODE == GATED_DW ? (a.K - kb < a.k_split ? a.K - kb : a.k_split) : a.K;
  // steps [first, last): of both halves for dx
  const int first = MODE == GATED_DX ? (int)(split * a.k_split) : 0;
  int last = MODE == GATED_DX ? 2 * half_steps : (int)((klen + TILE_K - 1) / TILE_K);
  if (MODE == GATED_DX && first + a.k_split < last) last = (int)(first + a.k_split);

  // -- loads into LDS: chunk c (1 KB) of an operand's part of a stage; wavefront w loads chunks w, w + 4, ... of each
  // along: chunk c is rows 8 c .. 8 c + 7, lane l row l / 8, LDS slot l % 8, which holds K segment slot ^ (row / 2 % 8)
  const int seg = (lane & 7) ^ (lane >> 4) ^ (4 * (wave & 1));
  // across: a row of the stage has BM / 8 slots; slot s of row k holds column segment s ^ 4 (k % 4)
  auto across_off = [&](int slots, int c, int64_t ld, int64_t cols) __attribute__((always_inline)) {
    const int k = c * (64 / slots) + lane / slots, s = (lane % slots) ^ ((k & 3) << 2);
    return s * 8 < cols ? (uint32_t)(k * ld + s * 8) * 2u : TILE_OOB;
  };
  uint32_t xo[CX], wo[CW];
  const int64_t xrows = a.M - m0, wrows = a.N - n0;
#pragma unroll
  for (int i = 0; i < CX; ++i) {
    const int c = wave + 4 * i, r = 8 * c + (lane >> 3);
    if constexpr (XT) xo[i] = across_off(BM / 8, c, a.ldx, a.xw - m0);
    else xo[i] = r < xrows ? (uint32_t)(r * a.ldx) * 2u + seg * 16 : TILE_OOB;
  }
#pragma unroll
  for (int i = 0; i < CW; ++i) {
    const int c = wave + 4 * i;
    int r = 8 * c + (lane >> 3);
    if (PAIR && i >= CW / 2) r -= BN / 2;
    if constexpr (WT) wo[i] = across_off(BN / 8, c, a.ldw, a.ww - n0);
    else wo[i] = r < wrows ? (uint32_t)(r * a.ldw) * 2u + seg * 16 : TILE_OOB;
  }
  // bytes from a tile's first element to the end of its operand
  auto rest = [](int64_t rows, int64_t ld, int64_t cols) __attribute__((always_inline)) {
    return rows <= 0 ? 0 : ((rows - 1) * ld + cols) * 2;
  };
  int step_at = first;  // the step whose loads are issued next
  auto load = [](const uint16_t* p, int records, uint8_t* to, uint32_t off) __attribute__((always_inline)) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), (short)0, __builtin_amdgcn_readfirstlane(records),
                                          0x00020000),
        (lds_void*)to, 16, off, 0, 0, 0);
  };
  const int64_t kw = (a.K + 7) / 8 * 8;  // whole loads: the operand's rows are padded to them
  const int xrec = XT ? 0 : (int)rest(xrows < BM ? xrows : BM, a.ldx, kw);
  const int wrec = WT ? 0 : (int)rest(wrows < BN ? wrows : BN, a.ldw, kw);
  // per step: the lane's K offset of an operand along the contraction; first row and bytes left of one across it
  const bool second = MODE == GATED_DX && first >= half_steps;
  const int64_t skip = MODE == GATED_DX ? (int64_t)(first - (second ? half_steps : 0)) * TILE_K : 0;
  uint32_t kbyte = (uint32_t)skip * 2u, kdead;
  const uint16_t *xp = XT ? a.x[0] + kb * a.ldx + m0 : a.x[second] + m0 * a.ldx;
  const uint16_t *wp = a.w[MODE == GATED_DX ? second : half] + (kb + skip) * a.ldw + n0;
  int64_t xleft = rest(klen, a.ldx, a.xw - m0), wleft = rest(klen - skip, a.ldw, a.ww - n0);
  auto bytes = [](int64_t left) __attribute__((always_inline)) {
    return (int)(left <= 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : left);
  };
  int xbytes = XT ? bytes(xleft) : xrec, wbytes = bytes(wleft);
  auto next_step = [&]() __attribute__((always_inline)) {
    ++step_at;
    kbyte += 2 * TILE_K;
    wp += TILE_K * a.ldw;
    wleft -= TILE_K * a.ldw * 2;
    if (MODE == GATED_DX && step_at == half_steps) {  // on to the other half
      kbyte = 0u;
      xp = a.x[1] + m0 * a.ldx;
      wp = a.w[1] + n0;
      wleft = rest(klen, a.ldw, a.ww - n0);
    }
    if constexpr (XT) {
      xp += TILE_K * a.ldx;
      xleft -= TILE_K * a.ldx * 2;
      xbytes = bytes(xleft);
    }
    // (past the last step nothing is read: zeros of one operand would meet infinities of the other)
    if constexpr (WT) wbytes = step_at < last ? bytes(wleft) : 0;
    kdead = step_at < last && kbyte + seg * 16 < (uint32_t)a.K * 2u ? 0u : TILE_OOB;
  };
  kdead = first < last && kbyte + seg * 16 < (uint32_t)a.K * 2u ? 0u : TILE_OOB;
  // load i of the step: x's, then w's
  auto issue = [&](uint8_t* st, int i) __attribute__((always_inline)) {
    if (i < CX) {
      uint8_t* to = st + (wave + 4 * i) * 1024;
      if constexpr (XT) load(xp, xbytes, to, xo[i]);
      else load(xp, xbytes, to, (xo[i] + kbyte) | kdead);
    } else if (i < CX + CW) {
      const int k = i - CX;
      uint8_t* to = st + BM * 2 * TILE_K + (wave + 4 * k) * 1024;
      if constexpr (WT) load(wp, wbytes, to, wo[k]);
      else
        load(a.w[k >= CW / 2] + n0 * a.ldw, wrec, to, (wo[k] + kbyte) | kdead);
    }
  };

  // -- operand fragments: lane l holds row (or column) l % 32 of a block, contraction 8 h .. 8 h + 7 of a 16-wide sub-step
  const int frow = lane & 31;
  const int fsw = (frow >> 1) & 7;
  const int tq = (lane & 15) >> 2;
  const int tcol = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  // (one addition to the stage's address: the compiler tells a stage's reads from the loads in flight into the other by the
  // pointers' origin, which it follows through few steps)
  auto read_along = [&](const uint8_t* st, int at, int row0, int kk) __attribute__((always_inline)) {
    const int off = at + (row0 + frow) * 2 * TILE_K + (((2 * kk + h) ^ fsw) << 4);
    return *reinterpret_cast<const s16x8*>(st + off);
  };
  auto read_across = [&](const uint8_t* st, int at, int rowb, int blk, int kk) __attribute__((always_inline)) {
    const int off = at + (kk * 16 + 8 * h + tq) * rowb + ((blk ^ tq) << 6) + tcol;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + off));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + (off + 4 * rowb)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  s16x8 fx[2][MB], fw[2][NB];
  // read r of a sub-step's MB + NB into set s
  auto read = [&](const uint8_t* st, int s, int kk, int r) __attribute__((always_inline)) {
    constexpr int W_AT = BM * 2 * TILE_K;
    if (r < NB) {
      if constexpr (WT) fw[s][r] = read_across(st, W_AT, BN * 2, wn * NB + r, kk);
      else if constexpr (PAIR)
        fw[s][r] = read_along(st, W_AT, (r / (NB / 2)) * (BN / 2) + (wn * (NB / 2) + r % (NB / 2)) * 32, kk);
      else fw[s][r] = read_along(st, W_AT, (wn * NB + r) * 32, kk);
    } else if (r < NB + MB) {
      if constexpr (XT) fx[s][r - NB] = read_across(st, 0, BM * 2, wm * MB + r - NB, kk);
      else fx[s][r - NB] = read_along(st, 0, (wm * MB + r - NB) * 32, kk);
    }
  };

  // accumulators: lane l, register q of block (i, j): row 32 j + l % 32, column 32 i + 8 (q / 4) + 4 h + q % 4; started at
  // the bias (all its loads on one side of the branch on its type: one latency). Columns past the end read the last bias and
  // start at 0: GRAD writes zeros there, and zero times an infinite bias is none
  v16f acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    v16f first;
#pragma unroll
    for (int q = 0; q < 16; ++q) first[q] = 0.0f;
    if constexpr (PAIR) {
      const void* b = a.bias[i / (NB / 2)];
      const int64_t c0 = n0 + (wn * (NB / 2) + i % (NB / 2)) * 32 + 4 * h;
      auto column = [&](int q) __attribute__((always_inline)) {
        const int64_t c = c0 + 8 * (q >> 2) + (q & 3);
        return c < a.N ? c : a.N - 1;
      };
      if (b != nullptr && a.bias_dtype == FIM_F32) {
#pragma unroll
        for (int q = 0; q < 16; ++q) first[q] = static_cast<const float*>(b)[column(q)];
      } else if (b != nullptr) {
        uint16_t e[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) e[q] = static_cast<const uint16_t*>(b)[column(q)];
#pragma unroll
        for (int q = 0; q < 16; ++q) first[q] = from16<DT>(e[q]);
      }
      if constexpr (MODE == GATED_GRAD) {
#pragma unroll
        for (int q = 0; q < 16; ++q) first[q] = c0 + 8 * (q >> 2) + (q & 3) < a.N ? first[q] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = first;
  }

  constexpr int T = MB * NB, READS = MB + NB, LOADS = CX + CW;
  // The MFMAs of sub-step kk from set s, with READS reads of the next one (from stage `rd`, into set 1 - s) and loads
  // [l0, l1) of the next step spread between them
  auto sub_step = [&](int s, const uint8_t* rd, int rkk, uint8_t* fill, int l0, int l1) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < T; ++m) {
      const int i = m % NB, j = m / NB;
      acc[i][j] = mfma16<DT>(fw[s][i], fx[s][j], acc[i][j]);
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * T / READS == m) read(rd, 1 - s, rkk, r);
#pragma unroll
      for (int l = 0; l < LOADS; ++l)
        if (l >= l0 && l < l1 && (l - l0) * T / (l1 - l0) == m) issue(fill, l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int L1 = (LOADS + 1) / 2;  // loads issued in the sub-step after the barrier; the others in the next
  // one step from stage cur, whose refill for two steps on begins after the barrier; the rest of nxt's loads first
  auto step = [&](uint8_t* cur, uint8_t* nxt) __attribute__((always_inline)) {
    sub_step(0, cur, 1, nxt, L1, LOADS);
    next_step();
    sub_step(1, cur, 2, nxt, 0, 0);
    sub_step(0, cur, 3, nxt, 0, 0);
    __builtin_amdgcn_s_waitcnt(tile_wait(0));  // nxt has landed, cur has been read
    asm volatile("s_barrier" ::: "memory");
    sub_step(1, nxt, 0, cur, 0, L1);
  };

#pragma unroll
  for (int l = 0; l < LOADS; ++l) issue(st0, l);
  next_step();
#pragma unroll
  for (int l = 0; l < L1; ++l) issue(st1, l);
  __builtin_amdgcn_s_waitcnt(tile_wait(L1));
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int r = 0; r < READS; ++r) read(st0, 0, 0, r);
  // pairs of steps: one exit; a step past the last multiplies zeros
  for (int k = first; k < last; k += 2) {
    step(st0, st1);
    step(st1, st0);
  }
  __builtin_amdgcn_s_waitcnt(tile_wait(0));
  asm volatile("s_barrier" ::: "memory");

  // -- epilogue
  const int64_t mw = m0 + wm * MB * 32;
  if constexpr (MODE == GATED_DW) {  // lanes are neighbouring columns of the weight: 128-byte runs
    float* to = a.part + (int64_t)(split * 2 + half) * a.N * a.M;
    const int64_t nw = n0 + wn * NB * 32 + 4 * h;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int64_t n = nw + 32 * i + 8 * (q >> 2) + (q & 3);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
          const int64_t m = mw + 32 * j + frow;
          if (n < a.N && m < a.M) to[n * a.M + m] = acc[i][j][q];
        }
      }
    return;
  }
  if (MODE == GATED_DX && a.part != nullptr) {
    float* to = a.part + (int64_t)split * a.M * a.N;
    const int64_t nw = n0 + wn * NB * 32 + 4 * h;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int64_t m = mw + 32 * j + frow;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const int64_t n = nw + 32 * i + 8 * (q >> 2) + (q & 3);
          if (n < a.N && m < a.M) to[m * a.N + n] = acc[i][j][q];
        }
    }
    return;
  }
  if constexpr (MODE != GATED_DW) {
    // 32 rows at a time through LDS (this wavefront's own part of the consumed stage): whole runs of the output's rows, by
    // buffer stores whose rows and columns past the end go out of range, without branches
    constexpr int NO = PAIR ? NB / 2 : NB, OC = 32 * NO, RB = OC * 2, SLOTS = RB / 16, PER = 64 / SLOTS;
    constexpr int AREA = 32 * RB, AREAS = MODE == GATED_GRAD ? 2 : 1, RUNS = 32 / PER;
    static_assert(4 * AREAS * AREA <= STAGE, "the wavefronts' areas lie in the first stage");
    uint8_t* area = st0 + wave * AREAS * AREA;
    auto place = [&](int row, int slot) __attribute__((always_inline)) {
      constexpr int RPL = RB >= 256 ? 1 : 256 / RB;
      return row * RB + ((slot ^ ((row / RPL) & (SLOTS - 1))) << 4);
    };
    const int64_t nw = n0 + wn * OC, rows_left = a.M - mw;
    const int slot = lane % SLOTS, prow = lane / SLOTS;
    const int cols_out = (int)(a.out_cols - nw < OC ? a.out_cols - nw : OC);
    const int cols_in = (int)(a.N - nw < OC ? a.N - nw : OC);
    auto buffer_bytes = [&](int64_t ld, int64_t cols) __attribute__((always_inline)) {
      const int64_t n = cols <= 0 ? 0 : rest(rows_left < 32 * MB ? rows_left : 32 * MB, ld, cols);
      return __builtin_amdgcn_readfirstlane((int)(n > 0x7fffffff ? 0x7fffffff : n));
    };
    const __amdgpu_buffer_rsrc_t o0 =
        __builtin_amdgcn_make_buffer_rsrc(a.out[0] + mw * a.ldo + nw, (short)0, buffer_bytes(a.ldo, cols_out), 0x00020000);
    const __amdgpu_buffer_rsrc_t o1 = __builtin_amdgcn_make_buffer_rsrc(
        (MODE == GATED_GRAD ? a.out[1] : a.out[0]) + mw * a.ldo + nw, (short)0, buffer_bytes(a.ldo, cols_out), 0x00020000);
    const __amdgpu_buffer_rsrc_t din = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.dout) + (MODE == GATED_GRAD ? mw * a.ldd + nw : 0), (short)0,
        MODE == GATED_GRAD ? buffer_bytes(a.ldd, cols_in) : 0, 0x00020000);
    float sums[MODE == GATED_GRAD ? NB : 1][16];
    if constexpr (MODE == GATED_GRAD) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) sums[i][q] = 0.0f;
    }
    auto epilogue = [&](auto wide_c) __attribute__((always_inline)) {
      constexpr bool WIDE = decltype(wide_c)::value;  // 16-byte rows of out (GRAD: of dout)
      const bool whole = rows_left >= 32 * MB;
      v4i grad[2][MODE == GATED_GRAD ? RUNS : 1];  // rows of the incoming gradient, 32 ahead
      auto load_grad = [&](int j) __attribute__((always_inline)) {
        if constexpr (MODE == GATED_GRAD) {
#pragma unroll
          for (int p = 0; p < RUNS; ++p) {
            if constexpr (WIDE) {
              const uint32_t at = (uint32_t)((32 * j + p * PER + prow) * a.ldd + slot * 8) * 2u;
              grad[j & 1][p] = __builtin_bit_cast(
                  v4i, __builtin_amdgcn_raw_buffer_load_b128(din, (int)(slot * 8 < cols_in ? at : TILE_OOB), 0, 0));
            }
          }
          if constexpr (!WIDE) {
            if (whole && slot * 8 + 8 <= cols_in) {
              const uint16_t* from = a.dout + (mw + 32 * j + prow) * a.ldd + nw + slot * 8;
#pragma unroll
              for (int p = 0; p < RUNS; ++p)
                grad[j & 1][p] = *reinterpret_cast<const v4i_any*>(from + (int64_t)p * PER * a.ldd);
            } else {
#pragma unroll
              for (int p = 0; p < RUNS; ++p) {
                const uint32_t at = (uint32_t)((32 * j + p * PER + prow) * a.ldd + slot * 8) * 2u;
                uint32_t e[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  e[c] = __builtin_amdgcn_raw_buffer_load_b16(din, (int)(slot * 8 + c < cols_in ? at + 2 * c : TILE_OOB), 0, 0);
#pragma unroll
                for (int c = 0; c < 4; ++c) grad[j & 1][p][c] = (int)(e[2 * c] | e[2 * c + 1] << 16);
              }
            }
          }
        }
      };
      load_grad(0);
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        if constexpr (MODE == GATED_GRAD) {
          if (j + 1 < MB) load_grad(j + 1);
#pragma unroll
          for (int p = 0; p < RUNS; ++p) *reinterpret_cast<v4i*>(area + place(p * PER + prow, slot)) = grad[j & 1][p];
          wave_lds_wait();
          if (rows_left < 32 * (j + 1)) {  // rows past the end: zero times anything
            const bool past = 32 * j + frow >= rows_left;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int q = 0; q < 16; ++q) acc[i][j][q] = past ? 0.0f : acc[i][j][q];
          }
        }
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint8_t* at = area + place(frow, 4 * o + q) + 8 * h;
            typedef int v2i __attribute__((ext_vector_type(2)));
            if constexpr (MODE == GATED_FORWARD) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = activate<ACT>(acc[o][j][4 * q + e]) * acc[o + NO][j][4 * q + e];
              *reinterpret_cast<v2i*>(at) = v2i{(int)to16x2<DT>(v[0], v[1]), (int)to16x2<DT>(v[2], v[3])};
            } else if constexpr (MODE == GATED_DX) {
              const v16f& s = acc[o][j];
              *reinterpret_cast<v2i*>(at) =
                  v2i{(int)to16x2<DT>(s[4 * q], s[4 * q + 1]), (int)to16x2<DT>(s[4 * q + 2], s[4 * q + 3])};
            } else {
              const v2i d2 = *reinterpret_cast<const v2i*>(at);
              const uint16_t d[4] = {(uint16_t)d2[0], (uint16_t)((uint32_t)d2[0] >> 16), (uint16_t)d2[1],
                                     (uint16_t)((uint32_t)d2[1] >> 16)};
              float dg[4], du[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float slope;
                const float act = activate<ACT, true>(acc[o][j][4 * q + e], slope);
                const float dv = from16<DT>(d[e]);
                dg[e] = dv * acc[o + NO][j][4 * q + e] * slope;
                du[e] = dv * act;
                sums[o][4 * q + e] += dg[e];
                sums[o + NO][4 * q + e] += du[e];
              }
              *reinterpret_cast<v2i*>(at) = v2i{(int)to16x2<DT>(dg[0], dg[1]), (int)to16x2<DT>(dg[2], dg[3])};
              *reinterpret_cast<v2i*>(at + AREA) = v2i{(int)to16x2<DT>(du[0], du[1]), (int)to16x2<DT>(du[2], du[3])};
            }
          }
        wave_lds_wait();
#pragma unroll
        for (int k = 0; k < AREAS; ++k) {
          auto run = [&](int p) __attribute__((always_inline)) {
            return *reinterpret_cast<const v4i*>(area + k * AREA + place(p * PER + prow, slot));
          };
          if constexpr (WIDE || MODE == GATED_GRAD) {
#pragma unroll
            for (int p = 0; p < RUNS; ++p) {
              typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
              const uint32_t at = (uint32_t)((32 * j + p * PER + prow) * a.ldo + slot * 8) * 2u;
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, run(p)), k ? o1 : o0,
                                                     (int)(slot * 8 < cols_out ? at : TILE_OOB), 0, MODE == GATED_GRAD ? 0 : STREAM_BIT);
            }
          } else if (whole && slot * 8 + 8 <= cols_out) {
            uint16_t* to = a.out[0] + (mw + 32 * j + prow) * a.ldo + nw + slot * 8;
#pragma unroll 2  // (whole, its addresses spill)
            for (int p = 0; p < RUNS; ++p) *reinterpret_cast<v4i_any*>(to + (int64_t)p * PER * a.ldo) = run(p);
          } else {
#pragma unroll
            for (int p = 0; p < RUNS; ++p) {
              const uint32_t at = (uint32_t)((32 * j + p * PER + prow) * a.ldo + slot * 8) * 2u;
              const v4i v = run(p);
#pragma unroll
              for (int c = 0; c < 8; ++c)
                __builtin_amdgcn_raw_buffer_store_b16((uint16_t)((uint32_t)v[c / 2] >> (16 * (c & 1))), o0,
                                                      (int)(slot * 8 + c < cols_out ? at + 2 * c : TILE_OOB), 0, 0);
            }
          }
        }
        wave_lds_wait();
      }
    };
    if (MODE == GATED_GRAD ? a.wide_dout : a.wide_out) epilogue(std::integral_constant<bool, true>{});
    else epilogue(std::integral_constant<bool, false>{});
    if constexpr (MODE == GATED_GRAD) {
      if (a.col_sums == nullptr) return;
      // lane l: value l % 32 of each 32: block (value / 16), register value % 16
#pragma unroll
      for (int i = 0; i < NB; i += 2) {
        float v[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = sums[i + (q >> 4)][q & 15];
        sum_lanes<16>(v, lane);
        const int blk = i + (frow >> 4), q = frow & 15;
        const int64_t n = nw + 32 * (blk % NO) + 8 * (q >> 2) + 4 * h + (q & 3);
        if (n < a.N) a.col_sums[((int64_t)(tm * 2 + wm) * 2 + blk / NO) * a.N + n] = v[0];
      }
    }
  }
}

}  // namespace fim
