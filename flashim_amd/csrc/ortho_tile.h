// The matrix products of the Newton-Schulz steps on tiles: operands of two FP16 halves, three products of halves each.
//
// A workgroup of four wavefronts (2 x 2) computes 64 MB x 64 MB products on 32 x 32 x 16 MFMAs. The contraction is walked 32 at a
// time: a row's 32 values are a line of 128 bytes, 32 hi and 32 lo, loaded straight into one of NS LDS stages and read in
// 16-byte pieces; X in P X runs across the contraction and is read transposed by the LDS (ds_read_tr16_b64). While the MFMAs of one
// 16-wide sub-step run, the operands of the next are read; the consumed stage is refilled behind the barrier, NS steps ahead.
//
// A and P are symmetric: only tiles on and below the diagonal are computed, and written twice. Where A's are few and its contraction
// is long, that is split, and the partial sums, which lie as the accumulators do, are joined by a launch that does the epilogue.
//
// Bound by the matrix pipes where tiles fill the card: P X of three matrices of 1024 x 4096 73 us, 1060 TFLOP/s of 16-bit
// products, what a library's 8192-cubed FP16 product reached on that card, whose power limit holds the clock to 1.5 to 1.8 GHz;
// of 96 matrices of 512 x 2048 and smaller 100 us, matrix pipes busy 69%. By prologue, epilogue and latency where there are few:
// one of 1024 x 4096 29 us (890), 523 x 196 5 to 7 us a launch.
#pragma once

#include "ortho.h"

namespace fim {

// GRAM: A = X X^T.  SQUARE: P = a I + b A + c A^2.  APPLY: X = P X.  LAST: O = P X, or the parameters' step.
enum { ORTHO_GRAM, ORTHO_SQUARE, ORTHO_APPLY, ORTHO_LAST };

__device__ __forceinline__ v16f mfma_halves(s16x8 a, s16x8 b, v16f c) { return mfma16<FIM_F16>(a, b, c); }

// Neighbouring tiles of an XCD. Whole eighths of the tiles gave some XCDs the long contractions of the first stacks (96 matrices:
// P X 110 us, the last one 192; 102 and 173 with runs of 16 or 32); runs of 4 and 8 share less in the L2 (111 and 110).
constexpr uint32_t ORTHO_RUN = 16;

// Scales of the accumulators, exact but for c's and b's own factors
struct OrthoOut {
  float gram, apply, last, square, old;
  __device__ explicit OrthoOut(const OrthoScalars& k)
      : gram(k.sa / (k.sx * k.sx)), apply(1.0f / k.sp), last(1.0f / (k.sp * k.sx)), square(k.c * k.sp / (k.sa * k.sa)),
        old(k.b * k.sp / k.sa) {}
};

// 32 x 32 products where they go, halves through 4 KB of LDS of this wavefront: whole lines are stored, and those on the other
// side of the diagonal are read transposed (2-byte stores there cost twice the product at m = 1024). Lane l, register q: row
// rb + l % 32, column cb + 8 (q / 4) + 4 (l / 32) + q % 4
template <int MODE>
__device__ __forceinline__ void ortho_block_out(const OrthoStack& s, const OrthoScalars& k, const OrthoOut& o, int b, int64_t at,
                                                int src, int rb, int cb, bool mirror, const v16f& acc,
                                                uint8_t* area) {
  constexpr bool SYM = MODE == ORTHO_GRAM || MODE == ORTHO_SQUARE;
  const int lane = threadIdx.x & 63, row = rb + (lane & 31), c0 = cb + 4 * (lane >> 5);
  if constexpr (MODE == ORTHO_LAST) {
    const int rows = (int)s.rows, cols = (int)s.cols;
    const int64_t base = (int64_t)b * rows * cols;
    // all loads before the stores, which may alias for all the compiler knows
    auto finish = [&](auto dt, auto step_c, auto tall_c) __attribute__((always_inline)) {
      constexpr int DT = decltype(dt)::value;
      constexpr bool STEP = decltype(step_c)::value, TALL = decltype(tall_c)::value;
      float v[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = c0 + 8 * q;
        float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (STEP && !TALL) {
          if (row < rows && col < cols) load4(s.out, base + (int64_t)row * cols + col, DT, cols - col, p);
        } else if constexpr (STEP) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (row < cols && col + u < rows) p[u] = load_elem<DT>(s.out, base + (int64_t)(col + u) * cols + row);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) v[4 * q + u] = p[u];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = c0 + 8 * q;
        float w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          w[u] = acc[4 * q + u] * o.last;
          if (STEP) w[u] = fmaf(-s.factor, w[u], k.keep * v[4 * q + u]);
        }
        if constexpr (!TALL) {
          if (row < rows && col < cols) store4(s.out, base + (int64_t)row * cols + col, DT, cols - col, w);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (row < cols && col + u < rows) store1(s.out, base + (int64_t)(col + u) * cols + row, w[u], DT);
        }
      }
    };
    auto by_side = [&](auto dt, auto step) __attribute__((always_inline)) {
      if (s.tall) finish(dt, step, std::integral_constant<bool, true>{});
      else finish(dt, step, std::integral_constant<bool, false>{});
    };
    auto by_step = [&](auto dt) __attribute__((always_inline)) {
      if (k.step) by_side(dt, std::integral_constant<bool, true>{});
      else by_side(dt, std::integral_constant<bool, false>{});
    };
    if (s.out_type == FIM_F32) by_step(std::integral_constant<int, FIM_F32>{});
    else if (s.out_type == FIM_BF16) by_step(std::integral_constant<int, FIM_BF16>{});
    else by_step(std::integral_constant<int, FIM_F16>{});
  } else {
    uint8_t* to = (MODE == ORTHO_GRAM ? s.a : MODE == ORTHO_SQUARE ? s.p : src ? s.x[0] : s.x[1]) + at;
    const int64_t ld = (int64_t)(SYM ? s.mp : s.np) * 4;
    v2i old[4][2];
    if constexpr (MODE == ORTHO_SQUARE) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint8_t* from = s.a + at + row * ld + line_of(c0 + 8 * q);
        old[q][0] = *reinterpret_cast<const v2i*>(from);
        old[q][1] = *reinterpret_cast<const v2i*>(from + 64);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = c0 + 8 * q;
      float v[4];
      if constexpr (MODE == ORTHO_SQUARE) {
        float z[4];
        join4(old[q][0], old[q][1], z);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[u] = fmaf(o.square, acc[4 * q + u], o.old * z[u]);
          if (row == col + u) v[u] += k.a * k.sp;
        }
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = acc[4 * q + u] * (MODE == ORTHO_GRAM ? o.gram : o.apply);
      }
      v2i hi, lo;
      split4(v, hi, lo);
      const int r = lane & 31;
      uint8_t* put = area + r * 128 + 8 * (lane >> 5);
      *reinterpret_cast<v2i*>(put + ((q ^ (r & 7)) << 4)) = hi;
      *reinterpret_cast<v2i*>(put + (((4 + q) ^ (r & 7)) << 4)) = lo;
    }
    wave_lds_wait();
    v4i w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const v4i*>(area + i * 1024 + lane * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 3);
      *reinterpret_cast<v4i*>(to + (rb + r) * ld + (cb >> 5) * 128 + (((lane & 7) ^ (r & 7)) << 4)) = w[i];
    }
    if (SYM && mirror) {
      const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // 16 columns of a plane: lane: column l % 16, rows 8 (l / 16) ..
        const int plane = i >> 1, c16 = i & 1, seg = 4 * plane + 2 * c16 + ((lane & 3) >> 1);
        s16x4 half[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int r = 8 * g + 4 * t + (l16 >> 2);
          half[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(area + r * 128 + ((seg ^ (r & 7)) << 4) + (lane & 1) * 8));
        }
        *reinterpret_cast<s16x8*>(to + (cb + 16 * c16 + l16) * ld + (rb >> 5) * 128 + plane * 64 + g * 16) =
            __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
    wave_lds_wait();  // (the area is written again)
  }
}

// Tile t of tm (tm + 1) / 2 + tn, tn <= tm
__device__ __forceinline__ void triangle(int t, int& tm, int& tn) {
  tm = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
  if ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
  if (tm * (tm + 1) / 2 > t) --tm;
  tm = __builtin_amdgcn_readfirstlane(tm);
  tn = t - tm * (tm + 1) / 2;
}

// splits > 1 (SYM): part[split][tile][64 MB x 64 MB] FP32 in place of the epilogue
template <int MODE, int MB, int NS>
__global__ __launch_bounds__(256, 128 * MB * 128 * NS > 80 * 1024 ? 1 : 2) void ortho_tile_kernel(
    const OrthoStack* __restrict__ table, int count, uint32_t tiles, int splits, float* __restrict__ part, int src, OrthoScalars k) {
  constexpr bool SYM = MODE == ORTHO_GRAM || MODE == ORTHO_SQUARE;
  constexpr bool WT = !SYM;  // the second operand runs across the contraction
  constexpr int NB = MB, BM = 64 * MB, BN = 64 * NB, OPERAND = BM * 128, STAGE = (BM + BN) * 128;
  constexpr int CX = BM / 32, CW = BN / 32;  // 1 KB loads of a stage per wavefront
  static_assert(NS == 2 || NS == 4, "stages");
  __shared__ __attribute__((aligned(16))) uint8_t st0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t st1[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t st2[NS > 2 ? STAGE : 16];
  __shared__ __attribute__((aligned(16))) uint8_t st3[NS > 2 ? STAGE : 16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, h = lane >> 5;

  // workgroups go round the 8 XCDs: each takes runs of ORTHO_RUN tiles, which share operands in its L2
  uint32_t t = ((blockIdx.x >> 3) / ORTHO_RUN * 8 + (blockIdx.x & 7)) * ORTHO_RUN + (blockIdx.x >> 3) % ORTHO_RUN;
  if (t >= tiles * (SYM ? splits : 1)) return;
  const int split = SYM ? __builtin_amdgcn_readfirstlane((int)(t / tiles)) : 0;
  t -= split * tiles;
  constexpr int PASS = MODE == ORTHO_GRAM ? 2 : MODE == ORTHO_SQUARE ? 3 : 4;
  const int e = stack_of(table, count, PASS, t);
  const OrthoStack s = table[e];  // (a copy: a reference would be read again after every store)
  const int mp = (int)s.mp, np = (int)s.np;
  const int mt = (mp + BM - 1) / BM, nt = (np + BN - 1) / BN, per = SYM ? mt * (mt + 1) / 2 : mt * nt;
  uint32_t local = t - s.first[PASS];
  const int b = __builtin_amdgcn_readfirstlane((int)(local / per));
  const int tile = __builtin_amdgcn_readfirstlane((int)(local - (uint32_t)b * per));
  int tm, tn;
  if constexpr (SYM) {
    triangle(tile, tm, tn);
  } else {  // m tiles of one column block follow each other
    tn = tile / mt;
    tm = tile - tn * mt;
    tn = __builtin_amdgcn_readfirstlane(tn);
    tm = __builtin_amdgcn_readfirstlane(tm);
  }
  const int m0 = tm * BM, n0 = tn * BN;
  const int64_t at = b * s.each;
  const uint8_t* X = (src ? s.x[1] : s.x[0]) + at;
  const uint8_t* first = MODE == ORTHO_GRAM ? X : MODE == ORTHO_SQUARE ? s.a + at : s.p + at;
  const uint8_t* second = MODE == ORTHO_SQUARE ? s.a + at : X;
  const int K = MODE == ORTHO_GRAM ? np : mp;  // multiples of 32
  const int all = K >> 5, from = all * split / splits, steps = all * (split + 1) / splits - from;  // (splits is 1 unless SYM)
  const int ld1 = (MODE == ORTHO_GRAM ? np : mp) * 4, ld2 = (MODE == ORTHO_SQUARE ? mp : np) * 4;  // bytes of a row

  // -- loads into LDS: chunk c (1 KB), wavefront w loads chunks w, w + 4, ...
  // along: lane l loads row 8 c + l / 8, LDS slot l % 8, which holds segment slot ^ (row / 2 % 8) of the line
  const int seg = (lane & 7) ^ (lane >> 4) ^ (4 * (wave & 1));
  const int xrows = mp - m0 < BM ? mp - m0 : BM, wrows = (SYM ? mp : np) - n0 < BN ? (SYM ? mp : np) - n0 : BN;
  uint32_t xo[CX], wo[CW];
#pragma unroll
  for (int i = 0; i < CX; ++i) {
    const int r = 8 * (wave + 4 * i) + (lane >> 3);
    xo[i] = r < xrows ? (uint32_t)(r * ld1) + seg * 16 : TILE_OOB;
  }
#pragma unroll
  for (int i = 0; i < CW; ++i) {
    const int c = wave + 4 * i, r = 8 * c + (lane >> 3);
    if constexpr (WT) {  // across: a row of the stage is BN / 32 lines; slot q of row r holds segment q ^ 4 (r % 4)
      constexpr int SLOTS = BN / 4;
      const int row = c * 64 / SLOTS + (SLOTS < 64 ? lane / SLOTS : 0), slot = lane % SLOTS;
      const int q = slot ^ ((row & 3) << 2);
      wo[i] = q * 4 < wrows ? (uint32_t)(row * ld2) + q * 16 : TILE_OOB;
    } else {
      wo[i] = r < wrows ? (uint32_t)(r * ld2) + seg * 16 : TILE_OOB;
    }
  }
  const uint8_t* xbase = first + (int64_t)m0 * ld1;
  const uint8_t* wbase = WT ? second + n0 * 4 : second + (int64_t)n0 * ld2;
  const int xbytes = xrows * ld1, wbytes = WT ? mp * ld2 - n0 * 4 : wrows * ld2;
  // (from is 0 where w runs across) past the last step everything reads as zero
  uint32_t xk = from * 128, wk = from * 128, dead = 0 < steps ? 0u : TILE_OOB;
  int step_at = 0;
  auto next_step = [&]() __attribute__((always_inline)) {
    ++step_at;
    xk += 128;
    wk += WT ? 32u * ld2 : 128u;
    dead = step_at < steps ? 0u : TILE_OOB;
  };
  auto load = [](const uint8_t* p, int records, uint8_t* to, uint32_t off) __attribute__((always_inline)) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, __builtin_amdgcn_readfirstlane(records), 0x00020000),
        (lds_void*)to, 16, off, 0, 0, 0);
  };
  auto issue = [&](uint8_t* st, int i) __attribute__((always_inline)) {
    if (i < CX) load(xbase, xbytes, st + (wave + 4 * i) * 1024, (xo[i] + xk) | dead);
    else if (i < CX + CW) load(wbase, wbytes, st + OPERAND + (wave + 4 * (i - CX)) * 1024, (wo[i - CX] + wk) | dead);
  };

  // -- operand fragments: lane l holds row (or column) l % 32 of a block, contraction 8 h .. 8 h + 7 of a 16-wide sub-step
  const int frow = lane & 31, fsw = (frow >> 1) & 7;
  const int tq = (lane & 15) >> 2, tcol = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  auto read_along = [&](const uint8_t* st, int from, int row0, int kk, int plane) __attribute__((always_inline)) {
    const int off = from + (row0 + frow) * 128 + (((4 * plane + 2 * kk + h) ^ fsw) << 4);
    return *reinterpret_cast<const s16x8*>(st + off);
  };
  auto read_across = [&](const uint8_t* st, int blk, int kk, int plane) __attribute__((always_inline)) {
    constexpr int ROWB = BN * 4;
    const int off = OPERAND + (kk * 16 + 8 * h + tq) * ROWB + (((2 * blk + plane) ^ tq) << 6) + tcol;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + off));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + (off + 4 * ROWB)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  s16x8 fx[2][MB][2], fw[2][NB][2];
  // read r of a sub-step's 2 (MB + NB) into set f
  auto read = [&](const uint8_t* st, int f, int kk, int r) __attribute__((always_inline)) {
    const int plane = r & 1;
    if (r < 2 * NB) {
      const int i = r >> 1;
      if constexpr (WT) fw[f][i][plane] = read_across(st, wn * NB + i, kk, plane);
      else fw[f][i][plane] = read_along(st, OPERAND, (wn * NB + i) * 32, kk, plane);
    } else {
      const int i = (r >> 1) - NB;
      fx[f][i][plane] = read_along(st, 0, (wm * MB + i) * 32, kk, plane);
    }
  };

  // accumulators: lane l, register q of block (i, j): row 32 j + l % 32, column 32 i + 8 (q / 4) + 4 h + q % 4
  v16f acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  constexpr int T = 3 * MB * NB, READS = 2 * (MB + NB), LOADS = CX + CW;
  auto sub_step = [&](int f, const uint8_t* rd, int rkk, uint8_t* fill, bool loads) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < T; ++m) {
      // the three products of a block lie MB NB apart: none waits for the one before
      const int i = m % NB, j = (m / NB) % MB, third = m / (MB * NB);
      acc[i][j] = mfma_halves(fw[f][i][third == 2], fx[f][j][third == 1], acc[i][j]);
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * T / READS == m) read(rd, 1 - f, rkk, r);
#pragma unroll
      for (int l = 0; l < LOADS; ++l)
        if (loads && l * T / LOADS == m) issue(fill, l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // one step from stage cur, which is refilled for NS steps on
  auto step = [&](uint8_t* cur, uint8_t* nxt) __attribute__((always_inline)) {
    sub_step(0, cur, 1, cur, false);
    __builtin_amdgcn_s_waitcnt(tile_wait((NS - 2) * LOADS));  // nxt has landed, cur has been read
    asm volatile("s_barrier" ::: "memory");
    sub_step(1, nxt, 0, cur, true);
    next_step();
  };
  uint8_t* const stages[4] = {st0, st1, st2, st3};
#pragma unroll
  for (int n = 0; n < NS; ++n) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) issue(stages[n], l);
    next_step();
  }
  __builtin_amdgcn_s_waitcnt(tile_wait((NS - 1) * LOADS));
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int r = 0; r < READS; ++r) read(st0, 0, 0, r);
  // NS steps a turn, one exit: a step past the last multiplies zeros
  for (int i = 0; i < steps; i += NS) {
    step(st0, st1);
    if constexpr (NS == 2) {
      step(st1, st0);
    } else {
      step(st1, st2);
      step(st2, st3);
      step(st3, st0);
    }
  }
  __builtin_amdgcn_s_waitcnt(tile_wait(0));
  asm volatile("s_barrier" ::: "memory");

  // -- epilogue
  if (SYM && splits > 1) {
    float* to = part + ((int64_t)split * tiles + t) * (BM * BN) + lane * 4;
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v4f*>(to + ((((wm * MB + j) * 2 * NB + wn * NB + i) * 4) + q) * 256) =
              v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    return;
  }
  const OrthoOut o(k);
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int rb = m0 + (wm * MB + j) * 32;
    if (rb >= mp) continue;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int cb = n0 + (wn * NB + i) * 32;
      if (cb >= (SYM ? mp : np)) continue;
      ortho_block_out<MODE>(s, k, o, b, at, src, rb, cb, tm != tn, acc[i][j], st0 + wave * 4096);
    }
  }
}

// The splits' partial sums of A's tiles of 128 added up in order, and the epilogue: a 32 x 32 block a wavefront
__global__ __launch_bounds__(256) void ortho_join_kernel(const OrthoStack* __restrict__ table, int count, uint32_t tiles, int splits,
                                                         const float* __restrict__ part, OrthoScalars k) {
  constexpr int BM = 128;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * 4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t t = blockIdx.x >> 2;
  const int block = (int)(blockIdx.x & 3) * 4 + wave;
  const OrthoStack s = table[stack_of(table, count, 2, t)];
  const int mp = (int)s.mp, mt = (mp + BM - 1) / BM, per = mt * (mt + 1) / 2;
  const uint32_t local = t - s.first[2];
  const int b = __builtin_amdgcn_readfirstlane((int)(local / per));
  int tm, tn;
  triangle(__builtin_amdgcn_readfirstlane((int)(local - (uint32_t)b * per)), tm, tn);
  const int rb = tm * BM + (block >> 2) * 32, cb = tn * BM + (block & 3) * 32;
  if (rb >= mp || cb >= mp) return;
  const float* from = part + (int64_t)t * (BM * BM) + block * 1024 + lane * 4;
  v16f acc;
#pragma unroll
  for (int q = 0; q < 16; ++q) acc[q] = 0.0f;
#pragma unroll 4
  for (int n = 0; n < splits; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const v4f v = *reinterpret_cast<const v4f*>(from + (int64_t)n * tiles * (BM * BM) + q * 256);
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[4 * q + u] += v[u];
    }
  ortho_block_out<ORTHO_GRAM>(s, k, OrthoOut(k), b, b * s.each, 0, rb, cb, tm != tn, acc, lds + wave * 4096);
}

}  // namespace fim
