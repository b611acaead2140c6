// The matrix products of the Newton-Schulz steps on tiles: operands of two FP16 halves, three products of halves each.
//
// A workgroup of four wavefronts (2 x 2) computes 64 MB x 64 MB products on 32 x 32 x 16 MFMAs. The contraction is walked 32 at a
// time: a row's 32 values are a line of 128 bytes, 32 hi and 32 lo, loaded straight into one of two LDS stages and read in
// 16-byte pieces; X in P X runs across the contraction and is read transposed by the LDS (ds_read_tr16_b64). While the MFMAs of one
// 16-wide sub-step run, the operands of the next are read; the consumed stage is refilled behind the barrier, two steps ahead.
//
// A and P are symmetric: only tiles on and below the diagonal are computed, and written twice.
#pragma once

#include "ortho.h"

namespace fim {

// GRAM: A = X X^T.  SQUARE: P = a I + b A + c A^2.  APPLY: X = P X.  LAST: O = P X, or the parameters' step.
enum { ORTHO_GRAM, ORTHO_SQUARE, ORTHO_APPLY, ORTHO_LAST };

__device__ __forceinline__ v16f mfma_halves(s16x8 a, s16x8 b, v16f c) { return mfma16<FIM_F16>(a, b, c); }

template <int MODE, int MB>
__global__ __launch_bounds__(256, MB > 2 ? 1 : 2) void ortho_tile_kernel(const OrthoStack* __restrict__ table, int count,
                                                                         uint32_t tiles, int src, OrthoScalars k) {
  constexpr bool SYM = MODE == ORTHO_GRAM || MODE == ORTHO_SQUARE;
  constexpr bool WT = !SYM;  // the second operand runs across the contraction
  constexpr int BM = 64 * MB, OPERAND = BM * 128, CH = BM / 32;  // CH: 1 KB loads of an operand's stage per wavefront
  __shared__ __attribute__((aligned(16))) uint8_t st0[2 * OPERAND];
  __shared__ __attribute__((aligned(16))) uint8_t st1[2 * OPERAND];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, h = lane >> 5;

  // workgroups go round the 8 XCDs: each takes a contiguous run of tiles
  const uint32_t t = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (t >= tiles) return;
  const int e = stack_of(table, count, SYM ? 2 : 3, t);
  const OrthoStack& s = table[e];
  const int mp = (int)s.mp, np = (int)s.np;
  const int mt = (mp + BM - 1) / BM, nt = (np + BM - 1) / BM, per = SYM ? mt * (mt + 1) / 2 : mt * nt;
  uint32_t local = t - s.first[SYM ? 2 : 3];
  const int b = __builtin_amdgcn_readfirstlane((int)(local / per));
  const int tile = __builtin_amdgcn_readfirstlane((int)(local - (uint32_t)b * per));
  int tm, tn;
  if constexpr (SYM) {  // tile = tm (tm + 1) / 2 + tn, tn <= tm
    tm = (int)((sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f);
    if ((tm + 1) * (tm + 2) / 2 <= tile) ++tm;
    if (tm * (tm + 1) / 2 > tile) --tm;
    tm = __builtin_amdgcn_readfirstlane(tm);
    tn = tile - tm * (tm + 1) / 2;
  } else {  // m tiles of one column block follow each other
    tn = tile / mt;
    tm = tile - tn * mt;
    tn = __builtin_amdgcn_readfirstlane(tn);
    tm = __builtin_amdgcn_readfirstlane(tm);
  }
  const int m0 = tm * BM, n0 = tn * BM;
  const int64_t at = b * s.each;
  const uint8_t* X = s.x[src] + at;
  const uint8_t* first = MODE == ORTHO_GRAM ? X : MODE == ORTHO_SQUARE ? s.a + at : s.p + at;
  const uint8_t* second = MODE == ORTHO_SQUARE ? s.a + at : X;
  const int K = MODE == ORTHO_GRAM ? np : mp;  // multiples of 32
  const int steps = K >> 5;
  const int ld1 = (MODE == ORTHO_GRAM ? np : mp) * 4, ld2 = (MODE == ORTHO_SQUARE ? mp : np) * 4;  // bytes of a row

  // -- loads into LDS: chunk c (1 KB), wavefront w loads chunks w, w + 4, ...
  // along: lane l loads row 8 c + l / 8, LDS slot l % 8, which holds segment slot ^ (row / 2 % 8) of the line
  const int seg = (lane & 7) ^ (lane >> 4) ^ (4 * (wave & 1));
  const int xrows = mp - m0 < BM ? mp - m0 : BM, wrows = (SYM ? mp : np) - n0 < BM ? (SYM ? mp : np) - n0 : BM;
  uint32_t xo[CH], wo[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = wave + 4 * i, r = 8 * c + (lane >> 3);
    xo[i] = r < xrows ? (uint32_t)(r * ld1) + seg * 16 : TILE_OOB;
    if constexpr (WT) {  // across: a row of the stage is BM / 32 lines; slot q of row r holds segment q ^ 4 (r % 4)
      constexpr int SLOTS = BM / 4;
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
  uint32_t xk = 0, wk = 0, dead = 0;  // past the last step everything reads as zero
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
    if (i < CH) load(xbase, xbytes, st + (wave + 4 * i) * 1024, (xo[i] + xk) | dead);
    else if (i < 2 * CH) load(wbase, wbytes, st + OPERAND + (wave + 4 * (i - CH)) * 1024, (wo[i - CH] + wk) | dead);
  };

  // -- operand fragments: lane l holds row (or column) l % 32 of a block, contraction 8 h .. 8 h + 7 of a 16-wide sub-step
  const int frow = lane & 31, fsw = (frow >> 1) & 7;
  const int tq = (lane & 15) >> 2, tcol = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  auto read_along = [&](const uint8_t* st, int from, int row0, int kk, int plane) __attribute__((always_inline)) {
    const int off = from + (row0 + frow) * 128 + (((4 * plane + 2 * kk + h) ^ fsw) << 4);
    return *reinterpret_cast<const s16x8*>(st + off);
  };
  auto read_across = [&](const uint8_t* st, int blk, int kk, int plane) __attribute__((always_inline)) {
    constexpr int ROWB = BM * 4;
    const int off = OPERAND + (kk * 16 + 8 * h + tq) * ROWB + (((2 * blk + plane) ^ tq) << 6) + tcol;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + off));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + (off + 4 * ROWB)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  s16x8 fx[2][MB][2], fw[2][MB][2];
  // read r of a sub-step's 4 MB into set f
  auto read = [&](const uint8_t* st, int f, int kk, int r) __attribute__((always_inline)) {
    const int i = (r >> 1) % MB, plane = r & 1;
    if (r < 2 * MB) {
      if constexpr (WT) fw[f][i][plane] = read_across(st, wn * MB + i, kk, plane);
      else fw[f][i][plane] = read_along(st, OPERAND, (wn * MB + i) * 32, kk, plane);
    } else {
      fx[f][i][plane] = read_along(st, 0, (wm * MB + i) * 32, kk, plane);
    }
  };

  // accumulators: lane l, register q of block (i, j): row 32 j + l % 32, column 32 i + 8 (q / 4) + 4 h + q % 4
  v16f acc[MB][MB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  constexpr int T = 3 * MB * MB, READS = 4 * MB, LOADS = 2 * CH;
  auto sub_step = [&](int f, const uint8_t* rd, int rkk, uint8_t* fill, bool loads) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < T; ++m) {
      // the three products of a block lie MB * MB apart: none waits for the one before
      const int i = m % MB, j = (m / MB) % MB, part = m / (MB * MB);
      acc[i][j] = mfma_halves(fw[f][i][part == 2], fx[f][j][part == 1], acc[i][j]);
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * T / READS == m) read(rd, 1 - f, rkk, r);
#pragma unroll
      for (int l = 0; l < LOADS; ++l)
        if (loads && l * T / LOADS == m) issue(fill, l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // one step from stage cur, which is refilled for the step after the next
  auto step = [&](uint8_t* cur, uint8_t* nxt) __attribute__((always_inline)) {
    sub_step(0, cur, 1, cur, false);
    __builtin_amdgcn_s_waitcnt(tile_wait(0));  // nxt has landed, cur has been read
    asm volatile("s_barrier" ::: "memory");
    sub_step(1, nxt, 0, cur, true);
    next_step();
  };
#pragma unroll
  for (int l = 0; l < LOADS; ++l) issue(st0, l);
  next_step();
#pragma unroll
  for (int l = 0; l < LOADS; ++l) issue(st1, l);
  next_step();
  __builtin_amdgcn_s_waitcnt(tile_wait(LOADS));
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int r = 0; r < READS; ++r) read(st0, 0, 0, r);
  // pairs of steps: one exit; a step past the last multiplies zeros
  for (int i = 0; i < steps; i += 2) {
    step(st0, st1);
    step(st1, st0);
  }
  __builtin_amdgcn_s_waitcnt(tile_wait(0));

  // -- epilogue; exact scales but for c's and b's own factors
  const float gram_scale = k.sa / (k.sx * k.sx), apply_scale = 1.0f / k.sp, last_scale = apply_scale / k.sx;
  const float sq_scale = k.c * k.sp / (k.sa * k.sa), old_scale = k.b * k.sp / k.sa;
  uint8_t* to = (MODE == ORTHO_GRAM ? s.a : MODE == ORTHO_SQUARE ? s.p : s.x[1 - src]) + at;
  const int cols = SYM ? mp : np, ld = cols * 4;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int rb = m0 + (wm * MB + j) * 32, row = rb + frow;
    if (rb >= mp) continue;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int cb = n0 + (wn * MB + i) * 32;
      if (cb >= cols) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = cb + 8 * q + 4 * h;
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = acc[i][j][4 * q + u];
        if constexpr (MODE == ORTHO_LAST) {
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] *= last_scale;
          const int64_t base = (int64_t)b * s.rows * s.cols;
          if (s.tall) {
            if (row < (int)s.cols) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (col + u < (int)s.rows) finish1(s, k, base + (int64_t)(col + u) * s.cols + row, v[u]);
            }
          } else if (row < (int)s.rows && col < (int)s.cols) {
            finish4(s, k, base + (int64_t)row * s.cols + col, (int)s.cols - col, v);
          }
        } else {
          const int off = line_of(col);
          if constexpr (MODE == ORTHO_SQUARE) {
            const uint8_t* from = s.a + at + (int64_t)row * ld + off;
            float old[4];
            join4(*reinterpret_cast<const v2i*>(from), *reinterpret_cast<const v2i*>(from + 64), old);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              v[u] = fmaf(sq_scale, v[u], old_scale * old[u]);
              if (row == col + u) v[u] += k.a * k.sp;
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] *= MODE == ORTHO_GRAM ? gram_scale : apply_scale;
          }
          v2i hi, lo;
          split4(v, hi, lo);
          uint8_t* p = to + (int64_t)row * ld + off;
          *reinterpret_cast<v2i*>(p) = hi;
          *reinterpret_cast<v2i*>(p + 64) = lo;
          if (SYM && tm != tn) {  // the tile on the other side of the diagonal
            const s16x4 a4 = __builtin_bit_cast(s16x4, hi), b4 = __builtin_bit_cast(s16x4, lo);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              int16_t* o = reinterpret_cast<int16_t*>(to + (int64_t)(col + u) * ld + line_of(row));
              o[0] = a4[u];
              o[32] = b4[u];
            }
          }
        }
      }
    }
  }
}

}  // namespace fim
