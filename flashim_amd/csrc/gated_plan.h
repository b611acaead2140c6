// The gated feed-forward product's plans, on the host: which form a call takes, on which tiles, in how many splits, and what
// lies where in its workspace.
#pragma once

#include "gated_few.h"
#include "gated_rows.h"
#include "gated_rows_grad.h"
#include "gated_tile.h"

namespace fim {

inline int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// A [rows, cols] operand as the caller has it
struct Matrix {
  const uint16_t* p;
  int64_t ld, rows, cols;
  // The tile kernels read 16-byte runs at 32-bit offsets inside a tile; other operands are copied first
  bool as_is() const {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld >= cols && ld < (1 << 22);
  }
  int64_t padded() const { return cdiv(cols, 8) * 8; }
  int64_t copy_bytes() const { return as_is() ? 0 : align256(rows * padded() * 2); }
};

inline Matrix matrix(const void* p, int64_t ld, int64_t rows, int64_t cols) {
  return {static_cast<const uint16_t*>(p), rows == 1 ? cols : ld, rows, cols};
}

struct Tile { int mb, nb; };

// The time of a product of `rows` x `cols` outputs over `k` on a tile, in steps of a 128 x 128 tile (0.9 us). A round of 256
// x 256 tiles, one per CU, measured 1.4 us a step and 9 us beside (prologue, epilogue); of 128 x 128 tiles, two per CU, which
// read the operands twice as often but cover each other's prologue and epilogue, 0.9 us and 3 us. (Large and small, 16384 x
// 1024 x 8192 outputs: 255 and 280 us; 20000 x 512 x 4096, which the estimate gives to the small ones: 99 and 101 with GELU, 90 and
// 94 with SiLU; 16384 x 8192 x 1024: 208 and 287, in FP16 237 and 292.)
inline double tile_time(Tile t, int64_t rows, int64_t cols, int64_t splits, int64_t k) {
  const int64_t cus = device_cus(), size = 64 * t.mb;
  const int64_t rounds = cdiv(cdiv(rows, size) * cdiv(cols, size) * splits, cus);
  const double steps = (double)cdiv(k, TILE_K);
  // (a last small tile alone on its CU takes more than half the time of two)
  return t.mb == 4 ? rounds * (1.6 * steps + 10.0) : (0.5 * rounds + 0.1 * (rounds & 1)) * (steps + 3.0);
}

inline Tile gated_tile(int64_t rows, int64_t cols, int64_t k) {
  const Tile large{4, 4}, small{2, 2};
  return tile_time(large, rows, cols, 1, k) < tile_time(small, rows, cols, 1, k) ? large : small;
}

struct Splits {
  Tile tile;
  int64_t n;
};

// Tile and splits of the contraction of `cols` x `rows` outputs over k, where splits are joined (their FP32 partials written
// and read once, at 4.5 TB/s, and a launch); `alone`: one split needs no join
inline Splits split_plan(int64_t rows, int64_t cols, int64_t k, bool alone) {
  Splits best{{2, 2}, 0};
  double best_time = 0.0;
  for (const Tile t : {Tile{4, 4}, Tile{2, 2}}) {
    for (int64_t s = 1; s <= 256 && (s == 1 || k / s >= 256); s += s < 8 ? 1 : s / 4) {
      const double join = s == 1 && alone ? 0.0 : (double)(s + 1) * rows * cols * 4.0 / 4.5e6 + 3.0;  // us
      const double time = 0.9 * tile_time(t, rows, cols, s, cdiv(k, s)) + join;
      if (best.n != 0 && time >= best_time) continue;
      best_time = time;
      best = {t, s};
    }
  }
  return best;
}

// Whether the backward pass is (gated_rows_grad.h): all weights fit one workgroup's LDS, any number of rows. (Kernels of a call,
// 1000 x 64 -> 256: 20 us, 29 on tiles; 24000: 38 and 45; 320000: 156 and 337.)
inline bool gated_rows_grad(int64_t K, int64_t H) { return K <= 64 && H <= GRAD_HIDDEN; }

// Hidden columns of a block of the forward pass by rows
inline int64_t rows_block(int64_t K) { return rows_hidden(K <= 64 ? 64 : 128); }

inline int64_t rows_blocks(int64_t K, int64_t H) { return cdiv(H, rows_block(K)); }

// Whether the forward pass is a stream of rows (gated_rows.h): a short contraction, and outputs enough that its workgroups' way
// through all hidden columns of 256 rows at a time fills the chip. On rows and on tiles (BF16, SiLU and GELU, us): 32768 x 64 ->
// 256, 15.0 and 11.3; 40000, 15.0 and 14.5; 49152, 15.6 and 16.3; 16384 x 64 -> 1024, 16.2 and 20.8; 8192, 13.6 and 12.3; 81920 x
// 16 -> 64, 8.9 and 10.8; 32768 x 128 -> 512, 21.7 and 20.8; 49152, 26.5 and 29.9; 24576 x 128 -> 1024, 26.6 and 29.5; 81920 x 128
// -> 128, 19.1 and 13.9; 196608, 29.7 and 33.6. Over 364 sizes the form it takes is 0.3% slower on average than the faster one
// (19% at most). Fewer rows than 8192 were not measured.
inline bool gated_rows(int64_t M, int64_t K, int64_t H) {
  const int64_t width = H > rows_block(K) ? H : rows_block(K);
  return K <= 128 && M >= 8192 && M * width >= (K <= 64 ? 40000 : 80000) * (int64_t)device_cus();
}

// Workgroups per hidden block: one per CU over all blocks
inline int64_t rows_groups(int64_t M, int64_t K, int64_t H) {
  const int64_t most = cdiv(M, 32 * ROWS_WAVES), n = device_cus() / rows_blocks(K, H);
  return n < 1 ? 1 : n < most ? n : most;
}

// Workgroups of a backward pass by rows: one per CU at most, fewer where the steps saved (3.7 us each) would cost less than the
// partial weight gradients they leave (written, then joined, at 5 TB/s)
inline int64_t rows_grad_groups(int64_t M, int64_t K, int64_t H) {
  const int64_t steps = cdiv(M, 32 * rows_grad_sub(H));
  const double part = rows_grad_sub(H) * 2.0 * H * K * 4 * 2 / 5e6;  // us
  int64_t best = 0;
  double best_time = 0.0;
  for (int64_t rounds = cdiv(steps, device_cus()), i = 0; i < 16; ++rounds, ++i) {
    const int64_t groups = cdiv(steps, rounds);
    const double time = 3.7 * rounds + part * groups;
    if (best != 0 && time >= best_time) continue;
    best_time = time;
    best = groups;
  }
  return best;
}

enum GatedForm { FORM_FEW, FORM_ROWS, FORM_TILES };

struct Gated {
  Matrix x, wg, wu;
  int64_t M, K, H;
  GatedForm form;  // of the forward pass
  Tile forward;
  // workspace, in bytes: copies of the operands; backward: dg and du [M, hp], bias partials, weight partials
  int64_t x_at, wg_at, wu_at, dgu_at, cols_at, part_at, total;
  int64_t hp, ldg, sum_rows;
  int64_t dw_splits, dw_rows, dx_splits, dx_steps;  // splits, and what each contracts over
  Tile grad, dw, dx;
  bool rows;  // backward by rows: no dg, du in memory
};

inline Gated gated_plan(const Matrix& x, const Matrix& wg, const Matrix& wu, bool backward) {
  Gated g{};
  g.x = x;
  g.wg = wg;
  g.wu = wu;
  g.M = x.rows;
  g.K = x.cols;
  g.H = wg.rows;
  // both weights are read with one stride
  const bool copy_w = !wg.as_is() || !wu.as_is() || wg.ld != wu.ld;
  g.x_at = 0;
  if (!backward) {
    g.form = g.M <= FEW_ROWS ? FORM_FEW : gated_rows(g.M, g.K, g.H) ? FORM_ROWS : FORM_TILES;
    g.forward = gated_tile(g.M, 2 * g.H, g.K);
    if (g.form == FORM_FEW) return g;  // any rows are read in place
  }
  g.wg_at = g.x_at + x.copy_bytes();
  g.wu_at = g.wg_at + (copy_w ? align256(g.H * wg.padded() * 2) : 0);
  g.total = g.wu_at + (copy_w ? align256(g.H * wg.padded() * 2) : 0);
  g.hp = cdiv(g.H, 8) * 8;
  // whole 128-byte lines, one more than fit: rows of a power of two apart would meet in the same cache sets and channels
  g.ldg = cdiv(g.H, 64) * 64 + 64;
  if (!backward) return g;
  g.dgu_at = g.total;
  g.rows = gated_rows_grad(g.K, g.H);
  if (g.rows) {
    g.sum_rows = g.dw_splits = rows_grad_groups(g.M, g.K, g.H) * rows_grad_sub(g.H);
    g.cols_at = g.dgu_at;
    g.part_at = g.cols_at + align256(g.sum_rows * 2 * g.H * 4);
    g.total = g.part_at + align256(g.dw_splits * 2 * g.H * g.K * 4);
    return g;
  }
  g.grad = {2, 2};  // (its epilogue has no registers left beside 256 x 256 accumulators)
  g.cols_at = g.dgu_at + align256(2 * g.M * g.ldg * 2);
  g.sum_rows = 2 * cdiv(g.M, 64 * g.grad.mb);
  g.part_at = g.cols_at + align256(g.sum_rows * 2 * g.H * 4);
  // (the weights' gradients have both halves' tiles)
  const Splits dw = split_plan(g.K, 2 * cdiv(g.H, 128) * 128, g.M, false);
  g.dw = dw.tile;
  g.dw_rows = cdiv(cdiv(g.M, dw.n), TILE_K) * TILE_K;
  g.dw_splits = cdiv(g.M, g.dw_rows);
  const int64_t steps = 2 * cdiv(g.H, TILE_K);
  const Splits dx = split_plan(g.M, g.K, steps * TILE_K, true);
  g.dx = dx.tile;
  g.dx_steps = cdiv(steps, dx.n);
  g.dx_splits = cdiv(steps, g.dx_steps);
  // one area for both products' partials, one after the other
  const int64_t dw_bytes = g.dw_splits * 2 * g.H * g.K * 4;
  const int64_t dx_bytes = g.dx_splits == 1 ? 0 : g.dx_splits * g.M * g.K * 4;
  g.total = g.part_at + align256(dw_bytes > dx_bytes ? dw_bytes : dx_bytes);
  return g;
}

}  // namespace fim
