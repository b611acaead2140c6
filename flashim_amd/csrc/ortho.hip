// Orthogonalized matrices by Newton-Schulz products, and the optimizer step made of them (formulas and precision: ortho.h).
//
// Matrices come as stacks of one shape, many stacks a call; a table of them goes through kernel arguments into the workspace
// (no upload: capturable), and every launch after that runs over all matrices at once. Small ones take one launch, a workgroup
// each, and longer ones of as few rows a launch a step (ortho_small.h); the others a pass that updates the momentum and sums
// squares, one that writes sx X0 as halves (transposing tall matrices), and three launches of products a step (ortho_tile.h), the
// last of which writes O or steps the parameters. The two passes are bound by memory, at what a large copy reaches: three
// matrices of 1024 x 4096 (BF16 gradients, FP32 momenta) 126 MB each way in 24 and 25 us, 5.1 TB/s; 96 matrices of 33M elements in
// FP32 401 MB in 68 and 75 us.
#include <string.h>

#include "ortho_small.h"
#include "ortho_tile.h"

namespace fim {

constexpr int ORTHO_T = 256, ORTHO_FILL = 28;
struct OrthoFill {
  OrthoStack s[ORTHO_FILL];
};
static_assert(sizeof(OrthoFill) <= 4000, "kernel arguments");

__global__ __launch_bounds__(ORTHO_T) void ortho_fill_kernel(const OrthoFill f, OrthoStack* table, int n) {
  constexpr int WORDS = sizeof(OrthoStack) / 4;
  const uint32_t* from = reinterpret_cast<const uint32_t*>(&f);
  uint32_t* to = reinterpret_cast<uint32_t*>(table);
  for (int i = threadIdx.x; i < n * WORDS; i += ORTHO_T) to[i] = from[i];
}

__device__ __forceinline__ double ortho_sum(double v) {
  __shared__ double red[ORTHO_T / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < ORTHO_T / 64; ++i) v += red[i];
  return v;
}

// Momentum in place, and each chunk's sum of squares of U
__global__ __launch_bounds__(ORTHO_T) void ortho_momentum_kernel(const OrthoStack* __restrict__ table, int count,
                                                                 const OrthoScalars k) {
  const OrthoStack s = table[stack_of(table, count, 0, blockIdx.x)];
  const uint32_t local = blockIdx.x - s.first[0], b = local / s.chunks, c = local - b * s.chunks;
  const int64_t n = (int64_t)s.rows * s.cols, begin = (int64_t)c * s.chunk;
  const int64_t base = b * n + begin;
  const int len = (int)(n - begin < s.chunk ? n - begin : s.chunk);
  double sq = 0.0;
#pragma unroll 2
  for (int i = threadIdx.x * 4; i < len; i += ORTHO_T * 4) {
    float u[4];
    load4(s.g, base + i, s.g_type, len - i, u);
    if (s.mom != nullptr) {
      float m[4];
      load4(s.mom, base + i, FIM_F32, len - i, m);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        m[q] = fmaf(k.momentum, m[q], u[q]);
        u[q] = k.nesterov ? fmaf(k.momentum, m[q], u[q]) : m[q];
      }
      store4(s.mom, base + i, FIM_F32, len - i, m);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < len - i) sq = fma((double)u[q], (double)u[q], sq);
  }
  sq = ortho_sum(sq);
  if (threadIdx.x == 0) s.part[local] = sq;
}

// sx U / (|U| + eps) as halves, 64 x 64 of X a workgroup; a tall matrix's through LDS
__global__ __launch_bounds__(ORTHO_T) void ortho_convert_kernel(const OrthoStack* __restrict__ table, int count,
                                                                const OrthoScalars k) {
  __shared__ float tile[64 * 65];
  const OrthoStack s = table[stack_of(table, count, 1, blockIdx.x)];
  const uint32_t rt = (s.mp + 63) / 64, ct = (s.np + 63) / 64, local = blockIdx.x - s.first[1];
  const uint32_t b = local / (rt * ct), in = local - b * rt * ct;
  const int r0 = (int)(in / ct) * 64, c0 = (int)(in % ct) * 64;  // of X
  double sq = 0.0;
  for (uint32_t i = threadIdx.x; i < s.chunks; i += ORTHO_T) sq += s.part[b * s.chunks + i];
  const OrthoScale scaled(sqrt(ortho_sum(sq)) + k.eps, k.sx);
  const int rows = (int)s.rows, cols = (int)s.cols;
  const int sr0 = s.tall ? c0 : r0, sc0 = s.tall ? r0 : c0;  // of the source
  const int64_t base = (int64_t)b * rows * cols;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int lr = (int)threadIdx.x / 16 + 16 * p, lc = (threadIdx.x % 16) * 4, r = sr0 + lr, c = sc0 + lc;
    float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r < rows && c < cols) {
      const int64_t at = base + (int64_t)r * cols + c;
      load4(s.g, at, s.g_type, cols - c, u);
      if (s.mom != nullptr) {
        float m[4];
        load4(s.mom, at, FIM_F32, cols - c, m);
#pragma unroll
        for (int q = 0; q < 4; ++q) u[q] = k.nesterov ? fmaf(k.momentum, m[q], u[q]) : m[q];
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) tile[s.tall ? (lc + q) * 65 + lr : lr * 65 + lc + q] = u[q];
  }
  __syncthreads();
  uint8_t* X = s.x[0] + b * s.each;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int lr = (int)threadIdx.x / 16 + 16 * p, lc = (threadIdx.x % 16) * 4, r = r0 + lr, c = c0 + lc;
    if (r >= (int)s.mp || c >= (int)s.np) continue;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = scaled(tile[lr * 65 + lc + q]);
    v2i hi, lo;
    split4(v, hi, lo);
    uint8_t* at = X + (int64_t)r * s.np * 4 + line_of(c);
    *reinterpret_cast<v2i*>(at) = hi;
    *reinterpret_cast<v2i*>(at + 64) = lo;
  }
}

// -- host --------------------------------------------------------------------------------------------------------------

struct OrthoCall {
  int64_t count;
  const void* const* g;
  const int* g_type;
  float* const* mom;  // null: none
  void* const* out;
  const int* out_type;
  const int64_t *batch, *rows, *cols;
  const float* factor;  // null: 1
};

struct OrthoShape {
  int64_t m, n, mp, np, each, chunk, chunks, slab, slabs;
  bool small, thin;  // one launch; a launch a step
  int T;
};

enum { ORTHO_TILES, ORTHO_HALF, ORTHO_WHOLE, ORTHO_THIN };  // how a matrix is computed

constexpr int64_t ORTHO_MOST = int64_t{1} << 29;  // padded elements of a matrix are fewer: 31-bit offsets into its halves

static OrthoShape ortho_shape(int64_t rows, int64_t cols) {
  OrthoShape s;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  s.mp = cdiv(s.m, 32) * 32;
  s.np = cdiv(s.n, 32) * 32;
  s.T = (int)cdiv(s.m, 16);
  s.small = s.m <= SMALL_ROWS && small_lds(s.m, s.np) <= SMALL_LDS;
  s.slab = s.slabs = 0;
  if (s.m <= SMALL_ROWS) {  // (more rows' sums leave no room for a line, and are on tiles)
    // about 16 workgroups a matrix, each of which reads all their parts; four lines a workgroup at least
    const int64_t lines = s.np / 32, most = (SMALL_LDS - small_region(s.T) - 64) / (16 * s.T * 128);
    s.slab = cdiv(lines, 16) < 4 ? 4 : cdiv(lines, 16) > most ? most : cdiv(lines, 16);
    s.slabs = cdiv(lines, s.slab);
  }
  // (all their reads of all parts grow with the slabs squared: at most 2 MB each. 64 x 65536 in 121 slabs 201 us, 367 on tiles;
  // 64 x 131072 in 241 slabs 596, 545; 16 x 262144 120, 549)
  s.thin = !s.small && s.m <= SMALL_ROWS && s.slabs * s.T * s.T <= 2048;
  s.each = s.small ? 0 : s.thin ? cdiv(s.mp * s.np * 4 + 2 * s.slabs * s.T * s.T * 1024, 256) * 256
                                : cdiv((2 * s.mp * s.np + 2 * s.mp * s.mp) * 4, 256) * 256;
  // at least 8192 elements, at most 512 chunks a matrix
  s.chunk = cdiv(cdiv(rows * cols, 512), 4096) * 4096;
  if (s.chunk < 8192) s.chunk = 8192;
  s.chunks = cdiv(rows * cols, s.chunk);
  return s;
}

static bool ortho_empty(const OrthoCall& c, int64_t i) { return c.batch[i] == 0 || c.rows[i] == 0 || c.cols[i] == 0; }

static int64_t ortho_part_bytes(const OrthoCall& c);

// Sizes and the workspace's bytes: the table, then sums of squares and halves of the matrices on tiles
static int ortho_bytes(const OrthoCall& c, int64_t* bytes) {
  if (c.count < 0 || (c.count > 0 && (c.batch == nullptr || c.rows == nullptr || c.cols == nullptr))) return FIM_ERR_INVALID;
  if (c.count > 1 << 20) return FIM_ERR_UNSUPPORTED;
  int64_t total = cdiv(c.count * (int64_t)sizeof(OrthoStack), 256) * 256;
  int64_t small = 0, tiles = 0;  // workgroups of a launch over all stacks, of 1024 and of 256 threads: below 2^32 threads
  for (int64_t i = 0; i < c.count; ++i) {
    if (c.batch[i] < 0 || c.rows[i] < 0 || c.cols[i] < 0) return FIM_ERR_INVALID;
    if (ortho_empty(c, i)) continue;
    if (c.batch[i] >= 1 << 24 || c.rows[i] >= 1 << 24 || c.cols[i] >= 1 << 24) return FIM_ERR_UNSUPPORTED;
    const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
    if (s.mp * s.np >= ORTHO_MOST) return FIM_ERR_UNSUPPORTED;
    small += s.small ? c.batch[i] : s.thin ? c.batch[i] * s.slabs : 0;
    tiles += s.small ? 0 : c.batch[i] * (cdiv(s.mp, 64) * cdiv(s.np, 64) + s.chunks);
    if (small >= 1 << 22 || tiles >= 1 << 24) return FIM_ERR_UNSUPPORTED;
    if (s.small) continue;
    total += c.batch[i] * s.each + cdiv(c.batch[i] * s.chunks * 8, 256) * 256;
    if (total > int64_t{1} << 46) return FIM_ERR_UNSUPPORTED;
  }
  total += cdiv(ortho_part_bytes(c), 256) * 256;
  *bytes = total;
  return FIM_OK;
}

static bool ortho_type(int t) { return t == FIM_F32 || t == FIM_BF16 || t == FIM_F16; }
static bool ortho_aligned(const void* p, int t) {
  return p != nullptr && reinterpret_cast<uintptr_t>(p) % (t == FIM_F32 ? 4 : 2) == 0;
}

// The largest power of two that keeps values up to `most` (and a little more) below FP16's largest
static float ortho_scale(double most) {
  int e;
  frexp(60000.0 / (most > 1e-6 ? most : 1e-6), &e);
  return ldexpf(1.0f, e - 1);
}

// The scales of X, A and P: no entry of a matrix is larger than its largest singular value. These lie in [0, x] with x = 1 at first,
// and a step's odd polynomial takes that interval onto another that holds 0: its end is the largest value at x or where the slope
// is zero. False where the path leaves the halves little room (or does not end at all).
static bool ortho_scales(OrthoScalars& k) {
  const double a = k.a, b = k.b, c = k.c;
  double flat[2] = {-1.0, -1.0};  // squares at which a + 3 b q + 5 c q^2 is zero
  const double root = 9.0 * b * b - 20.0 * a * c;
  if (c == 0.0 && b != 0.0) {
    flat[0] = -a / (3.0 * b);
  } else if (c != 0.0 && root >= 0.0) {
    flat[0] = (-3.0 * b - sqrt(root)) / (10.0 * c);
    flat[1] = (-3.0 * b + sqrt(root)) / (10.0 * c);
  }
  double most_x = 1.0, most_p = 0.0, x = 1.0;
  for (int it = 0; it < k.steps; ++it) {
    double next = 0.0, p = 0.0;
    bool fine = true;
    auto look = [&](double q) {  // at a square within the interval
      if (!(q >= 0.0 && q <= x * x)) return;
      const double at = fabs(a + q * (b + q * c));
      fine = fine && at <= 48.0 && sqrt(q) * at <= 6.0;  // (not of NaN, which fmax passes over)
      p = fmax(p, at);
      next = fmax(next, sqrt(q) * at);
    };
    look(0.0);
    look(x * x);
    look(flat[0]);
    look(flat[1]);
    if (c != 0.0) look(-b / (2.0 * c));
    if (!fine) return false;
    most_p = fmax(most_p, p);
    x = next;
    if (it + 1 < k.steps) most_x = fmax(most_x, x);
  }
  // (by rounding a little more)
  k.sx = ortho_scale(1.1 * most_x);
  k.sa = ortho_scale(1.25 * most_x * most_x);
  k.sp = ortho_scale(1.05 * most_p);
  return true;
}

static int ortho_check(const OrthoCall& c, OrthoScalars& k) {
  if (k.steps < 1 || k.steps > 100 || !(k.eps >= 0.0)) return FIM_ERR_INVALID;
  if (!ortho_scales(k)) return FIM_ERR_UNSUPPORTED;
  if (c.count > 0 && (c.g == nullptr || c.g_type == nullptr || c.out == nullptr || c.out_type == nullptr)) return FIM_ERR_INVALID;
  for (int64_t i = 0; i < c.count; ++i) {
    if (!ortho_type(c.g_type[i]) || !ortho_type(c.out_type[i])) return FIM_ERR_INVALID;
    if (ortho_empty(c, i)) continue;
    if (!ortho_aligned(c.g[i], c.g_type[i]) || !ortho_aligned(c.out[i], c.out_type[i])) return FIM_ERR_INVALID;
    if (c.mom != nullptr && !ortho_aligned(c.mom[i], FIM_F32)) return FIM_ERR_INVALID;
  }
  return FIM_OK;
}

template <int T, int LDS, int MODE>
static void launch_small(const OrthoFew& few, const OrthoStack* table, int count, uint32_t grid, int step, const OrthoScalars& k,
                         hipStream_t stream) {
  const auto kernel = table == nullptr ? ortho_small_kernel<T, LDS, MODE, true> : ortho_small_kernel<T, LDS, MODE, false>;
  kernel<<<dim3(grid), dim3(64 * SMALL_WAVES), 0, stream>>>(few, table, count, step, k);
}

// LDS classes: 160 KB is a CU's; matrices of at most half of it run two to a CU
template <int T>
static void launch_small(int kind, const OrthoFew& few, const OrthoStack* table, int count, const uint32_t (&grid)[2],
                         const OrthoScalars& k, hipStream_t stream) {
  if (kind == ORTHO_HALF) return launch_small<T, SMALL_LDS / 2, SMALL_WHOLE>(few, table, count, grid[0], 0, k, stream);
  if (kind == ORTHO_WHOLE) return launch_small<T, SMALL_LDS, SMALL_WHOLE>(few, table, count, grid[0], 0, k, stream);
  launch_small<T, SMALL_LDS, THIN_FIRST>(few, table, count, grid[1], 0, k, stream);
  for (int it = 0; it < k.steps; ++it) launch_small<T, SMALL_LDS, THIN_STEP>(few, table, count, grid[1], it, k, stream);
}

static void launch_small(int T, int kind, const OrthoFew& few, const OrthoStack* table, int count, const uint32_t (&grid)[2],
                         const OrthoScalars& k, hipStream_t stream) {
  switch (T) {
    case 1: return launch_small<1>(kind, few, table, count, grid, k, stream);
    case 2: return launch_small<2>(kind, few, table, count, grid, k, stream);
    case 3: return launch_small<3>(kind, few, table, count, grid, k, stream);
    default: return launch_small<4>(kind, few, table, count, grid, k, stream);
  }
}

// The products' tiles, of 64 `side` squared, and how many parts their contraction has; `deep`: four LDS stages, not two
struct OrthoTiles {
  int side;
  int64_t tiles, splits;
  bool deep;
};
struct OrthoPlan {
  OrthoTiles gram, square, apply;
};

// Tiles of 128 move half the operands of 64, but a product needs enough of them for the card. By time measured (us a product; m x n):
// * A = X X^T, three of 1024 x 4096: 128 in 4 parts 42 + 9 to join, in 2 parts 46 + 7, whole 75; 64 whole 55. One: 128 in 4 parts
//   20 + 5, 64 whole 28. 196 x 523: 64 whole 7, in parts 5 + 5. 96 matrices of 512 x 2048 and smaller: 128 whole 79, 64 whole 82.
// * P: its contraction is short, and the epilogue costs as much: three of 1024: 64 whole 21, 128 in 2 parts 18 + 9, whole 29; the 96
//   matrices: 64 whole 28, 128 whole 32.
// * P X: three of 1024 x 4096: 128 71, 64 97; the 96 matrices 107, 152; 196 x 523: 64 6, 128 10.
// Four stages cover a workgroup's latencies where it is alone on its CU; two leave room for another.
static OrthoPlan ortho_plan(const OrthoCall& c) {
  int64_t t1 = 0, t2 = 0, a1 = 0, a2 = 0, most = 0;  // tiles of 64 and 128: symmetric, all; the longest contraction
  const int64_t cus = device_cus();
  for (int64_t i = 0; i < c.count; ++i) {
    if (ortho_empty(c, i)) continue;
    const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
    if (s.small || s.thin) continue;
    const int64_t m1 = cdiv(s.mp, 64), m2 = cdiv(s.mp, 128);
    t1 += c.batch[i] * (m1 * (m1 + 1) / 2);
    t2 += c.batch[i] * (m2 * (m2 + 1) / 2);
    a1 += c.batch[i] * m1 * cdiv(s.np, 64);
    a2 += c.batch[i] * m2 * cdiv(s.np, 128);
    if (s.np > most) most = s.np;
  }
  auto of = [&](int side, int64_t tiles, int64_t splits) {
    const int64_t n = tiles * splits;
    return OrthoTiles{side, tiles, splits, n <= (side == 1 ? 2 * cus : cus)};
  };
  int64_t splits = cdiv(3 * cus / 2, t2 > 0 ? t2 : 1);
  if (splits > most / 256) splits = most / 256;  // (eight steps at least)
  OrthoPlan p;
  p.gram = t2 >= cus ? of(2, t2, 1) : most <= 1024 || splits <= 1 ? of(1, t1, 1) : of(2, t2, splits);
  p.square = t2 >= 2 * cus ? of(2, t2, 1) : of(1, t1, 1);
  p.apply = a2 >= cus / 2 ? of(2, a2, 1) : of(1, a1, 1);
  return p;
}

static int64_t ortho_part_bytes(const OrthoCall& c) {
  const OrthoTiles g = ortho_plan(c).gram;
  return g.splits > 1 ? g.splits * g.tiles * (64 * g.side) * (64 * g.side) * 4 : 0;
}

template <int MODE>
static void launch_product(const OrthoStack* table, int count, const OrthoTiles& t, float* part, int src, const OrthoScalars& k,
                           hipStream_t stream) {
  const dim3 grid((unsigned)(cdiv(t.tiles * t.splits, 8 * ORTHO_RUN) * 8 * ORTHO_RUN)), block(256);
  const uint32_t tiles = (uint32_t)t.tiles;
  const int splits = (int)t.splits;
  // (P on tiles of 128 has two a CU and more, and P X on tiles of 64 at most two: their stages are 2 and 4)
  constexpr bool ALWAYS_2 = MODE == ORTHO_SQUARE, ALWAYS_4 = MODE == ORTHO_APPLY || MODE == ORTHO_LAST;
  if (t.side == 2) {
    if constexpr (!ALWAYS_2)
      if (t.deep) return ortho_tile_kernel<MODE, 2, 4><<<grid, block, 0, stream>>>(table, count, tiles, splits, part, src, k);
    ortho_tile_kernel<MODE, 2, 2><<<grid, block, 0, stream>>>(table, count, tiles, splits, part, src, k);
  } else {
    if constexpr (!ALWAYS_4)
      if (!t.deep) return ortho_tile_kernel<MODE, 1, 2><<<grid, block, 0, stream>>>(table, count, tiles, splits, part, src, k);
    ortho_tile_kernel<MODE, 1, 4><<<grid, block, 0, stream>>>(table, count, tiles, splits, part, src, k);
  }
}

static void launch_products(const OrthoStack* table, int count, const OrthoPlan& p, float* part, const OrthoScalars& k,
                            hipStream_t stream) {
  for (int it = 0; it < k.steps; ++it) {
    const int src = it & 1;
    launch_product<ORTHO_GRAM>(table, count, p.gram, part, src, k, stream);
    if (p.gram.splits > 1)  // (tiles of 128)
      ortho_join_kernel<<<dim3((unsigned)(p.gram.tiles * 4)), dim3(256), 0, stream>>>(table, count, (uint32_t)p.gram.tiles,
                                                                                      (int)p.gram.splits, part, k);
    launch_product<ORTHO_SQUARE>(table, count, p.square, nullptr, src, k, stream);
    if (it + 1 < k.steps) launch_product<ORTHO_APPLY>(table, count, p.apply, nullptr, src, k, stream);
    else launch_product<ORTHO_LAST>(table, count, p.apply, nullptr, src, k, stream);
  }
}

// Stacks of one group (a size of small matrices, or all that go on tiles) share their launches
static int ortho_run(const OrthoCall& c, OrthoScalars k, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  int64_t need = 0;
  int rc = ortho_bytes(c, &need);
  if (rc == FIM_OK) rc = ortho_check(c, k);
  if (rc != FIM_OK) return rc;
  bool any = false;
  for (int64_t i = 0; i < c.count; ++i) any = any || !ortho_empty(c, i);
  if (!any) return FIM_OK;
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return FIM_ERR_INVALID;
  OrthoStack* table = static_cast<OrthoStack*>(workspace);
  uint8_t* free_at = static_cast<uint8_t*>(workspace) + cdiv(c.count * (int64_t)sizeof(OrthoStack), 256) * 256;

  OrthoFill fill;
  memset(&fill, 0, sizeof(fill));
  int filled = 0;  // entries of `fill` that the device's table does not hold yet
  int written = 0;
  auto flush = [&]() {
    if (filled > 0) ortho_fill_kernel<<<dim3(1), dim3(ORTHO_T), 0, stream>>>(fill, table + written, filled);
    written += filled;
    filled = 0;
  };
  // group: 4 T + kind, or 0 for tiles
  auto group_of = [&](int64_t i) {
    const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
    if (s.thin) return 4 * s.T + ORTHO_THIN;
    return !s.small ? 0 : 4 * s.T + (small_lds(s.m, s.np) <= SMALL_LDS / 2 ? ORTHO_HALF : ORTHO_WHOLE);
  };
  const OrthoPlan plan = ortho_plan(c);
  float* part = reinterpret_cast<float*>(free_at);
  free_at += cdiv(ortho_part_bytes(c), 256) * 256;
  for (int group = 0; group < 4 * (SMALL_ROWS / 16 + 1); ++group) {
    const int kind = group % 4;
    int64_t first[5] = {0, 0, 0, 0, 0};
    const int start = written + filled;
    for (int64_t i = 0; i < c.count; ++i) {
      if (ortho_empty(c, i) || group_of(i) != group) continue;
      const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
      const int64_t batch = c.batch[i];
      OrthoStack& e = fill.s[filled];
      memset(&e, 0, sizeof(e));
      e.g = c.g[i];
      e.mom = c.mom == nullptr ? nullptr : c.mom[i];
      e.out = c.out[i];
      e.rows = (uint32_t)c.rows[i];
      e.cols = (uint32_t)c.cols[i];
      e.batch = (uint32_t)batch;
      e.mp = (uint32_t)s.mp;
      e.np = (uint32_t)s.np;
      e.factor = c.factor == nullptr ? 1.0f : c.factor[i];
      e.g_type = (uint8_t)c.g_type[i];
      e.out_type = (uint8_t)c.out_type[i];
      e.tall = c.rows[i] > c.cols[i];
      for (int p = 0; p < 5; ++p) e.first[p] = (uint32_t)first[p];
      if (kind == ORTHO_TILES || kind == ORTHO_THIN) {
        e.part = reinterpret_cast<double*>(free_at);
        free_at += cdiv(batch * s.chunks * 8, 256) * 256;
        e.x[0] = free_at;
        e.x[1] = e.x[0] + s.mp * s.np * 4;  // (thin: the parts)
        e.a = kind == ORTHO_THIN ? e.x[1] : e.x[1] + s.mp * s.np * 4;
        e.p = e.a + (kind == ORTHO_THIN ? s.slabs * s.T * s.T * 1024 : s.mp * s.mp * 4);
        e.each = s.each;
        free_at += batch * s.each;
        e.chunk = (uint32_t)s.chunk;
        e.chunks = (uint32_t)s.chunks;
        e.slab = (uint32_t)s.slab;
        e.slabs = (uint32_t)s.slabs;
      }
      if (kind == ORTHO_THIN) {
        first[0] += batch * s.chunks;
        first[1] += batch * s.slabs;
      } else if (kind == ORTHO_TILES) {
        auto triangle = [&](int side) {
          const int64_t n = cdiv(s.mp, 64 * side);
          return n * (n + 1) / 2;
        };
        first[0] += batch * s.chunks;
        first[1] += batch * cdiv(s.mp, 64) * cdiv(s.np, 64);
        first[2] += batch * triangle(plan.gram.side);
        first[3] += batch * triangle(plan.square.side);
        first[4] += batch * cdiv(s.mp, 64 * plan.apply.side) * cdiv(s.np, 64 * plan.apply.side);
      } else {
        first[0] += batch;
      }
      if (++filled == ORTHO_FILL) flush();
    }
    const int n = written + filled - start;
    if (n == 0) continue;
    if (kind != ORTHO_TILES) {
      OrthoFew few;
      const bool args = n <= SMALL_FEW && n == filled;  // (no table: neither its launch nor its latency)
      memcpy(few.s, fill.s, sizeof(few));
      if (args && kind != ORTHO_THIN) filled = 0;
      else flush();
      const OrthoStack* t = table + start;
      if (kind == ORTHO_THIN) ortho_momentum_kernel<<<dim3((unsigned)first[0]), dim3(ORTHO_T), 0, stream>>>(t, n, k);
      const uint32_t grid[2] = {(uint32_t)first[0], (uint32_t)first[1]};
      launch_small(group / 4, kind, few, args ? nullptr : t, n, grid, k, stream);
      continue;
    }
    flush();
    const OrthoStack* t = table + start;
    ortho_momentum_kernel<<<dim3((unsigned)first[0]), dim3(ORTHO_T), 0, stream>>>(t, n, k);
    ortho_convert_kernel<<<dim3((unsigned)first[1]), dim3(ORTHO_T), 0, stream>>>(t, n, k);
    launch_products(t, n, plan, part, k, stream);
  }
  return launch_status();
}

}  // namespace fim

using namespace fim;

extern "C" int fim_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int64_t* bytes) {
  if (bytes == nullptr) return FIM_ERR_INVALID;
  return ortho_bytes(OrthoCall{1, nullptr, nullptr, nullptr, nullptr, nullptr, &batch, &rows, &cols, nullptr}, bytes);
}

extern "C" int fim_orthogonalize(const void* g, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
                                 float b, float c, double eps, void* out, int out_dtype, void* workspace,
                                 int64_t workspace_bytes, hipStream_t stream) {
  const OrthoScalars k{0.0f, 1.0f, a, b, c, 0.0f, 0.0f, 0.0f, eps, steps, 0, 0};
  return ortho_run(OrthoCall{1, &g, &dtype, nullptr, &out, &out_dtype, &batch, &rows, &cols, nullptr}, k, workspace,
                   workspace_bytes, stream);
}

extern "C" int fim_muon_step_workspace(int64_t count, const int64_t* batch, const int64_t* rows, const int64_t* cols,
                                       int64_t* bytes) {
  if (bytes == nullptr) return FIM_ERR_INVALID;
  return ortho_bytes(OrthoCall{count, nullptr, nullptr, nullptr, nullptr, nullptr, batch, rows, cols, nullptr}, bytes);
}

extern "C" int fim_muon_step(int64_t count, void* const* params, const int* param_dtypes, const void* const* grads,
                             const int* grad_dtypes, float* const* momenta, const int64_t* batch, const int64_t* rows,
                             const int64_t* cols, const float* factors, float momentum, int nesterov, float keep, int steps,
                             float a, float b, float c, double eps, void* workspace, int64_t workspace_bytes,
                             hipStream_t stream) {
  if (count > 0 && (momenta == nullptr || factors == nullptr)) return FIM_ERR_INVALID;
  const OrthoScalars k{momentum, keep, a, b, c, 0.0f, 0.0f, 0.0f, eps, steps, nesterov, 1};
  return ortho_run(OrthoCall{count, grads, grad_dtypes, momenta, params, param_dtypes, batch, rows, cols, factors}, k, workspace,
                   workspace_bytes, stream);
}
