// Orthogonalized matrices by Newton-Schulz products, and the optimizer step made of them (formulas and precision: ortho.h).
//
// Matrices come as stacks of one shape, many stacks a call; a table of them goes through kernel arguments into the workspace
// (no upload: capturable), and every launch after that runs over all matrices at once. Small ones take one launch, a workgroup each
// (ortho_small.h); the others a pass that updates the momentum and sums squares, one that writes sx X0 as halves (transposing tall
// matrices), and three launches of products a step (ortho_tile.h), the last of which writes O or steps the parameters.
#include <string.h>

#include "ortho_small.h"
#include "ortho_tile.h"

namespace fim {

constexpr int ORTHO_T = 256, ORTHO_FILL = 28;
struct OrthoFill {
  OrthoStack s[ORTHO_FILL];
};
static_assert(sizeof(OrthoFill) <= 4000, "kernel arguments");

__global__ __launch_bounds__(64) void ortho_fill_kernel(const OrthoFill f, OrthoStack* table, int n) {
  constexpr int WORDS = sizeof(OrthoStack) / 4;
  const uint32_t* from = reinterpret_cast<const uint32_t*>(&f);
  uint32_t* to = reinterpret_cast<uint32_t*>(table);
  for (int i = threadIdx.x; i < n * WORDS; i += 64) to[i] = from[i];
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
  const OrthoStack& s = table[stack_of(table, count, 0, blockIdx.x)];
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
  const OrthoStack& s = table[stack_of(table, count, 1, blockIdx.x)];
  const uint32_t rt = (s.mp + 63) / 64, ct = (s.np + 63) / 64, local = blockIdx.x - s.first[1];
  const uint32_t b = local / (rt * ct), in = local - b * rt * ct;
  const int r0 = (int)(in / ct) * 64, c0 = (int)(in % ct) * 64;  // of X
  double sq = 0.0;
  for (uint32_t i = threadIdx.x; i < s.chunks; i += ORTHO_T) sq += s.part[b * s.chunks + i];
  const float scale = (float)((double)k.sx / (sqrt(ortho_sum(sq)) + k.eps));
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
    for (int q = 0; q < 4; ++q) v[q] = tile[lr * 65 + lc + q] * scale;
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
  int64_t m, n, mp, np, each, chunk, chunks;
  bool small;
  int T;
};

constexpr int64_t ORTHO_MOST = int64_t{1} << 29;  // padded elements of a matrix: 31-bit offsets into its halves

static OrthoShape ortho_shape(int64_t rows, int64_t cols) {
  OrthoShape s;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  s.mp = cdiv(s.m, 32) * 32;
  s.np = cdiv(s.n, 32) * 32;
  s.T = (int)cdiv(s.m, 16);
  s.small = s.m <= SMALL_ROWS && small_lds(s.m, s.np) <= SMALL_LDS;
  s.each = s.small ? 0 : cdiv((2 * s.mp * s.np + 2 * s.mp * s.mp) * 4, 256) * 256;
  // at least 8192 elements, at most 512 chunks a matrix
  s.chunk = cdiv(cdiv(rows * cols, 512), 4096) * 4096;
  if (s.chunk < 8192) s.chunk = 8192;
  s.chunks = cdiv(rows * cols, s.chunk);
  return s;
}

static bool ortho_empty(const OrthoCall& c, int64_t i) { return c.batch[i] == 0 || c.rows[i] == 0 || c.cols[i] == 0; }

// Sizes and the workspace's bytes: the table, then sums of squares and halves of the matrices on tiles
static int ortho_bytes(const OrthoCall& c, int64_t* bytes) {
  if (c.count < 0 || (c.count > 0 && (c.batch == nullptr || c.rows == nullptr || c.cols == nullptr))) return FIM_ERR_INVALID;
  if (c.count > 1 << 20) return FIM_ERR_UNSUPPORTED;
  int64_t total = cdiv(c.count * (int64_t)sizeof(OrthoStack), 256) * 256;
  for (int64_t i = 0; i < c.count; ++i) {
    if (c.batch[i] < 0 || c.rows[i] < 0 || c.cols[i] < 0) return FIM_ERR_INVALID;
    if (ortho_empty(c, i)) continue;
    if (c.batch[i] >= 1 << 24 || c.rows[i] >= 1 << 24 || c.cols[i] >= 1 << 24) return FIM_ERR_UNSUPPORTED;
    const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
    if (s.mp * s.np > ORTHO_MOST) return FIM_ERR_UNSUPPORTED;
    if (s.small) continue;
    total += c.batch[i] * s.each + cdiv(c.batch[i] * s.chunks * 8, 256) * 256;
    if (total > int64_t{1} << 46) return FIM_ERR_UNSUPPORTED;
  }
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

// The scales of X, A and P: no entry of a matrix is larger than its largest singular value, whose path from any s <= 1 is
// followed here. False where it leaves the halves little room (or does not end at all).
static bool ortho_scales(OrthoScalars& k) {
  double most_x = 1.0, most_p = 0.0;
  for (int i = 0; i <= 256; ++i) {
    double x = i / 256.0;
    for (int it = 0; it < k.steps; ++it) {
      const double q = x * x, p = k.a + q * (k.b + q * k.c);
      most_p = fmax(most_p, fabs(p));
      x *= p;
      if (!(fabs(p) <= 48.0) || !(fabs(x) <= 6.0)) return false;
      if (it + 1 < k.steps) most_x = fmax(most_x, fabs(x));
    }
  }
  // (between the grid's points and by rounding a little more)
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

template <int T, int LDS>
static void launch_small(const OrthoStack* table, int count, uint32_t grid, const OrthoScalars& k, hipStream_t stream) {
  ortho_small_kernel<T, LDS><<<dim3(grid), dim3(64 * SMALL_WAVES), 0, stream>>>(table, count, k);
}

// LDS classes: 160 KB is a CU's; matrices of at most half of it run two to a CU
static void launch_small(int T, bool half, const OrthoStack* table, int count, uint32_t grid, const OrthoScalars& k,
                         hipStream_t stream) {
  switch (T * 2 + half) {
    case 2: return launch_small<1, SMALL_LDS>(table, count, grid, k, stream);
    case 3: return launch_small<1, SMALL_LDS / 2>(table, count, grid, k, stream);
    case 4: return launch_small<2, SMALL_LDS>(table, count, grid, k, stream);
    case 5: return launch_small<2, SMALL_LDS / 2>(table, count, grid, k, stream);
    case 6: return launch_small<3, SMALL_LDS>(table, count, grid, k, stream);
    case 7: return launch_small<3, SMALL_LDS / 2>(table, count, grid, k, stream);
    case 8: return launch_small<4, SMALL_LDS>(table, count, grid, k, stream);
    case 9: return launch_small<4, SMALL_LDS / 2>(table, count, grid, k, stream);
  }
}

template <int MB>
static void launch_products(const OrthoStack* table, int count, uint32_t sym, uint32_t all, const OrthoScalars& k,
                            hipStream_t stream) {
  const dim3 gs((unsigned)cdiv(sym, 8) * 8), ga((unsigned)cdiv(all, 8) * 8), block(256);
  for (int it = 0; it < k.steps; ++it) {
    const int src = it & 1;
    ortho_tile_kernel<ORTHO_GRAM, MB><<<gs, block, 0, stream>>>(table, count, sym, src, k);
    ortho_tile_kernel<ORTHO_SQUARE, MB><<<gs, block, 0, stream>>>(table, count, sym, src, k);
    if (it + 1 < k.steps) ortho_tile_kernel<ORTHO_APPLY, MB><<<ga, block, 0, stream>>>(table, count, all, src, k);
    else ortho_tile_kernel<ORTHO_LAST, MB><<<ga, block, 0, stream>>>(table, count, all, src, k);
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
  int filled = 0;  // entries of `fill` that the device's table does not hold yet
  int written = 0;
  auto flush = [&]() {
    if (filled > 0) ortho_fill_kernel<<<dim3(1), dim3(64), 0, stream>>>(fill, table + written, filled);
    written += filled;
    filled = 0;
  };
  // group 2 T + half: small matrices; 0: tiles, of 64 MB
  auto group_of = [&](int64_t i) {
    const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
    return s.small ? 2 * s.T + (small_lds(s.m, s.np) <= SMALL_LDS / 2) : 0;
  };
  // tiles of 64 or 128: the larger ones where they still cover the CUs
  int64_t tiles128 = 0;
  for (int64_t i = 0; i < c.count; ++i)
    if (!ortho_empty(c, i) && group_of(i) == 0) {
      const OrthoShape s = ortho_shape(c.rows[i], c.cols[i]);
      tiles128 += c.batch[i] * cdiv(s.mp, 128) * cdiv(s.np, 128);
    }
  const int mb = tiles128 >= device_cus() ? 2 : 1;
  for (int group = 0; group < 10; ++group) {
    int64_t first[4] = {0, 0, 0, 0};
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
      for (int p = 0; p < 4; ++p) e.first[p] = (uint32_t)first[p];
      if (group == 0) {
        e.part = reinterpret_cast<double*>(free_at);
        free_at += cdiv(batch * s.chunks * 8, 256) * 256;
        e.x[0] = free_at;
        e.x[1] = e.x[0] + s.mp * s.np * 4;
        e.a = e.x[1] + s.mp * s.np * 4;
        e.p = e.a + s.mp * s.mp * 4;
        e.each = s.each;
        free_at += batch * s.each;
        e.chunk = (uint32_t)s.chunk;
        e.chunks = (uint32_t)s.chunks;
        const int64_t bm = 64 * mb, mt = cdiv(s.mp, bm);
        first[0] += batch * s.chunks;
        first[1] += batch * cdiv(s.mp, 64) * cdiv(s.np, 64);
        first[2] += batch * (mt * (mt + 1) / 2);
        first[3] += batch * mt * cdiv(s.np, bm);
      } else {
        first[0] += batch;
      }
      for (int p = 0; p < 4; ++p)
        if (first[p] >= int64_t{1} << 31) return FIM_ERR_UNSUPPORTED;
      if (++filled == ORTHO_FILL) flush();
    }
    const int n = written + filled - start;
    if (n == 0) continue;
    flush();
    const OrthoStack* t = table + start;
    if (group > 0) {
      launch_small(group / 2, group & 1, t, n, (uint32_t)first[0], k, stream);
      continue;
    }
    ortho_momentum_kernel<<<dim3((unsigned)first[0]), dim3(ORTHO_T), 0, stream>>>(t, n, k);
    ortho_convert_kernel<<<dim3((unsigned)first[1]), dim3(ORTHO_T), 0, stream>>>(t, n, k);
    if (mb == 2) launch_products<2>(t, n, (uint32_t)first[2], (uint32_t)first[3], k, stream);
    else launch_products<1>(t, n, (uint32_t)first[2], (uint32_t)first[3], k, stream);
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
