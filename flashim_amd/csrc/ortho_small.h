// A whole Newton-Schulz iteration, or optimizer step, of a small matrix in one workgroup: X, A and P stay in LDS.
//
// At most 64 rows (of the shorter side) whose X fits: read once, written once, and no launch between the 3 `steps` products, which on
// tiles would be as many launches of one or two workgroups. Sixteen wavefronts on 16 x 16 x 32 MFMAs: X X^T is split over the
// columns of four (each fragment is read once, and is either operand), whose sums meet in LDS; each wavefront adds up one of the 16
// blocks, those above the diagonal from the ones below, read across; P X is split over the columns too, and each wavefront replaces
// the columns it has read.
//
// Bound by the chain of dependent products, each of LDS latencies and two or three barriers, and at four blocks of rows by X X^T on
// four of the sixteen wavefronts, ten pairs of blocks each: 64 x 256 32 us, about 6 a step; 64 matrices of 16 x 512 beside each
// other 16.
#pragma once

#include "ortho.h"

namespace fim {

// SUMS: wavefronts that X X^T is split over, and whose sums lie in LDS at once (64 matrices of 16 x 512 15.8 us; by 8 16.0, by 16
// 16.9; not measured by more at four blocks of rows). SMALL_FEW: stacks that travel in kernel arguments
constexpr int SMALL_WAVES = 16, SMALL_SUMS = 4, SMALL_FEW = 6, SMALL_ROWS = 64, SMALL_LDS = 160 * 1024;

// (Three blocks of 16 rows spill some 30 registers, and are still ahead: 48 x 600 49 us, 62 in slabs, which four would need.)
// LDS of a matrix: X [16 T][np] halves; the wavefronts' sums, or A and P (one block of 16 rows: both, so that A's and P's
// columns past 16 stay zero and no barrier parts them from the sums: 64 matrices of 16 x 512 16.2 -> 15.7 us)
inline int64_t small_region(int T) {
  const int64_t sums = SMALL_SUMS * (T * (T + 1) / 2) * 1024, ap = 2 * (16 * T) * (T > 2 ? 256 : 128);
  return T == 1 ? sums + ap : sums > ap ? sums : ap;
}
inline int64_t small_lds(int64_t m, int64_t np) {
  const int64_t T = cdiv(m, 16);
  return 16 * T * np * 4 + small_region((int)T) + 64;
}

// Where a row's 16-byte segments lie in each line, by XOR: eight rows read at one segment, and four rows by 32 bytes of a transposed
// read, meet different banks.
__device__ __forceinline__ int small_key(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }

__device__ __forceinline__ v4f mfma_small(s16x8 a, s16x8 b, v4f c) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

struct OrthoFew {
  OrthoStack s[SMALL_FEW];
};

// WHOLE: the iteration in one launch. A longer matrix goes through it in slabs of columns, a workgroup each, a launch a step:
// FIRST writes a slab of X0 and its part of X X^T; STEP adds up all slabs' parts, in order and in every workgroup, replaces its
// slab by P X and leaves its part of the next X X^T, or O. (Seven launches for the 17 of the tiles, whose products of such a
// matrix have a tile or two: 7 x 3696 120 -> 47 us.)
enum { SMALL_WHOLE, THIN_FIRST, THIN_STEP };

// FEW: the stacks are in the arguments, which takes less than a table's launch and its latency; else in `table`
template <int T, int LDS, int MODE, bool FEW>
__global__ __launch_bounds__(64 * SMALL_WAVES) void ortho_small_kernel(const OrthoFew few, const OrthoStack* __restrict__ table,
                                                                       int count, int step, OrthoScalars k) {
  constexpr int PASS = MODE == SMALL_WHOLE ? 0 : 1;
  constexpr int SUMS = SMALL_SUMS, MP = 16 * T, LINES = T > 2 ? 2 : 1, PAIRS = T * (T + 1) / 2;  // LINES: of a row of A and P
  __shared__ __attribute__((aligned(128))) uint8_t lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  int e = 0;
  if constexpr (FEW) {
#pragma unroll
    for (int i = 1; i < SMALL_FEW; ++i) e += i < count && few.s[i].first[PASS] <= blockIdx.x;
  } else {
    e = stack_of(table, count, PASS, blockIdx.x);
  }
  const OrthoStack s = FEW ? few.s[e] : table[e];
  const uint32_t local = blockIdx.x - s.first[PASS];
  const int b = (int)(MODE == SMALL_WHOLE ? local : local / s.slabs);
  const int line0 = MODE == SMALL_WHOLE ? 0 : (int)(local - (uint32_t)b * s.slabs) * (int)s.slab;  // this workgroup's lines
  const int rows = (int)s.rows, cols = (int)s.cols, np = (int)s.np;
  const int nb = MODE == SMALL_WHOLE || (np >> 5) - line0 < (int)s.slab ? (np >> 5) - line0 : (int)s.slab, ld = nb * 128;
  const int64_t n = (int64_t)rows * cols, base = b * n;
  uint8_t* X = lds;
  constexpr bool APART = T == 1 && MODE == SMALL_WHOLE;
  float* sums = reinterpret_cast<float*>(lds + MP * ld);
  uint8_t* A = lds + MP * ld + (APART ? SUMS * PAIRS * 1024 : 0);  // [MP][LINES] lines
  uint8_t* P = A + MP * LINES * 128;
  if constexpr (APART)
    for (int i = tid * 16; i < 2 * MP * LINES * 128; i += 64 * SMALL_WAVES * 16) *reinterpret_cast<v4i*>(A + i) = v4i{0, 0, 0, 0};

  if constexpr (MODE != THIN_STEP) {
  // -- U in 32 bits where X will lie: element (r, c) of X in 4 bytes, the columns of each line rotated by the row
  const int short_side = s.tall ? cols : rows, long_side = s.tall ? rows : cols;
  if (short_side < MP || long_side < (line0 + nb) * 32) {
    for (int i = tid * 16; i < MP * ld; i += 64 * SMALL_WAVES * 16) *reinterpret_cast<v4i*>(X + i) = v4i{0, 0, 0, 0};
    __syncthreads();
  }
  double sq = 0.0;
  auto load_all = [&](auto dt, auto mom_c) __attribute__((always_inline)) {
    constexpr int DT = decltype(dt)::value, STEP = 64 * SMALL_WAVES * 4, U = 4;  // U loads in flight: stores may alias them
    constexpr bool MOM = decltype(mom_c)::value;
    int r = tid * 4 / cols, c = tid * 4 - r * cols;
    const int dr = STEP / cols, dc = STEP - dr * cols;
    for (int i0 = tid * 4; i0 < (int)n; i0 += U * STEP) {
      float u[U][4], m[MOM ? U : 1][4];
#pragma unroll
      for (int t = 0; t < U; ++t) {
        const int i = i0 + t * STEP;
        if (i < (int)n) {
          load4(s.g, base + i, DT, (int)n - i, u[t]);
          if constexpr (MOM) load4(s.mom, base + i, FIM_F32, (int)n - i, m[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < U; ++t) {
        const int i = i0 + t * STEP, left = (int)n - i;
        if (left > 0) {
          if constexpr (MOM) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              m[t][q] = fmaf(k.momentum, m[t][q], u[t][q]);
              u[t][q] = k.nesterov ? fmaf(k.momentum, m[t][q], u[t][q]) : m[t][q];
            }
            store4(s.mom, base + i, FIM_F32, left, m[t]);
          }
          int rr = r, cc = c;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (q < left) {
              sq = fma((double)u[t][q], (double)u[t][q], sq);
              const int xr = s.tall ? cc : rr, xc = s.tall ? rr : cc;
              *reinterpret_cast<float*>(X + xr * ld + (xc >> 5) * 128 + (((xc ^ xr) & 31) << 2)) = u[t][q];
            }
            if (++cc == cols) {
              cc = 0;
              ++rr;
            }
          }
        }
        r += dr;
        c += dc;
        if (c >= cols) {
          c -= cols;
          ++r;
        }
      }
    }
  };
  // a slab's elements, row by row of the source; the momentum has been updated and the squares summed by a launch before
  auto load_slab = [&](auto dt, auto mom_c) __attribute__((always_inline)) {
    constexpr int DT = decltype(dt)::value, STEP = 64 * SMALL_WAVES, U = 4;
    constexpr bool MOM = decltype(mom_c)::value;
    const int slab_long = long_side - line0 * 32 < nb * 32 ? long_side - line0 * 32 : nb * 32;
    const int width = s.tall ? cols : slab_long, height = s.tall ? slab_long : rows, quads = (width + 3) / 4;
    const int64_t from = base + (s.tall ? (int64_t)line0 * 32 * cols : line0 * 32);
    for (int i0 = tid; i0 < height * quads; i0 += U * STEP) {
      float u[U][4], m[MOM ? U : 1][4];
#pragma unroll
      for (int t = 0; t < U; ++t) {
        const int i = i0 + t * STEP, r = i / quads, c = (i - r * quads) * 4;
        if (r < height) {
          load4(s.g, from + (int64_t)r * cols + c, DT, width - c, u[t]);
          if constexpr (MOM) load4(s.mom, from + (int64_t)r * cols + c, FIM_F32, width - c, m[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < U; ++t) {
        const int i = i0 + t * STEP, r = i / quads, c = (i - r * quads) * 4;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (r < height && c + q < width) {
            const float v = !MOM ? u[t][q] : k.nesterov ? fmaf(k.momentum, m[MOM ? t : 0][q], u[t][q]) : m[MOM ? t : 0][q];
            const int xr = s.tall ? c + q : r, xc = s.tall ? r : c + q;
            *reinterpret_cast<float*>(X + xr * ld + (xc >> 5) * 128 + (((xc ^ xr) & 31) << 2)) = v;
          }
      }
    }
  };
  auto load_of = [&](auto dt) __attribute__((always_inline)) {
    auto load = [&](auto mom) __attribute__((always_inline)) {
      if constexpr (MODE == SMALL_WHOLE) load_all(dt, mom);
      else load_slab(dt, mom);
    };
    if (s.mom != nullptr) load(std::integral_constant<bool, true>{});
    else load(std::integral_constant<bool, false>{});
  };
  if (s.g_type == FIM_F32) load_of(std::integral_constant<int, FIM_F32>{});
  else if (s.g_type == FIM_BF16) load_of(std::integral_constant<int, FIM_BF16>{});
  else load_of(std::integral_constant<int, FIM_F16>{});
  if constexpr (MODE == THIN_FIRST)
    for (uint32_t i = tid; i < s.chunks; i += 64 * SMALL_WAVES) sq += s.part[b * s.chunks + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sq += __shfl_xor(sq, o);
  double* red = reinterpret_cast<double*>(sums);
  if (lane == 0) red[wave] = sq;
  __syncthreads();
  sq = red[0];
#pragma unroll
  for (int i = 1; i < SMALL_WAVES; ++i) sq += red[i];
  const OrthoScale scaled(sqrt(sq) + k.eps, k.sx);
  // -- sx X0 as halves, line by line in place: 8 lanes a line, all of which read before one writes
#pragma unroll 4
  for (int i = tid; i < MP * nb * 8; i += 64 * SMALL_WAVES) {
    const int q = i & 7, line = i >> 3, r = line / nb;
    uint8_t* at = X + line * 128;
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = scaled(*reinterpret_cast<const float*>(at + (((4 * q + u) ^ (r & 31)) << 2)));
    v2i hi, lo;
    split4(v, hi, lo);
    const int key = small_key(r);
    wave_lds_wait();
    *reinterpret_cast<v2i*>(at + (((q >> 1) ^ key) << 4) + (q & 1) * 8) = hi;
    *reinterpret_cast<v2i*>(at + (((4 + (q >> 1)) ^ key) << 4) + (q & 1) * 8) = lo;
  }
  }

  // the slab's lines as the workspace has them, without the swizzle
  uint8_t* stored = MODE == SMALL_WHOLE ? nullptr : s.x[0] + b * s.each + line0 * 128;
  auto move_slab = [&](bool out) __attribute__((always_inline)) {
#pragma unroll 4
    for (int i = tid; i < MP * nb * 8; i += 64 * SMALL_WAVES) {
      const int line = i >> 3, r = line / nb;
      v4i* global = reinterpret_cast<v4i*>(stored + (int64_t)r * np * 4 + (line - r * nb) * 128 + (i & 7) * 16);
      v4i* local_at = reinterpret_cast<v4i*>(X + line * 128 + (((i & 7) ^ small_key(r)) << 4));
      if (out) *global = *local_at;
      else *local_at = *global;
    }
  };
  if constexpr (MODE == THIN_STEP) move_slab(false);

  // fragments: lane: row (or column) l % 16, contraction 8 (l / 16) .. + 7 of 32
  auto along = [&](const uint8_t* p, int row_bytes, int r0, int line, int plane) __attribute__((always_inline)) {
    const int r = r0 + l16;
    return *reinterpret_cast<const s16x8*>(p + r * row_bytes + line * 128 + (((4 * plane + g) ^ small_key(r)) << 4));
  };
  auto across = [&](int r0, int col16, int plane) __attribute__((always_inline)) {  // X's rows r0 .. r0 + 31 (past MP: any, P is 0)
    s16x4 half[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int r = r0 + 8 * g + 4 * q + (l16 >> 2);
      if (MP % 32 != 0) r = r < MP ? r : r - 16;
      const int seg = 4 * plane + 2 * (col16 & 1) + ((lane & 3) >> 1);
      half[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(X + r * ld + (col16 >> 1) * 128 + ((seg ^ small_key(r)) << 4) + (lane & 1) * 8));
    }
    return __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // a block's values (lane: row l % 16, columns 4 g ..) into A or P as halves
  auto put = [&](uint8_t* p, int r, int c, const float (&v)[4]) __attribute__((always_inline)) {
    v2i hi, lo;
    split4(v, hi, lo);
    uint8_t* at = p + r * (LINES * 128) + (c >> 5) * 128;
    const int key = small_key(r), seg = (c & 31) >> 3;
    *reinterpret_cast<v2i*>(at + ((seg ^ key) << 4) + (c & 7) * 2) = hi;
    *reinterpret_cast<v2i*>(at + (((4 + seg) ^ key) << 4) + (c & 7) * 2) = lo;
  };
  constexpr int OWN = (T * T + SMALL_WAVES - 1) / SMALL_WAVES;  // blocks of A and P of a wavefront
  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
  const float gram_scale = k.sa / (k.sx * k.sx), apply_scale = 1.0f / k.sp, last_scale = apply_scale / k.sx;
  const float sq_scale = k.c * k.sp / (k.sa * k.sa), old_scale = k.b * k.sp / k.sa;

  float own[OWN][4];  // this wavefront's blocks of X X^T
  auto gram = [&]() __attribute__((always_inline)) {
    // -- A = X X^T: this wavefront's lines, all pairs of row blocks
    v4f acc[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) acc[i] = zero;
    __syncthreads();
    for (int line = wave; line < nb && wave < SUMS; line += SUMS) {
      s16x8 f[T][2];
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) f[i][pl] = along(X, ld, 16 * i, line, pl);
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 0, q = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j <= i; ++j, ++q) acc[q] = mfma_small(f[j][part == 2], f[i][part == 1], acc[q]);
    }
    if (wave < SUMS) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) *reinterpret_cast<v4f*>(sums + (wave * PAIRS + i) * 256 + lane * 4) = acc[i];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
      const int q = wave + SMALL_WAVES * t, i = q / T, j = q % T;
#pragma unroll
      for (int u = 0; u < 4; ++u) own[t][u] = 0.0f;
      if (q < T * T) {
        const int hi = i > j ? i : j, lo = i > j ? j : i;
        const float* from = sums + (hi * (hi + 1) / 2 + lo) * 256;
#pragma unroll
        for (int w = 0; w < SUMS; ++w)
#pragma unroll
          for (int u = 0; u < 4; ++u)  // above the diagonal: row l % 16, column 4 g + u of the block below, across
            own[t][u] += from[w * PAIRS * 256 + (i >= j ? lane * 4 + u : ((l16 >> 2) * 16 + 4 * g + u) * 4 + (l16 & 3))];
      }
    }
  };
  auto polynomial = [&]() __attribute__((always_inline)) {
    if constexpr (!APART) __syncthreads();  // (A and P lie where the sums lay)
    if (!APART && (T == 1 || T == 3)) {  // columns past 16 T of the last line: zero
      for (int i = tid * 16; i < 2 * MP * LINES * 128; i += 64 * SMALL_WAVES * 16) *reinterpret_cast<v4i*>(A + i) = v4i{0, 0, 0, 0};
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
      const int q = wave + SMALL_WAVES * t;
#pragma unroll
      for (int u = 0; u < 4; ++u) own[t][u] *= gram_scale;
      if (q < T * T) put(A, 16 * (q / T) + l16, 16 * (q % T) + 4 * g, own[t]);
    }
    __syncthreads();
    // -- P = a I + b A + c A^2
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
      const int q = wave + SMALL_WAVES * t, i = q / T, j = q % T;
      if (q < T * T) {
        v4f w[3] = {zero, zero, zero};
#pragma unroll
        for (int line = 0; line < LINES; ++line) {
          s16x8 fi[2], fj[2];
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) {
            fi[pl] = along(A, LINES * 128, 16 * i, line, pl);
            fj[pl] = along(A, LINES * 128, 16 * j, line, pl);
          }
#pragma unroll
          for (int part = 0; part < 3; ++part) w[part] = mfma_small(fj[part == 2], fi[part == 1], w[part]);
        }
        const int r = 16 * i + l16, c = 16 * j + 4 * g;
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[u] = fmaf(sq_scale, w[0][u] + (w[1][u] + w[2][u]), old_scale * own[t][u]);
          if (r == c + u) v[u] += k.a * k.sp;
        }
        put(P, r, c, v);
      }
    }
    __syncthreads();
  };
  auto apply = [&](bool last) __attribute__((always_inline)) {
    // -- X = P X: 16 columns a turn
    for (int c16 = wave; c16 < 2 * nb; c16 += SMALL_WAVES) {
      v4f y[T];
#pragma unroll
      for (int i = 0; i < T; ++i) y[i] = zero;
#pragma unroll
      for (int line = 0; line < LINES; ++line) {
        const s16x8 xh = across(32 * line, c16, 0), xl = across(32 * line, c16, 1);
        s16x8 fp[T][2];
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) fp[i][pl] = along(P, LINES * 128, 16 * i, line, pl);
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
          for (int i = 0; i < T; ++i) y[i] = mfma_small(part == 2 ? xl : xh, fp[i][part == 1], y[i]);
      }
      const int c = 16 * c16 + 4 * g, cx = line0 * 32 + c;  // of the slab, of X
#pragma unroll
      for (int i = 0; i < T; ++i) {
        const int r = 16 * i + l16;
        float v[4];
        if (last) {
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = y[i][u] * last_scale;
          if (s.tall) {
            if (r < cols) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (cx + u < rows) finish1(s, k, base + (int64_t)(cx + u) * cols + r, v[u]);
            }
          } else if (r < rows && cx < cols) {
            finish4(s, k, base + (int64_t)r * cols + cx, cols - cx, v);
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = y[i][u] * apply_scale;
          v2i hi, lo;
          split4(v, hi, lo);
          uint8_t* at = X + r * ld + (c >> 5) * 128;
          const int key = small_key(r), seg = (c & 31) >> 3;
          *reinterpret_cast<v2i*>(at + ((seg ^ key) << 4) + (c & 7) * 2) = hi;
          *reinterpret_cast<v2i*>(at + (((4 + seg) ^ key) << 4) + (c & 7) * 2) = lo;
        }
      }
    }
  };

  if constexpr (MODE == SMALL_WHOLE) {
    for (int it = 0; it < k.steps; ++it) {
      gram();
      polynomial();
      apply(it == k.steps - 1);
    }
    return;
  }
  // parts of X X^T: [slab][T T][256], two of them in turn: a workgroup of this launch may still read the last ones
  auto parts = [&](int turn) __attribute__((always_inline)) {
    return reinterpret_cast<float*>((turn & 1 ? s.p : s.a) + b * s.each) + lane * 4;
  };
  if constexpr (MODE == THIN_STEP) {
#pragma unroll
    for (int t = 0; t < OWN; ++t) {
      const int q = wave + SMALL_WAVES * t;
      v4f sum = zero;
      if (q < T * T) {
#pragma unroll 8
        for (uint32_t i = 0; i < s.slabs; ++i) sum += *reinterpret_cast<const v4f*>(parts(step) + ((int64_t)i * (T * T) + q) * 256);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) own[t][u] = sum[u];
    }
    polynomial();
    const bool last = step == k.steps - 1;
    apply(last);
    if (last) return;
    __syncthreads();
  } else {
    __syncthreads();
  }
  move_slab(true);
  gram();
#pragma unroll
  for (int t = 0; t < OWN; ++t) {
    const int q = wave + SMALL_WAVES * t;
    if (q < T * T)
      *reinterpret_cast<v4f*>(parts(MODE == THIN_FIRST ? 0 : step + 1) + ((int64_t)(line0 / (int)s.slab) * (T * T) + q) * 256) =
          v4f{own[t][0], own[t][1], own[t][2], own[t][3]};
  }
}

}  // namespace fim
