// The backward pass of the gated feed-forward operator over many rows, of at most 64 channels and 256 hidden columns: one
// pass over x and dout that leaves dx and each workgroup's partial sums of the weights' and biases' gradients.
//
// dg and du never leave the CU: written and read again they were 0.6 of the bytes moved (320000 x 64 -> 256 with its joins, in turn:
// 156 us, 337 us on tiles). A workgroup keeps all weights in LDS and takes 32 rows at a time (64 where H is at most 128). Each of
// its eight wavefronts owns 32 hidden columns: it multiplies them, applies the epilogue, adds its dg^T x and du^T x to
// accumulators that stay in registers for the whole launch, and its column sums too. dg and du go to LDS in 16 bits (operands of
// 16-bit products, as everywhere in this operator); after one barrier each wavefront takes a 16 x 16 tile of dx, contracted over
// all of them. With two LDS copies of dg, du and x that is the only barrier of a step: a wavefront writes the next step's while
// others still read this one's.
//
// Measured (device time of this kernel alone, MI355X, BF16, SiLU): 320000 x 64 -> 256, 124 us after two hundred calls, 162 us in
// the first calls after a pause (246 MB are 48 us): vector work 50% of the cycles, matrix products 20%, LDS 42%, with two
// wavefronts per SIMD to overlap them. The joins of the weights' and the biases' partials take 7 + 5 us beside it.
#pragma once

#include "gated_few.h"
#include "gated_rows.h"

namespace fim {

constexpr int GRAD_HIDDEN = 256;  // hidden columns whose weights fit: 64 KB with 64 channels

// 32-row blocks of a step: as many as wavefronts per hidden block allow
inline int rows_grad_sub(int64_t H) { return H <= GRAD_HIDDEN / 2 ? 2 : 1; }

// Where a row's 16-byte slots go, by XOR: rows of 128 bytes (x, weights), and of 256 or more (dg, du). Sixteen rows read at
// one slot spread over all banks either way; and so do the four rows by 64 bytes, or eight by 32, of a transposed read.
__device__ __forceinline__ int swizzle8(int r) { return ((r << 1) & 4) | ((r >> 2) & 2) | ((r >> 2) & 1); }
__device__ __forceinline__ int swizzle16(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

template <int DT, int ACT, bool WIDE>
__global__ __launch_bounds__(64 * ROWS_WAVES, 2) void gated_rows_grad_kernel(const RowsArgs a) {
  constexpr int HB = GRAD_HIDDEN, XT = 2 * 4096, DT_BYTES = 32 * 2 * HB * 2;
  __shared__ __attribute__((aligned(16))) uint8_t wl[2 * HB * 128];
  __shared__ __attribute__((aligned(16))) uint8_t xl[2 * XT];
  __shared__ __attribute__((aligned(16))) uint8_t dl[2 * DT_BYTES];
  __shared__ __attribute__((aligned(16))) float bias[2 * HB];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = ROWS_WAVES / a.sub, hb = wave % nb, rs = wave / nb;  // this wavefront's hidden block and row block
  const int hbs = (a.H + 31) / 32, stride = nb * 128;                 // bytes of a row of dg and du in LDS
  const bool active = hb < hbs;

  // weights: 128 bytes a row
  for (int i = tid; i < 2 * HB * 8; i += 64 * ROWS_WAVES) {
    const int r = i >> 3, seg = i & 7, n = r % HB;
    v4i v = {0, 0, 0, 0};
    if (n < a.H && seg * 8 < a.kw) v = *reinterpret_cast<const v4i*>(a.w[r / HB] + (int64_t)n * a.ldw + seg * 8);
    *reinterpret_cast<v4i*>(wl + r * 128 + ((seg ^ swizzle8(r)) << 4)) = v;
  }
  for (int i = tid; i < 2 * HB; i += 64 * ROWS_WAVES) {
    const void* b = a.bias[i / HB];
    const int n = i % HB;
    bias[i] = b == nullptr || n >= a.H  ? 0.0f
              : a.bias_dtype == FIM_F32 ? static_cast<const float*>(b)[n]
                                        : from16<DT>(static_cast<const uint16_t*>(b)[n]);
  }
  // (hidden blocks past the end stay zero: dx's contraction runs over them)
  for (int i = tid; i < 2 * DT_BYTES / 16; i += 64 * ROWS_WAVES) *reinterpret_cast<v4i*>(dl + i * 16) = v4i{0, 0, 0, 0};

  const int rows_step = 32 * a.sub;
  const int64_t steps = (a.M + rows_step - 1) / rows_step;
  const int fsw = swizzle8(row);
  auto left_bytes = [&](int64_t r0, int most, int64_t ld, int64_t cols) __attribute__((always_inline)) {
    const int64_t rows = a.M - r0 < most ? a.M - r0 : most;
    return __builtin_amdgcn_readfirstlane(rows <= 0 ? 0 : (int)(((rows - 1) * ld + cols) * 2));
  };
  // 16 bytes of x a thread, and where they lie in LDS
  const int xrow = tid >> 3, xseg = tid & 7;
  const bool loads_x = xrow < rows_step;
  const int xat = xrow * 128 + ((xseg ^ swizzle8(xrow)) << 4);
  auto load_x = [&](int64_t step) __attribute__((always_inline)) {
    const int64_t r0 = step < steps ? step * rows_step : a.M;
    const auto src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.x) + r0 * a.ldx, (short)0,
                                                       left_bytes(r0, rows_step, a.ldx, a.kw), 0x00020000);
    const uint32_t at = (uint32_t)(xrow * a.ldx + xseg * 8) * 2u;
    return __builtin_bit_cast(
        v4i, __builtin_amdgcn_raw_buffer_load_b128(src, (int)(loads_x && xseg * 8 < a.kw ? at : TILE_OOB), 0, 0));
  };
  // the incoming gradient of this wavefront's 32 x 32: lane h loads 8 columns 16 p + 8 h
  auto load_d = [&](int64_t step, v4i (&d)[2]) __attribute__((always_inline)) {
    const int64_t at0 = step * rows_step + 32 * rs, r0 = step < steps && at0 < a.M ? at0 : a.M;
    const auto src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.dout) + r0 * a.ldd, (short)0,
                                                       left_bytes(r0, 32, a.ldd, a.H), 0x00020000);
    if constexpr (WIDE) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int col = hb * 32 + 16 * p + 8 * h;
        d[p] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
                                           src, (int)(col < a.H ? (uint32_t)(row * a.ldd + col) * 2u : TILE_OOB), 0, 0));
      }
    } else if (a.M - r0 >= 32 && hb * 32 + 32 <= a.H) {
      const uint16_t* from = a.dout + (r0 + row) * a.ldd + hb * 32 + 8 * h;
#pragma unroll
      for (int p = 0; p < 2; ++p) d[p] = *reinterpret_cast<const v4i_any*>(from + 16 * p);
    } else {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int col = hb * 32 + 16 * p + 8 * h;
        const uint32_t at = (uint32_t)(row * a.ldd + col) * 2u;
        uint32_t e[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          e[c] = __builtin_amdgcn_raw_buffer_load_b16(src, (int)(col + c < a.H ? at + 2 * c : TILE_OOB), 0, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c) d[p][c] = (int)(e[2 * c] | e[2 * c + 1] << 16);
      }
    }
  };

  // transposed reads: each 16 lanes read 4 rows of 16 columns and get a column each
  const int i16 = lane & 15, trow = 8 * h + (i16 >> 2), tcol = ((lane >> 4) & 1) * 16 + 4 * (i16 & 3);
  auto transposed = [&](const uint8_t* p) __attribute__((always_inline)) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  };

  v16f dw[2][2];    // [gate, up][channels 32 b ..]: lane: channel, registers: hidden column
  float sums[32];   // of dg and du over this lane's rows
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int q = 0; q < 16; ++q) dw[i >> 1][i & 1][q] = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) sums[i] = 0.0f;

  v4i xr, d[2];

  // A step's dg, du and their part of the weights' gradients; x and dout of the next ones are on their way meanwhile
  auto gradients = [&](int64_t step, int cur) __attribute__((always_inline)) {
    const uint8_t* xt = xl + cur * XT + rs * 4096;
    uint8_t* dt = dl + cur * DT_BYTES;
    if (active) {
      typedef int v2i __attribute__((ext_vector_type(2)));
      v2i dv[4];  // as an accumulator block lies: the halves exchange the 4 columns that are the other's
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)d[p][c], (uint32_t)d[p][c + 2], false, false);
          dv[2 * p][c] = (int)r[0];
          dv[2 * p + 1][c] = (int)r[1];
        }
      load_d(step + gridDim.x, d);
      v16f g, u;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v4f bg = *reinterpret_cast<const v4f*>(bias + hb * 32 + 8 * q + 4 * h);
        const v4f bu = *reinterpret_cast<const v4f*>(bias + HB + hb * 32 + 8 * q + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[4 * q + e] = bg[e];
          u[4 * q + e] = bu[e];
        }
      }
      const uint8_t* wrow = wl + (hb * 32 + row) * 128;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int off = ((2 * kk + h) ^ fsw) << 4;
        const s16x8 x = *reinterpret_cast<const s16x8*>(xt + row * 128 + off);
        g = mfma16<DT>(*reinterpret_cast<const s16x8*>(wrow + off), x, g);
        u = mfma16<DT>(*reinterpret_cast<const s16x8*>(wrow + HB * 128 + off), x, u);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w = (uint32_t)dv[i >> 2][(i >> 1) & 1];
        const float dd = from16<DT>((uint16_t)(i & 1 ? w >> 16 : w));
        float slope;
        const float act = activate<ACT, true>(g[i], slope);
        g[i] = dd * u[i] * slope;
        u[i] = dd * act;
      }
      const int64_t left = a.M - step * rows_step - 32 * rs;
      if (left < 32) {  // rows past the end: zero times anything
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          g[i] = row < left ? g[i] : 0.0f;
          u[i] = row < left ? u[i] : 0.0f;
        }
      }
      uint8_t* drow_at = dt + (32 * rs + row) * stride + 8 * h;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sums[4 * q + e] += g[4 * q + e];
          sums[16 + 4 * q + e] += u[4 * q + e];
        }
        *reinterpret_cast<v2i*>(drow_at + (((hb * 4 + q) ^ swizzle16(row)) << 4)) =
            v2i{(int)to16x2<DT>(g[4 * q], g[4 * q + 1]), (int)to16x2<DT>(g[4 * q + 2], g[4 * q + 3])};
        *reinterpret_cast<v2i*>(drow_at + (((nb * 4 + hb * 4 + q) ^ swizzle16(row)) << 4)) =
            v2i{(int)to16x2<DT>(u[4 * q], u[4 * q + 1]), (int)to16x2<DT>(u[4 * q + 2], u[4 * q + 3])};
      }
    }
    if (loads_x) *reinterpret_cast<v4i*>(xl + (cur ^ 1) * XT + xat) = xr;
    xr = load_x(step + 2 * (int64_t)gridDim.x);
    if (active && a.dw_part != nullptr) {  // this wavefront's dg^T x and du^T x: 32 rows are two sub-steps
      wave_lds_wait();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        s16x8 xf[2], df[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s16x4 t[2], td[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int r = 16 * s + 4 * k + trow, c = b * 32 + tcol;
            t[k] = transposed(xt + r * 128 + (((c >> 3) ^ swizzle8(r)) << 4) + (c & 7) * 2);
            td[k] = transposed(dt + (32 * rs + r) * stride + (((b * nb * 4 + hb * 4 + (tcol >> 3)) ^ swizzle16(r)) << 4) + (tcol & 7) * 2);
          }
          xf[b] = __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7);
          df[b] = __builtin_shufflevector(td[0], td[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int up = 0; up < 2; ++up)
#pragma unroll
          for (int b = 0; b < 2; ++b) dw[up][b] = mfma16<DT>(df[up], xf[b], dw[up][b]);
      }
    }
  };

  // This wavefront's tiles of a step's dx
  const int kg = lane >> 4, ct = wave & 3, col = ct * 16 + 4 * kg;
  auto products = [&](int64_t step, int cur) __attribute__((always_inline)) {
    const uint8_t* dt = dl + cur * DT_BYTES;
    const int64_t r0 = step * rows_step;
    const auto to = __builtin_amdgcn_make_buffer_rsrc(a.dx + r0 * a.K, (short)0, left_bytes(r0, rows_step, a.K, a.K),
                                                      0x00020000);
    const int c = ct * 16 + 4 * (i16 & 3), wr = 8 * kg + (i16 >> 2);
    const uint8_t* w_at[2];  // + 4 k rows; a swizzle that is the same 32 rows on
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w_at[k] = wl + (wr + 4 * k) * 128 + (((c >> 3) ^ swizzle8(wr + 4 * k)) << 4) + (c & 7) * 2;
    for (int rt = wave >> 2; rt < 2 * a.sub; rt += 2) {
      const int r = rt * 16 + i16;
      v4f acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll 1
      for (int st = 0; st < 2 * nb; st += 4) {  // four hidden blocks, of the gate's first: 256 bytes of a row
        const int on = (st < nb ? 32 * st : HB + 32 * (st - nb)) * 128;
        s16x8 df[4], wf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          df[j] = *reinterpret_cast<const s16x8*>(dt + r * stride + st * 64 + (((4 * j + kg) ^ swizzle16(i16)) << 4));
          wf[j] = __builtin_shufflevector(transposed(w_at[0] + on + j * 4096), transposed(w_at[1] + on + j * 4096), 0, 1, 2, 3,
                                          4, 5, 6, 7);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j & 1] = mfma16x16<DT>(wf[j], df[j], acc[j & 1]);
      }
      const v4f v = acc[0] + acc[1];  // lane: row, registers: channels 4 kg ..
      const uint32_t w[2] = {to16x2<DT>(v[0], v[1]), to16x2<DT>(v[2], v[3])};
      const uint32_t at = (uint32_t)(r * a.K + col) * 2u;
      if (a.wide_dx) {
        typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{w[0], w[1]}, to, (int)(col < a.K ? at : TILE_OOB), 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(w[e >> 1] >> (16 * (e & 1))), to,
                                                (int)(col + e < a.K ? at + 2 * e : TILE_OOB), 0, 0);
      }
    }
  };

  // Between two barriers: dx of one step and the gradients of the next, in either order. The two wavefronts of a SIMD take
  // them in opposite orders, so one's matrix and LDS work runs beside the other's vector work.
  const int64_t first = blockIdx.x;
  xr = load_x(first);
  load_d(first, d);
  if (loads_x) *reinterpret_cast<v4i*>(xl + xat) = xr;
  xr = load_x(first + gridDim.x);
  const bool late = wave >= 4;
  int cur = 1;
  for (int64_t next = first; next < steps + gridDim.x; next += gridDim.x, cur ^= 1) {  // (first: nothing to contract yet)
    __syncthreads();
    const bool contracts = a.dx != nullptr && next != first;
    if (contracts && !late) products(next - gridDim.x, cur);
    if (next < steps) gradients(next, cur ^ 1);
    if (contracts && late) products(next - gridDim.x, cur);
  }

  if (!active) return;
  const int64_t part = (int64_t)blockIdx.x * a.sub + rs;
  if (a.dw_part != nullptr) {
    float* to = a.dw_part + part * 2 * a.H * a.K;
#pragma unroll
    for (int up = 0; up < 2; ++up)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const int n = hb * 32 + 8 * (q >> 2) + 4 * h + (q & 3), k = b * 32 + row;
          if (n < a.H && k < a.K) to[((int64_t)up * a.H + n) * a.K + k] = dw[up][b][q];
        }
  }
  if (a.col_sums != nullptr) {  // lane l: the sum of value l % 32 (gate: 0..15, up) of its half's columns
    sum_lanes<16>(sums, lane);
    const int q = row & 15, n = hb * 32 + 8 * (q >> 2) + 4 * h + (q & 3);
    if (n < a.H) a.col_sums[(part * 2 + (row >> 4)) * a.H + n] = sums[0];
  }
}

}  // namespace fim
