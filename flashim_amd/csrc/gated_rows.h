// The gated feed-forward operator over many rows of few channels (a contraction of at most 128): a stream of rows.
//
// On tiles, a product with one or two steps of contraction is all prologue and epilogue, and a workgroup's phases follow each
// other. Here the weights of a block of hidden columns stay in LDS for the whole launch (64 KB), and each of a workgroup's
// eight wavefronts works alone on 32 rows at a time: it loads them straight into MFMA operand registers, the next 32 while it
// works, multiplies them by 32 hidden columns at a time, and writes whole 128-byte lines through its own LDS area. No barrier
// after the weights are in; the wavefronts of a SIMD drift apart, one's vector work covers another's loads.
//
// A stream: x read once, the output written once. Measured (device time, MI355X, BF16, SiLU): 320000 x 64 -> 256, 48 us (77 on
// tiles; 205 MB, 4.3 TB/s; 58 us in the first calls after a pause; the vector work of the activation and the stores' way through
// LDS are 55% of it); 160000 x 128 -> 512, 64 us (82 on tiles).
// Outputs are stored plainly: marked as streams, the product that read them next took 104 us in place of 97 with this one.
#pragma once

#include "gated_tile.h"

namespace fim {

struct RowsArgs {
  const uint16_t* x;      // [M, kw], 16-byte aligned rows
  const uint16_t* w[2];   // [H, kw]
  int64_t ldx, ldw, M;
  int K, kw, H;           // kw: K rounded up to 8
  const void* bias[2];
  int bias_dtype;
  uint16_t* out;          // [M, H] packed
  int blocks;             // hidden blocks; workgroup i takes block i % blocks
  // backward (gated_rows_grad.h)
  const uint16_t* dout;
  int64_t ldd;
  uint16_t* dx;           // [M, K] packed, or null
  float* dw_part;         // [workgroups * sub][2][H][K], or null
  float* col_sums;        // [workgroups * sub][2][H], or null
  int wide_dx;            // 8-byte stores of dx
  int sub;                // 32-row blocks of a step
};

constexpr int ROWS_WAVES = 8;
constexpr int rows_hidden(int kp) { return 16384 / kp; }  // hidden columns of a block: 64 KB of weights

// A wavefront's [32 rows, 64 columns] in its LDS area to rows of 128 bytes at `out` (rows `ld` apart, `rows` of them; `to`: the
// same as a buffer, where bytes and columns past the end go out of range)
template <bool WIDE>
__device__ __forceinline__ void store_rows64(const uint8_t* area, uint16_t* out, const __amdgpu_buffer_rsrc_t to, int64_t ld,
                                             int64_t rows, int col0, int cols, int lane) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const int slot = lane & 7, row0 = lane >> 3, col = col0 + slot * 8;
  v4i v[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = p * 8 + row0;
    v[p] = *reinterpret_cast<const v4i*>(area + row * 128 + ((slot ^ ((row >> 1) & 7)) << 4));
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[p]), to,
                                             (int)(col < cols ? (uint32_t)((p * 8 + row0) * ld + col) * 2u : TILE_OOB), 0, 0);
  } else if (rows >= 32 && col + 8 <= cols) {
#pragma unroll
    for (int p = 0; p < 4; ++p) *reinterpret_cast<v4i_any*>(out + (p * 8 + row0) * ld + col) = v[p];
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int c = 0; c < 8; ++c)
        __builtin_amdgcn_raw_buffer_store_b16(
            (uint16_t)((uint32_t)v[p][c / 2] >> (16 * (c & 1))), to,
            (int)(col + c < cols ? (uint32_t)((p * 8 + row0) * ld + col + c) * 2u : TILE_OOB), 0, 0);
  }
}

template <int DT, int ACT, int KP, bool WIDE>
__global__ __launch_bounds__(64 * ROWS_WAVES, 2) void gated_rows_kernel(const RowsArgs a) {
  constexpr int HB = rows_hidden(KP), KS = KP / 16, KB = KP / 32;
  constexpr int REGION = 2 * HB * 128;  // 64 channels of all weight rows
  __shared__ __attribute__((aligned(16))) uint8_t wl[KP / 64 * REGION];
  __shared__ __attribute__((aligned(16))) float bias[2 * HB];
  __shared__ __attribute__((aligned(16))) uint8_t areas[ROWS_WAVES * 4096];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = __builtin_amdgcn_readfirstlane((int)blockIdx.x % a.blocks);
  const int group = __builtin_amdgcn_readfirstlane((int)blockIdx.x / a.blocks);
  const int groups = __builtin_amdgcn_readfirstlane((int)gridDim.x / a.blocks);
  const int n0 = block * HB, hidden = a.H - n0 < HB ? a.H - n0 : HB;

  // the block's weights: row r (gate rows, then up rows), channels 64 s .. 64 s + 63 at region s, 16-byte slots swizzled by
  // the row as the tiles' stages are
  for (int i = tid; i < 2 * HB * (KP / 8); i += 64 * ROWS_WAVES) {
    const int r = i / (KP / 8), seg = i - r * (KP / 8), n = r % HB;
    v4i v = {0, 0, 0, 0};
    if (n < hidden && seg * 8 < a.kw) v = *reinterpret_cast<const v4i*>(a.w[r / HB] + (int64_t)(n0 + n) * a.ldw + seg * 8);
    *reinterpret_cast<v4i*>(wl + (seg >> 3) * REGION + r * 128 + (((seg & 7) ^ ((r >> 1) & 7)) << 4)) = v;
  }
  for (int i = tid; i < 2 * HB; i += 64 * ROWS_WAVES) {
    const void* b = a.bias[i / HB];
    const int n = i % HB;
    bias[i] = b == nullptr || n >= hidden ? 0.0f
              : a.bias_dtype == FIM_F32   ? static_cast<const float*>(b)[n0 + n]
                                          : from16<DT>(static_cast<const uint16_t*>(b)[n0 + n]);
  }
  __syncthreads();

  uint8_t* area = areas + wave * 4096;
  const int64_t row_blocks = (a.M + 31) / 32, step = (int64_t)groups * ROWS_WAVES;
  const int fsw = (row >> 1) & 7;
  auto left_bytes = [&](int64_t r0, int64_t ld, int64_t cols) __attribute__((always_inline)) {
    const int64_t rows = a.M - r0 < 32 ? a.M - r0 : 32;
    return __builtin_amdgcn_readfirstlane(rows <= 0 ? 0 : (int)(((rows - 1) * ld + cols) * 2));
  };
  // this lane's operands of 32 rows: channels 16 kk + 8 h .. + 7
  s16x8 xf[2][KS];
  auto load_x = [&](int64_t rb, s16x8 (&f)[KS]) __attribute__((always_inline)) {
    const int64_t r0 = rb < row_blocks ? rb * 32 : a.M;
    const auto src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.x) + r0 * a.ldx, (short)0,
                                                       left_bytes(r0, a.ldx, a.kw), 0x00020000);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const int k = 16 * kk + 8 * h;
      const uint32_t at = (uint32_t)(row * a.ldx + k) * 2u;
      f[kk] = __builtin_bit_cast(
          s16x8, __builtin_amdgcn_raw_buffer_load_b128(src, (int)(k < a.kw ? at : TILE_OOB), 0, 0));
    }
  };

  auto work = [&](int64_t rb, const s16x8 (&x)[KS]) __attribute__((always_inline)) {
    const int64_t r0 = rb * 32;
    const auto to = __builtin_amdgcn_make_buffer_rsrc(a.out + r0 * a.H + n0, (short)0, left_bytes(r0, a.H, hidden), 0x00020000);
    const int hbs = (hidden + 31) / 32;
    // 32 hidden columns; odd: the second half of a 64-column line
    auto part = [&](int hb, auto odd_c) __attribute__((always_inline)) {
      constexpr int ODD = decltype(odd_c)::value;
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
      for (int kk = 0; kk < KS; ++kk) {
        const int off = (kk >> 2) * REGION + (((2 * (kk & 3) + h) ^ fsw) << 4);
        g = mfma16<DT>(*reinterpret_cast<const s16x8*>(wrow + off), x[kk], g);
        u = mfma16<DT>(*reinterpret_cast<const s16x8*>(wrow + HB * 128 + off), x[kk], u);
      }
      typedef int v2i __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate<ACT>(g[4 * q + e]) * u[4 * q + e];
        *reinterpret_cast<v2i*>(area + row * 128 + (((ODD * 4 + q) ^ fsw) << 4) + 8 * h) =
            v2i{(int)to16x2<DT>(v[0], v[1]), (int)to16x2<DT>(v[2], v[3])};
      }
    };
    for (int hb = 0; hb < hbs; hb += 2) {
      part(hb, std::integral_constant<int, 0>{});
      if (hb + 1 < hbs) part(hb + 1, std::integral_constant<int, 1>{});
      wave_lds_wait();
      store_rows64<WIDE>(area, a.out + r0 * a.H + n0, to, a.H, a.M - r0, hb * 32, hidden, lane);
      wave_lds_wait();
    }
  };

  int64_t rb = (int64_t)group * ROWS_WAVES + wave;
  load_x(rb, xf[0]);
  for (; rb < row_blocks; rb += 2 * step) {
    load_x(rb + step, xf[1]);
    work(rb, xf[0]);
    if (rb + step >= row_blocks) break;
    load_x(rb + 2 * step, xf[0]);
    work(rb + step, xf[1]);
  }
}

}  // namespace fim
