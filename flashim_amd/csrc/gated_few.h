// The gated feed-forward product of a few rows (at most 64): the weights are the traffic, each read once.
//
// A workgroup takes 16 hidden columns; its eight wavefronts share the contraction, 64 channels at a time, and load both
// weights' rows straight into MFMA operands (lane l: row l % 16, channels 8 (l / 16) + 32 s), so a launch of H / 16 workgroups
// has all of a small layer's weights in flight at once. The wavefronts' sums are added through LDS in their order. Rows of any
// alignment are read in place: a copy to aligned rows, as the tiles take, would cost twice the product's own traffic.
//
// One row of 512 channels by 2 x 2048 hidden columns (4 MB of weights): 4.0 us, 7.4 us on a tile; the latency of a launch and
// of one round of loads, 0.8 us of traffic.
#pragma once

#include "gated_tile.h"

namespace fim {

struct FewArgs {
  const uint16_t* x;
  const uint16_t* w[2];
  int64_t ldx, ldw[2];
  int M, K, H;
  const void* bias[2];
  int bias_dtype;
  uint16_t* out;
  int wide_out;
};

constexpr int FEW_WAVES = 8, FEW_ROWS = 64;

// Eight channels from k on, zero past K, in loads of V
template <int V>
__device__ __forceinline__ s16x8 load_channels(const uint16_t* p, int k, int K) {
  s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if constexpr (V == 8) {
    const s16x8 got = *reinterpret_cast<const s16x8*>(p + (k < K ? k : 0));
    return k < K ? got : v;
  } else if constexpr (V == 2) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const s16x2 got = *reinterpret_cast<const s16x2*>(p + (k + 2 * i < K ? k + 2 * i : 0));
      v[2 * i] = k + 2 * i < K ? got[0] : (short)0;
      v[2 * i + 1] = k + 2 * i < K ? got[1] : (short)0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const short got = (short)p[k + i < K ? k + i : 0];
      v[i] = k + i < K ? got : (short)0;
    }
  }
  return v;
}

template <int DT>
__device__ __forceinline__ v4f mfma16x16(s16x8 a, s16x8 b, v4f c) {
  typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (DT == FIM_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// MT: blocks of 16 rows
template <int DT, int ACT, int MT, int V>
__global__ __launch_bounds__(64 * FEW_WAVES) void gated_few_kernel(const FewArgs a) {
  __shared__ v4f part[FEW_WAVES][2 * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4, n0 = blockIdx.x * 16;
  const int n = n0 + r < a.H ? n0 + r : a.H - 1;  // (rows past the end repeat the last; their sums are not stored)
  const uint16_t *wg = a.w[0] + n * a.ldw[0], *wu = a.w[1] + n * a.ldw[1];
  const uint16_t* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = a.x + (int64_t)(16 * t + r < a.M ? 16 * t + r : a.M - 1) * a.ldx;
  v4f g[MT], u[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) g[t] = u[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (int k0 = 64 * wave; k0 < a.K; k0 += 64 * FEW_WAVES) {
    s16x8 fg[2], fu[2], fx[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = k0 + 32 * s + 8 * c;
      fg[s] = load_channels<V>(wg, k, a.K);
      fu[s] = load_channels<V>(wu, k, a.K);
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[s][t] = load_channels<V>(x[t], k, a.K);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        g[t] = mfma16x16<DT>(fg[s], fx[s][t], g[t]);
        u[t] = mfma16x16<DT>(fu[s], fx[s][t], u[t]);
      }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    part[wave][t][lane] = g[t];
    part[wave][MT + t][lane] = u[t];
  }
  __syncthreads();
  // lane l of block t: row 16 t + l % 16, hidden columns 4 (l / 16) .. + 3
  for (int i = threadIdx.x; i < 64 * MT; i += 64 * FEW_WAVES) {
    const int t = i >> 6, l = i & 63, m = 16 * t + (l & 15), col = n0 + 4 * (l >> 4);
    if (m >= a.M || col >= a.H) continue;
    v4f v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = part[0][k * MT + t][l];
#pragma unroll
      for (int w = 1; w < FEW_WAVES; ++w) v[k] += part[w][k * MT + t][l];
    }
    uint16_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float b[2] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (a.bias[k] != nullptr && col + e < a.H)
          b[k] = a.bias_dtype == FIM_F32 ? static_cast<const float*>(a.bias[k])[col + e]
                                         : from16<DT>(static_cast<const uint16_t*>(a.bias[k])[col + e]);
      o[e] = to16<DT>(activate<ACT>(v[0][e] + b[0]) * (v[1][e] + b[1]));
    }
    uint16_t* to = a.out + (int64_t)m * a.H + col;
    if (a.wide_out) {
      *reinterpret_cast<uint2*>(to) = uint2{(uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < a.H) to[e] = o[e];
    }
  }
}

}  // namespace fim
