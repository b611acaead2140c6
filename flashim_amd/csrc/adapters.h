// What the low-rank adapters' kernels share: operands of any alignment, which adapter a row has, FP32 values as two of 16 bits.
#pragma once

#include "common.h"
#include "gated_tile.h"

namespace fim {

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef s16x4 s16x4_any __attribute__((aligned(2)));
typedef s16x8 s16x8_any __attribute__((aligned(2)));

// Row r's adapter: index[r / per] where that names one, else -1
struct AdapterIndex {
  const void* index;
  int wide;       // 64-bit values, else 32
  uint32_t per;   // rows of an entry
  int adapters;
};
__device__ __forceinline__ int adapter_of(const AdapterIndex& t, uint32_t row) {
  const uint32_t e = t.per == 1 ? row : row / t.per;
  if (t.wide) {
    const int64_t v = static_cast<const int64_t*>(t.index)[e];
    return v >= 0 && v < t.adapters ? (int)v : -1;
  }
  const int v = static_cast<const int*>(t.index)[e];
  return v >= 0 && v < t.adapters ? v : -1;
}

template <int DT>
__device__ __forceinline__ v4f mfma_rank(s16x8 a, s16x8 b, v4f c) {
  typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (DT == FIM_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// The first n of N neighbours, zeros after them
template <int N>
__device__ __forceinline__ auto load_some(const uint16_t* p, int n) {
  typedef short T __attribute__((ext_vector_type(N)));
  typedef T Any __attribute__((aligned(2)));
  if (n >= N) return (T) * reinterpret_cast<const Any*>(p);
  T v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? (short)p[i] : (short)0;
  return v;
}
template <int N, typename T>
__device__ __forceinline__ void store_some(uint16_t* p, int n, T v) {
  typedef T Any __attribute__((aligned(2)));
  if (n >= N) {
    *reinterpret_cast<Any*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (uint16_t)v[i];
}

// FP32 as hi + lo of 16 bits (16 or 22 bits of it). The compiler may not see where v comes from: it would round hi's two uses
// differently.
template <int DT>
__device__ __forceinline__ void split16(float v, short& hi, short& lo) {
  asm("" : "+v"(v));
  const uint16_t h = to16<DT>(v);
  const float rest = v - from16<DT>(h);
  hi = (short)h;
  lo = (short)to16<DT>(fabsf(rest) < __builtin_inff() ? rest : 0.0f);  // (infinity less infinity would be NaN)
}

// What lo meets of an operand that meets hi and lo: the same, but one in the place of an infinity. hi makes the infinity; lo, zero
// or of the other sign, would make NaN of it. (A NaN may become anything: hi makes it, too.)
template <int DT, typename T>
__device__ __forceinline__ T beside_hi(T v) {
  constexpr int N = sizeof(T) / 4;
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef int words __attribute__((ext_vector_type(N)));
  constexpr uint16_t most = DT == FIM_BF16 ? 0x7f7f : 0x7bff;
  words w = __builtin_bit_cast(words, v);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int both = w[i], size = both & 0x7fff7fff;
    const u16x2 past = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, size), u16x2{most, most});
    const u16x2 one = __builtin_bit_cast(u16x2, both) - (past << (uint16_t)14);
    w[i] = __builtin_bit_cast(int, one);
  }
  return __builtin_bit_cast(T, w);
}
// Four values of the second operand twice, for hi and lo of four of the first
template <int DT>
__device__ __forceinline__ s16x8 beside_halves(s16x4 v) {
  return __builtin_shufflevector(v, beside_hi<DT>(v), 0, 1, 2, 3, 4, 5, 6, 7);
}

// For the largest of finite values: an infinity or NaN beside them stays one whatever it is scaled by.
__device__ __forceinline__ float finite_abs(float v) { return fabsf(v) < __builtin_inff() ? fabsf(v) : 0.0f; }

// A power of two that brings values of at most `most` near FP16's upper end, and its inverse: FP16 has the range of neither large
// nor small FP32 values (gradients of 1e-6), and BF16 needs none.
__device__ __forceinline__ float half_scale(float most, float& inverse) {
  int up = 14 - ((int)(f2u(most) >> 23 & 255) - 127);
  up = up > 100 ? 100 : up;
  inverse = u2f((uint32_t)(127 - up) << 23);
  return u2f((uint32_t)(127 + up) << 23);
}

}  // namespace fim
