// What the Newton-Schulz kernels share: the table of matrices, their layout in 16-bit halves, loads and stores by type.
//
//   X0 = U / (|U|_F + eps), of the shorter side's rows (a tall matrix is transposed); `steps` times
//   A = X X^T,  P = a I + b A + c A^2,  X = P X;   O = X.   The optimizer's U = g + mu m after m = mu m + g.
//
// The products amplify what is small in X0 (by a^steps, 485 times at five steps), and with it any rounding of the large
// directions: operands of one BF16 each leave 1 to 5% of an output wrong, of one FP16 each 0.3 to 0.6%. So every operand is two FP16
// numbers, hi + lo, 22 bits, and a product is hi hi + hi lo + lo hi on the matrix cores with FP32 sums: errors of an FP32 product
// (1e-6 to 5e-6 of an output) at a third of the FP16 rate, which is five times the FP32 rate. X, A and P are stored times powers of
// two, as large as their entries' bounds (by the coefficients, computed on the host) allow, so that lo, too, is seldom below FP16's
// normal numbers.
#pragma once

#include <type_traits>

#include "common.h"
#include "gated_tile.h"

namespace fim {

// A stack of matrices of one shape, packed row-major; the table lies in the workspace. m <= n: sides, padded mp, np to 32.
struct OrthoStack {
  const void* g;
  float* mom;     // null: U = g
  void* out;      // O, or the parameters that are stepped in place
  uint8_t* x[2];  // sx X of the first matrix, [mp][np] halves; the others `each` bytes apart
  uint8_t* a;     // sa A, [mp][mp] halves
  uint8_t* p;     // sp P
  double* part;   // partial sums of squares, `chunks` a matrix
  int64_t each;
  uint32_t rows, cols, batch, mp, np, chunk, chunks;
  uint32_t slab, slabs;  // thin matrices: lines of 32 columns a workgroup, and workgroups a matrix; a and p: parts of X X^T
  float factor;     // O's factor in a step
  uint32_t first[5];  // first workgroup of a pass over: elements, conversion tiles, tiles of A, of P, of P X
  uint8_t g_type, out_type, tall, pad;
};
static_assert(sizeof(OrthoStack) % 8 == 0, "");

struct OrthoScalars {
  float momentum, keep;  // keep = 1 - lr * weight decay
  float a, b, c;
  float sx, sa, sp;  // powers of two that X, A and P are stored times
  double eps;
  int steps, nesterov, step;  // step: parameters are stepped; else O is written
};

// A row of halves: a line of 128 bytes for 32 columns, hi of all, then lo of all.
__device__ __forceinline__ uint32_t line_of(uint32_t col) { return (col >> 5) * 128 + (col & 31) * 2; }

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}
typedef int v2i __attribute__((ext_vector_type(2)));

// Four values as halves. The compiler may not see where they come from: it fuses a product and its conversion into one rounding
// for hi and not for lo's subtraction, and at a tie lo then belongs to the other neighbour.
__device__ __forceinline__ void split4(const float (&v)[4], v2i& hi, v2i& lo) {
  _Float16 h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = v[i];
    asm("" : "+v"(x));
    h[i] = (_Float16)x;
    l[i] = (_Float16)(x - (float)h[i]);
  }
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  hi = __builtin_bit_cast(v2i, (h4{h[0], h[1], h[2], h[3]}));
  lo = __builtin_bit_cast(v2i, (h4{l[0], l[1], l[2], l[3]}));
}
__device__ __forceinline__ void join4(v2i hi, v2i lo, float (&v)[4]) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  const h4 h = __builtin_bit_cast(h4, hi), l = __builtin_bit_cast(h4, lo);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)h[i] + (float)l[i];
}

// sx / (|U| + eps) as two FP32 factors, the first a power of two: 1 in the range where FP32 holds the quotient with room. (A sum
// below FP32's smallest number is eps beside a zero matrix, or zero, whose 0 / 0 is NaN.)
struct OrthoScale {
  float first, second;
  __device__ OrthoScale(double norm_eps, float sx) {
    const double s = (double)sx / (norm_eps > 0.0 && norm_eps < 1e-60 ? 1e-60 : norm_eps);
    const bool large = s > 0x1p100, small = s < 0x1p-100;
    first = large ? 0x1p100f : small ? 0x1p-60f : 1.0f;
    second = (float)(s * (large ? 0x1p-100 : small ? 0x1p60 : 1.0));
  }
  __device__ float operator()(float u) const { return u * first * second; }
};

// Up to four neighbours of a tensor of type dt, in one access where the address allows
__device__ __forceinline__ void load4(const void* p, int64_t i, int dt, int n, float (&v)[4]) {
  const int es = dt == FIM_F32 ? 4 : 2;
  const uint8_t* at = static_cast<const uint8_t*>(p) + i * es;
  if (n >= 4 && (reinterpret_cast<uintptr_t>(at) & (4 * es - 1)) == 0) {
    if (dt == FIM_F32) {
      const v4f w = *reinterpret_cast<const v4f*>(at);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = w[k];
    } else {
      const v2i w = *reinterpret_cast<const v2i*>(at);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t bits = (uint32_t)w[k >> 1] >> (16 * (k & 1)) & 0xffff;
        v[k] = dt == FIM_BF16 ? bf16_to_f32((uint16_t)bits) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = 0.0f;
    if (k < n)
      v[k] = dt == FIM_F32    ? load_elem<FIM_F32>(p, i + k)
             : dt == FIM_BF16 ? load_elem<FIM_BF16>(p, i + k)
                              : load_elem<FIM_F16>(p, i + k);
  }
}
__device__ __forceinline__ float load1(const void* p, int64_t i, int dt) {
  return dt == FIM_F32 ? load_elem<FIM_F32>(p, i) : dt == FIM_BF16 ? load_elem<FIM_BF16>(p, i) : load_elem<FIM_F16>(p, i);
}
__device__ __forceinline__ void store1(void* p, int64_t i, float v, int dt) {
  if (dt == FIM_F32) static_cast<float*>(p)[i] = v;
  else if (dt == FIM_BF16) static_cast<uint16_t*>(p)[i] = to16<FIM_BF16>(v);
  else static_cast<uint16_t*>(p)[i] = to16<FIM_F16>(v);
}
__device__ __forceinline__ void store4(void* p, int64_t i, int dt, int n, const float (&v)[4]) {
  const int es = dt == FIM_F32 ? 4 : 2;
  uint8_t* at = static_cast<uint8_t*>(p) + i * es;
  if (n >= 4 && (reinterpret_cast<uintptr_t>(at) & (4 * es - 1)) == 0) {
    if (dt == FIM_F32) *reinterpret_cast<v4f*>(at) = v4f{v[0], v[1], v[2], v[3]};
    else if (dt == FIM_BF16)
      *reinterpret_cast<v2i*>(at) = v2i{(int)to16x2<FIM_BF16>(v[0], v[1]), (int)to16x2<FIM_BF16>(v[2], v[3])};
    else
      *reinterpret_cast<v2i*>(at) = v2i{(int)to16x2<FIM_F16>(v[0], v[1]), (int)to16x2<FIM_F16>(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < n) store1(p, i + k, v[k], dt);
}

// O's elements where they go: O itself, or the parameter's step p = keep p - factor O.
__device__ __forceinline__ void finish4(const OrthoStack& s, const OrthoScalars& k, int64_t i, int n, float (&o)[4]) {
  if (k.step) {
    float p[4];
    load4(s.out, i, s.out_type, n, p);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(-s.factor, o[e], k.keep * p[e]);
  }
  store4(s.out, i, s.out_type, n, o);
}
__device__ __forceinline__ void finish1(const OrthoStack& s, const OrthoScalars& k, int64_t i, float o) {
  if (k.step) o = fmaf(-s.factor, o, k.keep * load1(s.out, i, s.out_type));
  store1(s.out, i, o, s.out_type);
}

// The last stack whose workgroups of pass `which` start at or before wg
__device__ __forceinline__ int stack_of(const OrthoStack* t, int count, int which, uint32_t wg) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i = 0; i < count; i += 64) {
    const int at = i + lane < count ? i + lane : count - 1;
    n += __popcll(__builtin_amdgcn_ballot_w64(i + lane < count && t[at].first[which] <= wg));
  }
  return __builtin_amdgcn_readfirstlane(n - 1);
}

}  // namespace fim
