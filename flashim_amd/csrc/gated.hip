// The gated feed-forward product and its backward pass, BF16 or FP16 on the matrix cores with FP32 sums.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  out = act(g) * u            x [M, K], Wg and Wu [H, K], out [M, H]
//   dg = dout * u * act'(g),  du = dout * act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg, dbu: column sums of dg, du
//
// Forward, one kernel: a workgroup multiplies a tile of x by the same columns of both weights and applies bias, activation
// and product to its accumulators. Backward, the same product again with another epilogue (g and u are not kept from the
// forward pass: with K below about 1000 their two writes and reads cost more than the products), which writes dg and du in
// x's type (they are operands of 16-bit matrix products next; FP32 sums for the bias gradients are taken before that
// rounding); then one product for dx over both halves and one for the weights, split over rows where its tiles are few.
#include "activation.h"

namespace fim {

typedef short s16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ v16f mfma16(s16x8 a, s16x8 b, v16f c) {
  typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (DT == FIM_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint16_t to16(float v) {
  return DT == FIM_BF16 ? (uint16_t)(pack_bf16x2(v, 0.0f) & 0xffff) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ float from16(uint16_t h) {
  return DT == FIM_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

enum { GATED_FORWARD, GATED_GRAD, GATED_DX, GATED_DW };

// One operand as rows x contraction: element (r, k) at p[r * rs + k * ks]
struct Operand {
  const uint16_t* p;
  int64_t rs, ks;
};

struct GatedArgs {
  Operand x, w[2];        // rows of x; rows of the weights (w[1]: up). The second half of dx's contraction is x1, w[1]
  Operand x1;
  int64_t M, N, K;        // output rows, columns, contraction
  const void* b[2];
  int bdt;
  const uint16_t* dout;
  int64_t dout_stride;
  uint16_t* out[2];       // out (or dx); dg and du; dWg and dWu
  int64_t out_stride;
  int64_t out_cols;       // columns written (dg, du: up to the padded width, with zeros)
  float* col_sums;        // GATED_GRAD: [M tiles][2][N] sums of dg, du
  float* part;            // GATED_DW: [splits][2][M][N]
  int splits;
};

constexpr int GT = 64, GK = 32, GP = GK + 8;  // tile, contraction step, LDS row

// 64 x 32 of an operand into LDS rows of GP
__device__ __forceinline__ void stage(uint16_t (*s)[GP], const Operand& o, int64_t r0, int64_t rows, int64_t k0, int64_t k1) {
  for (int i = threadIdx.x; i < GT * GK; i += 256) {
    const int r = i / GK, k = i - r * GK;
    uint16_t v = 0;
    if (r0 + r < rows && k0 + k < k1) v = o.p[(r0 + r) * o.rs + (k0 + k) * o.ks];
    s[r][k] = v;
  }
}

template <int DT, int MODE, int ACT>
__global__ __launch_bounds__(256) void gated_kernel(const GatedArgs a) {
  constexpr bool PAIR = MODE == GATED_FORWARD || MODE == GATED_GRAD;
  __shared__ __attribute__((aligned(16))) uint16_t xs[GT][GP], ws[PAIR ? 2 : 1][GT][GP];
  __shared__ float cols[2][2][GT];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = wave >> 1, wn = wave & 1, h = lane >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * GT, n0 = (int64_t)blockIdx.y * GT;
  const int half = MODE == GATED_DW ? blockIdx.z & 1 : 0, split = MODE == GATED_DW ? blockIdx.z >> 1 : 0;
  int64_t kb = 0, ke = a.K;
  if constexpr (MODE == GATED_DW) {
    const int64_t per = (a.K + a.splits - 1) / a.splits;
    kb = split * per;
    ke = kb + per < a.K ? kb + per : a.K;
  }
  v16f acc[PAIR ? 2 : 1];
#pragma unroll
  for (int i = 0; i < (PAIR ? 2 : 1); ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
  for (int part = 0; part < (MODE == GATED_DX ? 2 : 1); ++part) {
    const Operand& x = MODE == GATED_DX ? (part ? a.x1 : a.x) : half ? a.x1 : a.x;
    for (int64_t k = kb; k < ke; k += GK) {
      __syncthreads();
      stage(xs, x, m0, a.M, k, ke);
      stage(ws[0], MODE == GATED_DX ? a.w[part] : a.w[0], n0, a.N, k, ke);
      if constexpr (PAIR) stage(ws[1], a.w[1], n0, a.N, k, ke);
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < GK; kk += 16) {
        const s16x8 xv = *reinterpret_cast<const s16x8*>(&xs[wm * 32 + (lane & 31)][kk + 8 * h]);
#pragma unroll
        for (int i = 0; i < (PAIR ? 2 : 1); ++i)
          acc[i] = mfma16<DT>(*reinterpret_cast<const s16x8*>(&ws[i][wn * 32 + (lane & 31)][kk + 8 * h]), xv, acc[i]);
      }
    }
  }
  // lane: output row m, columns n0 + 32 wn + 8 (q / 4) + 4 h + q % 4
  const int64_t m = m0 + wm * 32 + (lane & 31);
  float sums[2][16];
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int nl = wn * 32 + 8 * (q >> 2) + 4 * h + (q & 3);
    const int64_t n = n0 + nl;
    const bool in = m < a.M && n < a.N;
    if constexpr (PAIR) {
      float bias[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (a.b[i] != nullptr && n < a.N)
          bias[i] = a.bdt == FIM_F32 ? static_cast<const float*>(a.b[i])[n]
                                     : from16<DT>(static_cast<const uint16_t*>(a.b[i])[n]);
      const float g = acc[0][q] + bias[0], u = acc[1][q] + bias[1];
      if constexpr (MODE == GATED_FORWARD) {
        if (in) a.out[0][m * a.out_stride + n] = to16<DT>(activate<ACT>(g) * u);
      } else {
        float slope, dg = 0.0f, du = 0.0f;
        const float act = activate<ACT, true>(g, slope);
        if (in) {
          const float d = from16<DT>(a.dout[m * a.dout_stride + n]);
          dg = d * u * slope;
          du = d * act;
        }
        if (m < a.M && n < a.out_cols) {
          a.out[0][m * a.out_stride + n] = to16<DT>(dg);
          a.out[1][m * a.out_stride + n] = to16<DT>(du);
        }
        sums[0][q] = dg;
        sums[1][q] = du;
      }
    } else if constexpr (MODE == GATED_DX) {
      if (in) a.out[0][m * a.out_stride + n] = to16<DT>(acc[0][q]);
    } else {
      if (in) a.part[((split * 2 + half) * a.M + m) * a.N + n] = acc[0][q];
    }
  }
  if constexpr (MODE == GATED_GRAD) {
    if (a.col_sums == nullptr) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        float v = sums[i][q];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor(v, o);
        if ((lane & 31) == 0) cols[i][wm][wn * 32 + 8 * (q >> 2) + 4 * h + (q & 3)] = v;
      }
    __syncthreads();
    if (threadIdx.x < 2 * GT) {
      const int i = threadIdx.x / GT, c = threadIdx.x % GT;
      if (n0 + c < a.N) a.col_sums[((int64_t)blockIdx.x * 2 + i) * a.N + n0 + c] = cols[i][0][c] + cols[i][1][c];
    }
  }
}

// out[i] = sum over s of part[s][i], in order
template <int DT>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* part, int64_t n, int64_t splits, uint16_t* out0,
                                                         uint16_t* out1) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
    for (int64_t s = 0; s < splits; ++s) v += part[s * 2 * n + i];
    uint16_t* out = i < n ? out0 : out1;
    if (out != nullptr) out[i < n ? i : i - n] = to16<DT>(v);
  }
}

// db[i][c] = sum over tiles of col_sums[tile][i][c]: one wavefront per value
template <int DT>
__global__ __launch_bounds__(256) void gated_bias_kernel(const float* col_sums, int64_t n, int64_t tiles, void* db0,
                                                         void* db1, int bdt) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= 2 * n) return;
  double v = 0.0;
  for (int64_t t = threadIdx.x & 63; t < tiles; t += 64) v += col_sums[t * 2 * n + at];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  void* db = at < n ? db0 : db1;
  if ((threadIdx.x & 63) != 0 || db == nullptr) return;
  const int64_t c = at < n ? at : at - n;
  if (bdt == FIM_F32) static_cast<float*>(db)[c] = (float)v;
  else static_cast<uint16_t*>(db)[c] = to16<DT>((float)v);
}

// -- launches ----------------------------------------------------------------------------------------------------------

static int64_t align16(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The backward pass's workspace: dg and du [M, Hp] in x's type, bias partials, weight partials
struct GatedSpace {
  int64_t hp, dgu, cols, part, total;
  int splits;
};

static GatedSpace gated_space(int64_t M, int64_t K, int64_t H) {
  GatedSpace s;
  s.hp = cdiv(H, 8) * 8;
  s.dgu = 0;
  s.cols = align16(2 * M * s.hp * 2);
  s.part = s.cols + align16(cdiv(M, GT) * 2 * H * 4);
  const int64_t tiles = 2 * cdiv(H, GT) * cdiv(K, GT);
  int64_t splits = cdiv(2 * (int64_t)device_cus(), tiles > 0 ? tiles : 1);
  const int64_t most = cdiv(M, 4 * GK);
  if (splits > most) splits = most > 0 ? most : 1;
  s.splits = (int)splits;
  s.total = s.part + align16(splits * 2 * H * K * 4);
  return s;
}

static int gated_check(int dtype, int64_t M, int64_t K, int64_t H, int bias_dtype, int act) {
  if (M < 0 || K <= 0 || H <= 0 || act < 0 || act >= ACT_COUNT) return FIM_ERR_INVALID;
  if (dtype != FIM_BF16 && dtype != FIM_F16) return FIM_ERR_UNSUPPORTED;
  if (bias_dtype != FIM_F32 && bias_dtype != dtype) return FIM_ERR_INVALID;
  if (cdiv(M, GT) > INT32_MAX || cdiv(H, GT) > 65535 || cdiv(K, GT) > 65535) return FIM_ERR_UNSUPPORTED;
  return FIM_OK;
}

template <typename F>
static void with_type(int dtype, F&& f) {
  if (dtype == FIM_BF16) f(std::integral_constant<int, FIM_BF16>{});
  else f(std::integral_constant<int, FIM_F16>{});
}

}  // namespace fim

using namespace fim;

extern "C" int fim_gated_linear_workspace(int64_t M, int64_t K, int64_t H, int backward, int64_t* bytes) {
  if (bytes == nullptr) return FIM_ERR_INVALID;
  const int rc = gated_check(FIM_BF16, M, K, H, FIM_F32, 0);
  if (rc != FIM_OK) return rc;
  *bytes = backward ? gated_space(M, K, H).total : 0;
  return FIM_OK;
}

extern "C" int fim_gated_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t x_stride, const void* w_gate,
                                int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, int64_t H,
                                const void* b_gate, const void* b_up, int bias_dtype, int act, void* out,
                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const int rc = gated_check(dtype, M, K, H, bias_dtype, act);
  if (rc != FIM_OK) return rc;
  if (M == 0) return FIM_OK;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || out == nullptr) return FIM_ERR_INVALID;
  GatedArgs a{};
  a.x = {static_cast<const uint16_t*>(x), x_stride, 1};
  a.w[0] = {static_cast<const uint16_t*>(w_gate), w_gate_stride, 1};
  a.w[1] = {static_cast<const uint16_t*>(w_up), w_up_stride, 1};
  a.M = M;
  a.N = H;
  a.K = K;
  a.b[0] = b_gate;
  a.b[1] = b_up;
  a.bdt = bias_dtype;
  a.out[0] = static_cast<uint16_t*>(out);
  a.out_stride = H;
  with_type(dtype, [&](auto dt) {
    with_activation(act, [&](auto act_c) {
      gated_kernel<decltype(dt)::value, GATED_FORWARD, decltype(act_c)::value>
          <<<dim3((unsigned)cdiv(M, GT), (unsigned)cdiv(H, GT)), dim3(256), 0, stream>>>(a);
    });
  });
  return launch_status();
}

extern "C" int fim_gated_linear_backward(const void* x, int dtype, int64_t M, int64_t K, int64_t x_stride,
                                         const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
                                         int64_t H, const void* b_gate, const void* b_up, int bias_dtype, int act,
                                         const void* d_out, int64_t d_out_stride, void* dx, void* dw_gate, void* dw_up,
                                         void* db_gate, void* db_up, void* workspace, int64_t workspace_bytes,
                                         hipStream_t stream) {
  const int rc = gated_check(dtype, M, K, H, bias_dtype, act);
  if (rc != FIM_OK) return rc;
  if (M == 0) return FIM_OK;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || d_out == nullptr) return FIM_ERR_INVALID;
  const GatedSpace s = gated_space(M, K, H);
  if (workspace == nullptr || workspace_bytes < s.total) return FIM_ERR_INVALID;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint16_t* dg = reinterpret_cast<uint16_t*>(ws + s.dgu);
  uint16_t* du = dg + M * s.hp;
  const bool biases = db_gate != nullptr || db_up != nullptr;
  const Operand xr = {static_cast<const uint16_t*>(x), x_stride, 1};
  const Operand wg = {static_cast<const uint16_t*>(w_gate), w_gate_stride, 1};
  const Operand wu = {static_cast<const uint16_t*>(w_up), w_up_stride, 1};
  GatedArgs a{};
  a.x = xr;
  a.w[0] = wg;
  a.w[1] = wu;
  a.M = M;
  a.N = H;
  a.K = K;
  a.b[0] = b_gate;
  a.b[1] = b_up;
  a.bdt = bias_dtype;
  a.dout = static_cast<const uint16_t*>(d_out);
  a.dout_stride = d_out_stride;
  a.out[0] = dg;
  a.out[1] = du;
  a.out_stride = s.hp;
  a.out_cols = s.hp;
  a.col_sums = biases ? reinterpret_cast<float*>(ws + s.cols) : nullptr;
  with_type(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    with_activation(act, [&](auto act_c) {
      gated_kernel<DT, GATED_GRAD, decltype(act_c)::value>
          <<<dim3((unsigned)cdiv(M, GT), (unsigned)cdiv(s.hp, GT)), dim3(256), 0, stream>>>(a);
    });
    if (biases)
      gated_bias_kernel<DT><<<dim3((unsigned)cdiv(2 * H, 4)), dim3(256), 0, stream>>>(a.col_sums, H, cdiv(M, GT), db_gate,
                                                                                      db_up, bias_dtype);
    if (dx != nullptr) {
      GatedArgs d{};
      d.x = {dg, s.hp, 1};
      d.x1 = {du, s.hp, 1};
      d.w[0] = {wg.p, 1, wg.rs};
      d.w[1] = {wu.p, 1, wu.rs};
      d.M = M;
      d.N = K;
      d.K = H;
      d.out[0] = static_cast<uint16_t*>(dx);
      d.out_stride = K;
      gated_kernel<DT, GATED_DX, ACT_NONE>
          <<<dim3((unsigned)cdiv(M, GT), (unsigned)cdiv(K, GT)), dim3(256), 0, stream>>>(d);
    }
    if (dw_gate != nullptr || dw_up != nullptr) {
      GatedArgs w{};
      w.x = {dg, 1, s.hp};
      w.x1 = {du, 1, s.hp};
      w.w[0] = {xr.p, 1, xr.rs};
      w.M = H;
      w.N = K;
      w.K = M;
      w.part = reinterpret_cast<float*>(ws + s.part);
      w.splits = s.splits;
      gated_kernel<DT, GATED_DW, ACT_NONE>
          <<<dim3((unsigned)cdiv(H, GT), (unsigned)cdiv(K, GT), (unsigned)(2 * s.splits)), dim3(256), 0, stream>>>(w);
      const int64_t blocks = cdiv(2 * H * K, 256);
      gated_join_kernel<DT><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream>>>(
          w.part, H * K, s.splits, static_cast<uint16_t*>(dw_gate), static_cast<uint16_t*>(dw_up));
    }
  });
  return launch_status();
}
