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
//
// Four forms, chosen by sizes (gated_plan.h): up to 64 rows forward (gated_few.h), many rows of at most 128 channels forward
// (gated_rows.h), backward of at most 64 channels and 256 hidden columns (gated_rows_grad.h), and tiles (gated_tile.h).
#include "gated_plan.h"

namespace fim {

// Operands copied to packed rows of `to_cols` elements, zeros past their own: 16-byte stores, up to three operands a launch
struct PackArgs {
  struct {
    const uint16_t* from;
    uint16_t* to;
    int64_t ld, rows;
    int cols, per_row;    // per_row: 16-byte runs of a packed row
    int64_t first_block;  // the operand's first workgroup
  } m[3];
  int count;
};

__global__ __launch_bounds__(256) void gated_pack_kernel(const PackArgs a) {
  int o = 0;
  while (o + 1 < a.count && (int64_t)blockIdx.x >= a.m[o + 1].first_block) ++o;
  const auto& m = a.m[o];
  // (one 64-bit division a workgroup)
  const int64_t run0 = ((int64_t)blockIdx.x - m.first_block) * 1024, row0 = run0 / m.per_row;
  const uint32_t rest = (uint32_t)(run0 - row0 * m.per_row);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t at = rest + k * 256 + threadIdx.x, down = at / (uint32_t)m.per_row;
    const int64_t r = row0 + down;
    const int c = (int)(at - down * m.per_row) * 8;
    if (r >= m.rows) return;
    const uint16_t* from = m.from + r * m.ld + c;
    v4i v;
    if (c + 8 <= m.cols) {
      v = *reinterpret_cast<const v4i_any*>(from);
    } else {
      uint32_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = c + i < m.cols ? from[i] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (int)(e[2 * i] | e[2 * i + 1] << 16);
    }
    reinterpret_cast<v4i*>(m.to)[r * m.per_row + (c >> 3)] = v;
  }
}

// The sums of `splits` parts of n values, in order: the first n0 to out0, the others to out1 (either may be null). Few
// splits: four values a thread where n, n0 and the outputs' addresses allow (wide)
template <int DT>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* part, int64_t n, int64_t n0, int splits, uint16_t* out0,
                                                         uint16_t* out1, int wide) {
  if (wide) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
      v4f v = *reinterpret_cast<const v4f*>(part + i);
      for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const v4f*>(part + s * n + i);
      uint16_t* out = i < n0 ? out0 : out1;
      if (out == nullptr) continue;
      *reinterpret_cast<uint2*>(out + (i < n0 ? i : i - n0)) = uint2{to16x2<DT>(v[0], v[1]), to16x2<DT>(v[2], v[3])};
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
      float v = part[i];
      for (int s = 1; s < splits; ++s) v += part[s * n + i];
      uint16_t* out = i < n0 ? out0 : out1;
      if (out != nullptr) out[i < n0 ? i : i - n0] = to16<DT>(v);
    }
  }
}

// Many splits: 64 values a workgroup, the splits dealt to its four wavefronts, whose sums are added in their order
template <int DT>
__global__ __launch_bounds__(256) void gated_join_many_kernel(const float* part, int64_t n, int64_t n0, int splits,
                                                              uint16_t* out0, uint16_t* out1) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int s = wave; s < splits; s += 4) v += part[s * n + i];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave != 0 || i >= n) return;
  uint16_t* out = i < n0 ? out0 : out1;
  if (out != nullptr) out[i < n0 ? i : i - n0] = to16<DT>(sums[0][lane] + sums[1][lane] + (sums[2][lane] + sums[3][lane]));
}

// db[i][c] = sum over tiles of col_sums[tile][i][c]: 16 values a workgroup, the tiles dealt to 64 rows of threads
template <int DT>
__global__ __launch_bounds__(1024) void gated_bias_kernel(const float* col_sums, int64_t n, int64_t tiles, void* db0,
                                                          void* db1, int bdt) {
  __shared__ double sums[64][16];
  const int c = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t at = (int64_t)blockIdx.x * 16 + c;
  double v = 0.0;
  if (at < 2 * n) {
#pragma unroll 8
    for (int64_t t = row; t < tiles; t += 64) v += col_sums[t * 2 * n + at];
  }
  sums[row][c] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (row < half) sums[row][c] += sums[row + half][c];
    __syncthreads();
  }
  void* db = at < n ? db0 : db1;
  if (row != 0 || at >= 2 * n || db == nullptr) return;
  const int64_t to = at < n ? at : at - n;
  if (bdt == FIM_F32) static_cast<float*>(db)[to] = (float)sums[0][c];
  else static_cast<uint16_t*>(db)[to] = to16<DT>((float)sums[0][c]);
}

// -- launches ----------------------------------------------------------------------------------------------------------

// Copies what has to be copied; g.x, g.wg and g.wu are readable by the tiles afterwards
static void gated_operands(Gated& g, uint8_t* ws, hipStream_t stream) {
  PackArgs a{};
  int64_t blocks = 0;
  auto copy = [&](Matrix& m, int64_t at) {
    uint16_t* to = reinterpret_cast<uint16_t*>(ws + at);
    a.m[a.count++] = {m.p, to, m.ld, m.rows, (int)m.cols, (int)(m.padded() / 8), blocks};
    blocks += cdiv(m.rows * m.padded() / 8, 1024);
    m = {to, m.padded(), m.rows, m.padded()};
  };
  const bool copy_w = g.wu_at != g.wg_at;
  if (!g.x.as_is()) copy(g.x, g.x_at);
  if (copy_w) {
    copy(g.wg, g.wg_at);
    copy(g.wu, g.wu_at);
  }
  if (a.count > 0) gated_pack_kernel<<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a);
}

template <int DT, int MODE, int ACT, int MB, int NB>
static void launch_tile(TileArgs a, int64_t splits, hipStream_t stream) {
  constexpr int64_t BM = 64 * MB, BN = MODE == GATED_FORWARD || MODE == GATED_GRAD ? 32 * NB : 64 * NB;
  a.mt = (int)cdiv(a.M, BM);
  a.nt = (int)cdiv(a.N, BN) * (MODE == GATED_DW ? 2 : 1);
  a.group = 4;
  const int64_t wgs = cdiv((int64_t)a.mt * a.nt * splits, 8) * 8;
  gated_tile_kernel<DT, MODE, ACT, MB, NB><<<dim3((unsigned)wgs), dim3(256), 0, stream>>>(a);
}

template <int DT, int MODE, int ACT>
static void launch_product(const TileArgs& a, Tile t, int64_t splits, hipStream_t stream) {
  if constexpr (MODE != GATED_GRAD) {
    if (t.mb == 4) return launch_tile<DT, MODE, ACT, 4, 4>(a, splits, stream);
  }
  launch_tile<DT, MODE, ACT, 2, 2>(a, splits, stream);
}

template <int DT>
static void launch_join(const float* part, int64_t n, int64_t n0, int64_t splits, void* out0, void* out1,
                        hipStream_t stream) {
  uint16_t *o0 = static_cast<uint16_t*>(out0), *o1 = static_cast<uint16_t*>(out1);
  if (splits <= 4) {
    const int wide = n % 4 == 0 && n0 % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(o0) | reinterpret_cast<uintptr_t>(o1)) % 8 == 0;
    const int64_t blocks = cdiv(n, wide ? 1024 : 256);
    gated_join_kernel<DT><<<dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream>>>(part, n, n0, (int)splits,
                                                                                                    o0, o1, wide);
  } else {
    gated_join_many_kernel<DT><<<dim3((unsigned)cdiv(n, 64)), dim3(256), 0, stream>>>(part, n, n0, (int)splits, o0, o1);
  }
}

template <int DT, int ACT, int KP>
static void launch_rows(const RowsArgs& a, bool wide, hipStream_t stream) {
  const dim3 grid((unsigned)(rows_groups(a.M, a.K, a.H) * a.blocks));
  if (wide) gated_rows_kernel<DT, ACT, KP, true><<<grid, dim3(64 * ROWS_WAVES), 0, stream>>>(a);
  else gated_rows_kernel<DT, ACT, KP, false><<<grid, dim3(64 * ROWS_WAVES), 0, stream>>>(a);
}

template <int DT, int ACT>
static void launch_rows_grad(const RowsArgs& a, bool wide, hipStream_t stream) {
  const dim3 grid((unsigned)rows_grad_groups(a.M, a.K, a.H));
  if (wide) gated_rows_grad_kernel<DT, ACT, true><<<grid, dim3(64 * ROWS_WAVES), 0, stream>>>(a);
  else gated_rows_grad_kernel<DT, ACT, false><<<grid, dim3(64 * ROWS_WAVES), 0, stream>>>(a);
}

// The same launch by rows, from the tiles' arguments
static RowsArgs rows_args(const TileArgs& a, int64_t K) {
  RowsArgs r{};
  r.x = a.x[0];
  r.ldx = a.ldx;
  r.ldw = a.ldw;
  r.M = a.M;
  r.K = (int)K;
  r.kw = (int)(cdiv(a.K, 8) * 8);
  r.H = (int)a.N;
  for (int i = 0; i < 2; ++i) {
    r.w[i] = a.w[i];
    r.bias[i] = a.bias[i];
  }
  r.bias_dtype = a.bias_dtype;
  r.dout = a.dout;
  r.ldd = a.ldd;
  r.out = a.out[0];
  r.col_sums = a.col_sums;
  r.blocks = (int)rows_blocks(K, a.N);
  r.sub = rows_grad_sub(a.N);
  return r;
}

template <int DT, int ACT, int V>
static void launch_few(const FewArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(a.H, 16)), block(64 * FEW_WAVES);
  if (a.M <= 16) gated_few_kernel<DT, ACT, 1, V><<<grid, block, 0, stream>>>(a);
  else if (a.M <= 32) gated_few_kernel<DT, ACT, 2, V><<<grid, block, 0, stream>>>(a);
  else gated_few_kernel<DT, ACT, 4, V><<<grid, block, 0, stream>>>(a);
}

// Elements per load that every row of the three operands allows: 8, 2 or 1
static int few_vector(const Matrix& x, const Matrix& wg, const Matrix& wu) {
  int v = 8;
  for (const Matrix* m : {&x, &wg, &wu}) {
    auto fits = [&](int w) {
      return reinterpret_cast<uintptr_t>(m->p) % (2 * w) == 0 && m->ld % w == 0 && m->cols % w == 0;
    };
    while (v > 1 && !fits(v)) v = v == 8 ? 2 : 1;
  }
  return v;
}

static int gated_check(int dtype, int64_t M, int64_t K, int64_t H, int bias_dtype, int act) {
  if (M < 0 || K <= 0 || H <= 0 || act < 0 || act >= ACT_COUNT) return FIM_ERR_INVALID;
  if (dtype != FIM_BF16 && dtype != FIM_F16) return FIM_ERR_UNSUPPORTED;
  if (bias_dtype != FIM_F32 && bias_dtype != dtype) return FIM_ERR_INVALID;
  // tile counts and offsets inside a tile are 32-bit
  if (K >= (1 << 21) || H >= (1 << 21) || cdiv(M, 128) * cdiv(K > H ? K : H, 64) >= (1LL << 30)) return FIM_ERR_UNSUPPORTED;
  return FIM_OK;
}

template <typename F>
static void with_type(int dtype, F&& f) {
  if (dtype == FIM_BF16) f(std::integral_constant<int, FIM_BF16>{});
  else f(std::integral_constant<int, FIM_F16>{});
}

static bool workspace_ok(const Gated& g, const void* workspace, int64_t bytes) {
  return workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && bytes >= g.total;
}

static bool rows_wide(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

static TileArgs gated_forward_args(const Gated& g, const void* b_gate, const void* b_up, int bias_dtype) {
  TileArgs a{};
  a.x[0] = g.x.p;
  a.w[0] = g.wg.p;
  a.w[1] = g.wu.p;
  a.ldx = g.x.ld;
  a.ldw = g.wg.ld;
  a.M = g.M;
  a.N = g.H;
  a.K = g.x.cols;
  a.bias[0] = b_gate;
  a.bias[1] = b_up;
  a.bias_dtype = bias_dtype;
  return a;
}

}  // namespace fim

using namespace fim;

extern "C" int fim_gated_linear_workspace(const void* x, int64_t M, int64_t K, int64_t x_stride, const void* w_gate,
                                          int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, int64_t H,
                                          int backward, int64_t* bytes) {
  if (bytes == nullptr) return FIM_ERR_INVALID;
  const int rc = gated_check(FIM_BF16, M, K, H, FIM_F32, 0);
  if (rc != FIM_OK) return rc;
  *bytes = gated_plan(matrix(x, x_stride, M, K), matrix(w_gate, w_gate_stride, H, K), matrix(w_up, w_up_stride, H, K),
                      backward != 0)
               .total;
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
  Gated g = gated_plan(matrix(x, x_stride, M, K), matrix(w_gate, w_gate_stride, H, K), matrix(w_up, w_up_stride, H, K), false);
  if (g.total > 0 && !workspace_ok(g, workspace, workspace_bytes)) return FIM_ERR_INVALID;
  if (g.form == FORM_FEW) {
    FewArgs f{};
    f.x = g.x.p;
    f.w[0] = g.wg.p;
    f.w[1] = g.wu.p;
    f.ldx = g.x.ld;
    f.ldw[0] = g.wg.ld;
    f.ldw[1] = g.wu.ld;
    f.M = (int)M;
    f.K = (int)K;
    f.H = (int)H;
    f.bias[0] = b_gate;
    f.bias[1] = b_up;
    f.bias_dtype = bias_dtype;
    f.out = static_cast<uint16_t*>(out);
    f.wide_out = H % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
    const int v = few_vector(g.x, g.wg, g.wu);
    with_type(dtype, [&](auto dt) {
      with_activation(act, [&](auto act_c) {
        constexpr int DT = decltype(dt)::value, ACT = decltype(act_c)::value;
        if (v == 8) launch_few<DT, ACT, 8>(f, stream);
        else if (v == 2) launch_few<DT, ACT, 2>(f, stream);
        else launch_few<DT, ACT, 1>(f, stream);
      });
    });
    return launch_status();
  }
  gated_operands(g, static_cast<uint8_t*>(workspace), stream);
  TileArgs a = gated_forward_args(g, b_gate, b_up, bias_dtype);
  a.out[0] = static_cast<uint16_t*>(out);
  a.ldo = a.out_cols = H;
  a.wide_out = rows_wide(out, H);
  with_type(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    with_activation(act, [&](auto act_c) {
      constexpr int ACT = decltype(act_c)::value;
      if (g.form == FORM_TILES) launch_product<DT, GATED_FORWARD, ACT>(a, g.forward, 1, stream);
      else if (K <= 64) launch_rows<DT, ACT, 64>(rows_args(a, K), a.wide_out, stream);
      else launch_rows<DT, ACT, 128>(rows_args(a, K), a.wide_out, stream);
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
  Gated g = gated_plan(matrix(x, x_stride, M, K), matrix(w_gate, w_gate_stride, H, K), matrix(w_up, w_up_stride, H, K), true);
  if (!workspace_ok(g, workspace, workspace_bytes)) return FIM_ERR_INVALID;
  if (M == 1) d_out_stride = H;
  if (d_out_stride >= (1 << 22)) return FIM_ERR_UNSUPPORTED;  // 32-bit offsets inside a tile
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  gated_operands(g, ws, stream);
  uint16_t* dg = reinterpret_cast<uint16_t*>(ws + g.dgu_at);
  uint16_t* du = dg + M * g.ldg;
  const bool biases = db_gate != nullptr || db_up != nullptr;
  TileArgs a = gated_forward_args(g, b_gate, b_up, bias_dtype);
  a.dout = static_cast<const uint16_t*>(d_out);
  a.ldd = d_out_stride;
  a.wide_dout = rows_wide(d_out, d_out_stride) && H % 8 == 0;
  a.out[0] = dg;
  a.out[1] = du;
  a.ldo = g.ldg;
  a.out_cols = g.hp;
  a.wide_out = 1;
  a.col_sums = biases ? reinterpret_cast<float*>(ws + g.cols_at) : nullptr;
  with_type(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    with_activation(act, [&](auto act_c) {
      constexpr int ACT = decltype(act_c)::value;
      if (g.rows) {
        RowsArgs r = rows_args(a, K);
        r.dx = static_cast<uint16_t*>(dx);
        r.wide_dx = K % 4 == 0 && reinterpret_cast<uintptr_t>(dx) % 8 == 0;
        if (dw_gate != nullptr || dw_up != nullptr) r.dw_part = reinterpret_cast<float*>(ws + g.part_at);
        launch_rows_grad<DT, ACT>(r, a.wide_dout, stream);
      } else {
        launch_product<DT, GATED_GRAD, ACT>(a, g.grad, 1, stream);
      }
    });
    if (biases)
      gated_bias_kernel<DT><<<dim3((unsigned)cdiv(2 * H, 16)), dim3(1024), 0, stream>>>(
          a.col_sums, H, g.sum_rows, db_gate, db_up, bias_dtype);
    if (dx != nullptr && !g.rows) {
      TileArgs d{};
      d.x[0] = dg;
      d.x[1] = du;
      d.w[0] = g.wg.p;
      d.w[1] = g.wu.p;
      d.ldx = g.ldg;
      d.ldw = g.wg.ld;
      d.M = M;
      d.N = K;
      d.K = H;
      d.ww = g.wg.padded();
      d.out[0] = static_cast<uint16_t*>(dx);
      d.ldo = d.out_cols = K;
      d.wide_out = rows_wide(dx, K);
      d.k_split = g.dx_steps;
      d.part = g.dx_splits > 1 ? reinterpret_cast<float*>(ws + g.part_at) : nullptr;
      launch_product<DT, GATED_DX, ACT_NONE>(d, g.dx, g.dx_splits, stream);
      if (g.dx_splits > 1) launch_join<DT>(d.part, M * K, M * K, g.dx_splits, dx, nullptr, stream);
    }
    if (dw_gate != nullptr || dw_up != nullptr) {
      TileArgs w{};
      w.x[0] = g.x.p;
      w.w[0] = dg;
      w.w[1] = du;
      w.ldx = g.x.ld;
      w.ldw = g.ldg;
      w.M = K;
      w.N = H;
      w.K = M;
      w.xw = g.x.padded();
      w.ww = g.hp;
      w.part = reinterpret_cast<float*>(ws + g.part_at);
      w.k_split = g.dw_rows;
      if (!g.rows) launch_product<DT, GATED_DW, ACT_NONE>(w, g.dw, g.dw_splits, stream);
      launch_join<DT>(w.part, 2 * H * K, H * K, g.dw_splits, dw_gate, dw_up, stream);
    }
  });
  return launch_status();
}
