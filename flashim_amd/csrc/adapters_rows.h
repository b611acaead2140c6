// Low-rank adapters over rows: h = s_j x A_j^T and out = base + h B_j^T in one pass, j the row's adapter. The gradient of x is the
// same pass over d_out with B_j^T and A_j^T in their places.
//
// A tile of 16 rows (or one) is a wavefront's, or four wavefronts' that split the contraction and then the columns. Operands go
// straight into registers: a tile's rows are read once, and A_j and B_j come from the caches. h stays in the accumulators' layout: a
// lane holds 4 ranks of its row, and the second product's contraction is ordered by what lanes hold, hi of the 4 and then lo of
// the 4 beside the same 4 of B_j twice; so h keeps 16 bits or more and nothing is exchanged. Rows of several adapters in a
// tile: once for each adapter that occurs, rows of others computed and not stored.
#pragma once

#include "adapters.h"

namespace fim {

struct AdapterArgs {
  const uint16_t *x, *base, *a, *b;  // x [M, K], base [M, N] or null, a [J, R, K], b [J, N, R]
  int64_t ldx, ld_base;
  uint16_t* out;  // packed [M, N]
  float* h;       // packed [M, 16 NR], or null
  AdapterIndex index;
  const float* scales;  // [J], or null
  float scale;
  uint32_t M;
  int K, N, R, parts;  // parts: of the columns
};

// QUADS: R is a multiple of 4, so that a lane's 4 ranks of B_j lie in one row.
template <int DT, int NR, int W, bool ONE, bool QUADS>
__global__ __launch_bounds__(256) void adapter_rows_kernel(const AdapterArgs p) {
  constexpr int GROUP = NR <= 2 && W > 1 ? 4 : 2;  // blocks of 32 columns whose operands are in flight
  __shared__ __attribute__((aligned(16))) float sums[W > 1 ? W * NR * 256 : 4];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t tile = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const uint32_t r0 = ONE ? tile : tile * 16;
  if (r0 >= p.M) return;
  const int part = W > 1 ? (int)blockIdx.y * W + wave : (int)blockIdx.y;
  const uint32_t mine = ONE ? r0 : r0 + l16;
  const bool there = mine < p.M;
  const uint32_t row = there ? mine : p.M - 1;
  const int which = there ? adapter_of(p.index, row) : -2;
  const uint16_t* x = p.x + (int64_t)row * p.ldx;
  const uint16_t* base = p.base == nullptr ? nullptr : p.base + (int64_t)row * p.ld_base;
  uint16_t* out = p.out + (int64_t)row * p.N;
  // this part's columns, in blocks of 32, and this wavefront's steps of the contraction
  const int blocks = (p.N + 31) / 32, n_from = (int)((int64_t)blocks * part / p.parts), n_to = (int)((int64_t)blocks * (part + 1) / p.parts);
  const int steps = (p.K + 31) / 32, k_from = W > 1 ? steps * wave / W : 0, k_to = W > 1 ? steps * (wave + 1) / W : steps;
  const int n_full = n_to < p.N / 32 ? n_to : p.N / 32;  // blocks before this one are whole
  const bool writes = !ONE || l16 == 0;

  s16x8 old[2][GROUP];
  auto load_base = [&](int nb, s16x8 (&v)[GROUP]) __attribute__((always_inline)) {  // of whole blocks; past them any
    if (base == nullptr) return;
#pragma unroll
    for (int u = 0; u < GROUP; ++u) {
      const int at = nb + u < n_full ? nb + u : n_full - 1;
      v[u] = *reinterpret_cast<const s16x8_any*>(base + 32 * at + 8 * g);
    }
  };
  if (n_from < n_full) load_base(n_from, old[0]);

  uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(there) & 0xffff;  // rows to do
  while (left != 0) {
    const int j = __builtin_amdgcn_readlane(which, __builtin_ctz(left));
    const bool own = which == j;
    left &= ~(uint32_t)__builtin_amdgcn_ballot_w64(own);
    if (j < 0) {  // no adapter: base, or zeros
#pragma unroll 4
      for (int nb = n_from; nb < n_to; ++nb) {
        const int n = 32 * nb + 8 * g;
        s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (base != nullptr && n < p.N) v = load_some<8>(base + n, p.N - n);
        if (own && n < p.N && writes) store_some<8>(out + n, p.N - n, v);
      }
      continue;
    }
    const uint16_t* b = p.b + (int64_t)j * p.N * p.R;
    // B_j's operands of column c: 4 ranks of each 16
    auto load_b = [&](int c, s16x4 (&v)[NR]) __attribute__((always_inline)) {
      const uint16_t* from = b + (int64_t)c * p.R;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int r = 16 * i + 4 * g;
        if constexpr (QUADS) {
          const s16x4 w = *reinterpret_cast<const s16x4_any*>(from + (r < p.R ? r : 0));
#pragma unroll
          for (int q = 0; q < 4; ++q) v[i][q] = r < p.R ? w[q] : (short)0;
        } else {
          v[i] = load_some<4>(from + r, p.R - r);
        }
      }
    };
    auto load_group = [&](int nb, s16x4 (&v)[GROUP][2][NR]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        const int at = nb + u < n_full ? nb + u : n_full - 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) load_b(32 * at + 8 * (l16 >> 2) + 4 * t + (l16 & 3), v[u][t]);
      }
    };
    s16x4 bv[2][GROUP][2][NR];
    if (n_from < n_full) load_group(n_from, bv[0]);

    // -- h: accumulators: lane: row l % 16, ranks 16 i + 4 (l / 16) ..
    v4f h[NR];
    const uint16_t* a[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      h[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      const int r = 16 * i + l16 < p.R ? 16 * i + l16 : p.R - 1;
      a[i] = p.a + ((int64_t)j * p.R + r) * p.K;
    }
    int s = k_from;
    const int whole = k_to < p.K / 32 ? k_to : p.K / 32;
#pragma unroll 4
    for (; s < whole; ++s) {
      const s16x8 v = *reinterpret_cast<const s16x8_any*>(x + 32 * s + 8 * g);
#pragma unroll
      for (int i = 0; i < NR; ++i) h[i] = mfma_rank<DT>(*reinterpret_cast<const s16x8_any*>(a[i] + 32 * s + 8 * g), v, h[i]);
    }
    if (s < k_to) {
      const int k = 32 * s + 8 * g;
      const s16x8 v = load_some<8>(x + k, p.K - k);
#pragma unroll
      for (int i = 0; i < NR; ++i) h[i] = mfma_rank<DT>(load_some<8>(a[i] + k, p.K - k), v, h[i]);
    }
    if constexpr (W > 1) {
      v4f* to = reinterpret_cast<v4f*>(sums);
      lds_barrier();  // (the sums of the adapter before have been read)
#pragma unroll
      for (int i = 0; i < NR; ++i) to[(wave * NR + i) * 64 + lane] = h[i];
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        h[i] = to[i * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) h[i] += to[(w * NR + i) * 64 + lane];
      }
    }
    const float scale = p.scales == nullptr ? p.scale : p.scale * p.scales[j];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[i][q] = 16 * i + 4 * g + q < p.R ? h[i][q] * scale : 0.0f;
        most = fmaxf(most, finite_abs(h[i][q]));
      }
    if (p.h != nullptr && part == 0 && own && writes) {
#pragma unroll
      for (int i = 0; i < NR; ++i) *reinterpret_cast<v4f*>(p.h + (int64_t)row * (16 * NR) + 16 * i + 4 * g) = h[i];
    }
    float up = 1.0f, down = 1.0f;
    if constexpr (DT == FIM_F16) {
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      up = half_scale(most, down);
    }
    s16x8 hf[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        short hi, lo;
        split16<DT>(DT == FIM_F16 ? h[i][q] * up : h[i][q], hi, lo);
        hf[i][q] = hi;
        hf[i][4 + q] = lo;
      }
    // -- out: two products of 16 columns whose rows interleave, so that a lane gets 8 neighbours
    auto block = [&](const s16x4 (&v)[2][NR], s16x8 from) __attribute__((always_inline)) {
      float o[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NR; ++i) d = mfma_rank<DT>(__builtin_shufflevector(v[t][i], v[t][i], 0, 1, 2, 3, 4, 5, 6, 7), hf[i], d);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float z = from16<DT>((uint16_t)from[4 * t + q]);
          if (base == nullptr) o[4 * t + q] = DT == FIM_F16 ? d[q] * down : d[q];
          else o[4 * t + q] = DT == FIM_F16 ? fmaf(d[q], down, z) : d[q] + z;
        }
      }
      const v4i w = {(int)to16x2<DT>(o[0], o[1]), (int)to16x2<DT>(o[2], o[3]), (int)to16x2<DT>(o[4], o[5]), (int)to16x2<DT>(o[6], o[7])};
      return __builtin_bit_cast(s16x8, w);
    };
    auto group = [&](int nb, int cur) __attribute__((always_inline)) {
      if (nb + GROUP < n_full) {
        load_base(nb + GROUP, old[cur ^ 1]);
        load_group(nb + GROUP, bv[cur ^ 1]);
      }
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        const s16x8 w = block(bv[cur][u], old[cur][u]);
        if (own && writes && nb + u < n_full) *reinterpret_cast<s16x8_any*>(out + 32 * (nb + u) + 8 * g) = w;
      }
    };
    for (int nb = n_from; nb < n_full; nb += 2 * GROUP) {
      group(nb, 0);
      if (nb + GROUP < n_full) group(nb + GROUP, 1);
    }
    if (n_full < n_to) {  // the last columns
      const int n = 32 * n_full + 8 * g;
      s16x4 v[2][NR];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int c = 32 * n_full + 8 * (l16 >> 2) + 4 * t + (l16 & 3);
        load_b(c < p.N ? c : p.N - 1, v[t]);
      }
      s16x8 from = {0, 0, 0, 0, 0, 0, 0, 0};
      if (base != nullptr && n < p.N) from = load_some<8>(base + n, p.N - n);
      const s16x8 w = block(v, from);
      if (own && writes && n < p.N) store_some<8>(out + n, p.N - n, w);
    }
    if (left != 0 && n_from < n_full) load_base(n_from, old[0]);  // for the next adapter's rows
  }
}

}  // namespace fim
