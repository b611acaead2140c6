// Low-rank adapters over rows: h = s_j x A_j^T and out = base + h B_j^T in one pass, j the row's adapter. The gradient of x is the
// same pass over d_out with B_j^T and A_j^T in their places.
//
// A tile of 32 or 16 rows (or one) is a wavefront's, or four wavefronts' that split the contraction and then the columns. Operands
// go straight into registers: a tile's rows are read once, and A_j and B_j come from the caches. h stays in the accumulators'
// layout: a lane holds 4 ranks of its row a block, and the second product's contraction is ordered by what lanes hold, hi of the 4
// and then lo of the 4 beside the same 4 of B_j twice; so h keeps 16 bits or more and nothing is exchanged. Rows of several
// adapters in a tile: once for each adapter that occurs, rows of others computed and not stored. (Indices in random order cost that
// many passes: 16384 rows of 512 -> 2048 at rank 16 and 64 adapters 330 us, sorted 47, of one adapter 31.)
//
// Bound by memory at low ranks: 40000 x 512 -> 2048 at rank 16, 369 MB in 92 us, 4.0 TB/s of the 5.1 of a large copy; 320000 x 64
// -> 256 at rank 8 as many in 84. By the caches' reads of A_j and B_j at high ones: rank 32 106 us, 64 152, 128 213 (171, 278 and
// 434 with 8-byte loads of B_j and 16 rows): every tile of 32 rows reads all of B_j. 64 rows of adapters of their own, 1024 -> 4096
// at rank 16: 12 MB in 7 us, latency.
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

// The first of the 4 ranks that group g of 16 lanes holds of block i: two blocks' lie side by side, for loads of 16 bytes of B_j
template <int NR>
__device__ __forceinline__ int rank_of(int i, int g) {
  return NR == 1 ? 4 * g : 32 * (i >> 1) + 8 * g + 4 * (i & 1);
}

// SETS: of 16 rows, which meet each operand of A_j and B_j as it is read (0: one row). EVEN: R is a multiple of 4, or of
// 8 past 16 ranks, so that the ranks a lane loads lie in one row of B_j.
template <int DT, int NR, int W, int SETS, bool EVEN>
__global__ __launch_bounds__(256, SETS == 2 && NR <= 4 ? 2 : 1) void adapter_rows_kernel(const AdapterArgs p) {
  constexpr bool ONE = SETS == 0;
  constexpr int S = ONE ? 1 : SETS;
  // blocks of 32 columns whose operands are in flight
  constexpr int GROUP = NR <= 2 && S == 1 ? 4 : NR == 4 || S * NR >= 8 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) float sums[W > 1 ? W * S * NR * 256 : 4];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t tile = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const uint32_t r0 = ONE ? tile : tile * (16 * S);
  if (r0 >= p.M) return;
  const int part = W > 1 ? (int)blockIdx.y * W + wave : (int)blockIdx.y;
  uint32_t row[S];
  int which[S];
  const uint16_t *x[S], *base[S];
  uint16_t* out[S];
  uint32_t left = 0;  // rows to do, 16 bits a set
#pragma unroll
  for (int z = 0; z < S; ++z) {
    const uint32_t mine = ONE ? r0 : r0 + 16 * z + l16;
    const bool there = mine < p.M;
    row[z] = there ? mine : p.M - 1;
    which[z] = there ? adapter_of(p.index, row[z]) : -2;
    x[z] = p.x + (int64_t)row[z] * p.ldx;
    base[z] = p.base + (p.base == nullptr ? 0 : (int64_t)row[z] * p.ld_base);
    out[z] = p.out + (int64_t)row[z] * p.N;
    left |= ((uint32_t)__builtin_amdgcn_ballot_w64(there) & 0xffff) << (16 * z);
  }
  // this part's columns, in blocks of 32, and this wavefront's steps of the contraction
  const int blocks = (p.N + 31) / 32;
  const int n_from = (int)((int64_t)blocks * part / p.parts), n_to = (int)((int64_t)blocks * (part + 1) / p.parts);
  const int steps = (p.K + 31) / 32, k_from = W > 1 ? steps * wave / W : 0, k_to = W > 1 ? steps * (wave + 1) / W : steps;
  const int n_full = n_to < p.N / 32 ? n_to : p.N / 32;  // blocks before this one are whole
  const bool writes = !ONE || l16 == 0;

  s16x8 old[2][S][GROUP];
  auto load_base = [&](int nb, s16x8 (&v)[S][GROUP]) __attribute__((always_inline)) {  // of whole blocks; past them any
    if (p.base == nullptr) return;
#pragma unroll
    for (int z = 0; z < S; ++z)
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        const int at = nb + u < n_full ? nb + u : n_full - 1;
        v[z][u] = *reinterpret_cast<const s16x8_any*>(base[z] + 32 * at + 8 * g);
      }
  };
  if (n_from < n_full) load_base(n_from, old[0]);

  while (left != 0) {
    const int first = __builtin_ctz(left);
    int j = __builtin_amdgcn_readlane(which[0], first & 15);
    if constexpr (S > 1) j = first < 16 ? j : __builtin_amdgcn_readlane(which[S - 1], first & 15);
    bool own[S];
#pragma unroll
    for (int z = 0; z < S; ++z) {
      own[z] = which[z] == j;
      left &= ~(((uint32_t)__builtin_amdgcn_ballot_w64(own[z]) & 0xffff) << (16 * z));
    }
    if (j < 0) {  // no adapter: base, or zeros
#pragma unroll
      for (int z = 0; z < S; ++z)
#pragma unroll 4
        for (int nb = n_from; nb < n_to; ++nb) {
          const int n = 32 * nb + 8 * g;
          s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
          if (p.base != nullptr && n < p.N) v = load_some<8>(base[z] + n, p.N - n);
          if (own[z] && n < p.N && writes) store_some<8>(out[z] + n, p.N - n, v);
        }
      continue;
    }
    const uint16_t* b = p.b + (int64_t)j * p.N * p.R;
    // B_j's operands of column c: this lane's ranks
    auto load_b = [&](int c, s16x4 (&v)[NR]) __attribute__((always_inline)) {
      const uint16_t* from = b + (int64_t)c * p.R;
      if constexpr (NR == 1) {
        const int r = rank_of<NR>(0, g);
        v[0] = EVEN ? (s16x4) * reinterpret_cast<const s16x4_any*>(from + (r < p.R ? r : 0)) : load_some<4>(from + r, p.R - r);
        if (EVEN && r >= p.R) v[0] = s16x4{0, 0, 0, 0};
      } else {
#pragma unroll
        for (int i = 0; i < NR; i += 2) {
          const int r = rank_of<NR>(i, g);
          if constexpr (EVEN) {
            s16x8 w = *reinterpret_cast<const s16x8_any*>(from + (r < p.R ? r : 0));
            if (r >= p.R) w = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
            v[i] = __builtin_shufflevector(w, w, 0, 1, 2, 3);
            v[i + 1] = __builtin_shufflevector(w, w, 4, 5, 6, 7);
          } else {
            v[i] = load_some<4>(from + r, p.R - r);
            v[i + 1] = load_some<4>(from + r + 4, p.R - r - 4);
          }
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

    // -- h: accumulators: lane: row l % 16, ranks rank_of(i, l / 16) ..
    v4f h[S][NR];
    const uint16_t* a[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int z = 0; z < S; ++z) h[z][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      const int r0 = rank_of<NR>(i, l16 >> 2) + (l16 & 3), r = r0 < p.R ? r0 : p.R - 1;
      a[i] = p.a + ((int64_t)j * p.R + r) * p.K;
    }
    int s = k_from;
    const int whole = k_to < p.K / 32 ? k_to : p.K / 32;
#pragma unroll 4
    for (; s < whole; ++s) {
      s16x8 v[S];
#pragma unroll
      for (int z = 0; z < S; ++z) v[z] = *reinterpret_cast<const s16x8_any*>(x[z] + 32 * s + 8 * g);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const s16x8 w = *reinterpret_cast<const s16x8_any*>(a[i] + 32 * s + 8 * g);
#pragma unroll
        for (int z = 0; z < S; ++z) h[z][i] = mfma_rank<DT>(w, v[z], h[z][i]);
      }
    }
    if (s < k_to) {
      const int k = 32 * s + 8 * g;
      s16x8 v[S];
#pragma unroll
      for (int z = 0; z < S; ++z) v[z] = load_some<8>(x[z] + k, p.K - k);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const s16x8 w = load_some<8>(a[i] + k, p.K - k);
#pragma unroll
        for (int z = 0; z < S; ++z) h[z][i] = mfma_rank<DT>(w, v[z], h[z][i]);
      }
    }
    if constexpr (W > 1) {
      v4f* to = reinterpret_cast<v4f*>(sums);
      lds_barrier();  // (the sums of the adapter before have been read)
#pragma unroll
      for (int z = 0; z < S; ++z)
#pragma unroll
        for (int i = 0; i < NR; ++i) to[((wave * S + z) * NR + i) * 64 + lane] = h[z][i];
      lds_barrier();
#pragma unroll
      for (int z = 0; z < S; ++z)
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          h[z][i] = to[(z * NR + i) * 64 + lane];
#pragma unroll
          for (int w = 1; w < W; ++w) h[z][i] += to[((w * S + z) * NR + i) * 64 + lane];
        }
    }
    const float scale = p.scales == nullptr ? p.scale : p.scale * p.scales[j];
    float up[S], down[S];
    s16x8 hf[S][NR];
#pragma unroll
    for (int z = 0; z < S; ++z) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          h[z][i][q] = rank_of<NR>(i, g) + q < p.R ? h[z][i][q] * scale : 0.0f;
          most = fmaxf(most, finite_abs(h[z][i][q]));
        }
      if (p.h != nullptr && part == 0 && own[z] && writes) {
#pragma unroll
        for (int i = 0; i < NR; ++i) *reinterpret_cast<v4f*>(p.h + (int64_t)row[z] * (16 * NR) + rank_of<NR>(i, g)) = h[z][i];
      }
      up[z] = down[z] = 1.0f;
      if constexpr (DT == FIM_F16) {
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        up[z] = half_scale(most, down[z]);
      }
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          short hi, lo;
          split16<DT>(DT == FIM_F16 ? h[z][i][q] * up[z] : h[z][i][q], hi, lo);
          hf[z][i][q] = hi;
          hf[z][i][4 + q] = lo;
        }
    }
    // -- out: two products of 16 columns whose rows interleave, so that a lane gets 8 neighbours
    auto block = [&](int z, const s16x4 (&v)[2][NR], s16x8 from) __attribute__((always_inline)) {
      float o[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NR; ++i)
          d = mfma_rank<DT>(beside_halves<DT>(v[t][i]), hf[z][i], d);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float y = from16<DT>((uint16_t)from[4 * t + q]);
          if (p.base == nullptr) o[4 * t + q] = DT == FIM_F16 ? d[q] * down[z] : d[q];
          else o[4 * t + q] = DT == FIM_F16 ? fmaf(d[q], down[z], y) : d[q] + y;
        }
      }
      const v4i w = {(int)to16x2<DT>(o[0], o[1]), (int)to16x2<DT>(o[2], o[3]), (int)to16x2<DT>(o[4], o[5]),
                     (int)to16x2<DT>(o[6], o[7])};
      return __builtin_bit_cast(s16x8, w);
    };
    auto group = [&](int nb, int cur) __attribute__((always_inline)) {
      if (nb + GROUP < n_full) {
        load_base(nb + GROUP, old[cur ^ 1]);
        load_group(nb + GROUP, bv[cur ^ 1]);
      }
#pragma unroll
      for (int u = 0; u < GROUP; ++u)
#pragma unroll
        for (int z = 0; z < S; ++z) {
          const s16x8 w = block(z, bv[cur][u], old[cur][z][u]);
          if (own[z] && writes && nb + u < n_full) *reinterpret_cast<s16x8_any*>(out[z] + 32 * (nb + u) + 8 * g) = w;
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
#pragma unroll
      for (int z = 0; z < S; ++z) {
        s16x8 from = {0, 0, 0, 0, 0, 0, 0, 0};
        if (p.base != nullptr && n < p.N) from = load_some<8>(base[z] + n, p.N - n);
        const s16x8 w = block(z, v, from);
        if (own[z] && writes && n < p.N) store_some<8>(out[z] + n, p.N - n, w);
      }
    }
    if (left != 0 && n_from < n_full) load_base(n_from, old[0]);  // for the next adapter's rows
  }
}

}  // namespace fim
