// The gradients of the adapters: dA_j = t^T x and dB_j = d_out^T h over the rows of each adapter, t = s_j d_out B_j and h in FP32
// from the passes over rows.
//
// A workgroup takes an adapter, 128 columns of x or d_out and a chunk of rows. It lists the chunk's rows of its adapter, then
// sums over them 32 at a time: their columns go through LDS and are read transposed (ds_read_tr16_b64), t's 32 rows go straight
// into the operand's registers, hi and lo. Each chunk leaves a partial sum and a launch adds them up in order: no atomics, equal
// bits from run to run. A chunk without rows of its adapter leaves none.
//
// 16800 x 196 -> 523 in FP16, rank 12, 6 adapters: 24 us (22 without beside_hi) and 5 to join for 24 MB of x and d_out, 1.0 TB/s: unaligned rows of 16-byte
// loads, listing, and prologues of 2772 workgroups of 12 to 24 turns.
#pragma once

#include "adapters.h"

namespace fim {

// GRAD_CHUNK: rows that the list has room for; a longer chunk's are listed and summed in pieces
constexpr int GRAD_COLS = 128, GRAD_ROWS = 32, GRAD_CHUNK = 4096;

struct AdapterGradArgs {
  const uint16_t *x, *d;  // [M, K], [M, N]
  int64_t ldx, ldd;
  const float *t, *h;  // packed [M, 16 NR]
  AdapterIndex index;
  uint16_t *da, *db;  // [J, R, K], [J, N, R]; written here where there is one chunk
  float* part;        // [J][chunks][R][K + N], or null
  int* counts;        // [J][chunks] rows
  uint32_t M, chunk;
  int chunks, K, N, R, xt, ct;  // column tiles of x, and of both
};

// PIECES: chunks are longer than the list (one piece, known as such: 16800 x 196 -> 523 21 us, 28 not)
template <int DT, int NR, bool PIECES>
__global__ __launch_bounds__(256) void adapter_grad_kernel(const AdapterGradArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t stage[2][GRAD_ROWS * GRAD_COLS * 2];
  __shared__ uint16_t rows[GRAD_CHUNK];
  __shared__ int counted[4];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ct = (int)(blockIdx.x % (unsigned)p.ct);
  const int slot = (int)(blockIdx.x / (unsigned)p.ct), j = slot / p.chunks, chunk = slot - j * p.chunks;
  const uint32_t begin = (uint32_t)chunk * p.chunk, end = begin + p.chunk < p.M ? begin + p.chunk : p.M;
  const uint32_t piece = PIECES ? GRAD_CHUNK : p.chunk;  // rows listed at a time
  uint32_t r0 = begin;
  int total = 0, all = 0;  // of this piece's rows, of all before it
  const bool of_x = ct < p.xt;
  const int width = of_x ? p.K : p.N, c0 = (of_x ? ct : ct - p.xt) * GRAD_COLS;
  const uint16_t* y = of_x ? p.x : p.d;
  const int64_t ld = of_x ? p.ldx : p.ldd;
  const float* t = of_x ? p.t : p.h;
  // loads: 16 bytes of two rows a thread; zeros past the list and past the columns
  const int seg = tid & 15, lrow = tid >> 4, cols = width - c0 - 8 * seg;
  auto load_y = [&](int from, s16x8 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = from + lrow + 16 * q;
      v[q] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (i < total && cols > 0) v[q] = load_some<8>(y + (int64_t)(r0 + rows[i]) * ld + c0 + 8 * seg, cols);
    }
  };
  auto put_y = [&](int buf, const s16x8 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = lrow + 16 * q;
      *reinterpret_cast<s16x8*>(stage[buf] + r * 256 + (((seg >> 2) ^ (r & 3)) << 6) + (seg & 3) * 16) = v[q];
    }
  };
  float tv[NR][8];  // ranks 16 i + l % 16 of rows 8 (l / 16) ..
  auto load_t = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int i = from + 8 * g + q;
      const float* src = t + (int64_t)(r0 + (i < total ? rows[i] : 0)) * (16 * NR) + l16;
#pragma unroll
      for (int b = 0; b < NR; ++b) tv[b][q] = i < total ? src[16 * b] : 0.0f;
    }
  };

  v4f acc[NR][2];
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) acc[i][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  s16x8 yv[2];
  int buf = 0;
  do {
    const uint32_t r1 = r0 + piece < end ? r0 + piece : end;
    if constexpr (PIECES) __syncthreads();  // (the list before has been read)
    // -- the piece's rows of this adapter, in order: each wavefront counts a quarter, then lists it
    const uint32_t quarter = piece / 4, q0 = r0 + wave * quarter < r1 ? r0 + wave * quarter : r1;
    const uint32_t q1 = q0 + quarter < r1 ? q0 + quarter : r1;
    int n = 0;
#pragma unroll 4
    for (uint32_t r = q0 + lane; r - lane < q1; r += 64)
      n += __popcll(__builtin_amdgcn_ballot_w64(r < q1 && adapter_of(p.index, r < q1 ? r : r0) == j));
    if (lane == 0) counted[wave] = n;
    __syncthreads();
    int at = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? counted[w] : 0;
      total += counted[w];
    }
    if (total == 0) continue;
#pragma unroll 4
    for (uint32_t r = q0 + lane; r - lane < q1; r += 64) {
      const bool own = r < q1 && adapter_of(p.index, r < q1 ? r : r0) == j;
      const uint64_t owned = __builtin_amdgcn_ballot_w64(own);
      if (own) rows[at + __popcll(owned & ((uint64_t{1} << lane) - 1))] = (uint16_t)(r - r0);
      at += __popcll(owned);
    }
    __syncthreads();
    total = __builtin_amdgcn_readfirstlane(total);
    all += total;
    load_y(0, yv);
    load_t(0);
    for (int from = 0; from < total; from += GRAD_ROWS, buf ^= 1) {
      put_y(buf, yv);
      float up = 1.0f, down = 1.0f;
      if constexpr (DT == FIM_F16) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int q = 0; q < 8; ++q) most = fmaxf(most, finite_abs(tv[i][q]));
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
        up = half_scale(most, down);
      }
      s16x8 th[NR], tl[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          short hi, lo;
          split16<DT>(DT == FIM_F16 ? tv[i][q] * up : tv[i][q], hi, lo);
          th[i][q] = hi;
          tl[i][q] = lo;
        }
      load_y(from + GRAD_ROWS, yv);
      load_t(from + GRAD_ROWS);
      lds_barrier();  // (two stages: one barrier a turn)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        s16x4 half[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int r = 8 * g + 4 * q + (l16 >> 2);
          half[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4*)(stage[buf] + r * 256 + ((wave ^ (r & 3)) << 6) + c * 32 + (lane & 3) * 8));
        }
        const s16x8 v = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7), vl = beside_hi<DT>(v);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          if constexpr (DT == FIM_F16) {
            v4f s = mfma_rank<DT>(th[i], v, v4f{0.0f, 0.0f, 0.0f, 0.0f});
            s = mfma_rank<DT>(tl[i], vl, s);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][c][q] = fmaf(s[q], down, acc[i][c][q]);
          } else {
            acc[i][c] = mfma_rank<DT>(th[i], v, acc[i][c]);
            acc[i][c] = mfma_rank<DT>(tl[i], vl, acc[i][c]);
          }
        }
      }
    }
  } while (PIECES && (r0 += piece) < end);
  if (ct == 0 && tid == 0 && p.counts != nullptr) p.counts[slot] = all;
  if (all == 0 && p.part != nullptr) return;
  // -- lane: column l % 16 of 16, ranks 4 (l / 16) ..
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = c0 + 32 * wave + 16 * c + l16;
    if (col >= width) continue;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 16 * i + 4 * g + q;
        if (r >= p.R) continue;
        const float v = acc[i][c][q];
        if (p.part != nullptr) p.part[((int64_t)slot * p.R + r) * (p.K + p.N) + (of_x ? col : p.K + col)] = v;
        else if (of_x) p.da[((int64_t)j * p.R + r) * p.K + col] = to16<DT>(v);
        else p.db[((int64_t)j * p.N + col) * p.R + r] = to16<DT>(v);
      }
  }
}

// The chunks' partial sums of 64 outputs of an adapter, added up in order: each wavefront a run of chunks, of which the empty ones
// (never written) are passed over, then the wavefronts' sums
constexpr int JOIN_WAVES = 16;
template <int DT>
__global__ __launch_bounds__(64 * JOIN_WAVES) void adapter_join_kernel(const float* __restrict__ part, const int* __restrict__ counts,
                                                                       int chunks, int J, int K, int N, int R, uint16_t* da,
                                                                       uint16_t* db) {
  __shared__ float sums[JOIN_WAVES][64];
  const int width = K + N, of = R * width, blocks = (of + 63) / 64, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int from = (int)((int64_t)chunks * wave / JOIN_WAVES), to = (int)((int64_t)chunks * (wave + 1) / JOIN_WAVES);
  for (int64_t block = blockIdx.x; block < (int64_t)J * blocks; block += gridDim.x) {
    const int j = (int)(block / blocks), i = (int)(block - (int64_t)j * blocks) * 64 + lane, at = i < of ? i : of - 1;
    const float* mine = part + (int64_t)j * chunks * of + at;
    float v = 0.0f;
    for (int k0 = from; k0 < to; k0 += 64) {
      const int mine_at = k0 + lane < to ? k0 + lane : k0;
      uint64_t some = __builtin_amdgcn_ballot_w64(k0 + lane < to && counts[(int64_t)j * chunks + mine_at] > 0);
      while (some != 0) {
        constexpr int U = 8;  // loads in flight
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          w[u] = 0.0f;
          if (some != 0) w[u] = mine[(int64_t)(k0 + __builtin_ctzll(some)) * of];
          some &= some - 1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) v += w[u];
      }
    }
    sums[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && i < of) {
#pragma unroll
      for (int w = 1; w < JOIN_WAVES; ++w) v += sums[w][lane];
      const int r = i / width, c = i - r * width;
      if (c < K) da[((int64_t)j * R + r) * K + c] = to16<DT>(v);
      else db[((int64_t)j * N + c - K) * R + r] = to16<DT>(v);
    }
    __syncthreads();
  }
}

// at[j][k][r] = a[j][r][k] and bt[j][r][n] = b[j][n][r]
__global__ __launch_bounds__(256) void adapter_transpose_kernel(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b,
                                                                uint16_t* __restrict__ at, uint16_t* __restrict__ bt, int K, int N,
                                                                int R, int64_t na, int64_t nb) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < na) {
    const int64_t jk = i / R, j = jk / K;
    at[i] = a[(j * R + (i - jk * R)) * K + (jk - j * K)];
  } else if (i < na + nb) {
    const int64_t o = i - na, jr = o / N, j = jr / R;
    bt[o] = b[(j * N + (o - jr * N)) * R + (jr - j * R)];
  }
}

}  // namespace fim
