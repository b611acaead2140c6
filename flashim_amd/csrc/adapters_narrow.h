// The whole backward pass of low-rank adapters beside a narrow projection in one pass over x and d_out: dx, and each workgroup's
// partial sums of dA_j and dB_j.
//
// A workgroup takes an adapter and a chunk of rows and lists the chunk's rows of its adapter (a long chunk's in pieces). A_j and
// B_j^T lie in LDS, and so do 64 rows of x and d_out at a time, read once from memory and used three times: each wavefront
// multiplies 16 of them into h and t and its rows of dx; then t and h (hi and lo) meet all 64 rows, read transposed, in
// accumulators that stay in registers for the chunk. Passes of their own (adapters_rows.h, adapters_grad.h) read d_out twice and
// write and read t and h in FP32: 320000 x 64 -> 256 at rank 8 took 77 + 55 us and 22 to join, this one 62 and 6 to join:
// 246 MB at 4.0 TB/s, of the 5.1 of a large copy; the rest is the turns' barriers, with two workgroups a CU to cover them.
#pragma once

#include "adapters.h"

namespace fim {

// NARROW_ROWS: a turn's; NARROW_CHUNK: rows that the list has room for
constexpr int NARROW_ROWS = 64, NARROW_CHUNK = 1024;

// Columns of x and d_out, each rounded up to 32, that a workgroup has room for
// (768 at 16 ranks leaves a CU one workgroup, and little beside its weights: 16800 x 196 -> 523 in FP16 55 us, 42 by passes)
constexpr int NARROW_WIDTH = 384;

struct AdapterNarrowArgs {
  const uint16_t *x, *d, *a, *b;  // [M, K], [M, N], [J, R, K], [J, N, R]
  int64_t ldx, ldd;
  AdapterIndex index;
  const float* scales;
  float scale;
  uint16_t *dx, *da, *db;  // dx null: not wanted; da and db null: not wanted, else written here where there is one chunk
  float* part;             // [J][chunks][R][K + N], or null
  int* counts;             // [J][chunks] rows
  uint32_t M, chunk;
  int chunks, K, N, R;
};

// WHOLE: K and N are multiples of 32. PIECES: chunks are longer than the list
template <int DT, int NR, bool WHOLE, bool PIECES>
__global__ __launch_bounds__(256) void adapter_narrow_kernel(const AdapterNarrowArgs p) {
  constexpr int W = NARROW_WIDTH, CB = W / 64;                          // 16-column blocks of a wavefront
  // bytes of a row; an odd number of 16s: rows at one column meet different banks
  constexpr int STRIDE = W * 2 + 16, TS = 128 * NR + 16;
  __shared__ __attribute__((aligned(16))) uint8_t rows_at[NARROW_ROWS * STRIDE];  // x, then d_out, then zeros up to 32 columns
  __shared__ __attribute__((aligned(16))) uint8_t weights[16 * NR * STRIDE];      // A_j, then B_j^T
  __shared__ __attribute__((aligned(16))) uint8_t ts[NARROW_ROWS * TS];           // t hi, t lo, h hi, h lo
  __shared__ uint16_t list[NARROW_CHUNK];
  __shared__ int counted[4];
  __shared__ float largest[2][4];
  __shared__ int infinities[4];  // whether a wavefront's rows hold some
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = (int)blockIdx.x, j = slot / p.chunks, chunk = slot - j * p.chunks;  // j = J: rows without an adapter
  const bool none = j == p.index.adapters;
  const uint32_t begin = (uint32_t)chunk * p.chunk, end = begin + p.chunk < p.M ? begin + p.chunk : p.M;
  const uint32_t piece = PIECES ? NARROW_CHUNK : p.chunk;  // rows listed at a time
  uint32_t r0 = begin;
  int total = 0, all = 0;  // of this piece's rows, of all so far
  const int kp = (p.K + 31) & ~31, np = (p.N + 31) & ~31;
  const float scale = p.scales == nullptr || none ? p.scale : p.scale * p.scales[j];
  v4f acc[NR][CB];
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[i][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};

  // This wavefront's 16 rows of a turn: a lane loads 16 bytes of row l % 16, which are an operand of h or t as they are. Zeros past
  // the list and past the columns; the next turn's are on their way while this one's sums are taken
  s16x8 v[W / 32];
  // (the compiler may not keep the outcome of every step's comparison: it spilled 330, and took 14% longer)
  auto fresh = [](int v) __attribute__((always_inline)) {
    asm("" : "+s"(v));
    return v;
  };
  auto load_rows = [&](int from) __attribute__((always_inline)) {
    const int i = from + 16 * wave + l16;
    const bool there = i < total;
    const int xsteps = fresh(kp / 32), steps = fresh((kp + np) / 32);
    const int64_t row = r0 + list[there ? i : 0];
    const uint16_t *x = p.x + row * p.ldx + 8 * g, *d = p.d + row * p.ldd + 8 * g;
    if constexpr (WHOLE) {
#pragma unroll
      for (int s = 0; s < W / 32; ++s)
        if (s < steps) v[s] = *reinterpret_cast<const s16x8_any*>(s < xsteps ? x + 32 * s : d + 32 * (s - xsteps));
    } else {
#pragma unroll
      for (int s = 0; s < W / 32; ++s)
        if (s < steps) {
          const int c = 32 * (s < xsteps ? s : s - xsteps);
          v[s] = load_some<8>(s < xsteps ? x + c : d + c, (s < xsteps ? p.K : p.N) - c - 8 * g);
        }
    }
    if (!there) {
#pragma unroll
      for (int s = 0; s < W / 32; ++s) v[s] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  };
  do {
    const uint32_t r1 = r0 + piece < end ? r0 + piece : end;
    if constexpr (PIECES) __syncthreads();  // (the list before has been read)
    // -- the piece's rows of this adapter, in order: each wavefront counts a quarter, then lists it
    const uint32_t quarter = piece / 4, q0 = r0 + wave * quarter < r1 ? r0 + wave * quarter : r1;
    const uint32_t q1 = q0 + quarter < r1 ? q0 + quarter : r1;
    uint64_t own[NARROW_CHUNK / 256];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NARROW_CHUNK / 256; ++i) {
      const uint32_t r = q0 + 64 * i + lane;
      own[i] = __builtin_amdgcn_ballot_w64(r < q1 && adapter_of(p.index, r < q1 ? r : r0) == (none ? -1 : j));
      n += __popcll(own[i]);
    }
    if (lane == 0) counted[wave] = n;
    __syncthreads();
    int at = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? counted[w] : 0;
      total += counted[w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (total == 0) continue;
#pragma unroll
    for (int i = 0; i < NARROW_CHUNK / 256; ++i) {
      if (own[i] >> lane & 1) list[at + __popcll(own[i] & ((uint64_t{1} << lane) - 1))] = (uint16_t)(q0 - r0 + 64 * i + lane);
      at += __popcll(own[i]);
    }
    __syncthreads();
    if (none) {
      const int segs = (p.K + 7) / 8;
      for (int i = tid; i < total * segs; i += 256) {
        const int r = i / segs, c = (i - r * segs) * 8;
        store_some<8>(p.dx + (int64_t)(r0 + list[r]) * p.K + c, p.K - c, s16x8{0, 0, 0, 0, 0, 0, 0, 0});
      }
      continue;
    }
    if (all == 0) {
      for (int i = tid; i < 16 * NR * (kp / 8); i += 256) {
        const int r = i / (kp / 8), c = (i - r * (kp / 8)) * 8;
        s16x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r < p.R) w = load_some<8>(p.a + ((int64_t)j * p.R + r) * p.K + c, p.K - c);
        *reinterpret_cast<s16x8*>(weights + r * STRIDE + c * 2) = w;
      }
      for (int i = tid; i < np * 2 * NR; i += 256) {  // eight ranks of a column of B_j, down the rows of LDS
        const int c = i / (2 * NR), r = (i - c * (2 * NR)) * 8;
        s16x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c < p.N) w = load_some<8>(p.b + ((int64_t)j * p.N + c) * p.R + r, p.R - r);
#pragma unroll
        for (int q = 0; q < 8; ++q) *reinterpret_cast<short*>(weights + (r + q) * STRIDE + (kp + c) * 2) = w[q];
      }
    }
    all += total;
    load_rows(0);
    __syncthreads();
    for (int from = 0; from < total; from += NARROW_ROWS) {
      // -- h and t of this wavefront's 16 rows: lane: row l % 16, ranks 16 i + 4 g ..; the rows go to LDS for the other products
      uint8_t* mine = rows_at + (16 * wave + l16) * STRIDE + 16 * g;
      const uint8_t* wl = weights + l16 * STRIDE + 16 * g;
      const int xsteps = fresh(kp / 32), steps = fresh((kp + np) / 32);
      v4f h[NR], t[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) h[i] = t[i] = zero;
#pragma unroll
      for (int s = 0; s < W / 32; ++s)
        if (s < steps) {
          *reinterpret_cast<s16x8*>(mine + 64 * s) = v[s];
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const s16x8 w = *reinterpret_cast<const s16x8*>(wl + 16 * i * STRIDE + 64 * s);
            if (s < xsteps) h[i] = mfma_rank<DT>(w, v[s], h[i]);
            else t[i] = mfma_rank<DT>(w, v[s], t[i]);
          }
        }
      if (from + NARROW_ROWS < total) load_rows(from + NARROW_ROWS);
      // (an infinity in a row makes one or NaN of all its sums)
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum += h[i][q] + t[i][q];
      const uint64_t found = __builtin_amdgcn_ballot_w64(!(fabsf(sum) < __builtin_inff()));
      if (lane == 0) infinities[wave] = found != 0;
      // (ranks past R and rows past the list are zero: an infinity times the zeros there is NaN, which would meet all sums)
      const bool there = from + 16 * wave + l16 < total;
      float most_t = 0.0f, most_h = 0.0f;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool part = there && 16 * i + 4 * g + q < p.R;
          h[i][q] = part ? h[i][q] * scale : 0.0f;
          t[i][q] = part ? t[i][q] * scale : 0.0f;
          most_t = fmaxf(most_t, finite_abs(t[i][q]));
          most_h = fmaxf(most_h, finite_abs(h[i][q]));
        }
      // FP16: t and h times a power of two, one for the 64 rows, and for dx t times the row's own
      float up_r = 1.0f, down_r = 1.0f, up_t = 1.0f, down_t = 1.0f, up_h = 1.0f, down_h = 1.0f;
      if constexpr (DT == FIM_F16) {
        most_t = fmaxf(most_t, __shfl_xor(most_t, 16));
        most_t = fmaxf(most_t, __shfl_xor(most_t, 32));
        up_r = half_scale(most_t, down_r);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          most_t = fmaxf(most_t, __shfl_xor(most_t, o));
          most_h = fmaxf(most_h, __shfl_xor(most_h, o));
        }
        if (lane == 0) {
          largest[0][wave] = most_t;
          largest[1][wave] = most_h;
        }
        lds_barrier();
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          most_t = fmaxf(most_t, largest[0][w]);
          most_h = fmaxf(most_h, largest[1][w]);
        }
        up_t = half_scale(most_t, down_t);
        up_h = half_scale(most_h, down_h);
      }
      s16x8 tf[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        s16x4 th, tl, hh, hl;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          short hi, lo;
          split16<DT>(DT == FIM_F16 ? t[i][q] * up_r : t[i][q], hi, lo);
          tf[i][q] = hi;
          tf[i][4 + q] = lo;
          if constexpr (DT == FIM_F16) split16<DT>(t[i][q] * up_t, hi, lo);
          th[q] = hi;
          tl[q] = lo;
          split16<DT>(DT == FIM_F16 ? h[i][q] * up_h : h[i][q], hi, lo);
          hh[q] = hi;
          hl[q] = lo;
        }
        uint8_t* to = ts + (16 * wave + l16) * TS + 32 * i + 8 * g;
        *reinterpret_cast<s16x4*>(to) = th;
        *reinterpret_cast<s16x4*>(to + 32 * NR) = tl;
        *reinterpret_cast<s16x4*>(to + 64 * NR) = hh;
        *reinterpret_cast<s16x4*>(to + 96 * NR) = hl;
      }
      // -- dx: columns interleaved as in adapters_rows.h, A_j's ranks read down its columns
      if (p.dx != nullptr) {
        uint16_t* out = p.dx + (int64_t)(r0 + (there ? list[from + 16 * wave + l16] : 0)) * p.K + 8 * g;
        for (int c = 0; c < p.K; c += 32) {
          float o[8];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            v4f d = zero;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
              const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lds_s16x4*)(weights + (16 * i + 4 * g + (l16 >> 2)) * STRIDE + (c + 8 * (lane & 3) + 4 * u) * 2));
              d = mfma_rank<DT>(beside_halves<DT>(v), tf[i], d);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) o[4 * u + q] = DT == FIM_F16 ? d[q] * down_r : d[q];
          }
          const v4i w = {(int)to16x2<DT>(o[0], o[1]), (int)to16x2<DT>(o[2], o[3]), (int)to16x2<DT>(o[4], o[5]),
                         (int)to16x2<DT>(o[6], o[7])};
          const int left = WHOLE ? 8 : p.K - c - 8 * g;
          if (there && left > 0) store_some<8>(out + c, left, __builtin_bit_cast(s16x8, w));
        }
      }
      lds_barrier();
      // -- dA and dB: 64 rows, 32 a product; this wavefront's 16-column blocks of x and d_out
      auto sums = [&](auto beside) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int r = 32 * s + 8 * g + (l16 >> 2), xcols = kp, most = kp + np;
          s16x8 f[4][NR];  // t hi, t lo, h hi, h lo: rank l % 16, rows 8 g ..
#pragma unroll
          for (int plane = 0; plane < 4; ++plane)
#pragma unroll
            for (int i = 0; i < NR; ++i) {
              const uint8_t* src = ts + r * TS + 32 * (plane * NR + i) + (lane & 3) * 8;
              const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src);
              const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 4 * TS));
              f[plane][i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
          for (int c = 0; c < CB; ++c) {
            const int col = 16 * (wave + 4 * c);
            if (col >= most) continue;
            const uint8_t* src = rows_at + r * STRIDE + col * 2 + (lane & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 4 * STRIDE));
            const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), vl = beside(v);
            const bool of_x = col < xcols;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
              const s16x8 fh = of_x ? f[0][i] : f[2][i], fl = of_x ? f[1][i] : f[3][i];
              if constexpr (DT == FIM_F16) {
                const v4f z = mfma_rank<DT>(fl, vl, mfma_rank<DT>(fh, v, zero));
                const float down = of_x ? down_t : down_h;
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][c][q] = fmaf(z[q], down, acc[i][c][q]);
              } else {
                acc[i][c] = mfma_rank<DT>(fl, vl, mfma_rank<DT>(fh, v, acc[i][c]));
              }
            }
          }
        }
      };
      if (p.da != nullptr) {  // (infinities apart: 320000 x 64 -> 256 62 us, 68 in one)
        if (__builtin_amdgcn_readfirstlane(infinities[0] | infinities[1] | infinities[2] | infinities[3]))
          sums([](s16x8 v) { return beside_hi<DT>(v); });
        else sums([](s16x8 v) { return v; });
      }
      lds_barrier();
    }
  } while (PIECES && (r0 += piece) < end);
  if (none) return;
  if (tid == 0 && p.counts != nullptr) p.counts[slot] = all;
  if (all == 0 && p.part != nullptr) return;
  if (p.da == nullptr) return;
  // -- lane: column l % 16 of 16, ranks 4 g ..
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int at16 = 16 * (wave + 4 * c);
    const bool of_x = at16 < kp;
    const int col = (of_x ? at16 : at16 - kp) + l16, width = of_x ? p.K : p.N;
    if (at16 >= kp + np || col >= width) continue;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 16 * i + 4 * g + q;
        if (r >= p.R) continue;
        if (p.part != nullptr) p.part[((int64_t)slot * p.R + r) * (p.K + p.N) + (of_x ? col : p.K + col)] = acc[i][c][q];
        else if (of_x) p.da[((int64_t)j * p.R + r) * p.K + col] = to16<DT>(acc[i][c][q]);
        else p.db[((int64_t)j * p.N + col) * p.R + r] = to16<DT>(acc[i][c][q]);
      }
  }
}

}  // namespace fim
