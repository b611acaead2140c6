// Group norm with an activation over channels-last maps, and its backward pass.
//
// x [B, P, C] (P pixels, C channels innermost), G groups of D = C / G channels. Per (image, group) over its P x D values
//   xhat = (x - mean) * rstd,  z = xhat * weight[c] + bias[c],  y = act(z)
// and with dz = dy * act'(z)
//   dbias[c] = sum dz, dweight[c] = sum dz * xhat  (over images and pixels)
//   dx = rstd * (dz * weight - s1 - xhat * s2),  s1, s2 the group's means of dz * weight and dz * weight * xhat.
//
// Both directions are streams: the floor is one read and one write forward (2 n bytes of the type's size), x and dy in and
// dx out backward. The statistics need all of a group before the first output, so each direction reads its inputs twice; a
// workgroup takes the same pixels in both passes, and so finds them in its XCD's L2 or the Infinity Cache where they fit.
//
// A workgroup of 512 threads takes a run of pixels ("chunk") of one image and all channels: thread t keeps the V channels
// of column t % (C / V) and every (512 / (C / V))th pixel, so a wavefront reads whole contiguous runs and the per-channel
// parameters and sums stay in registers. Forward sums are kept per thread and channel about the thread's first pixel (no
// cancellation where the mean is large), merged as (count, mean, squared deviations); nothing is summed by atomics, so
// results do not depend on the order of workgroups.
#include "activation.h"

namespace fim {

constexpr int NORM_T = 512;           // threads of a workgroup
constexpr int NORM_MAX_C = 8192;      // per-channel partials of a workgroup lie in LDS
constexpr int NORM_UNROLL = 4;        // pixels in flight per thread

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;            // y, or dx
  const void* weight;   // null: 1
  const void* bias;     // null: 0
  int wdt, bdt;         // their types
  float* stats;         // [B, G, 2]: mean, rstd
  float* part;          // [B, chunks, G, 2] forward; [B, chunks, C, 2] backward
  float* csum;          // backward: [B, C, 2] sums over pixels of dz, dz * xhat
  float* coef;          // backward: [B, G, 2]: s1, s2
  void* dweight;
  void* dbias;
  int64_t P, sb, sp, db, dp;  // image and pixel strides of x and of dy, in elements
  int B, C, G, D;
  int chunks;
  int64_t chunk;        // pixels of a chunk
  float eps;
};

__device__ __forceinline__ float param(const void* p, int dt, int i, float missing) {
  if (p == nullptr) return missing;
  return dt == FIM_F32 ? static_cast<const float*>(p)[i]
                       : dt == FIM_BF16 ? load_elem<FIM_BF16>(p, i) : load_elem<FIM_F16>(p, i);
}

__device__ __forceinline__ void store_param(void* p, int dt, int i, float v) {
  if (dt == FIM_F32) static_cast<float*>(p)[i] = v;
  else if (dt == FIM_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// V elements as they lie in memory, and as floats
template <int DT, int V>
struct Pack {
  static constexpr int BYTES = V * (DT == FIM_F32 ? 4 : 2);
  struct alignas(BYTES < 16 ? BYTES : 16) Raw { uint8_t b[BYTES]; };
  static __device__ __forceinline__ Raw load(const void* p, int64_t i) {
    return *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(p) + i * (BYTES / V));
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[V]) {
    if constexpr (DT == FIM_F32) {
      __builtin_memcpy(f, &r, BYTES);
    } else {
      uint16_t h[V];
      __builtin_memcpy(h, &r, BYTES);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = DT == FIM_BF16 ? bf16_to_f32(h[i]) : (float)__builtin_bit_cast(_Float16, h[i]);
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[V]) {
    Raw r;
    if constexpr (DT == FIM_F32) {
      __builtin_memcpy(&r, f, BYTES);
    } else if constexpr (DT == FIM_BF16 && V % 2 == 0) {
      uint32_t w[V / 2];
#pragma unroll
      for (int k = 0; k < V / 2; ++k) w[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
      __builtin_memcpy(&r, w, BYTES);
    } else {
      uint16_t h[V];
#pragma unroll
      for (int k = 0; k < V; ++k)
        h[k] = DT == FIM_BF16 ? (uint16_t)(pack_bf16x2(f[k], 0.0f) & 0xffff) : __builtin_bit_cast(uint16_t, (_Float16)f[k]);
      __builtin_memcpy(&r, h, BYTES);
    }
    *reinterpret_cast<Raw*>(static_cast<uint8_t*>(p) + i * (BYTES / V)) = r;
  }
};

// This thread's share of a workgroup: column `col` (V channels) of pixels row, row + rows, ... of [begin, end)
struct Share {
  int col, row, rows;
  bool live;
};

__device__ __forceinline__ Share share_of(int cols, int pass) {
  Share s;
  if (cols >= NORM_T) {
    s.col = pass * NORM_T + threadIdx.x;
    s.row = 0;
    s.rows = 1;
    s.live = s.col < cols;
  } else {
    s.rows = NORM_T / cols;
    s.row = threadIdx.x / cols;
    s.col = threadIdx.x - s.row * cols;
    s.live = s.row < s.rows;
  }
  return s;
}

__device__ __forceinline__ int passes_of(int cols) { return cols >= NORM_T ? (cols + NORM_T - 1) / NORM_T : 1; }

// f(pixel, unpacked...) over this thread's pixels of [begin, end), NORM_UNROLL loads in flight
template <int DT, int V, typename F>
__device__ __forceinline__ void for_pixels(const void* p, int64_t base, int64_t stride, int64_t begin, int64_t end,
                                           const Share& s, F&& f) {
  typedef Pack<DT, V> Pk;
  int64_t i = begin + s.row;
  const int64_t step = s.rows;
  for (; i + (NORM_UNROLL - 1) * step < end; i += NORM_UNROLL * step) {
    typename Pk::Raw r[NORM_UNROLL];
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u) r[u] = Pk::load(p, base + (i + u * step) * stride);
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u) {
      float v[V];
      Pk::unpack(r[u], v);
      f(i + u * step, v);
    }
  }
  for (; i < end; i += step) {
    float v[V];
    Pk::unpack(Pk::load(p, base + i * stride), v);
    f(i, v);
  }
}

template <int DT, int V, typename F>
__device__ __forceinline__ void for_pixels2(const NormArgs& a, int64_t xbase, int64_t dbase, int64_t begin, int64_t end,
                                            const Share& s, F&& f) {
  typedef Pack<DT, V> Pk;
  int64_t i = begin + s.row;
  const int64_t step = s.rows;
  for (; i + (NORM_UNROLL - 1) * step < end; i += NORM_UNROLL * step) {
    typename Pk::Raw r[NORM_UNROLL], q[NORM_UNROLL];
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u) {
      r[u] = Pk::load(a.x, xbase + (i + u * step) * a.sp);
      q[u] = Pk::load(a.dy, dbase + (i + u * step) * a.dp);
    }
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u) {
      float v[V], d[V];
      Pk::unpack(r[u], v);
      Pk::unpack(q[u], d);
      f(i + u * step, v, d);
    }
  }
  for (; i < end; i += step) {
    float v[V], d[V];
    Pk::unpack(Pk::load(a.x, xbase + i * a.sp), v);
    Pk::unpack(Pk::load(a.dy, dbase + i * a.dp), d);
    f(i, v, d);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// pixels of [begin, end) that row `row` of `rows` takes
__device__ __forceinline__ int64_t row_count(int64_t begin, int64_t end, int row, int rows) {
  const int64_t n = end - begin - row;
  return n <= 0 ? 0 : (n + rows - 1) / rows;
}

// Forward, first pass: per (chunk, group) the mean and the sum of squared deviations.
template <int DT, int V>
__global__ __launch_bounds__(NORM_T) void norm_stats_kernel(const NormArgs a) {
  extern __shared__ float lds[];  // [rows][C] means, then [rows][C] squared deviations
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int64_t begin = chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const int cols = a.C / V;
  int rows = 1;
  const int passes = passes_of(cols);
  for (int pass = 0; pass < passes; ++pass) {
    const Share s = share_of(cols, pass);
    rows = s.rows;
    if (!s.live) continue;
    const int c0 = s.col * V;
    const int64_t base = b * a.sb + c0;
    const int64_t n = row_count(begin, end, s.row, s.rows);
    float shift[V], s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) shift[k] = s1[k] = s2[k] = 0.0f;
    if (n > 0) Pack<DT, V>::unpack(Pack<DT, V>::load(a.x, base + (begin + s.row) * a.sp), shift);
    for_pixels<DT, V>(a.x, base, a.sp, begin, end, s, [&](int64_t, const float(&v)[V]) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = v[k] - shift[k];
        s1[k] += d;
        s2[k] = fmaf(d, d, s2[k]);
      }
    });
    const float inv = n > 0 ? 1.0f / (float)n : 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float m = s1[k] * inv;
      lds[s.row * a.C + c0 + k] = shift[k] + m;
      lds[(s.rows + s.row) * a.C + c0 + k] = fmaf(-m, s1[k], s2[k]);
    }
  }
  __syncthreads();
  const float* m2 = lds + rows * a.C;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float total = (float)(end - begin) * (float)a.D;
  for (int g = wave; g < a.G; g += NORM_T / 64) {
    float sum = 0.0f;
    for (int i = lane; i < rows * a.D; i += 64) {
      const int r = i / a.D, at = r * a.C + g * a.D + (i - r * a.D);
      sum += (float)row_count(begin, end, r, rows) * lds[at];
    }
    const float mean = wave_sum(sum) / total;
    float dev = 0.0f;
    for (int i = lane; i < rows * a.D; i += 64) {
      const int r = i / a.D, at = r * a.C + g * a.D + (i - r * a.D);
      const float n = (float)row_count(begin, end, r, rows), d = lds[at] - mean;
      if (n > 0) dev += fmaf(n * d, d, m2[at]);
    }
    dev = wave_sum(dev);
    if (lane == 0) {
      float* p = a.part + ((int64_t)blockIdx.x * a.G + g) * 2;
      p[0] = mean;
      p[1] = dev;
    }
  }
}

// One wavefront per (image, group): the chunks' means and deviations merged.
__global__ __launch_bounds__(256) void norm_merge_kernel(const NormArgs a) {
  const int64_t bg = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (bg >= (int64_t)a.B * a.G) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = bg / a.G, g = bg - b * a.G;
  const float* p = a.part + (b * a.chunks * a.G + g) * 2;
  const double total = (double)a.P * a.D;
  double sum = 0.0;
  for (int i = lane; i < a.chunks; i += 64) {
    const int64_t begin = i * a.chunk, n = (begin + a.chunk < a.P ? begin + a.chunk : a.P) - begin;
    sum += (double)(n * a.D) * p[(int64_t)i * a.G * 2];
  }
  const double mean = wave_sum(sum) / total;
  double dev = 0.0;
  for (int i = lane; i < a.chunks; i += 64) {
    const int64_t begin = i * a.chunk, n = (begin + a.chunk < a.P ? begin + a.chunk : a.P) - begin;
    const double d = p[(int64_t)i * a.G * 2] - mean;
    dev += (double)(n * a.D) * d * d + p[(int64_t)i * a.G * 2 + 1];
  }
  dev = wave_sum(dev);
  if (lane == 0) {
    a.stats[2 * bg] = (float)mean;
    a.stats[2 * bg + 1] = (float)(1.0 / sqrt(dev / total + (double)a.eps));
  }
}

template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T) void norm_apply_kernel(const NormArgs a) {
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int64_t begin = chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const int cols = a.C / V, passes = passes_of(cols);
  for (int pass = 0; pass < passes; ++pass) {
    const Share s = share_of(cols, pass);
    if (!s.live) continue;
    const int c0 = s.col * V;
    float mean[V], mul[V], add[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float* st = a.stats + ((int64_t)b * a.G + (c0 + k) / a.D) * 2;
      mean[k] = st[0];
      mul[k] = st[1] * param(a.weight, a.wdt, c0 + k, 1.0f);
      add[k] = param(a.bias, a.bdt, c0 + k, 0.0f);
    }
    const int64_t out = (int64_t)b * a.P * a.C + c0;
    for_pixels<DT, V>(a.x, b * a.sb + c0, a.sp, begin, end, s,
                      [&](int64_t i, const float(&v)[V]) __attribute__((always_inline)) {
                        float y[V];
#pragma unroll
                        for (int k = 0; k < V; ++k) y[k] = activate<ACT>(fmaf(v[k] - mean[k], mul[k], add[k]));
                        Pack<DT, V>::store(a.out, out + i * a.C, y);
                      });
  }
}

// Backward, first pass: per (chunk, channel) the sums of dz and dz * xhat.
template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T) void norm_grad_sums_kernel(const NormArgs a) {
  extern __shared__ float lds[];  // [rows][C][2]
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int64_t begin = chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const int cols = a.C / V, passes = passes_of(cols);
  int rows = 1;
  for (int pass = 0; pass < passes; ++pass) {
    const Share s = share_of(cols, pass);
    rows = s.rows;
    if (!s.live) continue;
    const int c0 = s.col * V;
    float mean[V], rstd[V], w[V], add[V], s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float* st = a.stats + ((int64_t)b * a.G + (c0 + k) / a.D) * 2;
      mean[k] = st[0];
      rstd[k] = st[1];
      w[k] = param(a.weight, a.wdt, c0 + k, 1.0f);
      add[k] = param(a.bias, a.bdt, c0 + k, 0.0f);
      s1[k] = s2[k] = 0.0f;
    }
    for_pixels2<DT, V>(a, b * a.sb + c0, b * a.db + c0, begin, end, s,
                       [&](int64_t, const float(&v)[V], const float(&d)[V]) __attribute__((always_inline)) {
#pragma unroll
                         for (int k = 0; k < V; ++k) {
                           const float xhat = (v[k] - mean[k]) * rstd[k];
                           float slope;
                           activate<ACT, true>(fmaf(xhat, w[k], add[k]), slope);
                           const float dz = d[k] * slope;
                           s1[k] += dz;
                           s2[k] = fmaf(dz, xhat, s2[k]);
                         }
                       });
#pragma unroll
    for (int k = 0; k < V; ++k) {
      lds[(s.row * a.C + c0 + k) * 2] = s1[k];
      lds[(s.row * a.C + c0 + k) * 2 + 1] = s2[k];
    }
  }
  __syncthreads();
  float* p = a.part + (int64_t)blockIdx.x * a.C * 2;
  for (int i = threadIdx.x; i < 2 * a.C; i += NORM_T) {
    float sum = 0.0f;
    for (int r = 0; r < rows; ++r) sum += lds[r * a.C * 2 + i];
    p[i] = sum;
  }
}

// One workgroup per (image, group): the chunks' sums per channel, and the group's two means.
__global__ __launch_bounds__(256) void norm_grad_merge_kernel(const NormArgs a) {
  __shared__ float red[4][2];
  const int b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float g1 = 0.0f, g2 = 0.0f;
  for (int d = wave; d < a.D; d += 4) {
    const int c = g * a.D + d;
    double s1 = 0.0, s2 = 0.0;
    for (int i = lane; i < a.chunks; i += 64) {
      const float* p = a.part + (((int64_t)b * a.chunks + i) * a.C + c) * 2;
      s1 += p[0];
      s2 += p[1];
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (lane == 0) {
      a.csum[((int64_t)b * a.C + c) * 2] = (float)s1;
      a.csum[((int64_t)b * a.C + c) * 2 + 1] = (float)s2;
    }
    const float w = param(a.weight, a.wdt, c, 1.0f);
    g1 = fmaf((float)s1, w, g1);
    g2 = fmaf((float)s2, w, g2);
  }
  if (lane == 0) {
    red[wave][0] = g1;
    red[wave][1] = g2;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const int k = threadIdx.x;
    a.coef[2 * (int64_t)blockIdx.x + k] = (red[0][k] + red[1][k] + red[2][k] + red[3][k]) / ((float)a.P * (float)a.D);
  }
}

// Parameter gradients: the images' per-channel sums, in the order of the images. One wavefront per channel.
__global__ __launch_bounds__(256) void norm_grad_params_kernel(const NormArgs a) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (c >= a.C) return;
  double s1 = 0.0, s2 = 0.0;
  for (int b = lane; b < a.B; b += 64) {
    s1 += a.csum[((int64_t)b * a.C + c) * 2];
    s2 += a.csum[((int64_t)b * a.C + c) * 2 + 1];
  }
  s1 = wave_sum(s1);
  s2 = wave_sum(s2);
  if (lane == 0) {
    if (a.dbias != nullptr) store_param(a.dbias, a.bdt, c, (float)s1);
    if (a.dweight != nullptr) store_param(a.dweight, a.wdt, c, (float)s2);
  }
}

template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T) void norm_grad_apply_kernel(const NormArgs a) {
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int64_t begin = chunk * a.chunk, end = begin + a.chunk < a.P ? begin + a.chunk : a.P;
  const int cols = a.C / V, passes = passes_of(cols);
  for (int pass = 0; pass < passes; ++pass) {
    const Share s = share_of(cols, pass);
    if (!s.live) continue;
    const int c0 = s.col * V;
    float mean[V], rstd[V], w[V], add[V], m1[V], m2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int64_t bg = (int64_t)b * a.G + (c0 + k) / a.D;
      mean[k] = a.stats[2 * bg];
      rstd[k] = a.stats[2 * bg + 1];
      m1[k] = a.coef[2 * bg];
      m2[k] = a.coef[2 * bg + 1];
      w[k] = param(a.weight, a.wdt, c0 + k, 1.0f);
      add[k] = param(a.bias, a.bdt, c0 + k, 0.0f);
    }
    const int64_t out = (int64_t)b * a.P * a.C + c0;
    for_pixels2<DT, V>(a, b * a.sb + c0, b * a.db + c0, begin, end, s,
                       [&](int64_t i, const float(&v)[V], const float(&d)[V]) __attribute__((always_inline)) {
                         float dx[V];
#pragma unroll
                         for (int k = 0; k < V; ++k) {
                           const float xhat = (v[k] - mean[k]) * rstd[k];
                           float slope;
                           activate<ACT, true>(fmaf(xhat, w[k], add[k]), slope);
                           dx[k] = rstd[k] * (fmaf(d[k] * slope, w[k], -m1[k]) - xhat * m2[k]);
                         }
                         Pack<DT, V>::store(a.out, out + i * a.C, dx);
                       });
  }
}

// -- launches ----------------------------------------------------------------------------------------------------------

// Chunks of an image: about two workgroups per CU over all images (each keeps 512 x 4 loads in flight), but at least
// 8 pixels per thread row of a workgroup.
static void norm_split(int64_t B, int64_t P, int64_t C, int64_t& chunk, int& chunks) {
  const int64_t want = cdiv(2 * (int64_t)device_cus(), B > 0 ? B : 1);
  int64_t least = cdiv(8 * NORM_T * 8, C);
  if (least < 1) least = 1;
  chunk = cdiv(P, want > 0 ? want : 1);
  if (chunk < least) chunk = least;
  if (chunk > P) chunk = P > 0 ? P : 1;
  chunks = (int)cdiv(P > 0 ? P : 1, chunk);
}

static int elem_size(int dtype) { return dtype == FIM_F32 ? 4 : 2; }

// Elements per load: the largest power of two that divides the channels, every stride and the base addresses, up to 16
// bytes.
static int norm_vector(int dtype, int64_t C, std::initializer_list<int64_t> strides, std::initializer_list<const void*> ptrs) {
  const int es = elem_size(dtype);
  int v = 16 / es;
  auto fits = [&](int w) {
    if (C % w) return false;
    for (int64_t s : strides)
      if (s % w) return false;
    for (const void* p : ptrs)
      if (reinterpret_cast<uintptr_t>(p) % (uintptr_t)(w * es)) return false;
    return true;
  };
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

// f(integral constants DT, V)
template <typename F>
static void with_vector(int dtype, int v, F&& f) {
#define FIM_V(DT, N) case N: f(std::integral_constant<int, DT>{}, std::integral_constant<int, N>{}); break;
  if (dtype == FIM_F32) {
    switch (v) { FIM_V(FIM_F32, 4) FIM_V(FIM_F32, 2) default: FIM_V(FIM_F32, 1) }
  } else if (dtype == FIM_BF16) {
    switch (v) { FIM_V(FIM_BF16, 8) FIM_V(FIM_BF16, 4) FIM_V(FIM_BF16, 2) default: FIM_V(FIM_BF16, 1) }
  } else {
    switch (v) { FIM_V(FIM_F16, 8) FIM_V(FIM_F16, 4) FIM_V(FIM_F16, 2) default: FIM_V(FIM_F16, 1) }
  }
#undef FIM_V
}

static bool dtype_ok(int dt) { return dt == FIM_F32 || dt == FIM_BF16 || dt == FIM_F16; }

static int norm_check(int dtype, int64_t B, int64_t P, int64_t C, int64_t groups, int wdt, int bdt, int act) {
  if (B < 0 || P < 0 || C <= 0 || groups <= 0 || C % groups) return FIM_ERR_INVALID;
  if (!dtype_ok(dtype) || !dtype_ok(wdt) || !dtype_ok(bdt) || act < 0 || act >= ACT_COUNT) return FIM_ERR_INVALID;
  if (C > NORM_MAX_C || B * groups > INT32_MAX || B * C > INT32_MAX) return FIM_ERR_UNSUPPORTED;
  return FIM_OK;
}

static size_t norm_lds(int64_t C, int v) {
  const int64_t cols = C / v, rows = cols >= NORM_T ? 1 : NORM_T / cols;
  return (size_t)(rows * C * 2 * 4);
}

}  // namespace fim

using namespace fim;

extern "C" int fim_group_norm_workspace(int64_t B, int64_t P, int64_t C, int64_t groups, int backward, int64_t* floats) {
  if (floats == nullptr) return FIM_ERR_INVALID;
  const int rc = norm_check(FIM_F32, B, P, C, groups, FIM_F32, FIM_F32, 0);
  if (rc != FIM_OK) return rc;
  int64_t chunk;
  int chunks;
  norm_split(B, P, C, chunk, chunks);
  *floats = 2 * B * (backward ? (int64_t)chunks * C + C + groups : (int64_t)chunks * groups);
  return FIM_OK;
}

extern "C" int fim_group_norm(const void* x, int dtype, int64_t B, int64_t P, int64_t C, int64_t stride_b,
                              int64_t stride_p, int64_t groups, const void* weight, int weight_dtype, const void* bias,
                              int bias_dtype, float eps, int act, void* out, float* stats, float* workspace,
                              hipStream_t stream) {
  const int rc = norm_check(dtype, B, P, C, groups, weight_dtype, bias_dtype, act);
  if (rc != FIM_OK) return rc;
  if (B * P == 0) return FIM_OK;
  if (x == nullptr || out == nullptr || stats == nullptr || workspace == nullptr) return FIM_ERR_INVALID;
  NormArgs a{};
  a.x = x;
  a.out = out;
  a.weight = weight;
  a.bias = bias;
  a.wdt = weight_dtype;
  a.bdt = bias_dtype;
  a.stats = stats;
  a.part = workspace;
  a.P = P;
  a.sb = stride_b;
  a.sp = stride_p;
  a.B = (int)B;
  a.C = (int)C;
  a.G = (int)groups;
  a.D = (int)(C / groups);
  a.eps = eps;
  norm_split(B, P, C, a.chunk, a.chunks);
  if (B * a.chunks > INT32_MAX) return FIM_ERR_UNSUPPORTED;
  const int v = norm_vector(dtype, C, {stride_b, stride_p}, {x, out});
  const dim3 grid((unsigned)(B * a.chunks));
  with_vector(dtype, v, [&](auto dt, auto vec) {
    constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
    norm_stats_kernel<DT, V><<<grid, dim3(NORM_T), norm_lds(C, V), stream>>>(a);
    norm_merge_kernel<<<dim3((unsigned)cdiv(B * groups, 4)), dim3(256), 0, stream>>>(a);
    with_activation(act, [&](auto act_c) {
      norm_apply_kernel<DT, V, decltype(act_c)::value><<<grid, dim3(NORM_T), 0, stream>>>(a);
    });
  });
  return launch_status();
}

extern "C" int fim_group_norm_backward(const void* x, const void* d_out, int dtype, int64_t B, int64_t P, int64_t C,
                                       int64_t stride_b, int64_t stride_p, int64_t d_stride_b, int64_t d_stride_p,
                                       int64_t groups, const void* weight, int weight_dtype, const void* bias,
                                       int bias_dtype, int act, const float* stats, void* dx, void* d_weight, void* d_bias,
                                       float* workspace, hipStream_t stream) {
  const int rc = norm_check(dtype, B, P, C, groups, weight_dtype, bias_dtype, act);
  if (rc != FIM_OK) return rc;
  if (B * P == 0) return FIM_OK;
  if (x == nullptr || d_out == nullptr || dx == nullptr || stats == nullptr || workspace == nullptr) return FIM_ERR_INVALID;
  NormArgs a{};
  a.x = x;
  a.dy = d_out;
  a.out = dx;
  a.weight = weight;
  a.bias = bias;
  a.wdt = weight_dtype;
  a.bdt = bias_dtype;
  a.stats = const_cast<float*>(stats);
  a.dweight = d_weight;
  a.dbias = d_bias;
  a.P = P;
  a.sb = stride_b;
  a.sp = stride_p;
  a.db = d_stride_b;
  a.dp = d_stride_p;
  a.B = (int)B;
  a.C = (int)C;
  a.G = (int)groups;
  a.D = (int)(C / groups);
  norm_split(B, P, C, a.chunk, a.chunks);
  if (B * a.chunks > INT32_MAX) return FIM_ERR_UNSUPPORTED;
  a.part = workspace;
  a.csum = workspace + 2 * B * (int64_t)a.chunks * C;
  a.coef = a.csum + 2 * B * C;
  const int v = norm_vector(dtype, C, {stride_b, stride_p, d_stride_b, d_stride_p}, {x, d_out, dx});
  const dim3 grid((unsigned)(B * a.chunks));
  with_vector(dtype, v, [&](auto dt, auto vec) {
    constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
    with_activation(act, [&](auto act_c) {
      constexpr int ACT = decltype(act_c)::value;
      norm_grad_sums_kernel<DT, V, ACT><<<grid, dim3(NORM_T), norm_lds(C, V), stream>>>(a);
      norm_grad_merge_kernel<<<dim3((unsigned)(B * groups)), dim3(256), 0, stream>>>(a);
      norm_grad_apply_kernel<DT, V, ACT><<<grid, dim3(NORM_T), 0, stream>>>(a);
    });
    if (d_weight != nullptr || d_bias != nullptr)
      norm_grad_params_kernel<<<dim3((unsigned)cdiv(C, 4)), dim3(256), 0, stream>>>(a);
  });
  return launch_status();
}
