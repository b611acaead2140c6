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
// parameters and sums stay in registers, and loads a batch of pixels ahead. The first pass writes one partial per
// (chunk, group), the second adds up its image's partials before it starts, while its first loads are on their way (a
// launch between the two for groups so many that every workgroup would read them for long). Nothing is summed by atomics:
// results do not depend on the order of workgroups. Forward sums are kept about the mean of a thread's first pixels (no
// cancellation where the mean is large) and merged as means and squared deviations. Small maps take one launch forward
// (norm_group_kernel).
//
// Measured (device time after a hundred calls, MI355X; a large copy reaches 5.1 TB/s): two maps of 160000 x 64 BF16 with GELU,
// 12 us for the statistics and 21 us for the apply forward, 23 us and 32 us backward, where their read or write is 8 us: the
// activation with its slope is 20 to 40 vector operations a value (8 to 16 us), and each pass starts with a launch, the
// partials of the pass before and its first round of loads (5 us). Two of 40000 x 128: 12 + 4 (merge) + 13 us. 1024 x 64: 7.6 us
// in one launch (13.8 in two), latencies alone.
#include "activation.h"

namespace fim {

constexpr int NORM_T = 512;           // threads of a workgroup
// Pixels of a batch of loads (the next batch is loaded while one is worked on), for four wavefronts per SIMD (128 registers, of
// which the applies of 16-bit maps with 8 channels a load spill up to 13 forward and 20 backward): backward, with two tensors and
// the activation's slope, 4 took 180 to 230 registers and ran half as many wavefronts
constexpr int NORM_U = 4, NORM_GRAD_U = 2;
constexpr int NORM_OWN = 8;           // loads of a thread that owns its values (small maps)
constexpr int NORM_MAX_C = 8192;      // per-channel partials of a workgroup lie in LDS
constexpr int NORM_MERGE_G = 512;     // groups, and partials, that the workgroups of the second pass add up themselves
constexpr int64_t NORM_MERGE = 2 << 20;  // (over all workgroups)
// Bytes of a map that is small. One workgroup per (image, group) reads D channels of each pixel, as little as 16 bytes of a line:
// against two launches 1024 x 64 in 8 groups, 7.6 and 13.8 us; 16 images of it (2 MB), 9.8 and 14.3; 32, 13.5 and 14.9; 40 (5 MB),
// 19.2 and 17.6; 64, 24.2 and 18.0; 20 images of 256 x 512 in 32 groups (5 MB), 17.8 and 19.1
constexpr int64_t NORM_SMALL = 5 << 20;

struct NormArgs {
  const uint8_t* x;
  const uint8_t* dy;
  uint8_t* out;         // y, or dx
  const void* weight;   // null: 1
  const void* bias;     // null: 0
  int wdt, bdt;         // their types
  float* stats;         // [B, G, 2]: mean, rstd
  float* gpart;         // [B, chunks, G, 2]: mean and squared deviations; backward sums of dz * weight, dz * weight * xhat
  float* cpart;         // backward: [B, chunks, C, 2]: sums of dz, dz * xhat
  float* coef;          // backward, merged between the passes: [B, G, 2]: s1, s2
  void* dweight;
  void* dbias;
  int64_t P, sb, sp, db, dp;  // image and pixel strides of x and of dy, in elements
  int B, C, G, D;
  int chunks, chunk;    // chunks of an image, and their pixels
  int merged;           // stats (coef) were merged by a launch between the passes
  int first;            // of the workgroups of a pass, the launch's first (launch_pass)
  float eps;
};

__device__ __forceinline__ float param(const void* p, int dt, int i, float missing) {
  if (p == nullptr) return missing;
  return dt == FIM_F32 ? static_cast<const float*>(p)[i]
                       : dt == FIM_BF16 ? load_elem<FIM_BF16>(p, i) : load_elem<FIM_F16>(p, i);
}

// V neighbouring parameters: all loads on one side of the branch on their type, so their latencies overlap
template <int V>
__device__ __forceinline__ void params(const void* p, int dt, int i, float missing, float (&f)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = missing;
  } else if (dt == FIM_F32) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = static_cast<const float*>(p)[i + k];
  } else {
    uint16_t h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = static_cast<const uint16_t*>(p)[i + k];
#pragma unroll
    for (int k = 0; k < V; ++k)
      f[k] = dt == FIM_BF16 ? bf16_to_f32(h[k]) : (float)__builtin_bit_cast(_Float16, h[k]);
  }
}

// g[k]: the group of channel c0 + k
template <int V>
__device__ __forceinline__ void groups_of(int c0, int D, int (&g)[V]) {
  int at = c0 / D, r = c0 - at * D;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    g[k] = at;
    ++r;
    at += r == D;
    r = r == D ? 0 : r;
  }
}

__device__ __forceinline__ void store_param(void* p, int dt, int i, float v) {
  if (dt == FIM_F32) static_cast<float*>(p)[i] = v;
  else if (dt == FIM_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// V elements as they lie in memory, and as floats
template <int DT, int V>
struct Pack {
  static constexpr int ES = DT == FIM_F32 ? 4 : 2, BYTES = V * ES;
  struct alignas(BYTES < 16 ? BYTES : 16) Raw { uint8_t b[BYTES]; };
  static __device__ __forceinline__ Raw load(const uint8_t* p) { return *reinterpret_cast<const Raw*>(p); }
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
  // STREAM: marked as not read again soon, so that the inputs stay in the caches. 16-bit types only (40000 x 128 forward 29.2 ->
  // 27.7 us a call, 160000 x 64 with its backward 98 -> 91, and with a gated product that reads the output after it 56.6 -> 54.0;
  // FP32 maps took two to three times as long: 22725 x 196, 10 -> 30 us for the apply)
  template <bool STREAM = false>
  static __device__ __forceinline__ void store(uint8_t* p, const float (&f)[V]) {
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
    if constexpr (STREAM && DT != FIM_F32 && BYTES == 16) {
      typedef uint32_t Words __attribute__((ext_vector_type(4)));
      __builtin_nontemporal_store(__builtin_bit_cast(Words, r), reinterpret_cast<Words*>(p));
    } else {
      *reinterpret_cast<Raw*>(p) = r;
    }
  }
};

// This thread's share of a chunk: V channels from `c0`, pixels row, row + rows, ...: `n` of them
struct Share {
  int c0, row, rows, n;
  bool live;
};

template <int V>
__device__ __forceinline__ Share share_of(const NormArgs& a, int pass, int pixels) {
  const int cols = a.C / V;
  Share s;
  int col;
  if (cols >= NORM_T) {
    col = pass * NORM_T + threadIdx.x;
    s.row = 0;
    s.rows = 1;
    s.live = col < cols;
  } else {
    s.rows = NORM_T / cols;
    s.row = threadIdx.x / cols;
    col = threadIdx.x - s.row * cols;
    s.live = s.row < s.rows;
  }
  s.c0 = col * V;
  s.n = s.row < pixels ? (pixels - s.row + s.rows - 1) / s.rows : 0;
  return s;
}
template <int V>
__device__ __forceinline__ int passes_of(const NormArgs& a) {
  return a.C / V >= NORM_T ? (a.C / V + NORM_T - 1) / NORM_T : 1;
}

// The workgroup's image, chunk and pixels
struct Chunk {
  int b, i, pixels;
  int64_t begin;
};
__device__ __forceinline__ int block_of(const NormArgs& a) { return a.first + (int)blockIdx.x; }  // (below 2^31)
__device__ __forceinline__ Chunk chunk_of(const NormArgs& a) {
  Chunk c;
  c.b = (int)((uint32_t)block_of(a) / (uint32_t)a.chunks);
  c.i = block_of(a) - c.b * a.chunks;
  c.begin = (int64_t)c.i * a.chunk;
  c.pixels = c.begin + a.chunk < a.P ? a.chunk : (int)(a.P - c.begin);
  return c;
}
__device__ __forceinline__ int pixels_of(const NormArgs& a, int chunk) {
  const int64_t begin = (int64_t)chunk * a.chunk;
  return begin + a.chunk < a.P ? a.chunk : (int)(a.P - begin);
}

// A thread's pixels of one tensor, U at a time; batch k's loads past the end repeat the last pixel
template <int DT, int V, int U>
struct Rows {
  typedef Pack<DT, V> Pk;
  const uint8_t* p;
  int64_t step;
  int n;
  __device__ __forceinline__ Rows(const uint8_t* base, int64_t image, int64_t sp, const Chunk& c, const Share& s) {
    p = base + (c.b * image + (c.begin + s.row) * sp + s.c0) * Pk::ES;
    step = s.rows * sp * Pk::ES;
    n = s.n;
  }
  __device__ __forceinline__ void load(int k, typename Pk::Raw (&r)[U]) const {
    const uint8_t* at = p + k * step;
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = Pk::load(at + (k + u < n ? u : n - 1 - k) * step);
  }
  // f(first pixel's index, batch) over all pixels; r[0] holds the first batch
  template <typename F>
  __device__ __forceinline__ void batches(typename Pk::Raw (&r)[2][U], F&& f) const {
    for (int i = 0;;) {
      if (i + U < n) load(i + U, r[1]);
      f(i, r[0]);
      i += U;
      if (i >= n) break;
      if (i + U < n) load(i + U, r[0]);
      f(i, r[1]);
      i += U;
      if (i >= n) break;
    }
  }
};

// the same over the rows of two tensors
template <int DT, int V, int U, typename F>
__device__ __forceinline__ void batches2(const Rows<DT, V, U>& x, const Rows<DT, V, U>& d,
                                         typename Pack<DT, V>::Raw (&rx)[2][U], typename Pack<DT, V>::Raw (&rd)[2][U],
                                         F&& f) {
  auto next = [&](int i, int k) __attribute__((always_inline)) {
    if (i >= x.n) return;
    x.load(i, rx[k]);
    d.load(i, rd[k]);
  };
  for (int i = 0;;) {
    next(i + U, 1);
    f(i, rx[0], rd[0]);
    i += U;
    if (i >= x.n) break;
    next(i + U, 0);
    f(i, rx[1], rd[1]);
    i += U;
    if (i >= x.n) break;
  }
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Forward, first pass: per (chunk, group) the mean and the sum of squared deviations.
template <int DT, int V>
__global__ __launch_bounds__(NORM_T, 4) void norm_stats_kernel(const NormArgs a) {
  extern __shared__ float2 lds2[];  // [rows][C]: mean and squared deviations of a thread's pixels
  const Chunk ch = chunk_of(a);
  int rows = 1;
  for (int pass = 0; pass < passes_of<V>(a); ++pass) {
    const Share s = share_of<V>(a, pass, ch.pixels);
    rows = s.rows;
    if (!s.live) continue;
    float s1[V], s2[V], shift[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s1[k] = s2[k] = shift[k] = 0.0f;
    if (s.n > 0) {
      const Rows<DT, V, NORM_U> x(a.x, a.sb, a.sp, ch, s);
      typename Pack<DT, V>::Raw r[2][NORM_U];
      x.load(0, r[0]);
#pragma unroll
      for (int u = 0; u < NORM_U; ++u) {  // the first pixels' mean (repeats weigh in: any value near will do)
        float v[V];
        Pack<DT, V>::unpack(r[0][u], v);
#pragma unroll
        for (int k = 0; k < V; ++k) shift[k] = fmaf(v[k], 1.0f / NORM_U, shift[k]);
      }
      x.batches(r, [&](int i, const typename Pack<DT, V>::Raw(&now)[NORM_U]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NORM_U; ++u) {
          if (i + u >= s.n) break;
          float v[V];
          Pack<DT, V>::unpack(now[u], v);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float d = v[k] - shift[k];
            s1[k] += d;
            s2[k] = fmaf(d, d, s2[k]);
          }
        }
      });
    }
    const float inv = s.n > 0 ? 1.0f / (float)s.n : 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float m = s1[k] * inv;
      lds2[s.row * a.C + s.c0 + k] = float2{shift[k] + m, fmaf(-m, s1[k], s2[k])};
    }
  }
  __syncthreads();
  // the threads' means and deviations about the group's first: rows of a channel by several threads, then a wavefront per
  // group over its channels' parts
  __shared__ float2 sums[NORM_T];
  const int q = ch.pixels / rows, more = ch.pixels - q * rows;  // row r has q + (r < more) pixels
  const int parts = a.C < NORM_T ? NORM_T / a.C : 1, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  auto add = [&](int part, int c, float& s1, float& s2) __attribute__((always_inline)) {
    const float centre = lds2[c - c % a.D].x;
    for (int r = part; r < rows; r += parts) {
      const float n = (float)(q + (r < more));
      const float2 v = lds2[r * a.C + c];
      const float d = v.x - centre;
      s1 = fmaf(n, d, s1);
      s2 += fmaf(n * d, d, v.y);
    }
  };
  auto put = [&](int g, float s1, float s2) __attribute__((always_inline)) {
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    const float m = s1 / ((float)ch.pixels * (float)a.D);
    if (lane == 0)
      reinterpret_cast<float2*>(a.gpart)[(int64_t)block_of(a) * a.G + g] = float2{lds2[g * a.D].x + m, fmaf(-m, s1, s2)};
  };
  if (parts > 1) {
    const int part = threadIdx.x / a.C, c = threadIdx.x - part * a.C;
    float s1 = 0.0f, s2 = 0.0f;
    if (part < parts) add(part, c, s1, s2);
    sums[threadIdx.x] = float2{s1, s2};
    __syncthreads();
    for (int g = wave; g < a.G; g += NORM_T / 64) {
      s1 = s2 = 0.0f;
      for (int i = lane; i < parts * a.D; i += 64) {
        const int p = i / a.D;
        const float2 v = sums[p * a.C + g * a.D + (i - p * a.D)];
        s1 += v.x;
        s2 += v.y;
      }
      put(g, s1, s2);
    }
  } else {
    for (int g = wave; g < a.G; g += NORM_T / 64) {
      float s1 = 0.0f, s2 = 0.0f;
      for (int d = lane; d < a.D; d += 64) add(0, g * a.D + d, s1, s2);
      put(g, s1, s2);
    }
  }
}

// 1 / deviation from the means of a group's deviations and of their squares. A NaN variance, as infinite values leave, stays NaN
// (fmax would make it 0, and the group's finite values the activation of an infinity).
__device__ __forceinline__ float deviation_inverse(double s1, double s2, float eps) {
  const double var = s2 - s1 * s1;
  return (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)eps));
}

// A workgroup adds up its image's partials: thread t takes group t % G of every (threads / G)th chunk, all loads at once,
// about the first chunk's mean; then the threads of a group through LDS. to[g]: mean and 1 / deviation, or, BACKWARD, the
// group's means of dz * weight and dz * weight * xhat.
template <bool BACKWARD>
__device__ __forceinline__ void merge_groups(const NormArgs& a, int b, float2* to) {
  __shared__ double2 part[NORM_T];
  const float2* p = reinterpret_cast<const float2*>(a.gpart) + (int64_t)b * a.chunks * a.G;
  const int slices = NORM_T / a.G, slice = threadIdx.x / a.G, g = threadIdx.x - slice * a.G;
  const double total = (double)a.P * a.D;
  double s1 = 0.0, s2 = 0.0;
  const float centre = BACKWARD ? 0.0f : p[g].x;
  if (slice < slices) {
    for (int i = slice; i < a.chunks; i += slices) {
      const float2 v = p[(int64_t)i * a.G + g];
      if constexpr (BACKWARD) {
        s1 += v.x;
        s2 += v.y;
      } else {
        const double n = (double)pixels_of(a, i) * a.D, d = (double)v.x - centre;
        s1 += n * d;
        s2 += n * d * d + v.y;
      }
    }
  }
  part[threadIdx.x] = double2{s1, s2};
  __syncthreads();
  if ((int)threadIdx.x < a.G) {
    s1 = s2 = 0.0;
    for (int k = 0; k < slices; ++k) {
      const double2 v = part[k * a.G + g];
      s1 += v.x;
      s2 += v.y;
    }
    s1 /= total;
    s2 /= total;
    to[g] = BACKWARD ? float2{(float)s1, (float)s2}
                     : float2{(float)(centre + s1), deviation_inverse(s1, s2, a.eps)};
  }
  __syncthreads();
}

// Between the passes, where an image's partials are many: one wavefront per (image, group), a row of partials a lane
template <bool BACKWARD>
__global__ __launch_bounds__(256) void norm_merge_kernel(const NormArgs a) {
  const int64_t bg = (int64_t)block_of(a) * 4 + (threadIdx.x >> 6);
  if (bg >= (int64_t)a.B * a.G) return;
  const int64_t b = bg / a.G;
  const float2* p = reinterpret_cast<const float2*>(a.gpart) + b * a.chunks * a.G + (bg - b * a.G);
  const double total = (double)a.P * a.D;
  const float centre = BACKWARD ? 0.0f : p[0].x;
  double s1 = 0.0, s2 = 0.0;
  for (int i = threadIdx.x & 63; i < a.chunks; i += 64) {
    const float2 v = p[(int64_t)i * a.G];
    if constexpr (BACKWARD) {
      s1 += v.x;
      s2 += v.y;
    } else {
      const double n = (double)pixels_of(a, i) * a.D, d = (double)v.x - centre;
      s1 += n * d;
      s2 += n * d * d + v.y;
    }
  }
  s1 = wave_sum(s1) / total;
  s2 = wave_sum(s2) / total;
  if ((threadIdx.x & 63) == 0)
    reinterpret_cast<float2*>(BACKWARD ? a.coef : a.stats)[bg] =
        BACKWARD ? float2{(float)s1, (float)s2}
                 : float2{(float)(centre + s1), deviation_inverse(s1, s2, a.eps)};
}

// Forward, second pass.
template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T, 4) void norm_apply_kernel(const NormArgs a) {
  typedef Pack<DT, V> Pk;
  __shared__ float2 stat[NORM_MERGE_G];
  const Chunk ch = chunk_of(a);
  for (int pass = 0; pass < passes_of<V>(a); ++pass) {
    const Share s = share_of<V>(a, pass, ch.pixels);
    const bool any = s.live && s.n > 0;
    const Rows<DT, V, NORM_U> x(a.x, a.sb, a.sp, ch, s);
    typename Pk::Raw r[2][NORM_U];
    float mean[V], mul[V], add[V];
    if (any) {
      x.load(0, r[0]);
      params<V>(a.weight, a.wdt, s.c0, 1.0f, mul);
      params<V>(a.bias, a.bdt, s.c0, 0.0f, add);
    }
    if (pass == 0 && !a.merged) {
      merge_groups<false>(a, ch.b, stat);
      if (ch.i == 0 && (int)threadIdx.x < a.G)
        reinterpret_cast<float2*>(a.stats)[(int64_t)ch.b * a.G + threadIdx.x] = stat[threadIdx.x];
    }
    if (!any) continue;
    int g[V];
    groups_of<V>(s.c0, a.D, g);
    float2 st[V];
    if (a.merged) {
#pragma unroll
      for (int k = 0; k < V; ++k) st[k] = reinterpret_cast<const float2*>(a.stats)[(int64_t)ch.b * a.G + g[k]];
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) st[k] = stat[g[k]];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      mean[k] = st[k].x;
      mul[k] *= st[k].y;
    }
    uint8_t* out = a.out + (((int64_t)ch.b * a.P + ch.begin + s.row) * a.C + s.c0) * Pk::ES;
    const int64_t step = (int64_t)s.rows * a.C * Pk::ES;
    x.batches(r, [&](int i, const typename Pk::Raw(&now)[NORM_U]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < NORM_U; ++u) {
        if (i + u >= s.n) break;
        float v[V];
        Pk::unpack(now[u], v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = activate<ACT>(fmaf(v[k] - mean[k], mul[k], add[k]));
        Pk::template store<true>(out + (i + u) * step, v);
      }
    });
  }
}

// Small maps, forward: one workgroup per (image, group), whose values all stay in registers between the statistics and the
// output, up to NORM_OWN loads a thread. The mean first, then the deviations about it (and their sum, which takes out what the
// mean's rounding left).
template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T) void norm_group_kernel(const NormArgs a) {
  typedef Pack<DT, V> Pk;
  __shared__ float red[3][NORM_T / 64];
  const int b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
  const int cols = a.D / V, rows = NORM_T / cols, row = threadIdx.x / cols, col = threadIdx.x - row * cols;
  const int P = (int)a.P, c0 = g * a.D + col * V;
  const int n = row < rows && row < P ? (P - row + rows - 1) / rows : 0;
  typename Pk::Raw r[NORM_OWN];
  const uint8_t* x = a.x + (b * a.sb + (n > 0 ? row : 0) * a.sp + (n > 0 ? c0 : 0)) * Pk::ES;
  const int64_t step = rows * a.sp * Pk::ES;
#pragma unroll
  for (int i = 0; i < NORM_OWN; ++i) r[i] = Pk::load(x + (i < n ? i : 0) * step);
  float mul[V], add[V];
  params<V>(a.weight, a.wdt, n > 0 ? c0 : 0, 1.0f, mul);
  params<V>(a.bias, a.bdt, n > 0 ? c0 : 0, 0.0f, add);
  auto all = [&](float v, float (&to)[NORM_T / 64]) __attribute__((always_inline)) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) to[threadIdx.x >> 6] = v;
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NORM_T / 64; ++i) sum += to[i];
    return sum;
  };
  const float count = (float)((int64_t)P * a.D);
  float s0 = 0.0f;
#pragma unroll
  for (int i = 0; i < NORM_OWN; ++i) {
    float v[V], t = 0.0f;
    Pk::unpack(r[i], v);
#pragma unroll
    for (int k = 0; k < V; ++k) t += v[k];
    s0 += i < n ? t : 0.0f;
  }
  const float shift = all(s0, red[0]) / count;
  float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int i = 0; i < NORM_OWN; ++i) {
    float v[V], t = 0.0f, q = 0.0f;
    Pk::unpack(r[i], v);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = v[k] - shift;
      t += d;
      q = fmaf(d, d, q);
    }
    s1 += i < n ? t : 0.0f;
    s2 += i < n ? q : 0.0f;
  }
  s2 = all(s2, red[1]);
  const float off = all(s1, red[2]) / count, mean = shift + off;
  const float var = s2 / count - off * off, rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
  if (threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[blockIdx.x] = float2{mean, rstd};
#pragma unroll
  for (int k = 0; k < V; ++k) mul[k] *= rstd;
  uint8_t* out = a.out + (((int64_t)b * P + row) * a.C + c0) * Pk::ES;
  const int64_t out_step = (int64_t)rows * a.C * Pk::ES;
#pragma unroll
  for (int i = 0; i < NORM_OWN; ++i) {
    if (i >= n) break;
    float v[V];
    Pk::unpack(r[i], v);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = activate<ACT>(fmaf(v[k] - mean, mul[k], add[k]));
    Pk::store(out + i * out_step, v);
  }
}

// The per-channel values of a backward pass in registers: z = (x - mean) * mul + add, mul = rstd * weight
template <int V>
struct GradParams {
  float mean[V], mul[V], add[V];
  __device__ __forceinline__ GradParams(const NormArgs& a, int b, int c0) {
    int g[V];
    groups_of<V>(c0, a.D, g);
    float2 st[V];
#pragma unroll
    for (int k = 0; k < V; ++k) st[k] = reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.G + g[k]];
    params<V>(a.weight, a.wdt, c0, 1.0f, mul);
    params<V>(a.bias, a.bdt, c0, 0.0f, add);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      mean[k] = st[k].x;
      mul[k] *= st[k].y;
    }
  }
};

// Backward, first pass: per (chunk, channel) the sums of dz and dz * xhat, per (chunk, group) those times the weight.
template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T, 4) void norm_grad_sums_kernel(const NormArgs a) {
  typedef Pack<DT, V> Pk;
  extern __shared__ float2 lds2[];  // [rows][C]
  const Chunk ch = chunk_of(a);
  int rows = 1;
  for (int pass = 0; pass < passes_of<V>(a); ++pass) {
    const Share s = share_of<V>(a, pass, ch.pixels);
    rows = s.rows;
    if (!s.live) continue;
    float s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.0f;
    if (s.n > 0) {
      const Rows<DT, V, NORM_GRAD_U> x(a.x, a.sb, a.sp, ch, s), d(a.dy, a.db, a.dp, ch, s);
      typename Pk::Raw rx[2][NORM_GRAD_U], rd[2][NORM_GRAD_U];
      x.load(0, rx[0]);
      d.load(0, rd[0]);
      const GradParams<V> p(a, ch.b, s.c0);
      batches2<DT, V, NORM_GRAD_U>(x, d, rx, rd, [&](int i, const typename Pk::Raw(&nx)[NORM_GRAD_U], const typename Pk::Raw(&nd)[NORM_GRAD_U])
                      __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NORM_GRAD_U; ++u) {
          if (i + u >= s.n) break;
          float v[V], e[V];
          Pk::unpack(nx[u], v);
          Pk::unpack(nd[u], e);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float c = v[k] - p.mean[k];
            float slope;
            activate<ACT, true>(fmaf(c, p.mul[k], p.add[k]), slope);
            const float dz = e[k] * slope;
            s1[k] += dz;
            s2[k] = fmaf(dz, c, s2[k]);  // (times rstd at the end)
          }
        }
      });
    }
#pragma unroll
    for (int k = 0; k < V; ++k) lds2[s.row * a.C + s.c0 + k] = float2{s1[k], s2[k]};
  }
  __syncthreads();
  __shared__ float2 sums[NORM_T];
  const int parts = a.C < NORM_T ? NORM_T / a.C : 1;
  if (parts > 1) {  // rows of a channel by several threads
    const int part = threadIdx.x / a.C, c = threadIdx.x - part * a.C;
    float s1 = 0.0f, s2 = 0.0f;
    if (part < parts) {
      for (int r = part; r < rows; r += parts) {
        s1 += lds2[r * a.C + c].x;
        s2 += lds2[r * a.C + c].y;
      }
    }
    sums[threadIdx.x] = float2{s1, s2};
    __syncthreads();
  }
  for (int c = threadIdx.x; c < a.C; c += NORM_T) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int p = 0; p < parts; ++p) {
      const float2 v = parts > 1 ? sums[p * a.C + c] : lds2[c];  // (one row where there is one part)
      s1 += v.x;
      s2 += v.y;
    }
    for (int r = 1; parts == 1 && r < rows; ++r) {
      s1 += lds2[r * a.C + c].x;
      s2 += lds2[r * a.C + c].y;
    }
    s2 *= a.stats[2 * ((int64_t)ch.b * a.G + c / a.D) + 1];
    reinterpret_cast<float2*>(a.cpart)[(int64_t)block_of(a) * a.C + c] = float2{s1, s2};
    const float w = param(a.weight, a.wdt, c, 1.0f);
    lds2[c] = float2{s1 * w, s2 * w};
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < a.G; g += NORM_T / 64) {
    float t1 = 0.0f, t2 = 0.0f;
    for (int d = lane; d < a.D; d += 64) {
      t1 += lds2[g * a.D + d].x;
      t2 += lds2[g * a.D + d].y;
    }
    t1 = wave_sum(t1);
    t2 = wave_sum(t2);
    if (lane == 0) reinterpret_cast<float2*>(a.gpart)[(int64_t)block_of(a) * a.G + g] = float2{t1, t2};
  }
}

// Parameter gradients: 8 channels a workgroup, all chunks of all images in order
__device__ __forceinline__ void norm_grad_params(const NormArgs& a, int block) {
  __shared__ double red[NORM_T / 8][8][2];
  const int c = block * 8 + (threadIdx.x & 7), row = threadIdx.x >> 3;
  double s1 = 0.0, s2 = 0.0;
  if (c < a.C) {
    for (int64_t i = row; i < (int64_t)a.B * a.chunks; i += NORM_T / 8) {
      const float2 v = reinterpret_cast<const float2*>(a.cpart)[i * a.C + c];
      s1 += v.x;
      s2 += v.y;
    }
  }
  red[row][threadIdx.x & 7][0] = s1;
  red[row][threadIdx.x & 7][1] = s2;
  __syncthreads();
  if (threadIdx.x < 16) {
    const int k = threadIdx.x & 1, ch = threadIdx.x >> 1;
    double sum = 0.0;
    for (int r = 0; r < NORM_T / 8; ++r) sum += red[r][ch][k];
    if (block * 8 + ch < a.C) {
      if (k == 0 && a.dbias != nullptr) store_param(a.dbias, a.bdt, block * 8 + ch, (float)sum);
      if (k == 1 && a.dweight != nullptr) store_param(a.dweight, a.wdt, block * 8 + ch, (float)sum);
    }
  }
}

// Backward, second pass: dx; the workgroups past the chunks', the parameters' gradients.
template <int DT, int V, int ACT>
__global__ __launch_bounds__(NORM_T, 4) void norm_grad_apply_kernel(const NormArgs a) {
  typedef Pack<DT, V> Pk;
  __shared__ float2 coef[NORM_MERGE_G];
  if (block_of(a) >= a.B * a.chunks) {
    norm_grad_params(a, block_of(a) - a.B * a.chunks);
    return;
  }
  const Chunk ch = chunk_of(a);
  for (int pass = 0; pass < passes_of<V>(a); ++pass) {
    const Share s = share_of<V>(a, pass, ch.pixels);
    const bool any = s.live && s.n > 0;
    const Rows<DT, V, NORM_GRAD_U> x(a.x, a.sb, a.sp, ch, s), d(a.dy, a.db, a.dp, ch, s);
    if (pass == 0 && !a.merged) merge_groups<true>(a, ch.b, coef);
    if (!any) continue;
    typename Pk::Raw rx[2][NORM_GRAD_U], rd[2][NORM_GRAD_U];
    x.load(0, rx[0]);
    d.load(0, rd[0]);
    const GradParams<V> p(a, ch.b, s.c0);
    float k1[V], k2[V];  // dx = mul dz - ((x - mean) rstd^2 s2 + rstd s1)
    int g[V];
    groups_of<V>(s.c0, a.D, g);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float rstd = a.stats[2 * ((int64_t)ch.b * a.G + g[k]) + 1];
      const float2 v = a.merged ? reinterpret_cast<const float2*>(a.coef)[(int64_t)ch.b * a.G + g[k]] : coef[g[k]];
      k1[k] = rstd * v.x;
      k2[k] = rstd * rstd * v.y;
    }
    uint8_t* out = a.out + (((int64_t)ch.b * a.P + ch.begin + s.row) * a.C + s.c0) * Pk::ES;
    const int64_t step = (int64_t)s.rows * a.C * Pk::ES;
    batches2<DT, V, NORM_GRAD_U>(x, d, rx, rd, [&](int i, const typename Pk::Raw(&nx)[NORM_GRAD_U], const typename Pk::Raw(&nd)[NORM_GRAD_U])
                    __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < NORM_GRAD_U; ++u) {
        if (i + u >= s.n) break;
        float v[V], e[V];
        Pk::unpack(nx[u], v);
        Pk::unpack(nd[u], e);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float c = v[k] - p.mean[k];
          float slope;
          activate<ACT, true>(fmaf(c, p.mul[k], p.add[k]), slope);
          v[k] = e[k] * slope * p.mul[k] - fmaf(c, k2[k], k1[k]);  // (equal products of a single value cancel)
        }
        Pk::template store<true>(out + (i + u) * step, v);
      }
    });
  }
}

// -- launches ----------------------------------------------------------------------------------------------------------

// Chunks of an image: about two workgroups per CU over all images, each thread at least two pixels (8 channels a load)
static void norm_split(int64_t B, int64_t P, int64_t C, int& chunk, int& chunks) {
  const int64_t want = cdiv(2 * (int64_t)device_cus(), B > 0 ? B : 1);
  const int64_t rows = C >= 8 * NORM_T ? 1 : 8 * NORM_T / C;
  int64_t size = cdiv(P, want);
  if (size < rows * 2) size = rows * 2;
  if (size > P) size = P;
  if (size < 1) size = 1;
  chunk = (int)(size > INT32_MAX ? INT32_MAX : size);
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

// Elements per load of a workgroup per (image, group), or 0: not a small map, or more than a workgroup's
// registers hold
static int norm_own_vector(const NormArgs& a, int v, int es) {
  while (a.D % v) v /= 2;
  const int64_t cols = a.D / v;
  if (cols > NORM_T || cdiv(a.P, NORM_T / cols) > NORM_OWN) return 0;
  return (int64_t)a.B * a.P * a.C * es <= NORM_SMALL ? v : 0;
}

// One pass of `blocks` workgroups: launch(arguments, grid), several times where there are more than a launch takes (2^32
// threads; every image of a map has a workgroup at least)
template <typename F>
static void launch_pass(NormArgs a, int64_t blocks, F&& launch) {
  constexpr int64_t MOST = 1 << 22;
  for (int64_t first = 0; first < blocks; first += MOST) {
    a.first = (int)first;
    launch(a, dim3((unsigned)(blocks - first < MOST ? blocks - first : MOST)));
  }
}

template <bool BACKWARD>
static void launch_merge(const NormArgs& a, hipStream_t stream) {
  launch_pass(a, cdiv((int64_t)a.B * a.G, 4), [&](const NormArgs& p, dim3 grid) {
    norm_merge_kernel<BACKWARD><<<grid, dim3(256), 0, stream>>>(p);
  });
}

// Sizes and chunks; false: too many
static bool norm_shape(NormArgs& a, int64_t B, int64_t P, int64_t C, int64_t groups) {
  a.P = P;
  a.B = (int)B;
  a.C = (int)C;
  a.G = (int)groups;
  a.D = (int)(C / groups);
  norm_split(B, P, C, a.chunk, a.chunks);
  a.merged = a.G > NORM_MERGE_G || B * a.chunks * a.chunks * a.G > NORM_MERGE;
  return B * a.chunks + C <= INT32_MAX;
}

}  // namespace fim

using namespace fim;

extern "C" int fim_group_norm_workspace(int64_t B, int64_t P, int64_t C, int64_t groups, int backward, int64_t* floats) {
  if (floats == nullptr) return FIM_ERR_INVALID;
  const int rc = norm_check(FIM_F32, B, P, C, groups, FIM_F32, FIM_F32, 0);
  if (rc != FIM_OK) return rc;
  int chunk, chunks;
  norm_split(B, P, C, chunk, chunks);
  *floats = 2 * B * ((int64_t)chunks * groups + (backward ? chunks * C + groups : 0));
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
  a.x = static_cast<const uint8_t*>(x);
  a.out = static_cast<uint8_t*>(out);
  a.weight = weight;
  a.bias = bias;
  a.wdt = weight_dtype;
  a.bdt = bias_dtype;
  a.stats = stats;
  a.gpart = workspace;
  a.sb = stride_b;
  a.sp = stride_p;
  a.eps = eps;
  if (!norm_shape(a, B, P, C, groups)) return FIM_ERR_UNSUPPORTED;
  const int v = norm_vector(dtype, C, {stride_b, stride_p}, {x, out});
  if (const int own = norm_own_vector(a, v, elem_size(dtype))) {
    with_vector(dtype, own, [&](auto dt, auto vec) {
      with_activation(act, [&](auto act_c) {
        norm_group_kernel<decltype(dt)::value, decltype(vec)::value, decltype(act_c)::value>
            <<<dim3((unsigned)(B * groups)), dim3(NORM_T), 0, stream>>>(a);
      });
    });
    return launch_status();
  }
  with_vector(dtype, v, [&](auto dt, auto vec) {
    constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
    launch_pass(a, B * a.chunks, [&](const NormArgs& p, dim3 grid) {
      norm_stats_kernel<DT, V><<<grid, dim3(NORM_T), norm_lds(C, V), stream>>>(p);
    });
    if (a.merged) launch_merge<false>(a, stream);
    with_activation(act, [&](auto act_c) {
      launch_pass(a, B * a.chunks, [&](const NormArgs& p, dim3 grid) {
        norm_apply_kernel<DT, V, decltype(act_c)::value><<<grid, dim3(NORM_T), 0, stream>>>(p);
      });
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
  a.x = static_cast<const uint8_t*>(x);
  a.dy = static_cast<const uint8_t*>(d_out);
  a.out = static_cast<uint8_t*>(dx);
  a.weight = weight;
  a.bias = bias;
  a.wdt = weight_dtype;
  a.bdt = bias_dtype;
  a.stats = const_cast<float*>(stats);
  a.dweight = d_weight;
  a.dbias = d_bias;
  a.sb = stride_b;
  a.sp = stride_p;
  a.db = d_stride_b;
  a.dp = d_stride_p;
  if (!norm_shape(a, B, P, C, groups)) return FIM_ERR_UNSUPPORTED;
  a.gpart = workspace;
  a.cpart = a.gpart + 2 * B * a.chunks * groups;
  a.coef = a.cpart + 2 * B * a.chunks * C;
  const int v = norm_vector(dtype, C, {stride_b, stride_p, d_stride_b, d_stride_p}, {x, d_out, dx});
  const int64_t chunks = B * a.chunks, params = d_weight != nullptr || d_bias != nullptr ? cdiv(C, 8) : 0;
  with_vector(dtype, v, [&](auto dt, auto vec) {
    constexpr int DT = decltype(dt)::value, V = decltype(vec)::value;
    with_activation(act, [&](auto act_c) {
      constexpr int ACT = decltype(act_c)::value;
      launch_pass(a, chunks, [&](const NormArgs& p, dim3 grid) {
        norm_grad_sums_kernel<DT, V, ACT><<<grid, dim3(NORM_T), norm_lds(C, V), stream>>>(p);
      });
      if (a.merged) launch_merge<true>(a, stream);
      launch_pass(a, chunks + params, [&](const NormArgs& p, dim3 grid) {
        norm_grad_apply_kernel<DT, V, ACT><<<grid, dim3(NORM_T), 0, stream>>>(p);
      });
    });
  });
  return launch_status();
}
