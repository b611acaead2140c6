// The global norm of many tensors (gradients), and scaling them to at most a given norm.
//
//   total = sqrt(sum over all elements of g^2), or max |g|;   out = g * min(1, max_norm / (total + 1e-6))
//
// A stream: every gradient is read for the norm, then read again and written, in place or elsewhere (the floor is one read
// and one write; the second read comes from the Infinity Cache for gradients of up to about its 256 MB). Tensors are
// handed over in kernel arguments, up to 168 or 248 a launch (no table to upload, capturable); a workgroup finds its
// tensor among their first workgroups and takes one run of its elements.
//
// Squares are summed in 64 bits: FP32 gradients above 1.8e19 would overflow in 32, and the conversions and FMAs hide behind
// the loads. Each workgroup writes one partial; every workgroup of the second launch adds them all up in the same order
// (at most 2048 of them: a few kilobytes from the L2, less than another launch; beyond that a launch of its own does), so
// results do not depend on the order of workgroups.
//
// Scaling takes the gradients from the last one back, whose lines the norm's pass left in the Infinity Cache, and from 128 MB
// marks its loads and stores as streams, which leave those lines there: 200 million BF16 gradients into FP32 ones, both launches,
// 355 us forward and plain, 345 with the marked stores alone, 355 backward alone, 320 with both, 316 with marked loads too (and
// with an optimizer's read of the outputs after it 799 -> 741 us); 320 FP32 tensors (181 MB) 69 -> 61 us. Smaller gradients fit
// the cache and gain nothing; marked stores to unaligned lines cost them (4 million BF16: 5.8 -> 9.5 us).
//
// Measured (MI355X): 200 million BF16 gradients into FP32 ones, norm 69 us and scaling 235 us (5.1 TB/s, a copy's rate; 310 us
// where a lane wrote 32 bytes in two stores instead of 16 in one). 320 FP32 tensors of 22.6 million elements: 19 + 4 us, 6 us
// for the total, 6 + 27 us, as long as the host takes for 640 tensors. Ten tensors of 35000 elements: 4 + 4 us.
#include <type_traits>

#include "common.h"

namespace fim {

constexpr int CLIP_T = 256;
constexpr int CLIP_PARTIALS = 2048;   // partials that every workgroup of the scaling launch adds up itself
constexpr int64_t CLIP_STREAM = 128 << 20;  // bytes of gradients and outputs from which scaling streams: half the Infinity Cache
constexpr int64_t CLIP_ENTRY = 1 << 30;  // elements of one table entry: 32-bit indexing inside it

template <int N, bool OUT>
struct ClipTable {
  static constexpr int ENTRIES = N;
  static constexpr bool OUTPUTS = OUT;
  const void* in[N];
  void* out[OUT ? N : 1];
  uint32_t n[N];      // elements
  uint32_t first[N];  // first workgroup
  uint32_t entries, chunk;
};
typedef ClipTable<248, false> NormTable;
typedef ClipTable<168, true> ScaleTable;
static_assert(sizeof(NormTable) <= 4000 && sizeof(ScaleTable) <= 4000 + 56, "kernel arguments");

// The entry whose workgroups hold wg: the entries that start at or before it, counted by the wavefront's lanes (one load
// latency; a bisection's dependent loads took eight)
template <typename Table>
__device__ __forceinline__ int entry_of(const Table& t, uint32_t wg) {
  const uint32_t lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (uint32_t i = 0; i < Table::ENTRIES; i += 64) {
    const uint32_t at = i + lane < Table::ENTRIES ? i + lane : Table::ENTRIES - 1;
    n += __popcll(__builtin_amdgcn_ballot_w64(i + lane < t.entries && t.first[at] <= wg));
  }
  return n - 1;
}

// A load of 16 bytes, or of the 8 bytes that become 16 as FP32
template <int DT, bool HALF = false>
struct Vec {
  static constexpr int WORDS = HALF ? 2 : 4, N = DT == FIM_F32 ? WORDS : 2 * WORDS;
  typedef uint32_t T __attribute__((ext_vector_type(WORDS)));
  static __device__ __forceinline__ void unpack(const T& w, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (DT == FIM_F32) {
        f[i] = u2f(w[i]);
      } else if constexpr (DT == FIM_BF16) {
        f[2 * i] = u2f(w[i] << 16);
        f[2 * i + 1] = u2f(w[i] & 0xffff0000u);
      } else {
        f[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
};

struct SumSquares {
  typedef double Acc;
  static __device__ __forceinline__ double zero() { return 0.0; }
  static __device__ __forceinline__ double add(double a, float v) { return fma((double)v, (double)v, a); }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
  static __device__ __forceinline__ float total(double a) { return (float)sqrt(a); }
};
struct MaxAbs {
  typedef double Acc;  // (partials share the sums' layout)
  static __device__ __forceinline__ double zero() { return 0.0; }
  static __device__ __forceinline__ double add(double a, float v) {
    return (double)__builtin_elementwise_maximum((float)a, fabsf(v));  // NaN stays NaN
  }
  static __device__ __forceinline__ double join(double a, double b) { return add(a, (float)b); }
  static __device__ __forceinline__ float total(double a) { return (float)a; }
};

template <typename R>
__device__ __forceinline__ double join_workgroup(double v) {
  __shared__ double red[CLIP_T / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = R::join(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < CLIP_T / 64; ++i) v = R::join(v, red[i]);
  return v;
}

template <int DT, typename R>
__global__ __launch_bounds__(CLIP_T) void grad_norm_kernel(const NormTable t, double* __restrict__ part) {
  constexpr int ES = DT == FIM_F32 ? 4 : 2, N = Vec<DT>::N, U = 4;
  typedef typename Vec<DT>::T V;
  const int e = entry_of(t, blockIdx.x);
  const uint32_t begin = (blockIdx.x - t.first[e]) * t.chunk;
  const uint32_t n = t.n[e] - begin < t.chunk ? t.n[e] - begin : t.chunk;
  const uint8_t* p = static_cast<const uint8_t*>(t.in[e]) + (int64_t)begin * ES;
  // elements before the first 16-byte boundary, whole 16-byte vectors, the rest
  uint32_t head = (uint32_t)(-(intptr_t)p & 15) / ES;
  if (head > n) head = n;
  const uint32_t vecs = (n - head) / N;
  const V* v = reinterpret_cast<const V*>(p + head * ES);
  double acc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) acc[u] = R::zero();
  uint32_t i = threadIdx.x;
  for (; i + (U - 1) * CLIP_T < vecs; i += U * CLIP_T) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = v[i + u * CLIP_T];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[N];
      Vec<DT>::unpack(r[u], f);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[u] = R::add(acc[u], f[k]);
    }
  }
  for (; i < vecs; i += CLIP_T) {
    float f[N];
    Vec<DT>::unpack(v[i], f);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[0] = R::add(acc[0], f[k]);
  }
  if (threadIdx.x < head) acc[1] = R::add(acc[1], load_elem<DT>(p, threadIdx.x));
  const uint32_t tail = head + vecs * N + threadIdx.x;
  if (tail < n) acc[2] = R::add(acc[2], load_elem<DT>(p, tail));
  const double sum = join_workgroup<R>(R::join(R::join(acc[0], acc[1]), R::join(acc[2], acc[3])));
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

template <typename R>
__device__ __forceinline__ float total_of(const double* __restrict__ part, int parts) {
  double v = R::zero();
  for (int i = threadIdx.x; i < parts; i += CLIP_T) v = R::join(v, part[i]);
  return R::total(join_workgroup<R>(v));
}

template <typename R>
__global__ __launch_bounds__(CLIP_T) void grad_total_kernel(const double* __restrict__ part, int parts, float* total) {
  const float v = total_of<R>(part, parts);
  if (threadIdx.x == 0) *total = v;
}

__device__ __forceinline__ void store_elem(void* p, int64_t i, float v, int dt) {
  if (dt == FIM_F32) static_cast<float*>(p)[i] = v;
  else if (dt == FIM_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)(pack_bf16x2(v, 0.0f) & 0xffff);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// DO: the outputs' type. STREAM: loads and stores marked as not read again soon.
// parts > 0: the total is added up here, and workgroup 0 writes it; else it is read.
template <int DT, int DO, typename R, bool STREAM>
__global__ __launch_bounds__(CLIP_T) void grad_scale_kernel(const ScaleTable t, const double* __restrict__ part, int parts,
                                                            float* total, float max_norm, int writes_total) {
  constexpr bool HALF = DT != FIM_F32 && DO == FIM_F32;
  typedef Vec<DT, HALF> In;
  typedef typename In::T V;
  constexpr int ES = DT == FIM_F32 ? 4 : 2, N = In::N, EO = DO == FIM_F32 ? 4 : 2, U = HALF ? 8 : 4;
  const float sum = parts > 0 ? total_of<R>(part, parts) : *total;
  if (parts > 0 && writes_total && blockIdx.x == 0 && threadIdx.x == 0) *total = sum;
  const float quotient = max_norm / (sum + 1e-6f);
  const float scale = __builtin_elementwise_minimum(quotient, 1.0f);  // NaN stays NaN
  const int e = entry_of(t, blockIdx.x);
  if (scale == 1.0f && t.out[e] == t.in[e] && DT == DO) return;  // in place, unclipped: nothing changes
  // runs from the last one: what the norm's pass read last is still in the Infinity Cache
  const uint32_t last = (e + 1 < (int)t.entries ? t.first[e + 1] : gridDim.x) - 1;
  const uint32_t begin = (last - blockIdx.x) * t.chunk;
  const uint32_t n = t.n[e] - begin < t.chunk ? t.n[e] - begin : t.chunk;
  const uint8_t* p = static_cast<const uint8_t*>(t.in[e]) + (int64_t)begin * ES;
  uint8_t* q = static_cast<uint8_t*>(t.out[e]) + (int64_t)begin * EO;
  uint32_t head = (uint32_t)(-(intptr_t)p & (sizeof(V) - 1)) / ES;
  if (head > n) head = n;
  uint32_t vecs = (n - head) / N;
  constexpr int WB = N * EO;  // bytes of a store: 16, or 8 of FP32 into 16 bits
  if ((reinterpret_cast<uintptr_t>(q) + head * EO) % WB) head = vecs = 0;  // unlike alignments: element by element
  const V* v = reinterpret_cast<const V*>(p + head * ES);
  auto put = [&](uint32_t at, const V& r) __attribute__((always_inline)) {
    float f[N];
    In::unpack(r, f);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] *= scale;
    typedef uint32_t Out __attribute__((ext_vector_type(N * EO / 4)));
    Out w;
    if constexpr (DO == FIM_F32) {
#pragma unroll
      for (int k = 0; k < N; ++k) w[k] = f2u(f[k]);
    } else {
#pragma unroll
      for (int k = 0; k < N / 2; ++k)
        w[k] = DO == FIM_BF16 ? pack_bf16x2(f[2 * k], f[2 * k + 1])
                              : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * k]) |
                                    (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * k + 1]) << 16;
    }
    Out* to = reinterpret_cast<Out*>(q + (int64_t)(head + at * N) * EO);
    if constexpr (STREAM) __builtin_nontemporal_store(w, to);
    else *to = w;
  };
  uint32_t i = threadIdx.x;
  for (; i + (U - 1) * CLIP_T < vecs; i += U * CLIP_T) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = STREAM ? __builtin_nontemporal_load(v + i + u * CLIP_T) : v[i + u * CLIP_T];
#pragma unroll
    for (int u = 0; u < U; ++u) put(i + u * CLIP_T, r[u]);
  }
  for (; i < vecs; i += CLIP_T) put(i, v[i]);
  for (uint32_t k = threadIdx.x; k < n - vecs * N; k += CLIP_T) {
    const uint32_t at = k < head ? k : k + vecs * N;
    store_elem(q, at, load_elem<DT>(p, at) * scale, DO);
  }
}

// Elements of a workgroup: about sixteen workgroups per CU over all tensors, in steps of 2048.
static uint32_t clip_chunk(int64_t elements) {
  const int64_t c = cdiv(cdiv(elements, 16 * (int64_t)device_cus()), 2048) * 2048;
  return (uint32_t)(c < 2048 ? 2048 : c > CLIP_ENTRY ? CLIP_ENTRY : c);
}

struct Grads {
  int64_t count;
  const void* const* in;
  void* const* out;  // null: no outputs
  const int* in_dtype;
  const int* out_dtype;
  const int64_t* numel;
};

static bool clip_dtype(int dt) { return dt == FIM_F32 || dt == FIM_BF16 || dt == FIM_F16; }
static int clip_size(int dt) { return dt == FIM_F32 ? 4 : 2; }

static int clip_check(const Grads& g, int norm) {
  if (g.count < 0 || (norm != 0 && norm != 2)) return FIM_ERR_INVALID;
  if (g.count > 0 && (g.in == nullptr || g.in_dtype == nullptr || g.numel == nullptr)) return FIM_ERR_INVALID;
  for (int64_t i = 0; i < g.count; ++i) {
    if (!clip_dtype(g.in_dtype[i]) || g.numel[i] < 0) return FIM_ERR_INVALID;
    if (g.out != nullptr && !clip_dtype(g.out_dtype[i])) return FIM_ERR_INVALID;
    if (g.numel[i] == 0) continue;
    if (g.in[i] == nullptr || reinterpret_cast<uintptr_t>(g.in[i]) % clip_size(g.in_dtype[i])) return FIM_ERR_INVALID;
    if (g.out != nullptr &&
        (g.out[i] == nullptr || reinterpret_cast<uintptr_t>(g.out[i]) % clip_size(g.out_dtype[i])))
      return FIM_ERR_INVALID;
  }
  return FIM_OK;
}

static int64_t clip_total(const Grads& g) {
  int64_t n = 0;
  for (int64_t i = 0; i < g.count; ++i) n += g.numel[i];
  return n;
}

// Workgroups over all tensors, one partial each
static int64_t clip_parts(const Grads& g, uint32_t chunk) {
  int64_t parts = 0;
  for (int64_t i = 0; i < g.count; ++i) {
    for (int64_t at = 0; at < g.numel[i]; at += CLIP_ENTRY)
      parts += cdiv(g.numel[i] - at < CLIP_ENTRY ? g.numel[i] - at : CLIP_ENTRY, chunk);
  }
  return parts;
}

// launch(table, workgroups) over the tensors of types (in, out), a table at a time; those with outputs from the last one
template <typename Table, typename Launch>
static void for_tables(const Grads& g, int in_dtype, int out_dtype, uint32_t chunk, Launch&& launch) {
  Table t;
  t.entries = 0;
  t.chunk = chunk;
  uint32_t wgs = 0;
  auto flush = [&]() {
    if (t.entries > 0) launch(t, wgs);
    t.entries = 0;
    wgs = 0;
  };
  for (int64_t j = 0; j < g.count; ++j) {
    const int64_t i = Table::OUTPUTS ? g.count - 1 - j : j;
    if (g.in_dtype[i] != in_dtype || (Table::OUTPUTS && g.out_dtype[i] != out_dtype)) continue;
    for (int64_t at = 0; at < g.numel[i]; at += CLIP_ENTRY) {
      const uint32_t n = (uint32_t)(g.numel[i] - at < CLIP_ENTRY ? g.numel[i] - at : CLIP_ENTRY);
      t.in[t.entries] = static_cast<const uint8_t*>(g.in[i]) + at * clip_size(in_dtype);
      if constexpr (Table::OUTPUTS) t.out[t.entries] = static_cast<uint8_t*>(g.out[i]) + at * clip_size(out_dtype);
      t.n[t.entries] = n;
      t.first[t.entries] = wgs;
      wgs += (uint32_t)cdiv(n, chunk);
      if (++t.entries == Table::ENTRIES) flush();
    }
  }
  flush();
}

template <typename R>
static void launch_norm(const Grads& g, uint32_t chunk, double* part, hipStream_t stream) {
  auto of_type = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    for_tables<NormTable>(g, DT, 0, chunk, [&](const NormTable& t, uint32_t wgs) {
      grad_norm_kernel<DT, R><<<dim3(wgs), dim3(CLIP_T), 0, stream>>>(t, part);
      part += wgs;
    });
  };
  of_type(std::integral_constant<int, FIM_F32>{});
  of_type(std::integral_constant<int, FIM_BF16>{});
  of_type(std::integral_constant<int, FIM_F16>{});
}

template <typename R>
static void launch_scale(const Grads& g, uint32_t chunk, const double* part, int parts, float* total, float max_norm,
                         hipStream_t stream) {
  int writes = 1;
  int64_t bytes = 0;
  for (int64_t i = 0; i < g.count; ++i) bytes += g.numel[i] * (clip_size(g.in_dtype[i]) + clip_size(g.out_dtype[i]));
  const bool streams = bytes >= CLIP_STREAM;
  auto of_types = [&](auto dt, auto dout) {
    constexpr int DT = decltype(dt)::value, DO = decltype(dout)::value;
    for_tables<ScaleTable>(g, DT, DO, chunk, [&](const ScaleTable& t, uint32_t wgs) {
      const auto kernel = streams ? grad_scale_kernel<DT, DO, R, true> : grad_scale_kernel<DT, DO, R, false>;
      kernel<<<dim3(wgs), dim3(CLIP_T), 0, stream>>>(t, part, parts, total, max_norm, writes);
      writes = 0;
    });
  };
  auto of_type = [&](auto dt) {
    of_types(dt, std::integral_constant<int, FIM_F32>{});
    of_types(dt, std::integral_constant<int, FIM_BF16>{});
    of_types(dt, std::integral_constant<int, FIM_F16>{});
  };
  of_type(std::integral_constant<int, FIM_F32>{});
  of_type(std::integral_constant<int, FIM_BF16>{});
  of_type(std::integral_constant<int, FIM_F16>{});
}

template <typename R>
static void launch_clip(const Grads& g, double* part, float* total, float max_norm, hipStream_t stream) {
  const int64_t n = clip_total(g);
  const uint32_t chunk = clip_chunk(n);
  const int parts = (int)clip_parts(g, chunk);
  launch_norm<R>(g, chunk, part, stream);
  const bool merged = g.out == nullptr || parts == 0 || parts > CLIP_PARTIALS;
  if (merged) grad_total_kernel<R><<<dim3(1), dim3(CLIP_T), 0, stream>>>(part, parts, total);
  if (g.out != nullptr) launch_scale<R>(g, chunk, part, merged ? 0 : parts, total, max_norm, stream);
}

static int clip_run(const Grads& g, float max_norm, int norm, float* total, double* workspace, hipStream_t stream) {
  const int rc = clip_check(g, norm);
  if (rc != FIM_OK) return rc;
  if (total == nullptr || (clip_total(g) > 0 && workspace == nullptr)) return FIM_ERR_INVALID;
  if (clip_parts(g, clip_chunk(clip_total(g))) > INT32_MAX) return FIM_ERR_UNSUPPORTED;
  if (norm == 2) launch_clip<SumSquares>(g, workspace, total, max_norm, stream);
  else launch_clip<MaxAbs>(g, workspace, total, max_norm, stream);
  return launch_status();
}

}  // namespace fim

using namespace fim;

extern "C" int fim_grad_norm_workspace(int64_t count, const int64_t* numel, int64_t* doubles) {
  if (count < 0 || (count > 0 && numel == nullptr) || doubles == nullptr) return FIM_ERR_INVALID;
  for (int64_t i = 0; i < count; ++i)
    if (numel[i] < 0) return FIM_ERR_INVALID;
  const Grads g{count, nullptr, nullptr, nullptr, nullptr, numel};
  *doubles = clip_parts(g, clip_chunk(clip_total(g)));
  return FIM_OK;
}

extern "C" int fim_grad_norm(int64_t count, const void* const* grads, const int* dtypes, const int64_t* numel, int norm,
                             float* total, double* workspace, hipStream_t stream) {
  return clip_run(Grads{count, grads, nullptr, dtypes, nullptr, numel}, 0.0f, norm, total, workspace, stream);
}

extern "C" int fim_clip_grad_norm(int64_t count, const void* const* grads, const int* dtypes, void* const* out,
                                  const int* out_dtypes, const int64_t* numel, float max_norm, int norm, float* total,
                                  double* workspace, hipStream_t stream) {
  if (count > 0 && (out == nullptr || out_dtypes == nullptr)) return FIM_ERR_INVALID;
  return clip_run(Grads{count, grads, out, dtypes, out_dtypes, numel}, max_norm, norm, total, workspace, stream);
}
