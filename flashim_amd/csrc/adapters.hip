// Low-rank adapters of many requests beside a shared projection: out = base + s_j (x A_j^T) B_j^T, j by row or by leading entry,
// and the gradients of x, A and B (formulas and layouts: adapters_rows.h, adapters_grad.h).
#include <type_traits>

#include "adapters_grad.h"
#include "adapters_narrow.h"
#include "adapters_rows.h"
#include "gated_plan.h"

namespace fim {

constexpr int ADAPTER_RANK = 128;

static int adapter_blocks(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }  // of 16 ranks, as compiled

struct AdapterSizes {
  int64_t M, K, N, J, R, entries;
};

static int adapter_check(const AdapterSizes& s, int dtype, int wide) {
  if (s.M < 0 || s.K < 1 || s.N < 1 || s.J < 1 || s.R < 1 || s.entries < 0 || (wide != 0 && wide != 1)) return FIM_ERR_INVALID;
  if (s.M > 0 && (s.entries < 1 || s.M % s.entries != 0)) return FIM_ERR_INVALID;
  if (dtype != FIM_BF16 && dtype != FIM_F16) return dtype == FIM_F32 ? FIM_ERR_UNSUPPORTED : FIM_ERR_INVALID;
  constexpr int64_t most = int64_t{1} << 31;  // (rows: 16 a workgroup, whose threads a launch counts in 32 bits)
  if (s.R > ADAPTER_RANK || s.M >= most / 8 || s.K >= 1 << 24 || s.N >= 1 << 24 || s.J >= 1 << 20 || s.J * s.R >= most ||
      s.J * (s.K + s.N) >= most)
    return FIM_ERR_UNSUPPORTED;
  return FIM_OK;
}

// Forms by size. One row a workgroup where entries are single rows and few: their adapters differ, and a tile of rows would go
// through them one after the other (512 rows of 512 -> 2048, each with one of 64 adapters: 12 us, 513 on tiles 50; of one adapter
// 11 either way). Else tiles, four wavefronts each until rows fill the CUs, and beyond that where all four have
// a part of either product (40000 x 512 -> 2048 at rank 16: 115 -> 92 us); narrow maps a wavefront a tile, which exchange nothing
// (320000 x 64 -> 256 77 us, 106 with four). A tile of two sets of 16 rows halves the reads of A_j and B_j from the caches, once
// there are enough: 512 -> 2048, 16384 rows of ranks 32, 64, 128: 30, 40 and 64 us, of one set 45, 52 and 113; 4096 rows 15, 21,
// 35 and 18, 19, 41. At rank 16 it gains where a wavefront has the tile (320000 x 64 -> 256: 92 -> 84 us; 40000 x 512 -> 2048: 94
// -> 97).
template <int DT, int NR>
static void launch_rows(AdapterArgs& p, hipStream_t stream) {
  const int64_t cus = device_cus(), blocks = cdiv(p.N, 32);
  const bool one = p.index.per < 16 && p.M <= 512;
  const bool four = one || p.M < 128 * cus || (blocks >= 16 && p.K >= 128);
  const bool two = !one && (NR == 1 ? !four : p.M >= (NR == 4 ? 64 : 8) * cus);
  const int64_t tiles = one ? p.M : cdiv(p.M, two ? 32 : 16);
  // parts of the columns: enough wavefronts for the card, each with four blocks at least
  int64_t parts = cdiv(8 * cus, tiles * (four ? 4 : 1));
  const int64_t most = cdiv(blocks, four ? 16 : 4);
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  p.parts = (int)(four ? 4 * parts : parts);
  const dim3 grid((unsigned)(four ? tiles : cdiv(tiles, 4)), (unsigned)parts);
  auto launch = [&](auto quads) {
    constexpr bool Q = decltype(quads)::value;
    if (one) adapter_rows_kernel<DT, NR, 4, 0, Q><<<grid, dim3(256), 0, stream>>>(p);
    else if (four && two) adapter_rows_kernel<DT, NR, 4, 2, Q><<<grid, dim3(256), 0, stream>>>(p);
    else if (four) adapter_rows_kernel<DT, NR, 4, 1, Q><<<grid, dim3(256), 0, stream>>>(p);
    else adapter_rows_kernel<DT, NR, 1, 2, Q><<<grid, dim3(256), 0, stream>>>(p);  // (so many rows are always two sets)
  };
  if (p.R % (NR == 1 ? 4 : 8) == 0) launch(std::integral_constant<bool, true>{});
  else launch(std::integral_constant<bool, false>{});
}

template <typename F>
static void by_type(int dtype, int64_t R, F&& f) {
  auto ranks = [&](auto dt) {
    switch (adapter_blocks(R)) {
      case 1: return f(dt, std::integral_constant<int, 1>{});
      case 2: return f(dt, std::integral_constant<int, 2>{});
      case 4: return f(dt, std::integral_constant<int, 4>{});
      default: return f(dt, std::integral_constant<int, 8>{});
    }
  };
  if (dtype == FIM_BF16) ranks(std::integral_constant<int, FIM_BF16>{});
  else ranks(std::integral_constant<int, FIM_F16>{});
}

static void adapter_rows(AdapterArgs& p, int dtype, hipStream_t stream) {
  by_type(dtype, p.R, [&](auto dt, auto nr) { launch_rows<decltype(dt)::value, decltype(nr)::value>(p, stream); });
}

struct AdapterGradPlan {
  int64_t chunk, chunks, at, bt, t, part, counts, bytes;
  int xt, ct;
  bool narrow;
};

// Whether the backward pass is one pass over x and d_out
static bool adapter_narrow(int64_t K, int64_t N, int64_t R) {
  return R <= 32 && cdiv(K, 32) * 32 + cdiv(N, 32) * 32 <= NARROW_WIDTH;
}

constexpr int64_t GRAD_GRID = 1 << 24;  // workgroups of 256 threads, which a launch counts in 32 bits: fewer

static AdapterGradPlan grad_plan(const AdapterSizes& s) {
  AdapterGradPlan g;
  g.xt = (int)cdiv(s.K, GRAD_COLS);
  g.ct = g.xt + (int)cdiv(s.N, GRAD_COLS);
  g.narrow = adapter_narrow(s.K, s.N, s.R);
  // workgroups for the card where a chunk's rows have one adapter (narrow: two a CU), lists no longer than their room if the partial
  // sums of all adapters are 256 MB or less then; else fewer and longer chunks (lists in pieces)
  int64_t chunks = g.narrow ? 2 * (int64_t)device_cus() : cdiv(4 * (int64_t)device_cus(), g.ct);
  const int64_t step = g.narrow ? NARROW_ROWS : 256, longest = g.narrow ? NARROW_CHUNK : GRAD_CHUNK;
  const int64_t most = (int64_t{256} << 20) / (s.J * s.R * (s.K + s.N) * 4), fits = cdiv(s.M, longest);
  if (chunks < fits) chunks = fits;
  const int64_t grid = (GRAD_GRID - 1) / ((s.J + 1) * (g.narrow ? 1 : g.ct));
  if (chunks > most) chunks = most;
  if (chunks > grid) chunks = grid;
  if (chunks < 1) chunks = 1;
  g.chunk = cdiv(cdiv(s.M, chunks), step) * step;
  if (g.chunk < 256) g.chunk = 256;  // (a workgroup's weights cost as much)
  if (g.chunk > longest) g.chunk = cdiv(g.chunk, longest) * longest;
  g.chunks = cdiv(s.M, g.chunk);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += align256(bytes);
    return from;
  };
  g.at = take(g.narrow ? 0 : s.J * s.R * s.K * 2);
  g.bt = take(g.narrow ? 0 : s.J * s.R * s.N * 2);
  g.t = take(g.narrow ? 0 : s.M * 16 * adapter_blocks(s.R) * 4);
  g.part = take(g.chunks > 1 ? s.J * g.chunks * s.R * (s.K + s.N) * 4 : 0);
  g.counts = take(g.chunks > 1 ? s.J * g.chunks * 4 : 0);
  g.bytes = at;
  return g;
}

// What one launch of the backward pass cannot hold
static int grad_check(const AdapterSizes& s, const AdapterGradPlan& g) {
  const bool no = s.J * s.R * (s.K + s.N) >= int64_t{1} << 32 || s.R * (s.K + s.N) >= int64_t{1} << 30 ||
                  (s.J + 1) * g.chunks * (g.narrow ? 1 : g.ct) >= GRAD_GRID;
  return no ? FIM_ERR_UNSUPPORTED : FIM_OK;
}

}  // namespace fim

using namespace fim;

extern "C" int fim_low_rank_adapters(const void* base, int64_t base_stride, const void* x, int64_t x_stride, int dtype, int64_t M,
                                     int64_t K, int64_t N, const void* a, const void* b, int64_t J, int64_t R,
                                     const void* index, int index_wide, int64_t entries, const float* scales, float scale,
                                     void* out, float* h, hipStream_t stream) {
  const AdapterSizes s{M, K, N, J, R, entries};
  const int rc = adapter_check(s, dtype, index_wide);
  if (rc != FIM_OK) return rc;
  if (M == 0) return FIM_OK;
  if (x == nullptr || a == nullptr || b == nullptr || index == nullptr || out == nullptr) return FIM_ERR_INVALID;
  for (const void* t : {base, x, a, b, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(t) % 2) return FIM_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(index) % (index_wide ? 8 : 4) || reinterpret_cast<uintptr_t>(h) % 16) return FIM_ERR_INVALID;
  AdapterArgs p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(base), static_cast<const uint16_t*>(a),
                static_cast<const uint16_t*>(b), x_stride, base_stride, static_cast<uint16_t*>(out),
                adapter_narrow(K, N, R) ? nullptr : h,  // (no columns are saved)
                AdapterIndex{index, index_wide, (uint32_t)(M / entries), (int)J}, scales, scale, (uint32_t)M, (int)K, (int)N,
                (int)R, 1};
  adapter_rows(p, dtype, stream);
  return launch_status();
}

extern "C" int fim_low_rank_adapters_saved(int64_t K, int64_t N, int64_t R, int64_t* columns) {
  if (K < 1 || N < 1 || R < 1 || columns == nullptr) return FIM_ERR_INVALID;
  if (R > ADAPTER_RANK || K >= 1 << 24 || N >= 1 << 24) return FIM_ERR_UNSUPPORTED;
  *columns = adapter_narrow(K, N, R) ? 0 : 16 * adapter_blocks(R);
  return FIM_OK;
}

extern "C" int fim_low_rank_adapters_backward_workspace(int64_t M, int64_t K, int64_t N, int64_t J, int64_t R, int64_t* bytes) {
  if (bytes == nullptr) return FIM_ERR_INVALID;
  const AdapterSizes s{M, K, N, J, R, M};
  const int rc = adapter_check(s, FIM_BF16, 0);
  if (rc != FIM_OK) return rc;
  *bytes = 0;
  if (M == 0) return FIM_OK;
  const AdapterGradPlan g = grad_plan(s);
  *bytes = g.bytes;
  return grad_check(s, g);
}

extern "C" int fim_low_rank_adapters_backward(const void* d_out, int64_t d_out_stride, const void* x, int64_t x_stride, int dtype,
                                              int64_t M, int64_t K, int64_t N, const void* a, const void* b, int64_t J, int64_t R,
                                              const void* index, int index_wide, int64_t entries, const float* scales, float scale,
                                              const float* h, void* dx, void* da, void* db, void* workspace,
                                              int64_t workspace_bytes, hipStream_t stream) {
  const AdapterSizes s{M, K, N, J, R, entries};
  int rc = adapter_check(s, dtype, index_wide);
  if (rc != FIM_OK) return rc;
  if (M == 0) return FIM_ERR_INVALID;  // (there is no row to sum over: the caller's zeros)
  if (d_out == nullptr || x == nullptr || a == nullptr || b == nullptr || index == nullptr || (da == nullptr) != (db == nullptr) ||
      (da != nullptr && h == nullptr && !adapter_narrow(K, N, R)))
    return FIM_ERR_INVALID;
  for (const void* t : {d_out, x, a, b, static_cast<const void*>(dx), static_cast<const void*>(da), static_cast<const void*>(db)})
    if (reinterpret_cast<uintptr_t>(t) % 2) return FIM_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(index) % (index_wide ? 8 : 4) || reinterpret_cast<uintptr_t>(h) % 16) return FIM_ERR_INVALID;
  const AdapterGradPlan g = grad_plan(s);
  if (g.bytes > 0 && (workspace == nullptr || workspace_bytes < g.bytes || reinterpret_cast<uintptr_t>(workspace) % 256))
    return FIM_ERR_INVALID;
  if (dx == nullptr && da == nullptr) return FIM_OK;
  rc = grad_check(s, g);
  if (rc != FIM_OK) return rc;
  const int64_t na = J * R * K, nb = J * R * N;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* part = da != nullptr && g.chunks > 1 ? reinterpret_cast<float*>(ws + g.part) : nullptr;
  int* counts = part != nullptr ? reinterpret_cast<int*>(ws + g.counts) : nullptr;
  auto join = [&]() {
    if (part == nullptr) return;
    const auto kernel = dtype == FIM_BF16 ? adapter_join_kernel<FIM_BF16> : adapter_join_kernel<FIM_F16>;
    const int64_t blocks = J * cdiv(R * (K + N), 64);
    kernel<<<dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), dim3(64 * JOIN_WAVES), 0, stream>>>(
        part, counts, (int)g.chunks, (int)J, (int)K, (int)N, (int)R,
        static_cast<uint16_t*>(da), static_cast<uint16_t*>(db));
  };
  if (g.narrow) {
    const AdapterNarrowArgs q{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(d_out), static_cast<const uint16_t*>(a),
                              static_cast<const uint16_t*>(b), x_stride, d_out_stride,
                              AdapterIndex{index, index_wide, (uint32_t)(M / entries), (int)J}, scales, scale,
                              static_cast<uint16_t*>(dx), static_cast<uint16_t*>(da), static_cast<uint16_t*>(db), part, counts,
                              (uint32_t)M, (uint32_t)g.chunk, (int)g.chunks, (int)K, (int)N, (int)R};
    const dim3 grid((unsigned)((J + (dx != nullptr)) * g.chunks));  // (rows without an adapter: zeros of dx)
    auto launch = [&](auto dt, auto whole, auto pieces) {
      constexpr int DT = decltype(dt)::value;
      constexpr bool W = decltype(whole)::value, P = decltype(pieces)::value;
      if (R > 16) adapter_narrow_kernel<DT, 2, W, P><<<grid, dim3(256), 0, stream>>>(q);
      else adapter_narrow_kernel<DT, 1, W, P><<<grid, dim3(256), 0, stream>>>(q);
    };
    const auto yes = std::integral_constant<bool, true>{};
    const auto no = std::integral_constant<bool, false>{};
    auto of_type = [&](auto dt) {
      const bool whole = K % 32 == 0 && N % 32 == 0, pieces = g.chunk > NARROW_CHUNK;
      if (whole) pieces ? launch(dt, yes, yes) : launch(dt, yes, no);
      else pieces ? launch(dt, no, yes) : launch(dt, no, no);
    };
    if (dtype == FIM_BF16) of_type(std::integral_constant<int, FIM_BF16>{});
    else of_type(std::integral_constant<int, FIM_F16>{});
    join();
    return launch_status();
  }
  uint16_t *at = reinterpret_cast<uint16_t*>(ws + g.at), *bt = reinterpret_cast<uint16_t*>(ws + g.bt);
  float* t = reinterpret_cast<float*>(ws + g.t);
  const AdapterIndex rows{index, index_wide, (uint32_t)(M / entries), (int)J};
  adapter_transpose_kernel<<<dim3((unsigned)cdiv(na + nb, 256)), dim3(256), 0, stream>>>(
      static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), at, bt, (int)K, (int)N, (int)R, na, nb);
  // t = s d_out B and dx = t A: the forward pass over d_out (without dx: over no columns)
  AdapterArgs p{static_cast<const uint16_t*>(d_out), nullptr, bt, at, d_out_stride, 0, static_cast<uint16_t*>(dx), t, rows, scales,
                scale, (uint32_t)M, (int)N, dx == nullptr ? 0 : (int)K, (int)R, 1};
  adapter_rows(p, dtype, stream);
  if (da != nullptr) {
    const AdapterGradArgs q{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(d_out), x_stride, d_out_stride, t, h, rows,
                            static_cast<uint16_t*>(da), static_cast<uint16_t*>(db), part, counts, (uint32_t)M, (uint32_t)g.chunk,
                            (int)g.chunks, (int)K, (int)N, (int)R, g.xt, g.ct};
    by_type(dtype, R, [&](auto dt, auto nr) {
      constexpr int DT = decltype(dt)::value;
      const auto kernel = g.chunk > GRAD_CHUNK ? adapter_grad_kernel<DT, decltype(nr)::value, true>
                                               : adapter_grad_kernel<DT, decltype(nr)::value, false>;
      kernel<<<dim3((unsigned)(J * g.chunks * g.ct)), dim3(256), 0, stream>>>(q);
    });
    join();
  }
  return launch_status();
}
