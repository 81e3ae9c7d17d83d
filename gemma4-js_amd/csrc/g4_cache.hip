// Rows of a KV cache's planes: kept in place after drafted tokens were checked,
// or copied into another cache.
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kMaxPlanes = G4_CACHE_MAX_PLANES;
constexpr int kMaxWidth = 1 << 24;

struct Planes {
  float *dst[kMaxPlanes];
  const float *src[kMaxPlanes];
  int width[kMaxPlanes];
};

constexpr int kChunk = 64;    // 16-byte units (WIDE; else floats) of a row that a wave moves at once
constexpr int kCopyRows = 4;  // chunks per wave of a copy, their loads together
constexpr int kPlaceRows = 64;  // rows that move in place in one launch
constexpr long kMaxBlocks = 1 << 23;  // of a launch, which has less than 2^32 threads

template <bool WIDE>
struct Unit {
  typedef f32x4 type;
  static constexpr int floats = 4;
};
template <>
struct Unit<false> {
  typedef float type;
  static constexpr int floats = 1;
};

// Unit `at` of source row rows[i] (row i itself without rows), or NaN for an entry outside
// [0, src_rows).
template <bool WIDE>
__device__ __forceinline__ typename Unit<WIDE>::type row_unit(const float *src, int units, const int *rows,
                                                              int i, int src_rows, int at) {
  typedef typename Unit<WIDE>::type T;
  const int r = rows ? rows[i] : i;
  const bool ok = r >= 0 && r < src_rows;
  const T v = __builtin_nontemporal_load(reinterpret_cast<const T *>(src) + (size_t)(ok ? r : 0) * units + at);
  return ok ? v : (T)(0.f) + __int_as_float(0x7fc00000);
}

// dst row dst_row + i = src row rows[i] for n rows from row0 on; blockIdx.y is the plane, a wave
// takes kCopyRows chunks one after the other.  Bound by memory: 4000 rows of 30 planes (147 MB
// read, as much written) 48 us, 6.2 TB/s; 8 chunks per wave 52, these through the caches 59, a
// block per row with 4 bytes per lane 94.
template <bool WIDE>
__global__ __launch_bounds__(256) void cache_copy_kernel(Planes p, const int *__restrict__ rows, int row0,
                                                         int n, int dst_row, int src_rows) {
  typedef typename Unit<WIDE>::type T;
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int plane = blockIdx.y, units = p.width[plane] / Unit<WIDE>::floats;
  const int chunks = (units + kChunk - 1) / kChunk;
  const float *src = p.src[plane];
  T *dst = reinterpret_cast<T *>(p.dst[plane]) + ((size_t)dst_row + row0) * units;
  const long first = (long)wave * kCopyRows, all = (long)n * chunks;
  if (first >= all) return;
  T v[kCopyRows];
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const long k = first + u < all ? first + u : all - 1;
    const int i = (int)(k / chunks), at = (int)(k - (long)i * chunks) * kChunk + lane;
    v[u] = row_unit<WIDE>(src, units, rows, row0 + i, src_rows, at < units ? at : units - 1);
  }
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const long k = first + u;
    const int i = (int)(k / chunks), at = (int)(k - (long)i * chunks) * kChunk + lane;
    if (k < all && at < units) __builtin_nontemporal_store(v[u], dst + (size_t)i * units + at);
  }
}

// The same in place for up to kPlaceRows rows: a block owns 64 units of every row of a
// plane and reads them all before it writes any.  Bound by the launch: 5 rows of 30 planes
// 5.7 us per call, 9.3 through scratch in two launches.
template <bool WIDE>
__global__ __launch_bounds__(256) void cache_place_kernel(Planes p, const int *__restrict__ rows, int n,
                                                          int dst_row, int src_rows) {
  typedef typename Unit<WIDE>::type T;
  constexpr int U = kPlaceRows / 4;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int plane = blockIdx.y, units = p.width[plane] / Unit<WIDE>::floats;
  const int at = blockIdx.x * kChunk + lane;
  if (blockIdx.x * kChunk >= units) return;  // whole blocks
  T v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (w + 4 * u < n)
      v[u] = row_unit<WIDE>(p.src[plane], units, rows, w + 4 * u, src_rows, at < units ? at : units - 1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the barrier waits for LDS only)
  __syncthreads();
  T *dst = reinterpret_cast<T *>(p.dst[plane]) + (size_t)dst_row * units;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (w + 4 * u < n && at < units) dst[(size_t)(w + 4 * u) * units + at] = v[u];
}

Workspace g_cache_ws;

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_cache_rows(float *const *dst, const float *const *src, const int *widths, int planes,
                         const int32_t *rows, int n, int dst_row, int src_rows) {
  if (planes < 1 || planes > kMaxPlanes || n < 0 || dst_row < 0 || src_rows < 0)
    return fail(G4_E_ARG, "g4_cache_rows: planes %d (1..%d), n %d, dst_row %d, src_rows %d", planes,
                kMaxPlanes, n, dst_row, src_rows);
  if (!dst || !src || !widths) return fail(G4_E_ARG, "g4_cache_rows: null argument");
  if (n > 0 && src_rows == 0) return fail(G4_E_ARG, "g4_cache_rows: %d rows from none", n);
  for (int p = 0; p < planes; ++p)
    if (widths[p] <= 0 || widths[p] > kMaxWidth)
      return fail(G4_E_ARG, "g4_cache_rows: plane %d width %d (1..%d)", p, widths[p], kMaxWidth);
  G4_CHECK_INIT();
  if (n == 0) return ok();
  int rc = check_device_range(rows, (size_t)n * 4, "g4_cache_rows rows");
  Planes out{}, in{};
  size_t staged = 0;
  bool place = false, shifted = false, wide = true;
  int widest = 0;
  for (int p = 0; p < planes && !rc; ++p) {
    const size_t w = (size_t)widths[p];
    rc = check_device_range(dst[p], ((size_t)dst_row + n) * w * 4, "g4_cache_rows dst");
    if (!rc) rc = check_device_range(src[p], (size_t)src_rows * w * 4, "g4_cache_rows src");
    out.dst[p] = dst[p];
    in.src[p] = src[p];
    out.width[p] = in.width[p] = widths[p];
    const uintptr_t d0 = reinterpret_cast<uintptr_t>(dst[p] + (size_t)dst_row * w);
    const uintptr_t s0 = reinterpret_cast<uintptr_t>(src[p]);
    if (d0 < s0 + src_rows * w * 4 && s0 < d0 + n * w * 4) {
      place = true;
      // a column's block would write what another one's reads
      shifted = shifted || (d0 > s0 ? d0 - s0 : s0 - d0) % (w * 4) != 0;
    }
    staged += n * w;
    if (widths[p] > widest) widest = widths[p];
    wide = wide && widths[p] % 4 == 0 &&
           ((reinterpret_cast<uintptr_t>(dst[p]) | reinterpret_cast<uintptr_t>(src[p])) & 15) == 0;
  }
  if (rc) return rc;
  if (place && !shifted && n <= kPlaceRows) {
    for (int p = 0; p < planes; ++p) in.dst[p] = out.dst[p];
    const int units = wide ? widest / 4 : widest;
    hipLaunchKernelGGL(wide ? cache_place_kernel<true> : cache_place_kernel<false>,
                       dim3((units + kChunk - 1) / kChunk, planes), dim3(256), 0, stream(), in, rows, n,
                       dst_row, src_rows);
    G4_LAUNCH_CHECK("cache_place_kernel");
    return ok();
  }
  auto copy = [&](const Planes &pl, const int32_t *from, int to, int limit) {
    const long units = wide ? widest / 4 : widest, chunks = (units + kChunk - 1) / kChunk;
    const long most = kMaxBlocks * 4 * kCopyRows / chunks;  // rows of a launch
    for (long row0 = 0; row0 < n; row0 += most) {
      const long count = n - row0 < most ? n - row0 : most;
      const long blocks = (count * chunks + 4 * kCopyRows - 1) / (4 * kCopyRows);
      hipLaunchKernelGGL(wide ? cache_copy_kernel<true> : cache_copy_kernel<false>,
                         dim3((unsigned)blocks, planes), dim3(256), 0, stream(), pl, from, (int)row0,
                         (int)count, to, limit);
      G4_LAUNCH_CHECK("cache_copy_kernel");
    }
    return G4_OK;
  };
  if (!place) {
    for (int p = 0; p < planes; ++p) in.dst[p] = out.dst[p];
    rc = copy(in, rows, dst_row, src_rows);
    return rc ? rc : ok();
  }
  // more rows in place: all of them to scratch, then to where they go
  void *mem = nullptr;
  if ((rc = g_cache_ws.get(staged * 4, &mem, "g4_cache_rows"))) return rc;
  float *to = static_cast<float *>(mem);
  for (int p = 0; p < planes; ++p) {
    in.dst[p] = to;
    out.src[p] = to;
    to += (size_t)n * widths[p];
  }
  rc = copy(in, rows, 0, src_rows);
  if (!rc) rc = copy(out, nullptr, dst_row, n);
  return rc ? rc : ok();
}
