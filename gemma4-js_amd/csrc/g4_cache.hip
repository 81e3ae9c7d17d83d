// Rows of a KV cache's planes: kept in place after drafted tokens were checked,
// or copied into another cache.
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kMaxPlanes = G4_CACHE_MAX_PLANES;

struct Planes {
  float *dst[kMaxPlanes];
  const float *src[kMaxPlanes];
  int width[kMaxPlanes];
};

// One block per (row, plane): dst row dst_row + i = src row rows[i], or NaN for an
// entry outside [0, src_rows).  rows == nullptr: row i itself.
__global__ __launch_bounds__(256) void cache_rows_kernel(Planes p, const int *__restrict__ rows,
                                                         int dst_row, int src_rows) {
  const int i = blockIdx.x, plane = blockIdx.y;
  const int r = rows ? rows[i] : i;
  const bool ok = r >= 0 && r < src_rows;
  const int width = p.width[plane];
  const float *s = p.src[plane] + (size_t)(ok ? r : 0) * width;
  float *d = p.dst[plane] + ((size_t)dst_row + i) * width;
  for (int c = threadIdx.x; c < width; c += 256) d[c] = ok ? s[c] : __int_as_float(0x7fc00000);
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
    if (widths[p] <= 0) return fail(G4_E_ARG, "g4_cache_rows: plane %d width %d", p, widths[p]);
  G4_CHECK_INIT();
  if (n == 0) return ok();
  int rc = check_device_range(rows, (size_t)n * 4, "g4_cache_rows rows");
  Planes out{}, in{};
  size_t staged = 0;
  bool place = false;
  for (int p = 0; p < planes && !rc; ++p) {
    const size_t w = (size_t)widths[p];
    rc = check_device_range(dst[p], ((size_t)dst_row + n) * w * 4, "g4_cache_rows dst");
    if (!rc) rc = check_device_range(src[p], (size_t)src_rows * w * 4, "g4_cache_rows src");
    out.dst[p] = dst[p];
    in.src[p] = src[p];
    out.width[p] = in.width[p] = widths[p];
    const uintptr_t d0 = reinterpret_cast<uintptr_t>(dst[p] + (size_t)dst_row * w);
    const uintptr_t s0 = reinterpret_cast<uintptr_t>(src[p]);
    place = place || (d0 < s0 + src_rows * w * 4 && s0 < d0 + n * w * 4);
    staged += n * w;
  }
  if (rc) return rc;
  const dim3 grid(n, planes);
  if (!place) {
    for (int p = 0; p < planes; ++p) in.dst[p] = out.dst[p];
    hipLaunchKernelGGL(cache_rows_kernel, grid, dim3(256), 0, stream(), in, rows, dst_row, src_rows);
    G4_LAUNCH_CHECK("cache_rows_kernel");
    return ok();
  }
  void *mem = nullptr;
  if ((rc = g_cache_ws.get(staged * 4, &mem, "g4_cache_rows"))) return rc;
  float *at = static_cast<float *>(mem);
  for (int p = 0; p < planes; ++p) {
    in.dst[p] = at;
    out.src[p] = at;
    at += (size_t)n * widths[p];
  }
  hipLaunchKernelGGL(cache_rows_kernel, grid, dim3(256), 0, stream(), in, rows, 0, src_rows);
  G4_LAUNCH_CHECK("cache_rows_kernel");
  hipLaunchKernelGGL(cache_rows_kernel, grid, dim3(256), 0, stream(), out, nullptr, dst_row, n);
  G4_LAUNCH_CHECK("cache_rows_kernel");
  return ok();
}
