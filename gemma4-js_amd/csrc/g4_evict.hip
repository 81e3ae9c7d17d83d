// The rows of a cache to keep: the first ones, the latest ones and the heaviest of the others.
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kBins = 2048;

struct EvictArgs {
  const float *w;
  float *kept;
  int *rows;
  size_t stride;
  int len, keep, first, recent;
};

// Weights in their order as whole numbers: NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  if (u == 0x80000000u) return 0x80000000u;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// The sum over the threads before this one, and of all.  `tmp`: one int per wave.
template <int NW>
__device__ __forceinline__ int before_me(int x, int *tmp, int &all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(s, o, 64);
    if (lane >= o) s += y;
  }
  if (lane == 63) tmp[w] = s;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int y = tmp[i];
    if (i < w) base += y;
    all += y;
  }
  __syncthreads();
  return base + s - x;
}

// A block per set: the threshold's bits, 11, 11 and 10 of them, from histograms of the weights
// that agree with the bits found before; then the rows above it and as many of the equal ones as
// are wanted, in order.
__global__ __launch_bounds__(1024) void evict_kernel(EvictArgs a) {
  constexpr int NW = 16;
  __shared__ int hist[kBins];
  __shared__ int tmp[NW];
  __shared__ int found[2];
  const int t = threadIdx.x, end = a.len - a.recent;
  const float *w = a.w + (size_t)blockIdx.x * a.stride;
  int want = a.keep - a.first - a.recent;
  uint32_t top = 0xffffffffu;  // threshold
  if (want > 0) {
    uint32_t mask = 0;
    top = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = t; i < kBins; i += 1024) hist[i] = 0;
      __syncthreads();
      for (int i = a.first + t; i < end; i += 1024) {
        const uint32_t k = order_of(w[i]);
        if ((k & mask) == top) atomicAdd(&hist[k >> shift & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // bins from the top: thread t has bins 2047 - 2 t and 2046 - 2 t
      const int b = kBins - 1 - 2 * t, h1 = hist[b], h0 = hist[b - 1];
      int all;
      const int above = before_me<NW>(h0 + h1, tmp, all);
      if (above < want && want <= above + h1 + h0) {
        const bool low = want > above + h1;
        found[0] = low ? b - 1 : b;
        found[1] = low ? above + h1 : above;
      }
      __syncthreads();
      top |= (uint32_t)found[0] << shift;
      want -= found[1];
      mask |= (uint32_t)((1 << bits) - 1) << shift;
      __syncthreads();
    }
  }
  // `want` of the rows equal to the threshold stay
  int *rows = a.rows + (size_t)blockIdx.x * a.keep;
  float *kept = a.kept ? a.kept + (size_t)blockIdx.x * a.stride : nullptr;
  int equal = 0, out = 0;
  for (int i0 = 0; i0 < a.len; i0 += 1024) {
    const int i = i0 + t;
    const float x = i < a.len ? w[i] : 0.f;
    const bool mid = i >= a.first && i < end;
    const uint32_t k = order_of(x);
    int all;
    const int e = before_me<NW>(mid && k == top, tmp, all);
    const bool stays = i < a.len && (!mid || k > top || (k == top && equal + e < want));
    equal += all;
    const int at = out + before_me<NW>(stays, tmp, all);
    out += all;
    // (row `at` lies at or before this turn's rows, which all have been read)
    if (stays) {
      rows[at] = i;
      if (kept) kept[at] = x;
    }
  }
  if (!kept) return;
  __syncthreads();
  for (int i = a.keep + t; i < a.len; i += 1024) kept[i] = 0.f;
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_cache_evict(const float *weights, size_t stride, int sets, int len, int keep, int first,
                          int recent, int32_t *rows, float *kept) {
  if (sets < 0 || sets > 256 || len < 0 || len > 1 << 24 || keep < 0 || keep > len || first < 0 ||
      recent < 0 || first > keep || recent > keep - first)
    return fail(G4_E_ARG,
                "g4_cache_evict: sets %d (<= 256), len %d (<= 2^24), keep %d, first %d, recent %d "
                "(first + recent <= keep <= len)",
                sets, len, keep, first, recent);
  if (stride < (size_t)len || stride > (size_t(1) << 60) / 256)
    return fail(G4_E_ARG, "g4_cache_evict: stride %zu of %d rows", stride, len);
  const size_t n = sets > 0 ? (sets - 1) * stride + len : 0;
  const uintptr_t w = reinterpret_cast<uintptr_t>(weights), k = reinterpret_cast<uintptr_t>(kept);
  if (kept && kept != weights && (w < k ? k - w : w - k) < n * 4)
    return fail(G4_E_ARG, "g4_cache_evict: kept overlaps weights");
  G4_CHECK_INIT();
  if (sets == 0 || len == 0) return ok();
  int rc = check_device_range(weights, n * 4, "g4_cache_evict weights");
  if (!rc && keep) rc = check_device_range(rows, (size_t)sets * keep * 4, "g4_cache_evict rows");
  if (!rc && kept) rc = check_device_range(kept, n * 4, "g4_cache_evict kept");
  if (rc) return rc;
  EvictArgs a{weights, kept, rows, stride, len, keep, first, recent};
  hipLaunchKernelGGL(evict_kernel, dim3(sets), dim3(1024), 0, stream(), a);
  G4_LAUNCH_CHECK("evict_kernel");
  return ok();
}
