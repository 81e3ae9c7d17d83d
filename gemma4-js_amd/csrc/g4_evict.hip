// The rows of a cache to keep: the first ones, the latest ones and the heaviest of the others.
#include "g4_internal.h"
#include "g4_kv4.h"

namespace g4 {
namespace {

constexpr int kMaxSets = 256;
constexpr int kBins = 2048;
constexpr int kOneBlock = 1024 * 8;             // the most that one block takes (15 sets of 16000: 21.4 us, 17.2 by several)
constexpr int kThreads = 1024;                  // of a block of several
constexpr int kPerThread = 4;                   // weights
constexpr int kSlice = kThreads * kPerThread;   // a block's weights

struct EvictArgs {
  const float *w;
  float *kept;
  int *rows;
  size_t stride;
  int len, keep, first, recent;
  // caches of several slices
  int slices;
  int *hist;        // [sets][2048], zero between calls
  int *count;       // [sets][slices][4]: above the bin, in the bin; then rows before, equal ones before
  uint32_t *top;    // [sets][2]: threshold, rows equal to it that stay
  uint32_t *cand;   // [sets][slices * kSlice]: each slice's weights in the bin
  float *copy;      // [sets][slices * kSlice]: the weights, where kept overwrites them
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
  s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xf, 0xf, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xf, 0xf, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xf, 0xf, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xa, 0xf, false);  // rows 1 and 3: the sum before them
  s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xc, 0xf, false);  // rows 2 and 3 likewise
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

// The bin, from the top, in which the want-th of the counted lies (found[0]), and how many lie in
// the bins above it (found[1]).  Ends with a barrier.
template <int NW>
__device__ __forceinline__ void find_bin(const int *hist, int want, int *tmp, int *found) {
  constexpr int PER = kBins / (64 * NW);
  const int b = kBins - 1 - PER * threadIdx.x;
  int h[PER], sum = 0, all;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += h[i] = hist[b - i];
  int above = before_me<NW>(sum, tmp, all);
  if (above < want && want <= above + sum) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < want && want <= above + h[i]) found[0] = b - i, found[1] = above;
      above += h[i];
    }
  }
  __syncthreads();
}

// The threshold's bits are found in three passes, 11, 11 and 10 of them.
__device__ __forceinline__ int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit(uint32_t key, int pass) {
  return key >> digit_shift(pass) & (pass == 2 ? 1023u : 2047u);
}

// Selection by digits: 11 bits of the order at a time, the histogram of those that agree so far gives the
// next; no sort, and the rows come out in their order by a scan.
// A block per set of up to P weights per thread, which stay in registers: histograms of the
// weights that agree with the bits found before, then one scan that counts the rows above the
// threshold (the first and last ones among them) and, in the upper half, those equal to it.  2112
// weights: 5.7 us traced, three histograms and four scans one after the other, each short of
// nothing but instructions to fetch: 256 threads of 16 weights each, four times the code, take 7.9.
template <int P>
__global__ __launch_bounds__(1024) void evict_kernel(EvictArgs a) {
  constexpr int NW = 16;
  __shared__ int hist[3][kBins];
  __shared__ int tmp[NW];
  __shared__ int found[2];
  const int t = threadIdx.x, end = a.len - a.recent;
  const int per = (a.len + 64 * NW - 1) / (64 * NW), i0 = t * per;
  const float *w = a.w + (size_t)blockIdx.x * a.stride;
  float x[P];
#pragma unroll
  for (int j = 0; j < P; ++j) x[j] = w[min(i0 + j, a.len - 1)];
  for (int i = t; i < 3 * kBins; i += 64 * NW) (&hist[0][0])[i] = 0;
  uint32_t key[P], in = 0;  // in: between the first and the last ones, and not yet decided
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = i0 + j;
    key[j] = order_of(x[j]);
    if (j < per && i >= a.first && i < end) in |= 1u << j;
    else key[j] = 0xffffffffu;  // (no weight's)
  }
  int want = a.keep - a.first - a.recent;
  uint32_t top = want > 0 ? 0 : 0xfffffffeu;  // the threshold (which no weight has)
  __syncthreads();
  if (want > 0) {
#pragma unroll 1  // (less code to fetch: 2112 weights, unrolled, 8.9 us for 8.35)
    for (int pass = 0; pass < 3; ++pass) {
#pragma unroll
      for (int j = 0; j < P; ++j)
        if (in >> j & 1) atomicAdd(&hist[pass][digit(key[j], pass)], 1);
      __syncthreads();
      find_bin<NW>(hist[pass], want, tmp, found);
      const uint32_t d = (uint32_t)found[0];
      top |= d << digit_shift(pass);
      want -= found[1];
#pragma unroll
      for (int j = 0; j < P; ++j)
        if (digit(key[j], pass) != d) in &= ~(1u << j);
    }
  }
  // `want` of the rows equal to the threshold stay
  int mine = 0;
#pragma unroll
  for (int j = 0; j < P; ++j)
    if (j < per && i0 + j < a.len) mine += key[j] > top ? 1 : key[j] == top ? 1 << 16 : 0;
  int all;
  const int before = before_me<NW>(mine, tmp, all);
  int above = before & 0xffff, equal = before >> 16;
  int *rows = a.rows + (size_t)blockIdx.x * a.keep;
  float *kept = a.kept ? a.kept + (size_t)blockIdx.x * a.stride : nullptr;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (j >= per || i0 + j >= a.len) break;
    const bool same = key[j] == top;
    if (key[j] > top || (same && equal < want)) {
      const int at = above + min(equal, want);
      rows[at] = i0 + j;
      if (kept) kept[at] = x[j];
    }
    above += key[j] > top ? 1 : 0;
    equal += same ? 1 : 0;
  }
  if (kept)
    for (int i = a.keep + t; i < a.len; i += 64 * NW) kept[i] = 0.f;
}

// Longer caches, a block per slice of 4096 weights (blockIdx.x), four launches: the
// histogram of the first 11 bits ...  131072 weights: 2.6, 3.6, 7.2 and 3.3 us traced (with 256
// threads of 16 weights each 3.5, 4.8, 7.1 and 5.3), each little more than its loads' latencies; 2^20
// weights 53 us in all.  Many equal weights meet in one counter, in the third kernel those of a whole
// cache: 131072 weights of which 9 in 10 are 0, half of them kept, 238 us in all, 2^24 30 ms (spread
// out 18.6 us and 0.84 ms).  (All of the bin's weights in the third kernel's
// registers, each with its slice looked up: 11.2 us.)
__global__ __launch_bounds__(kThreads) void evict_count_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  const int t = threadIdx.x, set = blockIdx.y, end = a.len - a.recent;
  const float *w = a.w + (size_t)set * a.stride;
  for (int i = t; i < kBins; i += kThreads) hist[i] = 0;
  __syncthreads();
  float x[kPerThread];
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) x[j] = w[min((int)blockIdx.x * kSlice + kThreads * j + t, a.len - 1)];
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = blockIdx.x * kSlice + kThreads * j + t;
    if (i >= a.first && i < end) atomicAdd(&hist[digit(order_of(x[j]), 0)], 1);
  }
  __syncthreads();
  for (int i = t; i < kBins; i += kThreads)
    if (hist[i]) atomicAdd(&a.hist[set * kBins + i], hist[i]);
}

// ... each slice's weights in the bin of the threshold, and how many lie above it ...
__global__ __launch_bounds__(kThreads) void evict_list_kernel(EvictArgs a) {
  __shared__ int tmp[kThreads / 64], found[2];
  const int t = threadIdx.x, set = blockIdx.y, slice = blockIdx.x, end = a.len - a.recent;
  const float *w = a.w + (size_t)set * a.stride;
  float x[kPerThread];
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) x[j] = w[min(slice * kSlice + kThreads * j + t, a.len - 1)];
  const int want = a.keep - a.first - a.recent;
  find_bin<kThreads / 64>(a.hist + set * kBins, want, tmp, found);
  const uint32_t bin = want > 0 ? (uint32_t)found[0] : (uint32_t)kBins;  // (none)
  const size_t base = ((size_t)set * a.slices + slice) * kSlice;
  int mine = 0, above = 0, all;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = slice * kSlice + kThreads * j + t;
    if (a.copy && i < a.len) a.copy[base + kThreads * j + t] = x[j];
    const uint32_t d = digit(order_of(x[j]), 0);
    const bool mid = i >= a.first && i < end;
    // the first and last rows count as above
    if (i < a.len && (!mid || d > bin)) ++above;
    if (mid && d == bin) ++mine;
  }
  int at = before_me<kThreads / 64>(mine | above << 16, tmp, all) & 0xffff;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int i = slice * kSlice + kThreads * j + t;
    const uint32_t k = order_of(x[j]);
    if (i >= a.first && i < end && digit(k, 0) == bin) a.cand[base + at++] = k;
  }
  if (t == 0) {
    int *c = a.count + ((size_t)set * a.slices + slice) * 4;
    c[0] = all >> 16;
    c[1] = all & 0xffff;
  }
}

// ... the threshold's other bits from those, and the rows before each slice.  A wave takes slices w,
// w + 16, .. and holds the first 256 of the bin's weights of two of them in registers, loaded beside
// the bin's search ...
__global__ __launch_bounds__(1024) void evict_threshold_kernel(EvictArgs a) {
  constexpr int NW = 16;
  __shared__ int hist[kBins];
  __shared__ int tmp[NW], found[2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, set = blockIdx.x;
  const uint32_t *cand = a.cand + (size_t)set * a.slices * kSlice;
  int *count = a.count + (size_t)set * a.slices * 4;
  constexpr int HELD = 2, PER = 4;
  int n_held[HELD];
  uint32_t held[HELD][PER];
#pragma unroll
  for (int i = 0; i < HELD; ++i) n_held[i] = wave + NW * i < a.slices ? count[4 * (wave + NW * i) + 1] : 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
#pragma unroll
    for (int j = 0; j < PER; ++j)
      held[i][j] = lane + 64 * j < n_held[i] ? cand[(size_t)(wave + NW * i) * kSlice + lane + 64 * j] : 0;
  // f(weight) for this lane's of the wave's turn-th slice
  auto each = [&](int turn, auto f) {
    const int s = wave + NW * turn;
    int i = lane, n;
    if (turn < HELD) {
      n = n_held[0];
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        if (h != turn) continue;
        n = n_held[h];
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (lane + 64 * j < n) f(held[h][j]);
      }
      i += 64 * PER;
    } else {
      n = count[4 * s + 1];
    }
    for (; i < n; i += 64) f(cand[(size_t)s * kSlice + i]);
  };
  const int turns = (a.slices - wave + NW - 1) / NW;
  int want = a.keep - a.first - a.recent;
  find_bin<NW>(a.hist + set * kBins, want, tmp, found);
  for (int i = t; i < kBins; i += 1024) a.hist[set * kBins + i] = 0;  // for the next call
  uint32_t top = 0xfffffffeu;  // (which no weight has)
  if (want > 0) {
    uint32_t mask = 2047u << digit_shift(0);
    top = (uint32_t)found[0] << digit_shift(0);
    want -= found[1];
    for (int pass = 1; pass < 3; ++pass) {
      for (int i = t; i < kBins; i += 1024) hist[i] = 0;
      __syncthreads();
      for (int turn = 0; turn < turns; ++turn)
        each(turn, [&](uint32_t k) {
          if ((k & mask) == top) atomicAdd(&hist[digit(k, pass)], 1);
        });
      __syncthreads();
      find_bin<NW>(hist, want, tmp, found);
      top |= (uint32_t)found[0] << digit_shift(pass);
      want -= found[1];
      mask |= (pass == 1 ? 2047u : 1023u) << digit_shift(pass);
      __syncthreads();
    }
  }
  // each slice's rows above the threshold and equal to it
  for (int turn = 0; turn < turns; ++turn) {
    const int s = wave + NW * turn;
    int above = 0, equal = 0;
    each(turn, [&](uint32_t k) {
      above += k > top ? 1 : 0;
      equal += k == top ? 1 : 0;
    });
    // (whole numbers below 2^24 as floats)
    above = (int)team_sum(64, (float)above);
    equal = (int)team_sum(64, (float)equal);
    if (lane == 0) {
      count[4 * s + 2] = count[4 * s] + above;
      count[4 * s + 3] = equal;
    }
  }
  __syncthreads();
  int above = 0, equal = 0;  // before the turn's slices
  for (int s0 = 0; s0 < a.slices; s0 += 1024) {
    const int s = s0 + t;
    const bool in = s < a.slices;
    int all;
    const int x = in ? count[4 * s + 2] : 0, y = in ? count[4 * s + 3] : 0;
    const int bx = above + before_me<NW>(x, tmp, all);
    above += all;
    const int by = equal + before_me<NW>(y, tmp, all);
    equal += all;
    if (in) {
      count[4 * s + 2] = bx + min(by, want);
      count[4 * s + 3] = by;
    }
  }
  if (t == 0) {
    a.top[2 * set] = top;
    a.top[2 * set + 1] = (uint32_t)want;
  }
}

// ... and the rows.
__global__ __launch_bounds__(kThreads) void evict_rows_kernel(EvictArgs a) {
  constexpr int P = kPerThread;
  __shared__ int tmp[kThreads / 64];
  __shared__ float sw[kSlice];
  const int t = threadIdx.x, set = blockIdx.y, slice = blockIdx.x, end = a.len - a.recent;
  const size_t base = ((size_t)set * a.slices + slice) * kSlice;
  const float *w = a.copy ? a.copy + base : a.w + (size_t)set * a.stride + (size_t)slice * kSlice;
  const int n = min(kSlice, a.len - slice * kSlice);
#pragma unroll
  for (int j = 0; j < P; ++j) sw[kThreads * j + t] = w[min(kThreads * j + t, n - 1)];
  const uint32_t top = a.top[2 * set];
  const int want = (int)a.top[2 * set + 1];
  const int *c = a.count + ((size_t)set * a.slices + slice) * 4;
  const int rows_before = c[2], equal_before = c[3];
  __syncthreads();
  // thread t has weights P t .. of the slice
  float x[P];
  uint32_t key[P];
  int mine = 0, all;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = slice * kSlice + P * t + j;
    x[j] = sw[P * t + j];
    key[j] = i >= a.first && i < end ? order_of(x[j]) : 0xffffffffu;
    if (P * t + j < n) mine += key[j] > top ? 1 : key[j] == top ? 1 << 16 : 0;
  }
  const int before = before_me<kThreads / 64>(mine, tmp, all);
  int above = before & 0xffff, equal = equal_before + (before >> 16);
  const int base_equal = min(equal_before, want);
  int *rows = a.rows + (size_t)set * a.keep;
  float *kept = a.kept ? a.kept + (size_t)set * a.stride : nullptr;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = slice * kSlice + P * t + j;
    if (P * t + j >= n) break;
    const bool same = key[j] == top;
    if (key[j] > top || (same && equal < want)) {
      const int at = rows_before + above + min(equal, want) - base_equal;
      if ((unsigned)at < (unsigned)a.keep) {  // (always, unless another stream changes the weights meanwhile)
        rows[at] = i;
        if (kept) kept[at] = x[j];
      }
    }
    above += key[j] > top ? 1 : 0;
    equal += same ? 1 : 0;
  }
  if (!kept) return;
  for (int j = t; j < n; j += kThreads)
    if (slice * kSlice + j >= a.keep) kept[slice * kSlice + j] = 0.f;
}

__global__ __launch_bounds__(kThreads) void evict_clear_kernel(int *hist) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) hist[blockIdx.x * kBins + i] = 0;
}

// The histograms, which each call leaves zero as it found them, and the rest.
Workspace g_hist_ws, g_evict_ws;

int launch_slices(const EvictArgs &a, int sets) {
  hipLaunchKernelGGL(evict_count_kernel, dim3(a.slices, sets), dim3(kThreads), 0, stream(), a);
  G4_LAUNCH_CHECK("evict_count_kernel");
  hipLaunchKernelGGL(evict_list_kernel, dim3(a.slices, sets), dim3(kThreads), 0, stream(), a);
  G4_LAUNCH_CHECK("evict_list_kernel");
  hipLaunchKernelGGL(evict_threshold_kernel, dim3(sets), dim3(1024), 0, stream(), a);
  G4_LAUNCH_CHECK("evict_threshold_kernel");
  hipLaunchKernelGGL(evict_rows_kernel, dim3(a.slices, sets), dim3(kThreads), 0, stream(), a);
  G4_LAUNCH_CHECK("evict_rows_kernel");
  return G4_OK;
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_cache_evict(const float *weights, size_t stride, int sets, int len, int keep, int first,
                          int recent, int32_t *rows, float *kept) {
  if (sets < 0 || sets > kMaxSets || len < 0 || len > 1 << 24 || keep < 0 || keep > len || first < 0 ||
      recent < 0 || first > keep || recent > keep - first)
    return fail(G4_E_ARG,
                "g4_cache_evict: sets %d (<= 256), len %d (<= 2^24), keep %d, first %d, recent %d "
                "(first + recent <= keep <= len)",
                sets, len, keep, first, recent);
  if (stride < (size_t)len || stride > (size_t(1) << 52))
    return fail(G4_E_ARG, "g4_cache_evict: stride %zu of %d rows", stride, len);
  const size_t n = sets > 0 ? (sets - 1) * stride + len : 0;
  if (kept && kept != weights && overlap(weights, n * 4, kept, n * 4))
    return fail(G4_E_ARG, "g4_cache_evict: kept overlaps weights");
  const size_t n_rows = (size_t)sets * keep * 4;
  if (overlap(rows, n_rows, weights, n * 4) || (kept && overlap(rows, n_rows, kept, n * 4)))
    return fail(G4_E_ARG, "g4_cache_evict: rows overlaps weights or kept");
  G4_CHECK_INIT();
  if (sets == 0 || len == 0) return ok();
  int rc = check_device_range(weights, n * 4, "g4_cache_evict weights");
  if (!rc && keep) rc = check_device_range(rows, (size_t)sets * keep * 4, "g4_cache_evict rows");
  if (!rc && kept) rc = check_device_range(kept, n * 4, "g4_cache_evict kept");
  if (rc) return rc;
  EvictArgs a{};
  a.w = weights;
  a.kept = kept;
  a.rows = rows;
  a.stride = stride;
  a.len = len;
  a.keep = keep;
  a.first = first;
  a.recent = recent;
  if (len <= kOneBlock) {
    hipLaunchKernelGGL(len <= 4096 ? evict_kernel<4> : evict_kernel<8>, dim3(sets),
                       dim3(1024), 0, stream(), a);
    G4_LAUNCH_CHECK("evict_kernel");
    return ok();
  }
  a.slices = (len + kSlice - 1) / kSlice;
  const size_t all = (size_t)sets * a.slices;
  const size_t n_copy = kept == weights ? all * kSlice : 0;
  void *mem = nullptr, *hist = nullptr;
  if ((rc = g_hist_ws.get((size_t)kMaxSets * kBins * 4, &hist, "g4_cache_evict"))) return rc;
  if ((rc = g_evict_ws.get((all * 4 + (size_t)sets * 2 + all * kSlice + n_copy) * 4, &mem, "g4_cache_evict")))
    return rc;
  a.hist = static_cast<int *>(hist);
  a.count = static_cast<int *>(mem);
  a.top = reinterpret_cast<uint32_t *>(a.count + all * 4);
  a.cand = a.top + (size_t)sets * 2;
  a.copy = n_copy ? reinterpret_cast<float *>(a.cand + all * kSlice) : nullptr;
  rc = launch_slices(a, sets);
  if (rc) {
    // The third kernel, which clears the histograms, may be missing behind the first one, which adds to
    // them: counts of this call would give later ones rows that do not exist.
    hipLaunchKernelGGL(evict_clear_kernel, dim3(sets), dim3(kThreads), 0, stream(), a.hist);
    if (hipGetLastError() != hipSuccess) g_hist_ws = Workspace();  // (the next call makes others)
  }
  return rc ? rc : ok();
}
