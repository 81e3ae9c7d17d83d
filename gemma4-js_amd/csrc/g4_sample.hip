// Tokens by temperature, top-k, top-p and min-p from given random numbers.
//
// With the finite logits x of a row ordered by value (equal ones by index), d =
// (x - max x) / temperature and p = e^d, each cut keeps a prefix of that order:
//   top-k  the first k
//   top-p  those with less than top_p * mass(top-k) before them
//   min-p  those with p >= min_p
// so the kept set is all tokens above one logit and the first `ties` (by index)
// of those that equal it.  The token is the first one, by index, up to which more
// than u * (kept mass) lies.
//
// Numerics.  d, e^d and the borders are computed in binary64 and masses are summed
// as integers, round(p * 2^s), 2^s * vocab < 2^62: a token's border may lie next to
// u, and integer sums do not depend on their order.
#include <math.h>

#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kThreads = 1024;

struct SampleArgs {
  const float *x;
  size_t stride;
  int vocab, top_k;
  double inv_t, top_p, log_min;
  double unit;  // 2^s
  const float *u;
  int *tokens;
  float *probs;
};

// Order-preserving key of a finite logit (zeros alike); 0 for any other.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!isfinite(x)) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ uint64_t mass_of(double d, double unit) {
  return (uint64_t)(exp(d) * unit + 0.5);
}

// One block per row.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ uint32_t cnt[256];
  __shared__ unsigned long long mass[256];
  __shared__ uint32_t s_key, s_n;
  __shared__ unsigned long long s_mass;
  __shared__ unsigned long long part[kThreads];
  const int t = threadIdx.x;
  const float *x = a.x + (size_t)blockIdx.x * a.stride;
  if (t == 0) s_key = 0;
  __syncthreads();
  uint32_t best = 0;
  for (int i = t; i < a.vocab; i += kThreads) best = max(best, key_of(x[i]));
  atomicMax(&s_key, best);
  __syncthreads();
  best = s_key;
  if (best == 0) {
    if (t == 0) {
      a.tokens[blockIdx.x] = -1;
      if (a.probs) a.probs[blockIdx.x] = 0.f;
    }
    return;
  }
  const double top = logit_of(best);
  auto d_of = [&](uint32_t key) { return ((double)logit_of(key) - top) * a.inv_t; };
  // the cut: keys above `cut`, and the first `ties` that equal it
  uint32_t cut = 1, ties = 0xffffffffu;
  // One digit after the other: the key at which `want` tokens (or `want` mass) are
  // reached from the top, and what is left of `want` there.
  auto select = [&](bool by_mass, unsigned long long want, uint32_t lim, uint32_t lim_ties) {
    uint32_t prefix = 0;
    unsigned long long left = want, w_tie = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (t < 256) cnt[t] = 0, mass[t] = 0;
      __syncthreads();
      for (int i = t; i < a.vocab; i += kThreads) {
        const uint32_t k = key_of(x[i]);
        if (k == 0 || k < lim || (k ^ prefix) >> shift >> 8) continue;
        const uint32_t bin = k >> shift & 255;
        atomicAdd(&cnt[bin], 1u);
        if (by_mass && k > lim) atomicAdd(&mass[bin], (unsigned long long)mass_of(d_of(k), a.unit));
      }
      __syncthreads();
      if (t == 0) {
        if (by_mass && lim > 1 && !((lim ^ prefix) >> shift >> 8)) {  // the ties that top-k kept
          const uint64_t n = cnt[lim >> shift & 255] ? lim_ties : 0;
          mass[lim >> shift & 255] += n * mass_of(d_of(lim), a.unit);
        }
        int b = 255;
        unsigned long long l = left;
        for (; b > 0; --b) {
          const unsigned long long m = by_mass ? mass[b] : cnt[b];
          if (m >= l) break;
          l -= m;
        }
        s_n = b;
        s_mass = l;
      }
      __syncthreads();
      prefix |= s_n << shift;
      left = s_mass;
    }
    cut = prefix;
    if (by_mass) {
      w_tie = mass_of(d_of(cut), a.unit);
      const unsigned long long n = w_tie ? (left + w_tie - 1) / w_tie : 0;
      ties = n < 0xffffffffull ? (uint32_t)n : 0xffffffffu;
      if (cut == lim && lim_ties < ties) ties = lim_ties;
    } else {
      ties = (uint32_t)left;
    }
    __syncthreads();
  };
  auto block_sum = [&](unsigned long long v) {  // exclusive sum before this thread; total in s_mass
    part[t] = v;
    __syncthreads();
    for (int o = 1; o < kThreads; o <<= 1) {
      const unsigned long long w = t >= o ? part[t - o] : 0;
      __syncthreads();
      part[t] += w;
      __syncthreads();
    }
    if (t == 0) s_mass = part[kThreads - 1];
    const unsigned long long before = part[t] - v;
    __syncthreads();
    return before;
  };
  // each thread's run of consecutive tokens
  const int per = (a.vocab + kThreads - 1) / kThreads;
  const int i0 = min(t * per, a.vocab), i1 = min(i0 + per, a.vocab);
  unsigned long long n_all = 0;
  for (int i = i0; i < i1; ++i) n_all += key_of(x[i]) != 0;
  block_sum(n_all);
  const unsigned long long finite = s_mass;
  if (a.top_k > 0 && (unsigned long long)a.top_k < finite) select(false, a.top_k, 1, 0);
  auto kept_mass = [&]() {
    unsigned long long eq = 0;
    for (int i = i0; i < i1; ++i) eq += key_of(x[i]) == cut;
    uint32_t rank = (uint32_t)block_sum(eq);
    unsigned long long m = 0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key_of(x[i]);
      if (k == 0 || k < cut || (k == cut && rank++ >= ties)) continue;
      const double d = d_of(k);
      if (d >= a.log_min) m += mass_of(d, a.unit);
    }
    return m;
  };
  if (a.top_p < 1.0) {
    const double log_min = a.log_min;
    a.log_min = -INFINITY;
    block_sum(kept_mass());
    const unsigned long long want = (unsigned long long)ceil(a.top_p * (double)s_mass);
    select(true, want, cut, ties);
    a.log_min = log_min;
  }
  const unsigned long long m = kept_mass();
  const unsigned long long before = block_sum(m), total = s_mass;
  const float u = a.u[blockIdx.x];
  unsigned long long want = 0;  // the token is the first with a running mass above this
  if (u >= 1.f) {
    want = total - 1;
  } else if (u > 0.f) {
    want = __umul64hi((unsigned long long)((double)u * 18446744073709551616.0), total);
  }
  if (want < before || want >= before + m) return;
  unsigned long long run = before;
  uint32_t rank = 0;
  if (ties != 0xffffffffu)
    for (int i = 0; i < i0; ++i) rank += key_of(x[i]) == cut;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = key_of(x[i]);
    if (k == 0 || k < cut || (k == cut && rank++ >= ties)) continue;
    const double d = d_of(k);
    if (d < a.log_min) continue;
    run += mass_of(d, a.unit);
    if (run > want) {
      a.tokens[blockIdx.x] = i;
      if (a.probs) a.probs[blockIdx.x] = (float)(exp(d) * a.unit / (double)total);
      return;
    }
  }
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_sample(const float *logits, size_t stride, int rows, int vocab,
                     const g4_sample_params *params, const float *u, int32_t *tokens, float *probs) {
  if (rows < 0 || vocab <= 0 || stride < (size_t)vocab)
    return fail(G4_E_ARG, "g4_sample: rows %d, vocab %d, stride %zu", rows, vocab, stride);
  if (!params) return fail(G4_E_ARG, "g4_sample: null params");
  const g4_sample_params &p = *params;
  if (!(p.temperature >= 0.f) || !isfinite(p.temperature) || p.top_k < 0 || !(p.top_p > 0.f) ||
      !(p.top_p <= 1.f) || !(p.min_p >= 0.f) || !(p.min_p <= 1.f))
    return fail(G4_E_ARG,
                "g4_sample: temperature %g (>= 0), top_k %d (>= 0), top_p %g (in (0, 1]), min_p %g "
                "(in [0, 1])",
                p.temperature, p.top_k, p.top_p, p.min_p);
  G4_CHECK_INIT();
  if (rows == 0) return ok();
  int rc = check_device_range(logits, ((size_t)(rows - 1) * stride + vocab) * 4, "g4_sample logits");
  if (!rc) rc = check_device_range(u, (size_t)rows * 4, "g4_sample u");
  if (!rc) rc = check_device_range(tokens, (size_t)rows * 4, "g4_sample tokens");
  if (!rc && probs) rc = check_device_range(probs, (size_t)rows * 4, "g4_sample probs");
  if (rc) return rc;
  SampleArgs a{};
  a.x = logits;
  a.stride = stride;
  a.vocab = vocab;
  // temperature 0: the first of the largest alone
  a.top_k = p.temperature > 0.f ? p.top_k : 1;
  a.inv_t = p.temperature > 0.f ? 1.0 / (double)p.temperature : 0.0;
  a.top_p = p.top_p;
  a.log_min = log((double)p.min_p);
  int bits = 0;
  while (bits < 31 && (1u << bits) < (unsigned)vocab) ++bits;
  a.unit = ldexp(1.0, 62 - bits < 52 ? 62 - bits : 52);
  a.u = u;
  a.tokens = tokens;
  a.probs = probs;
  hipLaunchKernelGGL(sample_row_kernel, dim3(rows), dim3(kThreads), 0, stream(), a);
  G4_LAUNCH_CHECK("sample_row_kernel");
  return ok();
}
