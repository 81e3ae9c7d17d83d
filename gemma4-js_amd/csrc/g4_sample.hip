// Tokens by temperature, top-k, top-p and min-p from given random numbers.
//
// With the finite logits x of a row ordered by value (equal ones by index), d =
// (x - max x) / temperature and p = e^d, each cut keeps a prefix of that order:
//   top-k  the first k
//   top-p  those with less than top_p * mass(top-k) before them
//   min-p  those with p >= min_p
// The token is the first one, by index, up to which more than u * (kept mass) lies.
//
// Numerics.  A token's border may lie next to u, so d is binary64 and masses are
// integers: round(p * 2^k), 2^k * vocab < 2^62, whose sums do not depend on their order.
// e^d is e^(-b/8) (a table) times e^((f-1)/8) (a polynomial, exact to 2^-53), b and f
// from x * 8 / temperature = whole part and fraction; below e^-31 a mass counts as 0
// (2^-44, a unit of the sums at 262144 tokens).
//
// Three launches, the first two over slices of the rows:
//   sample_plan_kernel    per slice the largest logit and, by whole part of x * 8 / T, count
//                         and mass; a row's last block finds the bins in which the cuts lie
//                         (bins above them are kept, those below dropped)
//   sample_pick_kernel    the kept mass of every slice, and a list of the tokens in those bins
//   sample_finish_kernel  per row the cuts among them, the slice and the token
// With the temperature alone there is nothing to pick, and a row of one slice takes it all in
// one launch (sample_row_kernel).
//
// Measured at 262144 logits: one row by top-k and top-p 26 us (the launches 13, 5 and 9),
// which is the latency of the steps; 64 rows by top-p 70 us (31, 21 and 21).  There the two
// passes over the 67 MB are bound by memory for some 25 us; the rest is the 64-bit arithmetic of
// the first pass (16.8 million exponentials; 8 us more with keys instead of floats in its
// loops), the histograms' join and the rows' ends.  With the ends left to the second launch's
// last blocks, which share its registers and LDS, 64 rows took 13 us more.
//
// A bin of 1/8 holds more of a flat row: of unit spread at temperature 1.5 some 20000 tokens, all
// listed.  The search's passes over them, by one block, are then most of the time: 67 us for one
// row by top-p (the last launch 53), 217 by top-k as well, 64 rows 118 and 316.  Flatter rows,
// which list more than a quarter of their tokens, are read again instead: 985 us at temperature 50.
#include <math.h>

#include <type_traits>

#include "g4_internal.h"

// A logit's bin and its place in the bin come from one rounded product, wherever they are
// computed: products are fused into sums only where fma() says so.
#pragma clang fp contract(off)

namespace g4 {
namespace {

constexpr int NT = 512;       // threads per block
constexpr int kWaves = NT / 64;
constexpr int kBins = 256;    // 31 units of d: below, 2^-44 of the largest; the last one holds the rest
constexpr int kRest = kBins - 1;
constexpr double kPerUnit = 8.0;   // bins per unit of d
constexpr int kShortList = 16384;  // listed tokens of a row, or a quarter of a longer row's: a bin
                                   // holds 7% of a row of unit spread at temperature 1.5
constexpr int kNear = 4096;        // of these in LDS
constexpr int kFew = 128;          // tokens that are compared with each other: 64 rows of 262144 by
                                   // top-p 70 us, with 512 of them 74; by top-k as well 59, with 32 60
constexpr int kMaxRows = 256;      // rows per launch, fewer where their lists pass
constexpr size_t kListBytes = 256 << 20;
constexpr int kMaxShortRows = 1 << 22;  // of one slice: a launch has less than 2^32 threads
constexpr int kIndexBits = 22;
constexpr int kMaxVocab = 1 << kIndexBits;
constexpr int kMaxSlices = 2 * NT;
constexpr int kOneSlice = 8192;    // longest row of one slice: 17 us for one row of 8192 and 18 for
                                   // 256; in slices of 4096 21 and 27
typedef unsigned long long u64;

// What the first launch leaves for the second.
struct Plan {
  double id;        // whole part of max * s
  u64 before_k;     // mass above top-k's bin
  u64 total;        // mass of all bins
  float top;        // largest logit
  int any;          // 0: no finite logit
  int sure;         // bins below this one are kept,
  int part;         // and from there to below this one what min-p leaves
  int lo, hi;       // bins in which top-p's cut may lie (lo > hi: no such cut)
  int kb;           // the bin of top-k's cut, or -1
  uint32_t k_left;  // tokens of it that top-k keeps
  uint32_t n;       // listed tokens
  uint32_t about;   // the same from the bins' masses, at least
  float x0[2], x1[2];  // logits that may lie in bins sure .. hi, and in kb
};

struct SampleArgs {
  const float *x;
  size_t stride;
  int vocab, top_k, slices, per, list_len;
  u64 top_p64;  // top_p * 2^64, 0: no such cut
  double inv_t, s, log_min, unit;
  const float *u;
  int *tokens;
  float *probs;
  Plan *plan;
  u64 *hist;        // [rows][slices][kBins] masses
  uint32_t *counts; // and counts
  uint32_t *maxes;  // [rows][slices] keys
  u64 *list;        // [rows][list_len]
  u64 *mass;        // [rows][slices]
  uint32_t *count;  // [kMaxRows] blocks that are done, 0 between launches
};

// Order-preserving key of a finite logit (zeros alike); 0 for any other.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return (b & 0x7f800000u) == 0x7f800000u ? 0u : k;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// e^z, z = (f - 1/2) / 8, f in [0, 1): the Taylor sum to z^8, its last term spread over the even
// ones below by the Chebyshev polynomial T8 on |z| <= h = 1/16, 128 y^8 ~ 256 y^6 - 160 y^4 +
// 32 y^2 - 1 for y = z / h: off by h^8 / (128 * 8!) and z^9 / 9!, 2^-53.4
__device__ __forceinline__ double exp_part(double f) {
  constexpr double h2 = 1.0 / 256, last = 1.0 / 40320;
  const double z = fma(f, 1.0 / kPerUnit, -0.5 / kPerUnit);
  double r = fma(z, 1.0 / 5040, 1.0 / 720 + 2 * h2 * last);
  r = fma(r, z, 1.0 / 120);
  r = fma(r, z, 1.0 / 24 - 1.25 * h2 * h2 * last);
  r = fma(r, z, 1.0 / 6);
  r = fma(r, z, 0.5 + 0.25 * h2 * h2 * h2 * last);
  r = fma(r, z, 1.0);
  return fma(r, z, 1.0 - h2 * h2 * h2 * h2 * last / 128);
}
constexpr double kHalfBin = 0.93941306281347579;  // e^(-1/16)

// Nearest integer of v in [0, 2^51)
__device__ __forceinline__ u64 to_units(double v) {
  return (u64)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull;
}

// A sum of masses below the upper edge of bin 0, given below that of bin b.  (Bin 0 as it
// is: equal logits alone have borders at round shares of their mass.)
__device__ __forceinline__ u64 from_bin(u64 mass, int b) {
  return b == 0 ? mass : b < kRest ? (u64)((double)mass * exp(-(double)b / kPerUnit) + 0.5) : 0;
}

// Accesses that other XCDs' L2s see without a fence.
template <typename T>
__device__ __forceinline__ void put(T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(const T *p) {
  return __hip_atomic_load(const_cast<T *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Shared {
  u64 bins[kBins];     // masses of a slice's bins; the digits' weights
  uint32_t cnt[kBins];
  double tab[kBins];   // unit * e^(-b/8) * e^(-1/16)
  u64 mass[kMaxSlices];
  u64 few[kFew], weight[kFew];
  u64 wave[kWaves], pick, lo, hi;
  uint32_t v[8], n;
  Plan plan;
};

// v of an earlier lane (0 where there is none), as DPP moves of its halves
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T lane_before(T v) {
  const u64 b = __builtin_bit_cast(u64, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(T, (u64)hi << 32 | lo);
}

// Inclusive sum over the wave's lanes.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += lane_before<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8 in rows of 16 lanes
  v += lane_before<0x112, 0xf>(v);
  v += lane_before<0x114, 0xf>(v);
  v += lane_before<0x118, 0xf>(v);
  v += lane_before<0x142, 0xa>(v);  // row_bcast:15 to rows 1 and 3
  v += lane_before<0x143, 0xc>(v);  // row_bcast:31 to rows 2 and 3
  return v;
}

// Inclusive sum over the block's threads; *total: all of them.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *wave, T *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();  // wave is free
  if (lane == 63) wave[w] = v;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += wave[i];
    all += wave[i];
  }
  *total = all;
  return before + v;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, Shared &sm) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  if ((threadIdx.x & 63) == 0) sm.v[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) v = max(v, sm.v[i]);
  return v;
}

// Whether this block is the last one of its row to get here (all of its coherent
// stores done before).
__device__ __forceinline__ bool last_block(uint32_t *count, int slices, Shared &sm) {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t n = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm.v[0] = n + 1 == (uint32_t)slices;
    if (n + 1 == (uint32_t)slices) *count = 0;
  }
  __syncthreads();
  const bool last = sm.v[0] != 0;
  __syncthreads();
  return last;
}

// The slice's logits in thread order, -inf for what is not finite, and the largest one's key.
template <int E>
__device__ __forceinline__ uint32_t load_slice(const SampleArgs &a, const float *x, int i0, int n,
                                               float (&v)[E], Shared &sm) {
  float best = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = threadIdx.x + NT * e;
    v[e] = i < n ? x[i0 + i] : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = fabsf(v[e]) < INFINITY ? v[e] : -INFINITY;
    best = fmaxf(best, v[e]);
  }
  return block_max(key_of(best), sm);
}

// Count (for top-k) and mass of the slice's logits by bins below the largest one's.  A mass
// is in units of 1 / a.unit of its bin's upper edge.
template <int E>
__device__ __forceinline__ void slice_bins(const SampleArgs &a, const float (&v)[E],
                                           uint32_t best, Shared &sm) {
  if (threadIdx.x < kBins) sm.bins[threadIdx.x] = 0, sm.cnt[threadIdx.x] = 0;
  __syncthreads();
  const double id = floor((double)logit_of(best) * a.s), unit = a.unit * kHalfBin;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double y = (double)v[e] * a.s, fl = floor(y), db = id - fl;
    if (db < kRest) {  // (not for -inf)
      atomicAdd(&sm.bins[(int)db], to_units(exp_part(y - fl) * unit));
      if (a.top_k) atomicAdd(&sm.cnt[(int)db], 1u);
    }
  }
  __syncthreads();
}

// The row's plan from the sums of its bins (thread t < kBins: bin t; the others 0), in
// sm.plan.
__device__ __forceinline__ void make_plan(const SampleArgs &a, float top, uint32_t n, u64 bin_mass,
                                          Shared &sm) {
  const int b = threadIdx.x;
  const u64 m = from_bin(bin_mass, b);
  u64 total, finite = 0;
  Plan &p = sm.plan;
  if (b == 0) {
    p.id = floor((double)top * a.s);
    p.top = top;
    p.any = 1;
    p.kb = -1;
    p.k_left = 0;
    p.lo = 1;
    p.hi = 0;
    p.sure = kBins;
    p.before_k = 0;
    p.n = p.about = 0;
  }
  const u64 upto = block_scan(m, sm.wave, &total), before = upto - m;
  if (b == 0) {
    p.total = total;
    sm.lo = sm.hi = total;  // mass of top-k's tokens: at least, at most
  }
  if (a.top_k) {
    const u64 own = b < kRest ? n : 0, k = a.top_k;
    const u64 n_upto = block_scan(own, sm.wave, &finite), n_before = n_upto - own;
    if (b < kRest && n_before < k && k <= n_upto) {
      p.kb = b;
      p.k_left = (uint32_t)(k - n_before);
      p.before_k = before;
      sm.lo = before;
      sm.hi = upto;
      p.sure = b;
    }
  }
  __syncthreads();
  if (a.top_p64) {
    // a bin's sum is off by what its tokens' masses are rounded by
    const u64 room = (total >> 30) + a.vocab;
    u64 lo = __umul64hi(a.top_p64, sm.lo);
    const u64 hi = __umul64hi(a.top_p64, sm.hi) + room;
    lo = lo > room ? lo - room : 0;
    const int last = p.kb >= 0 ? p.kb : kRest - 1;
    __syncthreads();
    if (b == 0) p.lo = p.sure = lo ? last : 0, p.hi = last;
    __syncthreads();
    if (b < last && before < lo && lo <= upto) p.lo = p.sure = b;
    if (b < last && before < hi && hi <= upto) p.hi = b;
    __syncthreads();
  }
  // (a token's mass is more than e^(-1/8) of a unit)
  if ((b >= p.lo && b <= p.hi) || b == p.kb)
    atomicAdd(&p.about, (uint32_t)((double)bin_mass / a.unit * 1.134) + 1);
  __syncthreads();
  if (b == 0) {
    // bin b holds (max - x) * s in (b - 1, b + 1), min-p keeps what is <= d
    const double d = -a.log_min * kPerUnit;
    int sure = p.sure;
    if (d + 0.01 <= sure - 1) {  // the other cuts lie below
      p.kb = -1;
      p.lo = 1;
      p.hi = 0;
      sure = kBins;
    }
    const int cut = sure;
    if (d - 1.01 < cut) sure = d > 1.01 ? (int)(d - 1.01) : 0;
    const int end = d + 1.01 < kRest ? (int)(d + 1.01) + 1 : kRest;
    p.sure = sure;
    p.part = end < cut ? end : cut;
    // (room for the roundings of x * s)
    auto range = [&](int i, int first, int past) {
      const double u = (p.id - (past - 1)) / a.s, v = (p.id - first + 1) / a.s;
      p.x0[i] = first < past ? (float)(u - fabs(u) * 1e-6) : INFINITY;
      p.x1[i] = first < past ? (float)(v + fabs(v) * 1e-6) : -INFINITY;
    };
    const bool listed = p.lo <= p.hi;
    range(0, sure < p.part || !listed ? sure : p.lo, listed ? p.hi + 1 : p.part);
    range(1, p.kb, p.kb >= 0 ? p.kb + 1 : p.kb);
  }
  __syncthreads();
}

// A logit's place in the plan.
struct Place {
  int b;
  double part, x;
  __device__ Place(const SampleArgs &a, const Plan &p, uint32_t key) {
    x = (double)logit_of(key);
    const double y = x * a.s, fl = floor(y), db = p.id - fl;
    b = db < kRest ? (int)db : kRest;
    part = y - fl;
  }
  // (bins below p.sure are kept as they are)
  __device__ bool partial(const Plan &p) const { return b >= p.sure && b < p.part; }
  __device__ bool listed(const Plan &p) const { return (b >= p.lo && b <= p.hi) || b == p.kb; }
  __device__ bool likely(const SampleArgs &a, const Plan &p) const {
    return (x - (double)p.top) * a.inv_t >= a.log_min;
  }
  __device__ double mass(const double *tab) const { return tab[b] * exp_part(part); }
};

// A token in the order of the cuts: larger is earlier.
__device__ __forceinline__ u64 rank_of(uint32_t key, int i) {
  return (u64)key << kIndexBits | (uint32_t)(kMaxVocab - 1 - i);
}
__device__ __forceinline__ uint32_t rank_key(u64 r) { return (uint32_t)(r >> kIndexBits); }
__device__ __forceinline__ int rank_index(u64 r) {
  return kMaxVocab - 1 - (int)((uint32_t)r & (kMaxVocab - 1));
}

// Of the ranks that each() visits, all in [lo, hi], the one at which the `want`-th unit of
// weight from the top lies (want >= 1; the last one if there is less).  A digit of 8 bits
// after the other until kFew are left (`few`: there are no more), which are then compared
// pairwise.
template <typename Each, typename Weight>
__device__ __forceinline__ u64 select(Each &&each, Weight &&weight, u64 lo, u64 hi, u64 want,
                                      bool few, Shared &sm) {
  const int t = threadIdx.x;
  int rem = 64;     // bits of r - lo below the digits taken
  u64 prefix = 0;   // and those digits
  if (!few) {
    rem = 64 - __clzll((hi - lo) | 1);
    uint32_t n = kFew + 1;
    while (rem > 0 && n > kFew) {
      const int w = rem < 8 ? rem : 8;
      rem -= w;
      __syncthreads();
      if (t < 256) sm.bins[t] = 0, sm.cnt[t] = 0;
      if (t == 0) sm.v[1] = 0, sm.v[2] = 0, sm.pick = 0;
      __syncthreads();
      each([&](u64 r) {
        const u64 c = (r - lo) >> rem;
        if (c >> w != prefix) return;
        const int d = (int)c & ((1 << w) - 1);
        atomicAdd(&sm.bins[d], weight(r));
        atomicAdd(&sm.cnt[d], 1u);
      });
      __syncthreads();
      const u64 own = t < 256 ? sm.bins[255 - t] : 0;
      u64 total;
      const u64 upto = block_scan(own, sm.wave, &total);
      if (want > total) want = total;
      if (upto - own < want && want <= upto) {
        sm.v[1] = 255 - t;
        sm.v[2] = sm.cnt[255 - t];
        sm.pick = upto - own;
      }
      __syncthreads();
      prefix = prefix << w | sm.v[1];
      n = sm.v[2];
      want -= sm.pick;
    }
    if (rem == 0) {
      __syncthreads();
      return lo + prefix;
    }
  }
  __syncthreads();
  if (t == 0) sm.n = 0;
  __syncthreads();
  if (t == 0) sm.pick = 0;
  each([&](u64 r) {
    if (rem < 64 && (r - lo) >> rem != prefix) return;
    const uint32_t at = atomicAdd(&sm.n, 1u);
    sm.few[at] = r;
    sm.weight[at] = weight(r);
  });
  __syncthreads();
  const int n = sm.n;
  if (t < n) {
    const u64 r = sm.few[t], own = sm.weight[t];
    u64 before = 0, total = 0;
    for (int i = 0; i < n; ++i) {
      const u64 w = sm.weight[i];
      total += w;
      if (sm.few[i] > r) before += w;
    }
    if (want > total) want = total;
    if (before < want && want <= before + own) sm.pick = r;
  }
  __syncthreads();
  const u64 got = sm.pick;
  __syncthreads();
  return got;
}

// Where the listed tokens are: nowhere (what lies in the cuts' bins is found in the row
// again), in a.list if they fit, in LDS if they fit there.
enum List { kNoList, kMemory, kLds };

// The end of a row, for one block: the cuts among the listed tokens, the slice that holds
// the picked mass, the token.  E: tokens of a slice per thread.  sm.plan and sm.tab are
// set; sm.mass holds the slices' mass outside the cuts' bins.
template <int E, List LIST>
__device__ __forceinline__ void finish_row(const SampleArgs &a, const float *x, int row, Shared &sm,
                                           u64 *listed) {
  const int t = threadIdx.x;
  const Plan &p = sm.plan;
  auto bin_of = [&](u64 r) { return Place(a, p, rank_key(r)).b; };
  auto mass_of = [&](u64 r) { return to_units(Place(a, p, rank_key(r)).mass(sm.tab)); };
  u64 cut = 0;
  if (p.kb >= 0 || p.lo <= p.hi) {
    const bool fits = LIST != kNoList && p.n <= (uint32_t)a.list_len, few = LIST != kNoList && p.n <= kFew;
    // the first of them in LDS, loaded together
    const u64 *list = a.list + (size_t)row * a.list_len;
    const int n = fits ? p.n : 0;
    if (LIST == kMemory) {  // (the caller has loaded the first NT)
      constexpr int R = kNear / NT - 1;
      if (n > NT) {
        u64 r[R];
#pragma unroll
        for (int i = 0; i < R; ++i) r[i] = list[min(NT * (i + 1) + t, n - 1)];
#pragma unroll
        for (int i = 0; i < R; ++i) listed[NT * (i + 1) + t] = r[i];
      }
    }
    auto each_listed = [&](auto &&f) {
      if (fits) {  // (each thread reads what it wrote)
#pragma unroll 1
        for (int i = t; i < min(n, kNear); i += NT) f(listed[i]);
        if (LIST == kMemory && n > kNear) {  // the rest, the next ones' loads under way
          constexpr int R = 8;
          u64 v[R];
          auto load = [&](int i) {
#pragma unroll
            for (int j = 0; j < R; ++j) v[j] = list[min(i + NT * j, n - 1)];
          };
          load(kNear + t);
#pragma unroll 1
          for (int i = kNear + t; i < n; i += R * NT) {
            u64 r[R];
#pragma unroll
            for (int j = 0; j < R; ++j) r[j] = v[j];
            if (i + R * NT < n) load(i + R * NT);
#pragma unroll 1
            for (int j = i; j < min(i + R * NT, n); j += NT) {
              f(r[0]);
#pragma unroll
              for (int m = 0; m + 1 < R; ++m) r[m] = r[m + 1];
            }
          }
        }
      } else {
#pragma unroll 1
        for (int i = t; i < a.vocab; i += NT) {
          const uint32_t k = key_of(x[i]);
          if (k && Place(a, p, k).listed(p)) f(rank_of(k, i));
        }
      }
    };
    auto sum = [&](u64 v) {
      u64 total;
      block_scan(v, sm.wave, &total);
      return total;
    };
    // a listed token is in top-k's bin, or in one where top-p may cut, or both
    const bool k_cuts = p.kb >= 0, p_cuts = p.lo <= p.hi, both = k_cuts && p_cuts;
    auto in_k = [&](u64 r) { return !both || bin_of(r) == p.kb; };
    auto in_p = [&](u64 r) { return !both || bin_of(r) <= p.hi; };
    const uint32_t top = key_of(p.top);
    auto low = [&](int i) { return rank_of(max(key_of(p.x0[i]), 1u), kMaxVocab - 1); };
    auto high = [&](int i) { return rank_of(p.x1[i] < p.top ? key_of(p.x1[i]) : top, 0); };
    u64 all = p.total, k_cut = 0;
    if (k_cuts) {
      k_cut = select([&](auto &&f) { each_listed([&](u64 r) { if (in_k(r)) f(r); }); },
                     [](u64) { return 1ull; }, low(1), high(1), p.k_left, few, sm);
      if (both) {
        u64 m = 0;
        each_listed([&](u64 r) { if (in_k(r) && r >= k_cut) m += mass_of(r); });
        all = p.before_k + sum(m);
      }
      cut = k_cut;
    }
    if (p_cuts) {
      // (where min-p drops any token above these bins, it drops all that lie in them, and
      // it does not matter that the slices' mass lacks what top-p counts)
      u64 above = 0;
      for (int i = t; i < a.slices; i += NT) above += sm.mass[i];
      above = sum(above);
      const u64 want = __umul64hi(a.top_p64, all) + (a.top_p64 * all != 0);  // rounded up
      const u64 w = want > above ? want - above : 1;
      cut = select([&](auto &&f) { each_listed([&](u64 r) { if (r >= k_cut && in_p(r)) f(r); }); },
                   mass_of, low(0), high(0), w, few, sm);
    }
    each_listed([&](u64 r) {
      if (r >= cut && Place(a, p, rank_key(r)).likely(a, p))
        atomicAdd(&sm.mass[(uint32_t)rank_index(r) / (uint32_t)a.per], mass_of(r));
    });
  }
  __syncthreads();
  if (t == 0) sm.v[0] = 0, sm.pick = 0;
  __syncthreads();
  // the slice
  const u64 m0 = 2 * t < a.slices ? sm.mass[2 * t] : 0, m1 = 2 * t + 1 < a.slices ? sm.mass[2 * t + 1] : 0;
  u64 total;
  const u64 upto = block_scan(m0 + m1, sm.wave, &total);
  const float u = a.u[row];
  u64 want = 0;  // the token is the first with a running mass above this
  if (u >= 1.f)
    want = total - 1;
  else if (u > 0.f)
    want = __umul64hi((u64)((double)u * 18446744073709551616.0), total);
  const u64 before = upto - m0 - m1;
  if (before <= want && want < upto) {
    const bool second = want >= before + m0;
    sm.v[0] = 2 * t + second;
    sm.pick = want - before - (second ? m0 : 0);
  }
  __syncthreads();
  // and in it the wave's part of consecutive tokens, and of that the thread's.  Kept is what
  // lies at the cut or before it in the order, in a bin that is not dropped, and min-p leaves.
  const float cut_x = cut ? logit_of(rank_key(cut)) : -INFINITY;
  const int cut_i = rank_index(cut);
  const int last = max(max(p.sure, p.part) - 1, max(p.lo <= p.hi ? p.hi : 0, p.kb));
  auto kept = [&](float v, int i, double *m) {
    const bool finite = fabsf(v) < INFINITY;
    const double y = (double)(finite ? v : p.top) * a.s, fl = floor(y), db = p.id - fl;
    const int b = db < kRest ? (int)db : kRest;
    *m = sm.tab[b] * exp_part(y - fl);
    const int before = (int)(v > cut_x) | ((int)(v == cut_x) & (int)(i <= cut_i));
    const int likely = ((double)v - (double)p.top) * a.inv_t >= a.log_min;
    return (before & (int)finite & (int)(b <= last) & likely) != 0;  // no branches
  };
  const int lane = t & 63, w = t >> 6;
  const int i0 = sm.v[0] * a.per, i1 = min(i0 + a.per, a.vocab);
  want = sm.pick;
  // A slice's mass was summed by bins and rounded otherwise: beyond its tokens' masses it
  // is the last one's, and tokens of less than half a unit count 1 where there are no others.
  u64 least = 0;
  auto units = [&](float x_i, int i) {
    double m;
    const bool is = kept(x_i, i, &m);
    const u64 v = to_units(m);
    return !is ? (u64)0 : v > least ? v : least;
  };
  constexpr int Q = E > 8 ? E / 8 : 1;  // tokens of a thread
  u64 in = 0;
  for (int turn = 0; turn < 2; ++turn) {
    const int j = i0 + w * (64 * E) + lane;
    float y[E];
    u64 own = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) y[k] = x[min(j + 64 * k, i1 - 1)];
#pragma unroll
    for (int k = 0; k < E; ++k) own += units(j + 64 * k < i1 ? y[k] : NAN, j + 64 * k);
    block_scan(own, sm.wave, &in);
    if (in) break;
    least = 1;
  }
  if (in == 0) return;
  if (want >= in) want = in - 1;
  u64 first = 0;
  for (int i = 0; i < w; ++i) first += sm.wave[i];
  if (lane == 0 && first <= want && want < first + sm.wave[w]) {
    sm.v[0] = w;
    sm.pick = want - first;
  }
  __syncthreads();
  const int j0 = i0 + (int)sm.v[0] * (64 * E), j1 = min(j0 + 64 * E, i1), j = j0 + Q * t;
  want = sm.pick;
  float y[Q];
  u64 v[Q], own = 0;
#pragma unroll
  for (int k = 0; k < Q; ++k) y[k] = x[min(j + k, j1 - 1)];
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    v[k] = units(j + k < j1 ? y[k] : NAN, j + k);
    own += v[k];
  }
  u64 left = want - (block_scan(own, sm.wave, &in) - own);
  if (left >= own) return;  // (also where what lies before is more than want)
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    if (left < v[k]) {
      double m;
      kept(y[k], j + k, &m);
      a.tokens[row] = j + k;
      if (a.probs) a.probs[row] = (float)(m / (double)total);
      return;
    }
    left -= v[k];
  }
}

__device__ __forceinline__ void none_finite(const SampleArgs &a, int row) {
  if (threadIdx.x == 0) {
    a.tokens[row] = -1;
    if (a.probs) a.probs[row] = 0.f;
  }
}

__device__ __forceinline__ void make_table(const SampleArgs &a, double *tab) {
  if (threadIdx.x < kBins)
    tab[threadIdx.x] =
        threadIdx.x < kRest ? exp(-(double)threadIdx.x / kPerUnit) * (a.unit * kHalfBin) : 0.0;
}

// From the row's largest logit, of whole part id, to a slice's: bins, at most kBins.
__device__ __forceinline__ int shift_of(const SampleArgs &a, double id, uint32_t key) {
  const double d = key ? id - floor((double)logit_of(key) * a.s) : kBins;
  return d < kBins ? (int)d : kBins;
}

// ALONE: nothing is cut.
template <int E, bool ALONE>
__global__ __launch_bounds__(NT, E > 8 ? 8 : 6) void sample_plan_kernel(SampleArgs a) {
  __shared__ Shared sm;
  const int t = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
  const float *x = a.x + (size_t)row * a.stride;
  float v[E];
  const int i0 = slice * (E * NT);
  uint32_t best = load_slice<E>(a, x, i0, min((E * NT), a.vocab - i0), v, sm);
  uint32_t *maxes = a.maxes + (size_t)row * a.slices;
  u64 *hist = a.hist + (size_t)row * a.slices * kBins;
  uint32_t *counts = a.counts + (size_t)row * a.slices * kBins;
  if (best) {
    slice_bins<E>(a, v, best, sm);
    if (ALONE) {
      u64 total;
      block_scan(t < kBins ? from_bin(sm.bins[t], t) : 0, sm.wave, &total);
      if (t == 0) a.mass[(size_t)row * a.slices + slice] = total;
    } else if (t < kBins) {
      put(hist + (size_t)slice * kBins + t, sm.bins[t]);
      if (a.top_k) put(counts + (size_t)slice * kBins + t, sm.cnt[t]);
    }
  }
  if (ALONE) {
    if (t == 0) maxes[slice] = best;
    return;
  }
  if (t == 0) put(maxes + slice, best);
  if (!last_block(a.count + row, a.slices, sm)) return;
  uint32_t *shift = reinterpret_cast<uint32_t *>(sm.mass);
  best = 0;
  for (int i = t; i < a.slices; i += NT) {
    shift[i] = get(maxes + i);
    best = max(best, shift[i]);
  }
  best = block_max(best, sm);
  if (best == 0) {
    if (t == 0) a.plan[row].any = 0;
    return;
  }
  const float top = logit_of(best);
  const double id = floor((double)top * a.s);
  uint32_t n = 0;
  u64 m = 0;
  for (int i = t; i < a.slices; i += NT) shift[i] = shift_of(a, id, shift[i]);
  __syncthreads();
  // threads t and t + kBins take every other slice's bin t, a batch of loads at a time;
  // bins that a slice does not have re-read its bin t
  constexpr int U = E > 8 ? 8 : 16;
  const int bin = t & (kBins - 1);
  for (int i0 = t / kBins; i0 < a.slices; i0 += 2 * U) {
    u64 v[U];
    uint32_t c[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = min(i0 + 2 * j, a.slices - 1), b = bin - (int)shift[i];
      const size_t at = (size_t)i * kBins + (b >= 0 ? b : bin);
      v[j] = get(hist + at);
      c[j] = a.top_k ? get(counts + at) : 0;
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (i0 + 2 * j < a.slices && bin >= (int)shift[min(i0 + 2 * j, a.slices - 1)]) {
        m += v[j];
        n += c[j];
      }
  }
  __syncthreads();
  if (t >= kBins) sm.bins[bin] = m, sm.cnt[bin] = n;
  __syncthreads();
  if (t < kBins)
    m += sm.bins[t], n += sm.cnt[t];
  else
    m = n = 0;
  make_plan(a, top, n, m, sm);
  if (t == 0) a.plan[row] = sm.plan;
}

template <int E>
__global__ __launch_bounds__(NT, 8) void sample_pick_kernel(SampleArgs a) {
  __shared__ double tab[kBins];
  __shared__ u64 near[kNear], wave[kWaves];
  __shared__ Plan p;
  __shared__ uint32_t found, base;
  const int t = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
  const float *x = a.x + (size_t)row * a.stride;
  Plan *plan = a.plan + row;
  constexpr int C = 8;  // logits per thread at a time
  const int i0 = slice * (E * NT), n = min(E * NT, a.vocab - i0);
  float v[C];
  auto load = [&](int c) {
#pragma unroll
    for (int e = 0; e < C; ++e) {
      const int i = t + NT * (c * C + e);
      v[e] = i < n ? x[i0 + i] : NAN;
    }
  };
  u64 *list = a.list + (size_t)row * a.list_len;
  load(0);
  const uint32_t best = a.maxes[(size_t)row * a.slices + slice];
  const u64 bin = a.hist[((size_t)row * a.slices + slice) * kBins + (t & (kBins - 1))];
  make_table(a, tab);
  if (t == 0) p = *plan, found = 0;
  __syncthreads();
  if (!p.any) return;
  u64 m = 0;
  if (best && t < kBins) {
    const double d = p.id - floor((double)logit_of(best) * a.s) + t;
    if (d < p.sure) m = from_bin(bin, (int)d);
  }
  const float x0 = p.x0[0], x1 = p.x1[0], k0 = p.x0[1], k1 = p.x1[1];
  // From `near` to the list (for the whole block); the row is read again at its end if more than
  // fit are found.
  auto put_list = [&] {
    __syncthreads();
    const uint32_t n = found;
    if (t == 0 && n) base = atomicAdd(&plan->n, n <= kNear ? n : a.list_len + 1u);
    __syncthreads();
    if (n <= kNear)
      for (uint32_t i = t; i < n && base + i < (uint32_t)a.list_len; i += NT) list[base + i] = near[i];
  };
  for (int c = 0;;) {
    uint32_t near_by = 0;
    float u[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
      u[e] = v[e];
      if ((u[e] >= x0 && u[e] <= x1) || (u[e] >= k0 && u[e] <= k1)) near_by |= 1u << e;
    }
    const bool more = ++c < E / C;
    if (more) load(c);
#pragma unroll
    for (int e = 0; e < C; ++e) {
      if (!(near_by >> e & 1)) continue;
      const uint32_t key = key_of(u[e]);
      if (!key) continue;
      const Place at(a, p, key);
      if (at.partial(p)) {
        if (at.likely(a, p)) m += to_units(at.mass(tab));
      } else if (at.listed(p)) {
        const uint32_t pos = atomicAdd(&found, 1u);
        if (pos < kNear) near[pos] = rank_of(key, i0 + t + NT * ((c - 1) * C + e));
      }
    }
    if (!more) break;
    if (p.about <= kNear) continue;
    put_list();  // so that the next ones fit
    __syncthreads();
    if (t == 0) found = 0;
    __syncthreads();
  }
  u64 total;
  block_scan(m, wave, &total);
  if (t == 0) a.mass[(size_t)row * a.slices + slice] = total;
  put_list();
}

// A block per row.
template <int E, bool ALONE>
__global__ __launch_bounds__(NT, 2) void sample_finish_kernel(SampleArgs a) {
  __shared__ Shared sm;
  __shared__ u64 near[ALONE ? 1 : kNear];
  const int t = threadIdx.x, row = blockIdx.x;
  const float *x = a.x + (size_t)row * a.stride;
  const u64 *mass = a.mass + (size_t)row * a.slices;
  if (ALONE) {
    const uint32_t *maxes = a.maxes + (size_t)row * a.slices;
    uint32_t key[2], best = 0;
    u64 m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = min(t + NT * j, a.slices - 1);
      key[j] = maxes[i];
      m[j] = mass[i];
      best = max(best, key[j]);
    }
    make_table(a, sm.tab);
    best = block_max(best, sm);
    if (best == 0) return none_finite(a, row);
    const float top = logit_of(best);
    const double id = floor((double)top * a.s);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      sm.mass[t + NT * j] =
          t + NT * j < a.slices && key[j] ? from_bin(m[j], shift_of(a, id, key[j])) : 0;
    make_plan(a, top, 0, 0, sm);
    finish_row<E, kNoList>(a, x, row, sm, nullptr);
  } else {
    const u64 first = a.list[(size_t)row * a.list_len + t];
    for (int i = t; i < a.slices; i += NT) sm.mass[i] = mass[i];
    if (t == 0) sm.plan = a.plan[row];
    make_table(a, sm.tab);
    near[t] = first;
    __syncthreads();
    if (!sm.plan.any) return none_finite(a, row);
    finish_row<E, kMemory>(a, x, row, sm, near);
  }
}

// All of it for rows of one slice.
template <int E>
__global__ __launch_bounds__(NT) void sample_row_kernel(SampleArgs a) {
  __shared__ Shared sm;
  __shared__ u64 near[E * NT < kNear ? E * NT : kNear];
  const int t = threadIdx.x, row = blockIdx.x;
  const float *x = a.x + (size_t)row * a.stride;
  float v[E];
  const uint32_t best = load_slice<E>(a, x, 0, a.vocab, v, sm);
  if (best == 0) {
    none_finite(a, row);
    return;
  }
  make_table(a, sm.tab);
  slice_bins<E>(a, v, best, sm);
  make_plan(a, logit_of(best), t < kBins ? sm.cnt[t] : 0,
            t < kBins ? sm.bins[t] : 0, sm);
  Plan &p = sm.plan;
  u64 m = t < p.sure && t < kBins ? from_bin(sm.bins[t], t) : 0, total;
  if (p.sure < p.part || p.lo <= p.hi || p.kb >= 0) {
    if (t == 0) sm.n = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t key = key_of(v[e]);
      if (!key) continue;
      const Place at(a, p, key);
      if (at.partial(p)) {
        if (at.likely(a, p)) m += to_units(at.mass(sm.tab));
      } else if (at.listed(p)) {
        const uint32_t pos = atomicAdd(&sm.n, 1u);
        if (pos < kNear) near[pos] = rank_of(key, t + NT * e);
      }
    }
    __syncthreads();
    if (t == 0) p.n = sm.n <= kNear ? sm.n : a.list_len + 1u;  // more than fit: the row is read again
  }
  block_scan(m, sm.wave, &total);
  if (t == 0) sm.mass[0] = total;
  __syncthreads();
  finish_row<E, kLds>(a, x, row, sm, near);
}

Workspace g_sample_ws, g_sample_count;

int cdiv(int a, int b) { return (a + b - 1) / b; }

// Rows of several slices, at most kMaxRows of them.
int launch_slices(SampleArgs a, int rows) {
  const bool alone = !a.top_k && !a.top_p64 && a.log_min == -INFINITY;
  // 4096 logits to a slice, for few rows' latency; 16384 where these fill the GPU and there are
  // histograms, a quarter as many then.  us per call at 262144 logits, slices of 4096 / 16384, with
  // top-p: 8 rows 38 / 45, 16 rows 48 / 48, 32 rows 64 / 55, 64 rows 94 / 70 (of 8192: 72); by
  // the temperature alone 64 rows 29 / 36
  const int e = !alone && (long)rows * cdiv(a.vocab, 32 * NT) >= 512 ? 32 : 8;
  a.per = e * NT;
  a.slices = cdiv(a.vocab, a.per);
  const size_t n = (size_t)rows * a.slices;
  const size_t plan = ((size_t)rows * sizeof(Plan) + 15) & ~size_t(15), max = (n * 4 + 15) & ~size_t(15);
  const size_t bytes = plan + max + n * 8 + (size_t)rows * a.list_len * 8 + n * kBins * 12;
  void *mem = nullptr, *count = nullptr;
  int rc = g_sample_count.get(kMaxRows * 4, &count, "g4_sample");  // zeros when new
  if (!rc) rc = g_sample_ws.get(bytes, &mem, "g4_sample");
  if (rc) return rc;
  uint8_t *at = static_cast<uint8_t *>(mem);
  a.plan = reinterpret_cast<Plan *>(at);
  a.maxes = reinterpret_cast<uint32_t *>(at + plan);
  a.mass = reinterpret_cast<u64 *>(at + plan + max);
  a.list = a.mass + n;
  a.hist = a.list + (size_t)rows * a.list_len;
  a.counts = reinterpret_cast<uint32_t *>(a.hist + n * kBins);
  a.count = static_cast<uint32_t *>(count);
  const dim3 grid(a.slices, rows);
  hipLaunchKernelGGL((alone    ? sample_plan_kernel<8, true>
                      : e == 8 ? sample_plan_kernel<8, false>
                               : sample_plan_kernel<32, false>),
                     grid, dim3(NT), 0, stream(), a);
  G4_LAUNCH_CHECK("sample_plan_kernel");
  if (!alone) {
    hipLaunchKernelGGL(e == 8 ? sample_pick_kernel<8> : sample_pick_kernel<32>, grid, dim3(NT), 0,
                       stream(), a);
    G4_LAUNCH_CHECK("sample_pick_kernel");
  }
  hipLaunchKernelGGL((alone    ? sample_finish_kernel<8, true>
                      : e == 8 ? sample_finish_kernel<8, false>
                               : sample_finish_kernel<32, false>),
                     dim3(rows), dim3(NT), 0, stream(), a);
  G4_LAUNCH_CHECK("sample_finish_kernel");
  return G4_OK;
}

// The call without its first r rows.
SampleArgs from_row(SampleArgs a, int r) {
  a.x += (size_t)r * a.stride;
  a.u += r;
  a.tokens += r;
  if (a.probs) a.probs += r;
  return a;
}

int launch_sample(SampleArgs a, int rows) {
  if (a.vocab <= kOneSlice) {
    a.slices = 1;
    a.per = kOneSlice;
    a.list_len = kNear;
    const auto kernel = a.vocab <= 4 * NT   ? sample_row_kernel<4>
                        : a.vocab <= 8 * NT ? sample_row_kernel<8>
                                            : sample_row_kernel<kOneSlice / NT>;
    for (int r = 0; r < rows;) {
      const int n = min(rows - r, kMaxShortRows);
      hipLaunchKernelGGL(kernel, dim3(n), dim3(NT), 0, stream(), from_row(a, r));
      G4_LAUNCH_CHECK("sample_row_kernel");
      r += n;
    }
    return G4_OK;
  }
  // Two cuts may lie in three bins.  us per call at 262144 logits of unit spread, temperature 1.5,
  // with lists of 16384 / 65536: by top-p 0.75 one row 635 / 68, 64 rows 1072 / 118; by top-k
  // 131072 and top-p 0.9 one row 1340 / 217, 64 rows 2159 / 317.
  a.list_len = max(kShortList, a.vocab / 4);
  const int most = min(kMaxRows, (int)(kListBytes / 8 / a.list_len));
  for (int r = 0; r < rows; r += most)
    if (int rc = launch_slices(from_row(a, r), min(rows - r, most))) return rc;
  return G4_OK;
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_sample(const float *logits, size_t stride, int rows, int vocab,
                     const g4_sample_params *params, const float *u, int32_t *tokens, float *probs) {
  // (sizes in bytes stay far from 64 bits)
  if (rows < 0 || vocab <= 0 || vocab > kMaxVocab || stride < (size_t)vocab ||
      stride > (size_t(1) << 60) / (rows > 0 ? rows : 1))
    return fail(G4_E_ARG, "g4_sample: rows %d, vocab %d (1..%d), stride %zu", rows, vocab, kMaxVocab,
                stride);
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
  const bool greedy = p.temperature == 0.f;
  a.top_k = greedy ? 1 : p.top_k < vocab ? p.top_k : 0;
  a.inv_t = greedy ? 1.0 : 1.0 / (double)p.temperature;
  a.s = kPerUnit * a.inv_t;
  if (!greedy && p.top_p < 1.f) {
    a.top_p64 = (u64)ldexp((double)p.top_p, 64);
    if (a.top_p64 == 0) a.top_p64 = 1;
  }
  a.log_min = greedy ? -INFINITY : log((double)p.min_p);
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  a.unit = ldexp(1.0, bits > 12 ? 62 - bits : 50);
  a.u = u;
  a.tokens = tokens;
  a.probs = probs;
  rc = launch_sample(a, rows);
  return rc ? rc : ok();
}
