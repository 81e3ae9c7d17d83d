// The weight that each key of a cache got, summed over query rows and heads: from kept scores, and
// the scores of FP32 keys.
#include <math.h>

#include "g4_gemv.h"
#include "g4_internal.h"
#include "g4_key_weights.h"
#include "g4_kv4.h"

namespace g4 {

constexpr size_t kScoreFloats = size_t(64) << 20;  // kept at once, unless a few rows take more

int check_weighted(int qrows, int heads, int keylen, int qpos0, int sliding, int window,
                   const float *before, const float *weights, const char *who) {
  if (qrows < 0 || qrows > 1 << 20 || heads <= 0 || heads > 8 || keylen < 0 || keylen > 1 << 28)
    return fail(G4_E_ARG, "%s: qrows %d (<= 2^20), heads %d (<= 8), keylen %d (<= 2^28)", who, qrows,
                heads, keylen);
  if (qpos0 < 0 || qpos0 > keylen - qrows || (sliding && window <= 0))
    return fail(G4_E_ARG, "%s: keylen %d must cover query positions %d.. + %d (window %d)", who,
                keylen, qpos0, qrows, window);
  if (before && weights && before != weights && overlap(before, (size_t)keylen * 4, weights, (size_t)keylen * 4))
    return fail(G4_E_ARG, "%s: before overlaps weights", who);
  return G4_OK;
}

// The most rows r with r * heads * keys <= kScoreFloats, where they see no more than the call's keys, or
// than window + r of them.
int weighted_rows(int qrows, int heads, int qpos0, int window) {
  const double most = (double)(kScoreFloats / heads), w = window;
  double rows = most / (qpos0 + qrows);
  if (window > 0) rows = fmax(rows, (sqrt(w * w + 4 * most) - w) / 2);
  return rows >= qrows ? qrows : rows < 8 ? 8 : (int)rows;
}

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSplits = 512;

__global__ __launch_bounds__(256) void weights_kernel(SumArgs a) { add_weights(a, blockIdx.x, blockIdx.y); }

// (A single launch for any rows, 32 keys per block of 1024 threads, takes 15.8 us where these two take
// 8.1 and 3.9: 2048 rows over 4096 keys.)
// Adds the groups of a key, 16 of them under way together.
__global__ __launch_bounds__(64) void weights_join_kernel(SumArgs a, int groups) {
  const int key = a.key0 + blockIdx.x * 64 + threadIdx.x;
  if (key >= a.keylen) return;
  const float before = a.before ? a.before[key] : 0.f;
  float sum = 0.f;
  if (key >= a.s.first && key < a.s.end) {
    const size_t step = a.s.end - a.s.first;
    const float *p = a.part + (key - a.s.first);
    for (int g = 0; g < groups; g += kBatch) {
      float x[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) x[i] = p[min(g + i, groups - 1) * step];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (g + i < groups) sum += x[i];
    }
  }
  a.weights[key] = before + sum;
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

}  // namespace

size_t score_stride(int keys) { return (size_t)((keys + 3) & ~3) + 32; }
Scores scores_of(int qrows, int heads, int pos0, int window) {
  Scores s{};
  s.rows = qrows * heads;
  s.heads = heads;
  s.pos0 = pos0;
  s.window = window;
  s.first = window > 0 && pos0 >= window ? pos0 - window + 1 : 0;
  s.end = pos0 + qrows;
  s.stride = score_stride(s.end - s.first);
  return s;
}
int growing_scratch(Workspace &ws, size_t need, void **p, const char *who) {
  const size_t ahead = ws.bytes + ws.bytes / 2;
  if (need > ws.bytes && need < ahead && !encoding()) {
    const int rc = ws.get(ahead, p, who);
    if (rc != G4_E_NOMEM) return rc;
  }
  return ws.get(need, p, who);
}
size_t weight_part_floats(int rows, int keys) {
  return rows > kGroup ? (size_t)cdiv(rows, kGroup) * keys : 0;
}

int launch_weights_join(const Scores &s, int key0, int keylen, float *part, const float *before, float *weights) {
  hipLaunchKernelGGL(weights_join_kernel, dim3(cdiv(keylen - key0, 64)), dim3(64), 0, stream(),
                     (SumArgs{s, key0, keylen, before, weights, part}), cdiv(s.rows, kGroup));
  G4_LAUNCH_CHECK("weights_join_kernel");
  return G4_OK;
}

int launch_weights(const Scores &s, int key0, int keylen, float *part, const float *before, float *weights) {
  const bool several = s.rows > kGroup;
  hipLaunchKernelGGL(weights_kernel, dim3(cdiv(several ? s.end - s.first : keylen - key0, 256), several ? cdiv(s.rows, kGroup) : 1),
                     dim3(256), 0, stream(), (SumArgs{s, key0, keylen, before, weights, several ? part : nullptr}));
  G4_LAUNCH_CHECK("weights_kernel");
  return several ? launch_weights_join(s, key0, keylen, part, before, weights) : G4_OK;
}

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;

struct ScoreArgs {
  const float *q, *k;
  Scores s;
};

// Eight FP32 values, times `up`, as sums of two FP16 values.
__device__ __forceinline__ void halves(const f32x4 &a, const f32x4 &b, float up, half8_t &h, half8_t &l) {
  u32x4 x, y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2_t z = {(i < 2 ? a[2 * i] : b[2 * i - 4]) * up, (i < 2 ? a[2 * i + 1] : b[2 * i - 3]) * up};
    const half2_t u = __builtin_convertvector(z, half2_t);
    x[i] = __builtin_bit_cast(uint32_t, u);
    y[i] = __builtin_bit_cast(uint32_t,
                              __builtin_convertvector(z - __builtin_convertvector(u, f32x2_t), half2_t));
  }
  h = __builtin_bit_cast(half8_t, x);
  l = __builtin_bit_cast(half8_t, y);
}
__device__ __forceinline__ float largest(const f32x4 &a, const f32x4 &b) {
  float m = fmaxf(fabsf(a[0]), fabsf(a[1]));
  m = fmaxf(m, fmaxf(fabsf(a[2]), fabsf(a[3])));
  m = fmaxf(m, fmaxf(fabsf(b[0]), fabsf(b[1])));
  return fmaxf(m, fmaxf(fabsf(b[2]), fabsf(b[3])));
}
// max over the lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float group_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Scores of 16 RT rows and a run of steps of 16 NT keys, which the block's KG key groups take in
// turn; the DQ waves of a group share the head dim and add their scores through LDS, in order.
// q and k enter the FP16 matrix cores as two values each (hi hi, hi lo and lo hi; lo lo is below
// 2^-22 of a product), q with its row's largest at the exponent 13, k times 2^8; a wave in which a
// key's largest then is outside 2^-2 .. 2^15 does its step again with these keys' exponents.  (The
// attention over FP32 caches takes three BF16 parts of each, all 24 bits, in six products.  What these sums
// decide is which rows are heavier; with three products they are about as near to 64 bits as sums of FP32
// products, 5.1e-7 for 5.2e-7 and 4.2e-8 for 1.0e-7 of one and of 256 rows, and small values beside large
// ones keep what the header says.)
// One token over 8001 keys of 512 (16.4 MB): 6.1 us without the sums, a step per wave whose loads are all
// under way before q is ready; over 131072 keys 268 MB in 56 us with the sums, 4.8 TB/s: memory.
template <int HD, int DQ, int NT, int RT, int W>
struct ScoreSmem {
  static constexpr int KG = W / DQ, R = 16 * RT;
  u32x4 q[2][RT][HD / 32][64];
  f32x4 sx[DQ > 1 ? 2 : 1][KG][DQ][DQ > 1 ? RT : 1][DQ > 1 ? NT : 1][DQ > 1 ? 64 : 1];
  int xq[R];
  float2 wml[KG][R];
};
template <int HD, int DQ, int NT, int RT, int W>
__device__ __forceinline__ void few_scores(const ScoreArgs &a, int R0, int split, const Run &run,
                                           ScoreSmem<HD, DQ, NT, RT, W> &sm) {
  constexpr int KG = W / DQ, DW = HD / DQ, KN = DW / 32, R = 16 * RT, KEYS = 16 * NT;
  constexpr int AHEAD = NT * KN <= 4 ? KN : 2;  // a step's loads that are under way together
  const Scores &S = a.s;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kg = w / DQ, dq = w % DQ, c = lane & 15, g = lane >> 4;
  const int pa = S.pos0 + R0 / S.heads, pb = S.pos0 + (min(R0 + R, S.rows) - 1) / S.heads;
  const int lo = run.lo, hi = run.hi, steps = run.steps, t0 = run.t0, t1 = run.t1;

  f32x4 kr[AHEAD][NT][2];
  auto load_k = [&](int step, int n, f32x4 (&x)[NT][2]) {
    const int k0 = lo + min(step, steps - 1) * KEYS, last = hi - 1 - k0;
    const char *p = reinterpret_cast<const char *>(a.k + (size_t)k0 * HD + dq * DW);
#pragma unroll
    for (int T = 0; T < NT; ++T) {
      const uint32_t at = (uint32_t)(min(16 * T + c, last) * HD + 4 * g) * 4;
      x[T][0] = *reinterpret_cast<const f32x4 *>(p + at + 128 * n);
      x[T][1] = *reinterpret_cast<const f32x4 *>(p + at + 128 * n + 64);
    }
  };
  {
    constexpr int TW = HD / 8, PASS = 64 * W / TW;
    constexpr int N = (R + PASS - 1) / PASS < 4 ? (R + PASS - 1) / PASS : 4;  // rows of a thread under way together
    const int wd = t % TW;
    for (int first = 0; first < R; first += PASS * N) {
      const int r0 = first + t / TW;
      f32x4 x[N][2];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = min(R0 + min(r0 + PASS * i, R - 1), S.rows - 1);
        const f32x4 *p = reinterpret_cast<const f32x4 *>(a.q + (size_t)row * HD + 32 * (wd >> 2) + 4 * (wd & 3));
        x[i][0] = p[0];
        x[i][1] = p[4];
      }
      if (first == 0) {  // (q's loads first: it is worked on while k's are under way)
        asm volatile("" ::: "memory");
#pragma unroll
        for (int n = 0; n < (AHEAD == KN ? KN : 1); ++n) load_k(t0 + kg, n, kr[n]);
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = r0 + PASS * i;
        f32x4 x0 = x[i][0], x1 = x[i][1];
        int top = 0;  // as bits, where NaN > infinity > numbers
#pragma unroll
        for (int d = 0; d < 4; ++d)
          top = max(top, max(__float_as_int(x0[d]) & 0x7fffffff, __float_as_int(x1[d]) & 0x7fffffff));
        top = team_max<TW>(top);
        const int e = top == 0 || top >= 0x7f800000 ? 0 : max((top >> 23) - 127, -126);
        if (r >= R) break;
        if (wd == 0) sm.xq[r] = e - 13;
#pragma unroll
        for (int d = 0; d < 4; ++d) x0[d] = ldexpf(x0[d], 13 - e), x1[d] = ldexpf(x1[d], 13 - e);
        half8_t h, l;
        halves(x0, x1, 1.f, h, l);
        sm.q[0][r >> 4][wd >> 2][(r & 15) + 16 * (wd & 3)] = __builtin_bit_cast(u32x4, h);
        sm.q[1][r >> 4][wd >> 2][(r & 15) + 16 * (wd & 3)] = __builtin_bit_cast(u32x4, l);
      }
    }
  }
  __syncthreads();

  int pos[RT], xe[RT];
  float m[RT], l[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    pos[r] = S.pos0 + min(R0 + 16 * r + c, S.rows - 1) / S.heads;
    xe[r] = sm.xq[16 * r + c];
    m[r] = kNoScore;
    l[r] = 0.f;
  }
  const int turns = (t1 - t0 + KG - 1) / KG;
  for (int it = 0; it < turns; ++it) {
    const int step = t0 + kg + it * KG, key0 = lo + step * KEYS;
    const bool mine = step < t1;
    f32x4 s[RT][NT];
    float up[NT], top[NT];
#pragma unroll
    for (int T = 0; T < NT; ++T) up[T] = 256.f;
    bool again = false;
    for (int turn = 0; turn < 2; ++turn) {
#pragma unroll
      for (int T = 0; T < NT; ++T) top[T] = 0.f;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < NT; ++T) s[r][T] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int n0 = 0; n0 < KN; n0 += AHEAD)
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int n = n0 + e;
        const bool more = n + 1 < KN;
        if constexpr (AHEAD < KN) load_k(more ? step : step + KG, more ? n + 1 : 0, kr[1 - e]);
        half8_t kh[NT], kl[NT];
#pragma unroll
        for (int T = 0; T < NT; ++T) {
          top[T] = fmaxf(top[T], largest(kr[e][T][0], kr[e][T][1]));
          halves(kr[e][T][0], kr[e][T][1], up[T], kh[T], kl[T]);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const half8_t qh = __builtin_bit_cast(half8_t, sm.q[0][r][dq * KN + n][lane]);
          const half8_t ql = __builtin_bit_cast(half8_t, sm.q[1][r][dq * KN + n][lane]);
#pragma unroll
          for (int T = 0; T < NT; ++T)
            s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[T], ql, s[r][T], 0, 0, 0);
#pragma unroll
          for (int T = 0; T < NT; ++T)
            s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[T], qh, s[r][T], 0, 0, 0);
#pragma unroll
          for (int T = 0; T < NT; ++T)
            s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[T], qh, s[r][T], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (turn == 1) break;
      bool fits = true;
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        top[T] = group_max(top[T]);
        // (rows without numbers give scores that are none either way)
        fits = fits && (top[T] == 0.f || (top[T] >= 0x1p-10f && top[T] < 128.f) || !(top[T] < INFINITY));
      }
      again = !__all(fits);
      if (!again) break;
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        const int e = top[T] < INFINITY ? min(max((int)(__float_as_uint(top[T]) >> 23) - 127, -100), 127) : 0;
        up[T] = __int_as_float((127 + 8 - e) << 23);
      }
      if constexpr (AHEAD < KN) load_k(step, 0, kr[0]);
    }
    if constexpr (AHEAD == KN) {
      if (it + 1 < turns)
#pragma unroll
        for (int n = 0; n < KN; ++n) load_k(step + KG, n, kr[n]);
    }
#pragma unroll
    for (int T = 0; T < NT; ++T) {
      int ke[4] = {-8, -8, -8, -8};
      if (again)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ke[i] = 127 - (int)(__shfl((int)__float_as_uint(up[T]), 4 * g + i, 64) >> 23);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][T][i] = ldexpf(s[r][T][i] * kLog2e, xe[r] + ke[i]);
    }
    if constexpr (DQ > 1) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < NT; ++T) sm.sx[it & 1][kg][dq][r][T][lane] = s[r][T];
      __syncthreads();
      if (dq > 0) continue;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < NT; ++T)
#pragma unroll
          for (int d = 1; d < DQ; ++d) s[r][T] += sm.sx[it & 1][kg][d][r][T][lane];
    }
    if (!mine) continue;
    const bool inner = key0 + KEYS - 1 <= pa && (S.window == 0 || key0 > pb - S.window);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (!inner) {
#pragma unroll
        for (int T = 0; T < NT; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * T + 4 * g + i;
            if (key > pos[r] || (S.window > 0 && key <= pos[r] - S.window)) s[r][T][i] = -INFINITY;
          }
      }
      const int row = min(R0 + 16 * r + c, S.rows - 1);
      float tm = kNoScore;
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        *reinterpret_cast<f32x4 *>(S.score + (size_t)row * S.stride + (key0 + 16 * T + 4 * g - S.first)) = s[r][T];
        tm = fmaxf(tm, fmaxf(fmaxf(s[r][T][0], s[r][T][1]), fmaxf(s[r][T][2], s[r][T][3])));
      }
      // (fmaxf drops a NaN score, whose weight is NaN.)
      const float mn = fmaxf(m[r], group_max(tm));
      float sum = 0.f;
#pragma unroll
      for (int T = 0; T < NT; ++T)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(s[r][T][i] - mn);
      l[r] = fmaf(l[r], __builtin_amdgcn_exp2f(m[r] - mn), sum);
      m[r] = mn;
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    if (g == 0 && dq == 0) sm.wml[kg][16 * r + c] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  for (int r = t; r < R; r += 64 * W) {
    if (R0 + r >= S.rows) break;
    float M = kNoScore, L = 0.f;
    for (int i = 0; i < KG; ++i) M = fmaxf(M, sm.wml[i][r].x);
    for (int i = 0; i < KG; ++i) L = fmaf(sm.wml[i][r].y, __builtin_amdgcn_exp2f(sm.wml[i][r].x - M), L);
    S.ml[(size_t)(R0 + r) * S.splits + split] = make_float2(M, L);
  }
}

template <int HD, int DQ, int NT, int RT>
__global__ __launch_bounds__(64 * kWaves) void scores_kernel(ScoreArgs a) {
  __shared__ ScoreSmem<HD, DQ, NT, RT, kWaves> sm;
  const int R0 = blockIdx.x * sm.R;
  few_scores<HD, DQ, NT, RT, kWaves>(a, R0, blockIdx.y, Run(a.s, R0, sm.R, blockIdx.y, 16 * NT), sm);
}

// Many rows: a block owns 16 RT rows and a run of 32-key steps; its W waves share the head dim, so that
// each k is split into its two values once for all rows, with q in registers.  The waves' partial
// scores go through LDS; wave w adds those of rows 16 (w % RT) .. and, of these, keys 16 (w / RT) ..
// in order and keeps the running maximum and sum of its own.
// k times 2^8 in FP16 ends at 2^-24: what is lost of each is 2^-33, which 512 q below 16 make less
// than 10^-6 of a score.  A block with a k of 128 or more, with larger q and a key that is below
// 2^-10 throughout, or with a q below 2^-99, does its rows again, as scores_kernel does.
// 256 rows over 4096 keys of 512 (8 heads, 25 GFLOP with the three products): 45.9 us without the sums.
// Before its first step a block needs 10 us (its 128 KB of q 3.7, their parts 1.8, the first keys and
// products 3); a step takes 2.3: without its loads the call would take 11 us less, without two of its
// three products 4, without a third of its vector instructions nothing.  The whole call, 55, when it took
// 57: with 32 rows per block 85; with blocks of 4 waves, two per CU, alike.
template <int HD, int RT, int W>
__global__ __launch_bounds__(64 * W, 2) void scores_rows_kernel(ScoreArgs a) {
  constexpr int DW = HD / W, KN = DW / 32, R = 16 * RT, NT = W / RT, KEYS = 16 * NT;
  static_assert(W % RT == 0, "a tile per wave");
  union Smem {
    f32x4 sx[2][W][RT][NT][64];
    float rows[R][HD + 4];  // q, on its way from whole lines of memory
    ScoreSmem<HD, 1, NT, RT, W> general;
  };
  __shared__ Smem sm;
  __shared__ float stop[2][W][KEYS];  // the keys' largest values
  __shared__ int sq[W][R], sxq[R];    // q's largest, q's exponents
  __shared__ float2 wml[NT][R];
  const Scores &S = a.s;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int R0 = blockIdx.x * R, split = blockIdx.y;
  const Run run(S, R0, R, split, KEYS);
  const int lo = run.lo, hi = run.hi, steps = run.steps, t0 = run.t0, t1 = run.t1;
  bool fits = true, large = false;  // large: some q of 16 or more, for which small k matter

  struct Keys {
    f32x4 x[NT][KN][2];
  };
  Keys ka, kb;  // of the next step and the one after it
  auto load_k = [&](int step, Keys &kr) {
    const int k0 = __builtin_amdgcn_readfirstlane(lo + min(step, steps - 1) * KEYS), last = hi - 1 - k0;
    const char *p = reinterpret_cast<const char *>(a.k + (size_t)k0 * HD + w * DW);
#pragma unroll
    for (int T = 0; T < NT; ++T) {
      const uint32_t at = (uint32_t)(min(16 * T + c, last) * HD + 4 * g) * 4;
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        kr.x[T][n][0] = *reinterpret_cast<const f32x4 *>(p + at + 128 * n);
        kr.x[T][n][1] = *reinterpret_cast<const f32x4 *>(p + at + 128 * n + 64);
      }
    }
  };
  load_k(t0, ka);
  // q: lane (c, g) holds its row's dims 32 n + 4 g .. + 3 and + 16 .. + 19 of the wave's, k alike: a
  // load takes 64 consecutive bytes of each key
  half8_t qh[RT][KN], ql[RT][KN];
  {
    constexpr int U = R * HD / 4 / (64 * W);
    f32x4 y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + 64 * W * i, row = min(R0 + u / (HD / 4), S.rows - 1);
      y[i] = *reinterpret_cast<const f32x4 *>(a.q + (size_t)row * HD + u % (HD / 4) * 4);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = t + 64 * W * i;
      *reinterpret_cast<f32x4 *>(&sm.rows[u / (HD / 4)][u % (HD / 4) * 4]) = y[i];
    }
    __syncthreads();
    f32x4 x[RT][KN][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(&sm.rows[16 * r + c][w * DW + 32 * n + 4 * g]);
        x[r][n][0] = p[0];
        x[r][n][1] = p[4];
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      int top = 0;  // as bits, where NaN > infinity > numbers
#pragma unroll
      for (int n = 0; n < KN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = max(top, max(__float_as_int(x[r][n][0][i]) & 0x7fffffff, __float_as_int(x[r][n][1][i]) & 0x7fffffff));
      top = max(top, __shfl_xor(top, 16, 64));
      top = max(top, __shfl_xor(top, 32, 64));
      if (g == 0) sq[w][16 * r + c] = top;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      int top = 0;
#pragma unroll
      for (int d = 0; d < W; ++d) top = max(top, sq[d][16 * r + c]);
      const int e = top == 0 || top >= 0x7f800000 ? 0 : max((top >> 23) - 127, -126);
      if (w == 0 && g == 0) sxq[16 * r + c] = e - 21;  // (8 of k's)
      fits = fits && e >= -99;
      large = large || e >= 4;
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        f32x4 x0 = x[r][n][0], x1 = x[r][n][1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x0[i] = ldexpf(x0[i], 13 - e), x1[i] = ldexpf(x1[i], 13 - e);
        halves(x0, x1, 1.f, qh[r][n], ql[r][n]);
      }
    }
  }
  large = __any(large);
  auto scores = [&](int step, const Keys &kr, Keys &next) {
    load_k(step + 1, next);
    __builtin_amdgcn_sched_barrier(0);  // (before this step's are split)
    f32x4 s[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int T = 0; T < NT; ++T) s[r][T] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int at = (step - t0) & 1;
#pragma unroll
    for (int T = 0; T < NT; ++T) {
      float top = 0.f;
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        half8_t kh, kl;
        top = fmaxf(top, largest(kr.x[T][n][0], kr.x[T][n][1]));
        halves(kr.x[T][n][0], kr.x[T][n][1], 256.f, kh, kl);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[r][n], s[r][T], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[r][n], s[r][T], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[r][n], s[r][T], 0, 0, 0);
      }
      fits = fits && (top < 128.f || !(top < INFINITY));  // (what is no number gives scores that are none)
      if (large) {
        top = group_max(top);
        if (g == 0) stop[at][w][16 * T + c] = top;
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int T = 0; T < NT; ++T) sm.sx[at][w][r][T][lane] = s[r][T];
  };

  // this wave's rows and keys
  const int mr = w % RT, mt = w / RT;
  const int my_row = min(R0 + 16 * mr + c, S.rows - 1), my_pos = S.pos0 + my_row / S.heads;
  float m = kNoScore, l = 0.f;
  if (t0 < t1) scores(t0, ka, kb);
  asm volatile("" ::: "memory");  // (else loads move into the loop, with an address of 64 bits each)
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the waits in the loop then count its own loads
  __syncthreads();
  const float factor = ldexpf(kLog2e, sxq[16 * mr + c]);
  auto turn = [&](int step, const Keys &kr, Keys &next) {
    const int key0 = lo + step * KEYS, at = (step - t0) & 1;
    f32x4 y[W];  // (loaded before the next step's products)
#pragma unroll
    for (int d = 0; d < W; ++d) y[d] = sm.sx[at][d][mr][mt][lane];
    // (behind the last one: keys of no score of this block, which may send it the general way all the same)
    scores(step + 1, kr, next);
    f32x4 x = y[0];
#pragma unroll
    for (int d = 1; d < W; ++d) x += y[d];
    x *= factor;
    if (large && lane < KEYS) {
      float top = stop[at][0][lane];
      for (int d = 1; d < W; ++d) top = fmaxf(top, stop[at][d][lane]);
      fits = fits && (top == 0.f || top >= 0x1p-10f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key0 + 16 * mt + 4 * g + i;
      if (key > my_pos || (S.window > 0 && key <= my_pos - S.window)) x[i] = -INFINITY;
    }
    // (stored by all: behind a condition, the next wait for a load would wait for it too)
    *reinterpret_cast<f32x4 *>(S.score + (size_t)my_row * S.stride + (key0 + 16 * mt + 4 * g - S.first)) = x;
    // (fmaxf drops a NaN score, whose weight is NaN; a lane's maximum is its own until the end)
    const float mn = fmaxf(fmaxf(fmaxf(m, x[0]), fmaxf(x[1], x[2])), x[3]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(x[i] - mn);
    l = fmaf(l, __builtin_amdgcn_exp2f(m - mn), sum);
    m = mn;
    __syncthreads();
  };
  for (int step = t0; step < t1; step += 2) {
    turn(step, kb, ka);
    if (step + 1 < t1) turn(step + 1, ka, kb);
  }
  const bool odd = !__all(fits);
  __syncthreads();
  if (lane == 0) sq[w][0] = odd;
  __syncthreads();
  int again = 0;
#pragma unroll
  for (int d = 0; d < W; ++d) again |= sq[d][0];
  if (__builtin_amdgcn_readfirstlane(again)) {
    few_scores<HD, 1, NT, RT, W>(a, R0, split, run, sm.general);
    return;
  }
  const float M = group_max(m);
  l *= __builtin_amdgcn_exp2f(m - M);
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) wml[mt][16 * mr + c] = make_float2(M, l);
  __syncthreads();
  if (t < R && R0 + t < S.rows) {
    float Mx = kNoScore, L = 0.f;
    for (int i = 0; i < NT; ++i) Mx = fmaxf(Mx, wml[i][t].x);
    for (int i = 0; i < NT; ++i) L = fmaf(wml[i][t].y, __builtin_amdgcn_exp2f(wml[i][t].x - Mx), L);
    S.ml[(size_t)(R0 + t) * S.splits + split] = make_float2(Mx, L);
  }
}

// The kernel for the call's rows: its rows per block, keys per step of all its waves, blocks per CU
// and threads.
struct ScorePlan {
  void (*kernel)(ScoreArgs);
  int rows, keys, per_cu, threads;
};
// 17 to 32 rows take the kernel of few rows, two tiles of them, where it has a block per CU at most: 32
// rows, us, in this and the other way, over 1000 / 8001 / 32000 keys of 256 10.5 / 14.3 / 21.7 and 14.8 /
// 16.8 / 21.3 (32, 251 and 1000 blocks), of 512 12.2 / 25.3 / 33.9 and 17.3 / 22.4 / 29.7 (63, 501, 2000).
template <int HD>
ScorePlan score_plan(int rows, int keys) {
  constexpr int DQ = HD >= 128 ? HD / 128 : 1, FEW = 16 * kWaves / DQ;
  if (rows <= 16) return {scores_kernel<HD, DQ, 1, 1>, 16, FEW, 2, 64 * kWaves};
  if (rows <= 32 && cdiv(keys, FEW) <= cu_count())
    return {scores_kernel<HD, DQ, 1, 2>, 32, FEW, 2, 64 * kWaves};
  if constexpr (HD == 512)
    return {scores_rows_kernel<HD, 4, 8>, 64, 32, 1, 512};
  else
    return {scores_kernel<HD, 1, 2, 4>, 64, 32 * kWaves, 2, 64 * kWaves};
}

// What one launch over s takes.
struct ScoreNeeds {
  ScorePlan plan;
  int blocks, splits;
  size_t score, ml, sum;  // floats
  size_t bytes() const { return (score + ml + sum) * 4; }
};
ScoreNeeds needs_of(const Scores &s, int head_dim) {
  const int keys = s.end - s.first;
  ScoreNeeds n;
  n.plan = head_dim == 64    ? score_plan<64>(s.rows, keys)
           : head_dim == 128 ? score_plan<128>(s.rows, keys)
           : head_dim == 256 ? score_plan<256>(s.rows, keys)
                             : score_plan<512>(s.rows, keys);
  const int steps = cdiv(keys, n.plan.keys);
  n.blocks = cdiv(s.rows, n.plan.rows);
  n.splits = n.plan.per_cu * cu_count() / n.blocks;
  if (n.splits > steps) n.splits = steps;
  if (n.splits > kMaxSplits) n.splits = kMaxSplits;
  if (n.splits < 1) n.splits = 1;
  n.score = s.rows * s.stride;
  n.ml = (size_t)n.splits * s.rows * 2;
  n.sum = weight_part_floats(s.rows, keys);
  return n;
}

Workspace g_weights_ws;

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_attention_weights(const float *q, const float *k, int qrows, int heads, int head_dim,
                                int keylen, int qpos0, int sliding, int window,
                                const float *before, float *weights) {
  const char *who = "g4_attention_weights";
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return fail(G4_E_ARG, "%s: head_dim %d (64, 128, 256 or 512)", who, head_dim);
  if (int rc = check_weighted(qrows, heads, keylen, qpos0, sliding, window, before, weights, who)) return rc;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k)) & 15)
    return fail(G4_E_ARG, "%s: q and k must be 16-byte aligned", who);
  if (overlap(weights, (size_t)keylen * 4, q, (size_t)qrows * heads * head_dim * 4) ||
      overlap(weights, (size_t)keylen * 4, k, (size_t)keylen * head_dim * 4))
    return fail(G4_E_ARG, "%s: weights overlaps q or k", who);
  G4_CHECK_INIT();
  if (keylen == 0) return ok();
  int rc = check_device_range(weights, (size_t)keylen * 4, "g4_attention_weights weights");
  if (!rc && before) rc = check_device_range(before, (size_t)keylen * 4, "g4_attention_weights before");
  if (!rc && qrows) rc = check_device_range(q, (size_t)qrows * heads * head_dim * 4, "g4_attention_weights q");
  if (!rc) rc = check_device_range(k, (size_t)keylen * head_dim * 4, "g4_attention_weights k");
  if (rc) return rc;
  const int win = sliding ? (window < keylen ? window : keylen) : 0;
  if (qrows == 0) {
    Scores s{};
    s.heads = 1;
    rc = launch_weights(s, 0, keylen, nullptr, before, weights);
    return rc ? rc : ok();
  }
  const int most = weighted_rows(qrows, heads, qpos0, win);
  auto scores_at = [&](int r0) { return scores_of(qrows - r0 < most ? qrows - r0 : most, heads, qpos0 + r0, win); };
  size_t need = 0;  // of the chunk that takes most, before the first one
  for (int r0 = 0; r0 < qrows; r0 += most) {
    const size_t n = needs_of(scores_at(r0), head_dim).bytes();
    if (n > need) need = n;
  }
  void *mem = nullptr;
  if ((rc = growing_scratch(g_weights_ws, need, &mem, who))) return rc;
  for (int r0 = 0; r0 < qrows; r0 += most) {
    ScoreArgs a{};
    a.q = q + (size_t)r0 * heads * head_dim;
    a.k = k;
    Scores &s = a.s = scores_at(r0);
    const ScoreNeeds n = needs_of(s, head_dim);
    s.splits = n.splits;
    s.score = static_cast<float *>(mem);
    s.ml = reinterpret_cast<float2 *>(s.score + n.score);
    hipLaunchKernelGGL(n.plan.kernel, dim3(n.blocks, n.splits), dim3(n.plan.threads), 0, stream(), a);
    G4_LAUNCH_CHECK("scores_kernel");
    // (later chunks add to the keys that they see)
    float *part = s.score + n.score + n.ml;
    rc = r0 ? launch_weights(s, s.first, s.end, part, weights, weights)
            : launch_weights(s, 0, keylen, part, before, weights);
    if (rc) return rc;
  }
  return ok();
}
