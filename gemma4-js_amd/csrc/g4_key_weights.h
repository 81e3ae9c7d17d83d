// The sums of the keys' weights over the rows whose scores were kept, for the kernels that form them.
#pragma once

#include <math.h>

#include "g4_kv4.h"

namespace g4 {
namespace {

constexpr float kNoScore = -3.4028235e38f;  // where a row's maximum starts
constexpr int kGroup = 32;                  // rows that a block adds up

struct SumArgs {
  Scores s;
  int key0, keylen;  // weights of keys key0 .. keylen - 1 are written
  const float *before;
  float *weights;
  float *part;  // [groups][end - first], or null
};

constexpr int kBatch = 16;  // loads of a thread that are under way together

// A thread per key adds up to 32 rows; `by` counts these groups, `bx` 256 keys each.  The first rows'
// scores are loaded before the rows' maxima and sums are known.  2048 rows over 4096 keys: 33.5 MB in
// 8.1 us, 4.1 TB/s; 8 rows over 8001 keys: 4.0 us, two loads and a launch.
__device__ __forceinline__ void add_weights(const SumArgs &a, int bx, int by) {
  __shared__ float4 stat[kGroup];  // maximum, 1 / sum, last and (window) first key as bits
  const Scores &s = a.s;
  const int t = threadIdx.x, r0 = by * kGroup, n = min(kGroup, s.rows - r0);
  const int key = bx * 256 + t + (a.part ? s.first : a.key0);
  const bool any = key >= s.first && key < s.end;
  const float *p = s.score + (size_t)r0 * s.stride + (any ? key - s.first : 0);
  float x[kBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x[i] = p[(size_t)min(i0 + i, n - 1) * s.stride];
  };
  const float before = !a.part && a.before && key < a.keylen ? a.before[key] : 0.f;
  if (n > 0) {
    load(0);
    int lanes = 4;  // per row
    while (lanes < 64 && lanes * 2 * n <= 256) lanes *= 2;
    const int i = t / lanes, row = r0 + min(i, n - 1);
    const float2 *ml = s.ml + (size_t)row * s.splits;
    float m = kNoScore, l = 0.f;
    for (int p0 = t % lanes; p0 < s.splits; p0 += 4 * lanes) {
      float2 y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = ml[min(p0 + e * lanes, s.splits - 1)];
      float mn = m;
#pragma unroll
      for (int e = 0; e < 4; ++e) mn = fmaxf(mn, y[e].x);
      l *= __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (p0 + e * lanes < s.splits) l = fmaf(y[e].y, __builtin_amdgcn_exp2f(y[e].x - mn), l);
      m = mn;
    }
    const float mine = m;
    m = team_max(lanes, m);
    l = team_sum(lanes, l * __builtin_amdgcn_exp2f(mine - m));
    if (t % lanes == 0 && i < n) {
      const int pos = s.pos0 + row / s.heads;
      stat[i] = make_float4(m, 1.f / l, __int_as_float(pos),
                            __int_as_float(s.window > 0 ? pos - s.window : -1));
    }
  }
  __syncthreads();
  float sum = 0.f;
  for (int i0 = 0; i0 < n; i0 += kBatch) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float4 st = stat[min(i0 + i, n - 1)];
      const bool sees = i0 + i < n && key <= __float_as_int(st.z) && key > __float_as_int(st.w);
      const float w = __builtin_amdgcn_exp2f(x[i] - st.x) * st.y;
      if (sees) sum += w;
    }
    if (i0 + kBatch < n) load(i0 + kBatch);
  }
  if (!any) sum = 0.f;
  if (a.part) {
    if (any) a.part[(size_t)by * (s.end - s.first) + (key - s.first)] = sum;
  } else if (key < a.keylen) {
    a.weights[key] = before + sum;
  }
}

}  // namespace
}  // namespace g4
