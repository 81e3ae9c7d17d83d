// The weight that each key of a cache got, summed over query rows and heads: from kept scores, and
// the scores of FP32 keys.
#include <math.h>

#include "g4_gemv.h"
#include "g4_internal.h"
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
  const uintptr_t b = reinterpret_cast<uintptr_t>(before), w = reinterpret_cast<uintptr_t>(weights);
  const uintptr_t bytes = (uintptr_t)keylen * 4;
  if (before && weights && before != weights && (b < w ? w - b : b - w) < bytes)
    return fail(G4_E_ARG, "%s: before overlaps weights", who);
  return G4_OK;
}

int weighted_rows(int qrows, int heads, int keylen, int qpos0, int window) {
  const size_t keys = window > 0 && window + qrows < keylen ? window + qrows : keylen;
  size_t rows = kScoreFloats / (keys * heads);
  if (rows < 8) rows = 8;
  return rows < (size_t)qrows ? (int)rows : qrows;
}

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3.4028235e38f;  // where a row's maximum starts
constexpr int kGroup = 64;                  // rows that a block adds up

struct SumArgs {
  Scores s;
  int keylen;
  const float *before;
  float *weights;
  float *part;  // [groups][end - first], or null
};

__global__ __launch_bounds__(256) void weights_kernel(SumArgs a) {
  __shared__ float2 stat[kGroup];  // maximum, 1 / sum
  const Scores &s = a.s;
  const int t = threadIdx.x, r0 = blockIdx.y * kGroup;
  const int key = blockIdx.x * 256 + t + (a.part ? s.first : 0);
  {
    const int row = min(r0 + t / 4, s.rows - 1);
    float m = kNoScore, l = 0.f;
    for (int p = t & 3; p < s.splits; p += 4) {
      const float2 x = s.ml[(size_t)p * s.rows + row];
      const float mn = fmaxf(m, x.x);
      l = l * __builtin_amdgcn_exp2f(m - mn) + x.y * __builtin_amdgcn_exp2f(x.x - mn);
      m = mn;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64), mn = fmaxf(m, m2);
      const float x = l * __builtin_amdgcn_exp2f(m - mn), y = l2 * __builtin_amdgcn_exp2f(m2 - mn);
      l = (t & o) ? y + x : x + y;
      m = mn;
    }
    if ((t & 3) == 0) stat[t / 4] = make_float2(m, 1.f / l);
  }
  __syncthreads();
  const int n = min(kGroup, s.rows - r0);
  float sum = 0.f;
  if (key >= s.first && key < s.end) {
    const float *p = s.score + (size_t)r0 * s.stride + (key - s.first);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const int pos = s.pos0 + (r0 + i) / s.heads;
      const bool sees = key <= pos && (s.window == 0 || key > pos - s.window);
      const float w = __builtin_amdgcn_exp2f(p[(size_t)i * s.stride] - stat[i].x) * stat[i].y;
      if (sees) sum += w;
    }
  }
  if (a.part) {
    if (key < s.end) a.part[(size_t)blockIdx.y * (s.end - s.first) + (key - s.first)] = sum;
  } else if (key < a.keylen) {
    a.weights[key] = (a.before ? a.before[key] : 0.f) + sum;
  }
}

__global__ __launch_bounds__(256) void weights_join_kernel(SumArgs a, int groups) {
  const int key = blockIdx.x * 256 + threadIdx.x;
  if (key >= a.keylen) return;
  float sum = 0.f;
  if (key >= a.s.first && key < a.s.end)
    for (int g = 0; g < groups; ++g) sum += a.part[(size_t)g * (a.s.end - a.s.first) + (key - a.s.first)];
  a.weights[key] = (a.before ? a.before[key] : 0.f) + sum;
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

}  // namespace

size_t weight_part_floats(int rows, int keys) {
  return rows > kGroup ? (size_t)cdiv(rows, kGroup) * keys : 0;
}

int launch_weights(const Scores &s, int keylen, float *part, const float *before, float *weights) {
  SumArgs a{s, keylen, before, weights, s.rows > kGroup ? part : nullptr};
  const int groups = s.rows > 0 ? cdiv(s.rows, kGroup) : 1;
  hipLaunchKernelGGL(weights_kernel, dim3(cdiv(a.part ? s.end - s.first : keylen, 256), groups), dim3(256), 0,
                     stream(), a);
  G4_LAUNCH_CHECK("weights_kernel");
  if (!a.part) return G4_OK;
  hipLaunchKernelGGL(weights_join_kernel, dim3(cdiv(keylen, 256)), dim3(256), 0, stream(), a, groups);
  G4_LAUNCH_CHECK("weights_join_kernel");
  return G4_OK;
}

namespace {

struct ScoreArgs {
  const float *q, *k;
  Scores s;
};

// A block per row; a wave takes every fourth key.
template <int HD>
__global__ __launch_bounds__(256) void scores_kernel(ScoreArgs a) {
  constexpr int D = HD / 64;
  __shared__ float2 sml[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = blockIdx.x;
  const int pos = a.s.pos0 + row / a.s.heads;
  const int lo = a.s.window > 0 ? max(a.s.first, pos - a.s.window + 1) : a.s.first;
  float q[D];
#pragma unroll
  for (int d = 0; d < D; ++d) q[d] = a.q[(size_t)row * HD + lane * D + d];
  float m = kNoScore, l = 0.f;
  for (int key = lo + w; key <= pos; key += 4) {
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) x = fmaf(q[d], a.k[(size_t)key * HD + lane * D + d], x);
    x = wave_sum(x) * kLog2e;
    if (lane == 0) a.s.score[(size_t)row * a.s.stride + (key - a.s.first)] = x;
    const float mn = fmaxf(m, x);
    l = l * __builtin_amdgcn_exp2f(m - mn) + __builtin_amdgcn_exp2f(x - mn);
    m = mn;
  }
  if (lane == 0) sml[w] = make_float2(m, l);
  __syncthreads();
  if (threadIdx.x == 0) {
    float M = kNoScore, L = 0.f;
    for (int i = 0; i < 4; ++i) M = fmaxf(M, sml[i].x);
    for (int i = 0; i < 4; ++i) L += sml[i].y * __builtin_amdgcn_exp2f(sml[i].x - M);
    a.s.ml[row] = make_float2(M, L);
  }
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
    rc = launch_weights(s, keylen, nullptr, before, weights);
    return rc ? rc : ok();
  }
  const int most = weighted_rows(qrows, heads, keylen, qpos0, win);
  for (int r0 = 0; r0 < qrows; r0 += most) {
    const int n = qrows - r0 < most ? qrows - r0 : most;
    ScoreArgs a{};
    a.q = q + (size_t)r0 * heads * head_dim;
    a.k = k;
    Scores &s = a.s;
    s.rows = n * heads;
    s.heads = heads;
    s.splits = 1;
    s.pos0 = qpos0 + r0;
    s.window = win;
    s.first = win > 0 && s.pos0 >= win ? s.pos0 - win + 1 : 0;
    s.end = s.pos0 + n;
    s.stride = (size_t)((s.end - s.first + 3) & ~3);
    const size_t scores = s.rows * s.stride, ml = (size_t)s.splits * s.rows * 2;
    void *mem = nullptr;
    if ((rc = g_weights_ws.get((scores + ml + weight_part_floats(s.rows, s.end - s.first)) * 4, &mem, who)))
      return rc;
    s.score = static_cast<float *>(mem);
    s.ml = reinterpret_cast<float2 *>(s.score + scores);
    switch (head_dim) {
      case 64: hipLaunchKernelGGL(scores_kernel<64>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      case 128: hipLaunchKernelGGL(scores_kernel<128>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      case 256: hipLaunchKernelGGL(scores_kernel<256>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      default: hipLaunchKernelGGL(scores_kernel<512>, dim3(s.rows), dim3(256), 0, stream(), a); break;
    }
    G4_LAUNCH_CHECK("scores_kernel");
    rc = launch_weights(s, keylen, s.score + scores + ml, r0 ? weights : before, weights);
    if (rc) return rc;
  }
  return ok();
}
