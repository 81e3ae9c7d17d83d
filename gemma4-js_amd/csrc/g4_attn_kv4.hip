// Attention over a cache held in 4 bits, with the weight that each key got if asked for.
#include <math.h>

#include "g4_gemv.h"
#include "g4_internal.h"
#include "g4_kv4.h"

namespace g4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3.4028235e38f;  // where a row's maximum starts

struct Kv4Args {
  const float *q;
  const uint32_t *k, *v;
  const uint16_t *ks, *vs;
  float *y;
  Scores s;  // score null: not kept
};

// Values 8 l .. of a row at lane l's share of D of them.
template <int D>
__device__ __forceinline__ void values4(const uint32_t *codes, const uint16_t *scales, size_t row, int hd,
                                        int d0, float (&x)[D]) {
  const float s = bf16_to_f32(scales[(row * hd + d0) / 32]);
  const uint32_t w = codes[(row * hd + d0) / 8] >> (4 * (d0 & 7));
#pragma unroll
  for (int d = 0; d < D; ++d) x[d] = (float)((int)(w >> (4 * d) & 15u) - 8) * s;
}

// A block per row; a wave takes every fourth key, a lane HD / 64 values of it.
template <int HD>
__global__ __launch_bounds__(256) void attn_kv4_kernel(Kv4Args a) {
  constexpr int D = HD / 64;
  __shared__ float2 sml[4];
  __shared__ float so[4][HD];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = blockIdx.x, d0 = lane * D;
  const int pos = a.s.pos0 + row / a.s.heads;
  const int lo = a.s.window > 0 ? max(a.s.first, pos - a.s.window + 1) : a.s.first;
  float q[D], o[D] = {};
#pragma unroll
  for (int d = 0; d < D; ++d) q[d] = a.q[(size_t)row * HD + d0 + d];
  float m = kNoScore, l = 0.f;
  for (int key = lo + w; key <= pos; key += 4) {
    float kk[D], vv[D], x = 0.f;
    values4<D>(a.k, a.ks, key, HD, d0, kk);
    values4<D>(a.v, a.vs, key, HD, d0, vv);
#pragma unroll
    for (int d = 0; d < D; ++d) x = fmaf(q[d], kk[d], x);
    x = wave_sum(x) * kLog2e;
    if (a.s.score && lane == 0) a.s.score[(size_t)row * a.s.stride + (key - a.s.first)] = x;
    const float mn = fmaxf(m, x), c = __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(x - mn);
    l = l * c + p;
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = fmaf(p, vv[d], o[d] * c);
    m = mn;
  }
  if (lane == 0) sml[w] = make_float2(m, l);
#pragma unroll
  for (int d = 0; d < D; ++d) so[w][d0 + d] = o[d];
  __syncthreads();
  float M = kNoScore, L = 0.f, f[4];
  for (int i = 0; i < 4; ++i) M = fmaxf(M, sml[i].x);
  for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_exp2f(sml[i].x - M), L += sml[i].y * f[i];
  for (int d = threadIdx.x; d < HD; d += 256) {
    float x = 0.f;
    for (int i = 0; i < 4; ++i) x += so[i][d] * f[i];
    a.y[(size_t)row * HD + d] = x / L;
  }
  if (a.s.ml && threadIdx.x == 0) a.s.ml[row] = make_float2(M, L);
}

Workspace g_kv4_ws;

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_attention_kv4(const float *q, const g4_kv4 *cache, int qrows, int heads, int keylen,
                            int qpos0, int sliding, int window, float *y, const float *before,
                            float *weights) {
  const char *who = "g4_attention_kv4";
  if (int rc = check_kv4(cache, 0, keylen, who)) return rc;
  if (int rc = check_weighted(qrows, heads, keylen, qpos0, sliding, window, before, weights, who)) return rc;
  if (before && !weights) return fail(G4_E_ARG, "%s: before without weights", who);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(y)) & 15)
    return fail(G4_E_ARG, "%s: q and y must be 16-byte aligned", who);
  G4_CHECK_INIT();
  if (keylen == 0) return ok();
  const int head_dim = cache->head_dim;
  const size_t qn = (size_t)qrows * heads * head_dim * 4;
  int rc = check_kv4_memory(cache, keylen, true, true, "g4_attention_kv4 cache");
  if (!rc && qrows) rc = check_device_range(q, qn, "g4_attention_kv4 q");
  if (!rc && qrows) rc = check_device_range(y, qn, "g4_attention_kv4 y");
  if (!rc && weights) rc = check_device_range(weights, (size_t)keylen * 4, "g4_attention_kv4 weights");
  if (!rc && before) rc = check_device_range(before, (size_t)keylen * 4, "g4_attention_kv4 before");
  if (rc) return rc;
  const int win = sliding ? window : 0;
  if (qrows == 0) {
    Scores s{};
    s.heads = 1;
    if (weights) rc = launch_weights(s, keylen, nullptr, before, weights);
    return rc ? rc : ok();
  }
  const int most = weights ? weighted_rows(qrows, heads, keylen, qpos0, win) : qrows;
  for (int r0 = 0; r0 < qrows; r0 += most) {
    const int n = qrows - r0 < most ? qrows - r0 : most;
    Kv4Args a{};
    a.q = q + (size_t)r0 * heads * head_dim;
    a.y = y + (size_t)r0 * heads * head_dim;
    a.k = cache->k;
    a.v = cache->v;
    a.ks = cache->k_scales;
    a.vs = cache->v_scales;
    Scores &s = a.s;
    s.rows = n * heads;
    s.heads = heads;
    s.splits = 1;
    s.pos0 = qpos0 + r0;
    s.window = win;
    s.first = win > 0 && s.pos0 >= win ? s.pos0 - win + 1 : 0;
    s.end = s.pos0 + n;
    s.stride = (size_t)((s.end - s.first + 3) & ~3);
    const size_t scores = weights ? s.rows * s.stride : 0, ml = weights ? (size_t)s.splits * s.rows * 2 : 0;
    if (weights) {
      void *mem = nullptr;
      if ((rc = g_kv4_ws.get((scores + ml + weight_part_floats(s.rows, s.end - s.first)) * 4, &mem, who)))
        return rc;
      s.score = static_cast<float *>(mem);
      s.ml = reinterpret_cast<float2 *>(s.score + scores);
    }
    switch (head_dim) {
      case 64: hipLaunchKernelGGL(attn_kv4_kernel<64>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      case 128: hipLaunchKernelGGL(attn_kv4_kernel<128>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      case 256: hipLaunchKernelGGL(attn_kv4_kernel<256>, dim3(s.rows), dim3(256), 0, stream(), a); break;
      default: hipLaunchKernelGGL(attn_kv4_kernel<512>, dim3(s.rows), dim3(256), 0, stream(), a); break;
    }
    G4_LAUNCH_CHECK("attn_kv4_kernel");
    if (weights) rc = launch_weights(s, keylen, s.score + scores + ml, r0 ? weights : before, weights);
    if (rc) return rc;
  }
  return ok();
}
