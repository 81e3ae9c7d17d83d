// Attention of a tree of drafted tokens over the FP32 KV cache: node i, at position
// prefix + depth(i), sees the prefix, itself and its ancestors (within the window).
#include <math.h>

#include "g4_gemv.h"
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kMaxNodes = 256;

struct TreeArgs {
  const float *q, *k, *v;
  float *y;
  const int *parents;
  int nodes, heads, prefix, window;  // window 0: none
};

// One block per (node, head); its waves take turns over the keys, lane l holding dims
// DPL l .. of q, k, v and the output, with a running maximum and sum each.
template <int DPL>
__global__ __launch_bounds__(256) void attn_tree_kernel(TreeArgs a) {
  constexpr int HD = 64 * DPL;
  __shared__ uint32_t sees[kMaxNodes / 32];
  __shared__ int s_depth;
  __shared__ float sm[4], sl[4], so[4][HD];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int node = blockIdx.x / a.heads;
  if (t < kMaxNodes / 32) sees[t] = 0;
  __syncthreads();
  if (t == 0) {
    int depth = 0;
    for (int i = node;;) {
      sees[i >> 5] |= 1u << (i & 31);
      const int p = a.parents[i];
      if (p < -1 || p >= i) depth = -1;
      if (p < 0 || p >= i) break;
      ++depth;
      i = p;
    }
    s_depth = depth;
  }
  __syncthreads();
  const int depth = s_depth;
  float *y = a.y + (size_t)blockIdx.x * HD;
  if (depth < 0) {
    for (int i = t; i < HD; i += 256) y[i] = __int_as_float(0x7fc00000);
    return;
  }
  float q[DPL], o[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < DPL; ++j) {
    q[j] = a.q[(size_t)blockIdx.x * HD + DPL * lane + j];
    o[j] = 0.f;
  }
  auto key = [&](size_t at) {
    const float *k = a.k + at * HD + DPL * lane, *v = a.v + at * HD + DPL * lane;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) s = fmaf(q[j], k[j], s);
    s = wave_sum(s);
    const float mn = fmaxf(m, s);
    const float c = expf(m - mn), p = expf(s - mn);
    l = fmaf(l, c, p);
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = fmaf(p, v[j], o[j] * c);
    m = mn;
  };
  // positions above `low` are seen
  const int low = a.window > 0 ? a.prefix + depth - a.window : -1;
  for (int i = (low >= 0 ? low + 1 : 0) + w; i < a.prefix; i += 4) key(i);
  if (w == 0) {
    int at = depth;
    for (int i = node; i >= 0; --i)
      if (sees[i >> 5] >> (i & 31) & 1)
        if (a.prefix + at-- > low) key((size_t)a.prefix + i);
  }
  if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
  for (int j = 0; j < DPL; ++j) so[w][DPL * lane + j] = o[j];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], L = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = sl[i] != 0.f ? expf(sm[i] - M) : 0.f;
    L += f[i] * sl[i];
  }
  for (int i = t; i < HD; i += 256) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += f[j] != 0.f ? f[j] * so[j][i] : 0.f;
    y[i] = s / L;
  }
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_attention_tree(const float *q, const float *k, const float *v, int nodes, int heads,
                             int head_dim, int prefix, const int32_t *parents, int sliding,
                             int window, float *y) {
  if (nodes < 0 || nodes > kMaxNodes || heads <= 0 || heads > 8 || prefix < 0 ||
      prefix > 0x7fffffff - kMaxNodes ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) ||
      (sliding && window <= 0))
    return fail(G4_E_ARG,
                "g4_attention_tree: nodes %d (<= %d), heads %d (<= 8), head_dim %d (64, 128, 256 or "
                "512), prefix %d, window %d",
                nodes, kMaxNodes, heads, head_dim, prefix, window);
  G4_CHECK_INIT();
  if (nodes == 0) return ok();
  const size_t qn = (size_t)nodes * heads * head_dim * 4;
  const size_t kn = ((size_t)prefix + nodes) * head_dim * 4;
  int rc = check_device_range(q, qn, "g4_attention_tree q");
  if (!rc) rc = check_device_range(k, kn, "g4_attention_tree k");
  if (!rc) rc = check_device_range(v, kn, "g4_attention_tree v");
  if (!rc) rc = check_device_range(parents, (size_t)nodes * 4, "g4_attention_tree parents");
  if (!rc) rc = check_device_range(y, qn, "g4_attention_tree y");
  if (rc) return rc;
  TreeArgs a{q, k, v, y, parents, nodes, heads, prefix, sliding ? window : 0};
  const dim3 grid(nodes * heads);
  switch (head_dim / 64) {
    case 1: hipLaunchKernelGGL(attn_tree_kernel<1>, grid, dim3(256), 0, stream(), a); break;
    case 2: hipLaunchKernelGGL(attn_tree_kernel<2>, grid, dim3(256), 0, stream(), a); break;
    case 4: hipLaunchKernelGGL(attn_tree_kernel<4>, grid, dim3(256), 0, stream(), a); break;
    default: hipLaunchKernelGGL(attn_tree_kernel<8>, grid, dim3(256), 0, stream(), a); break;
  }
  G4_LAUNCH_CHECK("attn_tree_kernel");
  return ok();
}
