// Attention of a tree of drafted tokens over the FP32 KV cache: node i, at position
// prefix + depth(i), sees the prefix, itself and its ancestors (within the window).
#include <math.h>

#include "g4_gemv.h"
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr int kMaxNodes = 256, kNodeWords = kMaxNodes / 32;
constexpr int kTile = 16;  // keys per tile
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3.4028235e38f;  // where a row's maximum starts

struct TreeArgs {
  const float *q, *k, *v;
  float *y;
  const int *parents;
  int nodes, heads, prefix, window;  // window 0: none
  int first;    // first prefix key of the first tile
  int ptiles;   // tiles of the prefix; those of the tree follow
  int tiles, tps, splits;
  bool one_l2;  // the row blocks of a split go to one XCD
  float *part;  // [splits][rows][hd] unnormalised outputs
  float2 *ml;   // [splits][rows] (max, sum)
};

// Ancestors of the nodes as bits (themselves among them) and their number.
struct Tree {
  uint32_t sees[kMaxNodes][kNodeWords];
  int up[kMaxNodes];         // -1: none left
  short depth[kMaxNodes];    // -1: some parent on the way is not an earlier node
};

// Every node at once, the distance to the ancestor `up` doubling in each round.
template <int NTH>
__device__ __forceinline__ void make_tree(const TreeArgs &a, Tree &tr) {
  const int t = threadIdx.x;
  static_assert(NTH >= 256, "a thread per node");
  const bool mine = t < a.nodes;
  uint32_t s[kNodeWords];
  int up = -1, depth = 0;
#pragma unroll
  for (int w = 0; w < kNodeWords; ++w) s[w] = 0;
  if (mine) {
    up = a.parents[t];
    if (up < -1 || up >= t) up = -1, depth = -1;
    if (up >= 0) depth = 1;
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w) s[w] = t >> 5 == w ? 1u << (t & 31) : 0u;
  }
  bool more = true;
  while (more) {
    if (mine) {
#pragma unroll
      for (int w = 0; w < kNodeWords; ++w) tr.sees[t][w] = s[w];
      tr.up[t] = up;
      tr.depth[t] = (short)depth;
    }
    more = __syncthreads_or(up >= 0);
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kNodeWords; ++w) s[w] |= tr.sees[up][w];
      const int d = tr.depth[up];
      depth = d < 0 || depth < 0 ? -1 : depth + d;
      up = tr.up[up];
    }
    __syncthreads();
  }
}

// max over the lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float group_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int HD>
constexpr int kDimWaves = HD >= 256 ? 4 : HD / 64;

// A block owns 16 rows of [nodes * heads, hd] and a run of key tiles, which its KG key groups
// take in turn; the DQ waves of a group share the head dim.  On the FP32 matrix cores
// (v_mfma_f32_16x16x4f32), lane (c, g) of a wave working for row c throughout:
//   S^T = K . Q^T     a wave's dims; the group's waves add theirs through LDS, in wave order,
//                     so that they hold the same scores: keys 4 g .. + 3 per lane
//   softmax           running maximum and sum per row
//   O^T += V^T . P^T  the lane's probabilities are its operand as they are (step i takes keys
//                     4 g + i); output tile 4 q + e holds dims 64 q + 4 c + e, so V and O
//                     move as 16-byte vectors
// The next tile's K is loaded once the scores are formed, its V once the outputs are.
//
// Over long caches the FP32 products bound it: 64 nodes x 8 heads of 512 over 16000 keys, 16.8
// GFLOP, take 156 us (107 TFLOP/s) with two blocks per CU.  What a wave does between its products
// is what is left: rows of V that are not finite, dealt with in a branch of its own beside the
// products, cost 32 register moves per tile (182 us, without 171); 64-bit addresses per lane
// instead of a scalar base 15 us more.  Of 182 to 184, 32 rows per block (half the loads of K and
// V) took 209, two such groups of 16 in step 217, the next tile's scores ahead of the softmax 210.
// Short caches wait for their loads: 4 nodes over 203 keys 8.9 us, two launches.
// Head dims of 64 and 128: 4 and 2 key groups; twice as many take 9.8 us instead of 8.5 for 4
// nodes over 200 keys of dim 64, 31.4 instead of 28.6 for 64 nodes over 16000.
template <int HD, int KG>
__global__ __launch_bounds__(64 * kDimWaves<HD> * KG, 2) void attn_tree_kernel(TreeArgs a) {
  constexpr int DQ = kDimWaves<HD>, DW = HD / DQ, NJ = DW / 16, NQ = DW / 64;
  constexpr int NTH = 64 * DQ * KG, R = 16;
  struct Loop {
    Tree tree;
    f32x4 sx[2][KG][DQ][64];  // the waves' scores, two buffers
  };
  union Smem {
    Loop loop;
    float o[R][HD + 4];
  };
  __shared__ Smem sm;
  __shared__ float2 wml[KG][R];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int w = wave % DQ, kg = wave / DQ;
  const int c = lane & 15, g = lane >> 4;
  const int nrows = a.nodes * a.heads, d0 = w * DW;
  int split = blockIdx.y, R0 = blockIdx.x * R;
  if (a.one_l2) {  // blocks are dealt to the 8 XCDs in turn; there are multiples of 8 splits
    const int b = blockIdx.y * gridDim.x + blockIdx.x, n = b / 8;
    split = n / (int)gridDim.x * 8 + b % 8;
    R0 = n % (int)gridDim.x * R;
    if (split >= a.splits) return;
  }
  const int t0 = split * a.tps, t1 = min(t0 + a.tps, a.tiles);
  // (rows past the last: the last one again, not stored)
  const int row = min(R0 + c, nrows - 1), node = row / a.heads;
  const int last = a.prefix + a.nodes - 1;  // last cache row
  const bool has_tree = t1 > a.ptiles;
  auto key0_of = [&](int tile) {
    return tile < a.ptiles ? a.first + tile * kTile : a.prefix + (tile - a.ptiles) * kTile;
  };
  auto end_of = [&](int tile) { return tile < a.ptiles ? a.prefix - 1 : last; };
  float4 kr[NJ], vr[4][NQ];
  // (the tile's first key is the same for the wave: a scalar base, 32-bit offsets within the tile)
  auto load_k = [&](int tile) {
    tile = min(tile, t1 - 1);
    const int k0 = key0_of(tile);
    const char *p = reinterpret_cast<const char *>(a.k + (size_t)k0 * HD + d0);
    const uint32_t at = (uint32_t)(min(c, end_of(tile) - k0) * HD + 4 * g) * 4;
#pragma unroll
    for (int j = 0; j < NJ; ++j) kr[j] = *reinterpret_cast<const float4 *>(p + at + 64 * j);
  };
  auto load_v = [&](int tile) {
    tile = min(tile, t1 - 1);
    const int k0 = key0_of(tile);
    const char *p = reinterpret_cast<const char *>(a.v + (size_t)k0 * HD + d0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = (uint32_t)(min(4 * g + i, end_of(tile) - k0) * HD + 4 * c) * 4;
#pragma unroll
      for (int q = 0; q < NQ; ++q) vr[i][q] = *reinterpret_cast<const float4 *>(p + at + 256 * q);
    }
  };
  load_k(t0 + kg);
  load_v(t0 + kg);
  float4 qr[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    qr[j] = *reinterpret_cast<const float4 *>(a.q + (size_t)row * HD + d0 + 16 * j + 4 * g);
  if (has_tree || a.window > 0) make_tree<NTH>(a, sm.loop.tree);
  // keys at positions > low are in the row's window
  const int depth = has_tree || a.window > 0 ? sm.loop.tree.depth[node] : 0;
  const bool bad = depth < 0;
  const int low = a.window > 0 ? a.prefix + depth - a.window : -1;
  int high = low;  // the highest of the 16 rows
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) high = max(high, __shfl_xor(high, o, 64));
  high = __builtin_amdgcn_readfirstlane(high);

  float m = kNoScore, l = 0.f;  // l: this lane's keys only
  f32x4 o[4 * NQ];
#pragma unroll
  for (int n = 0; n < 4 * NQ; ++n) o[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // Everything loaded so far has to be there: a wait in the loop counts the loads behind the one
  // it is for, and would count by the loop's entry, q among them, in every turn.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  const int steps = (t1 - t0 + KG - 1) / KG;
  for (int it = 0; it < steps; ++it) {
    const int tile = t0 + kg + it * KG;
    const bool mine = tile < t1;
    const int key0 = key0_of(min(tile, t1 - 1));
    f32x4 s;
    {
      f32x4 sa[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float kk[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
        const float qq[4] = {qr[j].x, qr[j].y, qr[j].z, qr[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sa[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[i], qq[i], sa[i & 1], 0, 0, 0);
      }
      s = sa[0] + sa[1];
    }
    load_k(tile + KG);
    __builtin_amdgcn_s_setprio(1);  // before the other block's products (2% at head dim 256)
    if (DQ > 1) {
      sm.loop.sx[it & 1][kg][w][lane] = s;
      __syncthreads();
      s = sm.loop.sx[it & 1][kg][0][lane];
#pragma unroll
      for (int d = 1; d < DQ; ++d) s += sm.loop.sx[it & 1][kg][d][lane];
    }
    // whether every row sees every key of the tile
    const bool inner = mine && tile < a.ptiles && key0 > high && key0 + kTile <= a.prefix;
    uint32_t seen = 15u;  // bit i: row c sees key 4 g + i
    if (!inner) {
      uint32_t bits = 0;
      if (tile >= a.ptiles) {
        const int j0 = key0 - a.prefix;  // of 16 within 32 nodes
        bits = mine ? sm.loop.tree.sees[node][j0 >> 5] >> (j0 & 16) >> (4 * g) & 15u : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = min(j0 + 4 * g + i, a.nodes - 1);
          if (a.prefix + sm.loop.tree.depth[j] <= low) bits &= ~(1u << i);
        }
      } else if (mine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 4 * g + i;
          if (key < a.prefix && key > low) bits |= 1u << i;
        }
      }
      seen = bits;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(bits >> i & 1)) s[i] = -INFINITY;
    }
    float p[4];
    const float tm = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    // (fmaxf drops a NaN score, whose p is NaN.)
    const float mn = fmaxf(m, group_max(tm));
    const float corr = __builtin_amdgcn_exp2f((m - mn) * kLog2e);
    m = mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f((s[i] - mn) * kLog2e);
    l = fmaf(l, corr, (p[0] + p[1]) + (p[2] + p[3]));
    if (__any(corr != 1.f)) {
#pragma unroll
      for (int n = 0; n < 4 * NQ; ++n) o[n] *= corr;
    }
    __builtin_amdgcn_s_setprio(0);
    // a weight of 0 times a value that is not finite would reach rows that do not see the key
    bool odd = false;
    if (!inner) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float4 x = vr[i][q];
          odd = odd || !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w));
        }
      odd = __any(odd);
    }
    if (odd) {  // keys that the row sees, one by one; then nothing is left of the tile
      for (int kk = 0; mine && kk < kTile; ++kk) {
        const int from = 16 * (kk >> 2) + c, i = kk & 3;
        const float pi = i == 0 ? p[0] : i == 1 ? p[1] : i == 2 ? p[2] : p[3];
        const float pk = __shfl(pi, from, 64);
        const uint32_t see = (uint32_t)__shfl((int)seen, from, 64) >> i & 1u;
        if (see) {
          // lane (c, g): tile n, register v holds dim 64 q + 4 (4 g + v) + e
          const float *vp = a.v + (size_t)min(key0 + kk, end_of(tile)) * HD + d0 + 16 * g;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float4 x = *reinterpret_cast<const float4 *>(vp + 64 * q + 4 * v);
              o[4 * q][v] = fmaf(pk, x.x, o[4 * q][v]);
              o[4 * q + 1][v] = fmaf(pk, x.y, o[4 * q + 1][v]);
              o[4 * q + 2][v] = fmaf(pk, x.z, o[4 * q + 2][v]);
              o[4 * q + 3][v] = fmaf(pk, x.w, o[4 * q + 3][v]);
              __builtin_amdgcn_sched_barrier(0);  // few registers: this is rare
            }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < NQ; ++q) vr[i][q] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const float vv[4] = {vr[i][q].x, vr[i][q].y, vr[i][q].z, vr[i][q].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[4 * q + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[e], p[i], o[4 * q + e], 0, 0, 0);
      }
    load_v(tile + KG);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (bad) l = __int_as_float(0x7fc00000);
  if (w == 0 && g == 0) wml[kg][c] = make_float2(m, l);
  __syncthreads();
  // the key groups, added in order
  float M = kNoScore, L = 0.f;
#pragma unroll
  for (int k = 0; k < KG; ++k) M = fmaxf(M, wml[k][c].x);
#pragma unroll
  for (int k = 0; k < KG; ++k)
    L = fmaf(wml[k][c].y, __builtin_amdgcn_exp2f((wml[k][c].x - M) * kLog2e), L);
  const float f = __builtin_amdgcn_exp2f((m - M) * kLog2e);
  if (KG > 1)
#pragma unroll
    for (int n = 0; n < 4 * NQ; ++n) o[n] *= f;
  for (int k = KG - 1; k >= 1; --k) {
    if (kg == k)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float4 *dst = reinterpret_cast<float4 *>(&sm.o[c][d0 + 64 * q + 16 * g + 4 * v]);
          *dst = make_float4(o[4 * q][v], o[4 * q + 1][v], o[4 * q + 2][v], o[4 * q + 3][v]);
        }
    __syncthreads();
    if (kg == 0)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float4 x = *reinterpret_cast<const float4 *>(&sm.o[c][d0 + 64 * q + 16 * g + 4 * v]);
          o[4 * q][v] += x.x;
          o[4 * q + 1][v] += x.y;
          o[4 * q + 2][v] += x.z;
          o[4 * q + 3][v] += x.w;
        }
    __syncthreads();
  }
  if (kg > 0) return;
  const bool whole = a.splits == 1;
  float *out = whole ? a.y : a.part + (size_t)split * nrows * HD;
  if (R0 + c >= nrows) return;
  if (!whole && w == 0 && g == 0) a.ml[(size_t)split * nrows + row] = make_float2(M, L);
  float *p = out + (size_t)row * HD + d0 + 16 * g;
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float4 x = make_float4(o[4 * q][v], o[4 * q + 1][v], o[4 * q + 2][v], o[4 * q + 3][v]);
      if (whole) x = make_float4(x.x / L, x.y / L, x.z / L, x.w / L);
      *reinterpret_cast<float4 *>(p + 64 * q + 4 * v) = x;
    }
}

// Adds the key splits of a row: y = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.  A block is
// one row; thread (g, t) adds splits g, g + 4, .. of 16-byte unit t in order, then the 4 sums
// are added in order.  Bound by latency, so the first loads leave before the weights are known.
template <int HD>
__global__ __launch_bounds__(HD) void attn_tree_merge_kernel(TreeArgs a) {
  constexpr int G = 4, U = 8;
  const int t = threadIdx.x % (HD / G), g = threadIdx.x / (HD / G);
  const int row = blockIdx.x, nrows = a.nodes * a.heads;
  __shared__ float wt[kMaxSplits];
  __shared__ float sum;
  __shared__ f32x4 sums[G][HD / G];
  const f32x4 *p = reinterpret_cast<const f32x4 *>(a.part + (size_t)row * HD) + t;
  const size_t step = (size_t)nrows * HD / 4;
  f32x4 x[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = p[min(s0 + G * u, a.splits - 1) * step];
  };
  load(g);
  if (threadIdx.x < 64) {  // a lane per split
    const int lane = threadIdx.x;
    const float2 ml = a.ml[(size_t)min(lane, a.splits - 1) * nrows + row];
    float M = ml.x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float e = lane < a.splits ? __builtin_amdgcn_exp2f((ml.x - M) * kLog2e) : 0.f;
    wt[lane] = e;
    const float L = wave_sum(lane < a.splits ? e * ml.y : 0.f);
    if (lane == 0) sum = L;
  }
  __syncthreads();
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < a.splits; s0 += G * U) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + G * u < a.splits) y += wt[s0 + G * u] * x[u];
    if (s0 + G * U < a.splits) load(s0 + G * U);
  }
  sums[g][t] = y;
  __syncthreads();
  if (g > 0) return;
  y = (sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t]);
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] /= sum;
  reinterpret_cast<f32x4 *>(a.y + (size_t)row * HD)[t] = y;
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

Workspace g_tree_ws;

template <int HD, int KG>
int launch_tree(TreeArgs a) {
  const int rows = a.nodes * a.heads, blocks = cdiv(rows, 16);
  // A block per CU; two, whose waits overlap, where each then has many tiles and the splits'
  // outputs are little beside them.  16 nodes of 8 heads of 512 over 1900 keys (4 tiles per
  // block): 18.6 us, with two blocks 24.3; 64 nodes of 256 over 1500 (13 tiles): 20.0, with two
  // 23.9; 64 nodes of 512 over 16000 (126 tiles): 178, with two 157.
  const int one = cu_count() / blocks, two = 2 * cu_count() / blocks;
  int splits = one < 1 ? 1 : one;
  if (cdiv(a.tiles, splits) > 16) splits = two < 1 ? 1 : two;
  if (splits > kMaxSplits) splits = kMaxSplits;
  // Splits of its own for each XCD, whose L2 then is filled with its part of k and v alone: where
  // few row blocks are done with a tile sooner than all 8 L2s get it, and where k and v pass the 8
  // L2s (4 MB each); not where that would leave more than an eighth of the blocks out.  us per
  // call, heads 8 x 512: 16 nodes (8 blocks) over 1900 keys 18.6, else 19.8, over 16000 53, else
  // 81; 20 nodes over 16000 63, else 83; 32 nodes 88, else 96.  With more blocks over short caches
  // their loads of the same lines at the same time cost more: 32 nodes over 2000 keys 25, else 22.7;
  // 48 nodes over 9000 (16 of 21 splits) 93, else 79.
  const bool past_l2 = (size_t)a.tiles * kTile * HD * 8 > size_t(32) << 20;
  a.one_l2 = (blocks <= 8 || past_l2) && splits >= 8 && splits % 8 <= splits / 8;
  if (a.one_l2) splits = splits / 8 * 8;
  a.tps = cdiv(a.tiles, splits);
  if (a.tps < KG) a.tps = KG;
  a.splits = cdiv(a.tiles, a.tps);
  if (a.splits > 1) {
    void *mem = nullptr;
    const size_t part = (size_t)a.splits * rows * HD;
    if (int rc = g_tree_ws.get((part + (size_t)a.splits * rows * 2) * 4, &mem, "g4_attention_tree"))
      return rc;
    a.part = static_cast<float *>(mem);
    a.ml = reinterpret_cast<float2 *>(a.part + part);
  }
  hipLaunchKernelGGL((attn_tree_kernel<HD, KG>), dim3(blocks, a.one_l2 ? cdiv(a.splits, 8) * 8 : a.splits),
                     dim3(64 * kDimWaves<HD> * KG), 0, stream(), a);
  G4_LAUNCH_CHECK("attn_tree_kernel");
  if (a.splits == 1) return G4_OK;
  hipLaunchKernelGGL(attn_tree_merge_kernel<HD>, dim3(rows), dim3(HD), 0, stream(), a);
  G4_LAUNCH_CHECK("attn_tree_merge_kernel");
  return G4_OK;
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_attention_tree(const float *q, const float *k, const float *v, int nodes, int heads,
                             int head_dim, int prefix, const int32_t *parents, int sliding,
                             int window, float *y) {
  if (nodes < 0 || nodes > kMaxNodes || heads <= 0 || heads > 8 || prefix < 0 ||
      prefix > 0x7fffffff - 2 * kMaxNodes ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512) ||
      (sliding && window <= 0))
    return fail(G4_E_ARG,
                "g4_attention_tree: nodes %d (<= %d), heads %d (<= 8), head_dim %d (64, 128, 256 or "
                "512), prefix %d, window %d",
                nodes, kMaxNodes, heads, head_dim, prefix, window);
  const void *ptrs[] = {q, k, v, y};
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15)
      return fail(G4_E_ARG, "g4_attention_tree: q, k, v and y must be 16-byte aligned");
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
  TreeArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.y = y;
  a.parents = parents;
  a.nodes = nodes;
  a.heads = heads;
  a.prefix = prefix;
  a.window = sliding ? window : 0;
  // a root sees the most of the prefix: positions > prefix - window
  a.first = a.window > 0 && prefix >= a.window ? prefix - a.window + 1 : 0;
  a.ptiles = a.first < prefix ? cdiv(prefix - a.first, kTile) : 0;
  a.tiles = a.ptiles + cdiv(nodes, kTile);
  switch (head_dim) {
    case 64: rc = launch_tree<64, 4>(a); break;
    case 128: rc = launch_tree<128, 2>(a); break;
    case 256: rc = launch_tree<256, 1>(a); break;
    default: rc = launch_tree<512, 1>(a); break;
  }
  return rc ? rc : ok();
}
