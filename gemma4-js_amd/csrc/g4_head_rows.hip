// The tied BF16 head for several hidden states:
//   out[j, r] = softcap * tanh((scale * sum_k x[j, k] * E[r, k]) / softcap)
//
// Memory-bound: the table is read once for up to 64 states.  Numerics: the BF16 matrix form
// takes E as it is and a state as three BF16 parts, whose sum is the FP32 value (3 x 8 bits
// of its 24), so every product is exact and only the FP32 sums round.
#include "g4_internal.h"
#include "g4_ops.h"

namespace g4 {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxTiles = 4;  // 16-state tiles of a block
constexpr int kSteps = 2;     // steps of 32 k per stage
constexpr int kMaxStates = 65536, kMaxRows = 1 << 30;

int cdiv(int a, int b) { return (a + b - 1) / b; }

struct HeadArgs {
  const float *x;
  const uint16_t *E;
  float *out;
  u32x4 *parts;  // [tile][step][part][64 lanes]
  size_t out_stride;
  int n, rows, K;
  int steps;  // of 32 k, a multiple of a stage's
  float scale, softcap;
};

// 8 values as three BF16 parts each, truncations whose sum is the value: they have its sign
// and cannot overflow.  The first part holds what is not finite.  `in` false: zeros.
__device__ __forceinline__ void split8(const float (&v)[8], bool in, uint32_t (&w)[3][4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t p[2][3];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float u = in ? v[2 * e + h] : 0.f;
      const uint32_t b = __float_as_uint(u);
      const bool finite = (b & 0x7f800000u) != 0x7f800000u;
      p[h][0] = b & 0xffff0000u;
      const float r = u - __uint_as_float(p[h][0]);
      p[h][1] = finite ? __float_as_uint(r) & 0xffff0000u : 0u;
      p[h][2] = finite ? __float_as_uint(r - __uint_as_float(p[h][1])) : 0u;
      if (!finite && (b & 0x7fffffu)) p[h][0] |= 0x400000u;  // a NaN stays one
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i][e] = (p[0][i] >> 16) | (p[1][i] & 0xffff0000u);
  }
}

// States as parts in the order the matrix instructions read them: step s, part p of tile
// m holds, for lane (c, g), state 16 m + c, k = 32 s + 8 g .. + 7.  Zeros past n and K.
__global__ __launch_bounds__(256) void head_parts_kernel(HeadArgs a, int tiles) {
  const int u = blockIdx.x * 256 + threadIdx.x, lane = u & 63, c = lane & 15, g = lane >> 4;
  const int step = (u >> 6) % a.steps, m = (u >> 6) / a.steps;
  if (m >= tiles) return;
  const int j = 16 * m + c, k = 32 * step + 8 * g;
  const bool in = j < a.n && k < a.K;
  const float *src = a.x + (in ? (size_t)j * a.K + k : 0);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = src[e];
  uint32_t w[3][4];
  split8(v, in, w);
#pragma unroll
  for (int i = 0; i < 3; ++i)
    a.parts[(((size_t)m * a.steps + step) * 3 + i) * 64 + lane] = (u32x4){w[i][0], w[i][1], w[i][2], w[i][3]};
}

// Logits r .. r + 3 of state j from their sums, as g4_bf16_head computes them.
__device__ __forceinline__ void store_logits(const HeadArgs &a, f32x4 v, int j, int r) {
  if (j >= a.n) return;
  v *= a.scale;
  if (a.softcap > 0.f)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = tanhf(v[k] / a.softcap) * a.softcap;
  float *o = a.out + (size_t)j * a.out_stride + r;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.out) & 15) | (a.out_stride & 3)) == 0;
  if (wide && r + 3 < a.rows) {
    *reinterpret_cast<f32x4 *>(o) = v;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r + k < a.rows) o[k] = v[k];
  }
}

// A block takes tiles of 16 RT rows of E per wave, one after the other, and MT 16-state
// tiles.  D = E . X^T: lane (c, g) feeds row c of a row tile and state c, k 8 g .. + 7 of a
// step, and gets state c of rows 4 g .. + 3.  A stage is two steps, 128 bytes of each row.
// It reaches LDS by direct loads that leave as soon as the stage before has been read to
// registers (a wave's rows, one buffer) or is being multiplied (the states' parts for all
// waves, two buffers), also across tiles.  An instruction loads whole lines of 8 rows, past
// the caches.  A row's 16-byte units are stored at unit ^ (row & 7), so that lanes reading
// one unit of 8 rows meet all banks.
// Measured over 262144 x 1536 (us per call, the parts' launch of 5 among them): 5 states
// 133, 20 states 154, 40 states 168, 64 states 186 (4.7 TB/s of the table and its logits);
// with rows loaded straight to registers (64 bytes of 16 rows to an instruction) 5 and 64
// states took 154 and 216, with one tile per block 138 and 241.  At 64 states the loads of E
// alone take 120 us, the matrix instructions 61 at their peak; without the states' loads,
// two thirds of the products or the stores it is 169 to 172 of 194 (4 waves per block).
template <int MT, int RT, int WV>
__global__ __launch_bounds__(64 * WV, 2) void head_rows_kernel(HeadArgs a) {
  constexpr int P = kSteps * MT * 3;  // 1 KB pieces of the states in a stage
  constexpr int W = (P + WV - 1) / WV;      // and loads of a wave for them
  constexpr int R = 2 * RT;           // its loads of rows
  __shared__ u32x4 es[WV][R * 64];
  __shared__ u32x4 xs[2][P * 64];
  typedef __attribute__((address_space(3))) void *lds_ptr;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * kMaxTiles;
  const int chunks = a.K / 8, stages = a.steps / kSteps;
  const int tiles = (a.rows + 16 * RT * WV - 1) / (16 * RT * WV);
  const int unit = (lane & 7) ^ (lane >> 3);
  auto load_rows = [&](int tile, int st) {
    const int k = st * 8 + unit, at = k < chunks ? k : chunks - 1;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = tile * (16 * RT * WV) + w * (16 * RT) + 8 * i + (lane >> 3);
      const uint16_t *row = a.E + (size_t)(r < a.rows ? r : a.rows - 1) * a.K;
      __builtin_amdgcn_global_load_lds((const void *)(reinterpret_cast<const u32x4 *>(row) + at),
                                       (lds_ptr)(es[w] + i * 64), 16, 0, 2);
    }
  };
  auto load_states = [&](int st, int buf) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int p = w + WV * i < P ? w + WV * i : P - 1;  // the last one again, same bytes
      const int m = p / (kSteps * 3), q = p - m * (kSteps * 3);
      __builtin_amdgcn_global_load_lds(
          (const void *)(a.parts + (((size_t)(m0 + m) * a.steps + st * kSteps) * 3 + q) * 64 + lane),
          (lds_ptr)(xs[buf] + p * 64), 16, 0, 0);
    }
  };
  int buf = 0;
  load_rows(blockIdx.x, 0);
  load_states(0, 0);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    f32x4 d[RT][MT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) d[i][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int st = 0; st < stages; ++st, buf ^= 1) {
      // the stage has landed everywhere, and the other buffer is free
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      bf16x8 e[kSteps][RT];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < RT; ++i)
          e[s][i] = __builtin_bit_cast(bf16x8, es[w][(16 * i + c) * 8 + ((4 * s + g) ^ (c & 7))]);
      const bool last = st + 1 == stages;
      load_states(last ? 0 : st + 1, buf ^ 1);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the rows are in registers
      const int next = last ? tile + (int)gridDim.x : tile;
      load_rows(next < tiles ? next : tile, last ? 0 : st + 1);
      const u32x4 *x = xs[buf] + lane;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 2; p >= 0; --p) {
            const bf16x8 b = __builtin_bit_cast(bf16x8, x[((m * kSteps + s) * 3 + p) * 64]);
#pragma unroll
            for (int i = 0; i < RT; ++i)
              d[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e[s][i], b, d[i][m], 0, 0, 0);
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i)
        store_logits(a, d[i][m], 16 * (m0 + m) + c, (tile * WV + w) * (16 * RT) + 16 * i + 4 * g);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into LDS outlives its block
}

// Few rows: a block owns 16 rows and its W waves take turns over the stages, which they read
// straight to registers (states as FP32 rows, split here), the next one under way; the
// waves' sums meet in LDS.  Bound by the latency of those loads and the launch: 17 states, 4096
// rows of 1536 10.1 us.
template <int MT, int W>
__global__ __launch_bounds__(64 * W, 2) void head_split_kernel(HeadArgs a) {
  __shared__ f32x4 sums[W][MT][64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * kMaxTiles, r0 = blockIdx.x * 16;
  const int chunks = a.K / 8;
  const u32x4 *row =
      reinterpret_cast<const u32x4 *>(a.E + (size_t)(r0 + c < a.rows ? r0 + c : a.rows - 1) * a.K);
  const float *x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int j = 16 * (m0 + m) + c;
    x[m] = a.x + (size_t)(j < a.n ? j : a.n - 1) * a.K;
  }
  u32x4 e[kSteps];
  float v[kSteps][MT][8];
  auto load = [&](int st) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = (st * kSteps + s) * 4 + g, at = k < chunks ? k : chunks - 1;
      e[s] = row[at];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[s][m][i] = x[m][8 * at + i];
    }
  };
  f32x4 d[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) d[m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int stages = a.steps / kSteps;
  load(w < stages ? w : 0);
  for (int st = w; st < stages; st += W) {
    bf16x8 er[kSteps], xr[kSteps][MT][3];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bool in = (st * kSteps + s) * 4 + g < chunks;  // past K: zeros
      er[s] = __builtin_bit_cast(bf16x8, e[s]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t p[3][4];
        split8(v[s][m], in, p);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          xr[s][m][i] = __builtin_bit_cast(bf16x8, (u32x4){p[i][0], p[i][1], p[i][2], p[i][3]});
      }
    }
    load(st + W < stages ? st + W : st);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          d[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(er[s], xr[s][m][p], d[m], 0, 0, 0);
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) sums[w][m][lane] = d[m];
  __syncthreads();
  if (w >= MT) return;
  f32x4 sum = sums[0][w][lane];
#pragma unroll
  for (int i = 1; i < W; ++i) sum += sums[i][w][lane];
  store_logits(a, sum, 16 * (m0 + w) + c, r0 + 4 * g);
}

Workspace g_head_ws;

template <int MT, int RT, int WV, int PER_CU>
int launch_tiles(const HeadArgs &a, int groups) {
  // as many blocks as are resident, an equal number of tiles each
  const int tiles = cdiv(a.rows, 16 * RT * WV);
  const int slots = cdiv(PER_CU * cu_count(), groups), rounds = cdiv(tiles, slots);
  hipLaunchKernelGGL((head_rows_kernel<MT, RT, WV>), dim3(cdiv(tiles, rounds), groups), dim3(64 * WV),
                     0, stream(), a);
  G4_LAUNCH_CHECK("head_rows_kernel");
  return G4_OK;
}

template <int MT>
int launch_split(const HeadArgs &a, int groups) {
  // 8 waves where there is no more than a block per CU, for latency; 4 where blocks share a CU.  us
  // per call, 8 / 4: 17 states 4096 rows 10.1 / 13.7, 64 states 2048 rows 18 / 23, 8192 rows 36 / 31
  const dim3 grid(cdiv(a.rows, 16), groups);
  if ((int)(grid.x * grid.y) <= cu_count())
    hipLaunchKernelGGL((head_split_kernel<MT, 8>), grid, dim3(512), 0, stream(), a);
  else
    hipLaunchKernelGGL((head_split_kernel<MT, 4>), grid, dim3(256), 0, stream(), a);
  G4_LAUNCH_CHECK("head_split_kernel");
  return G4_OK;
}

int launch_head_rows(HeadArgs a) {
  const int tiles = cdiv(a.n, 16);
  const int groups = cdiv(tiles, kMaxTiles), mt = groups > 1 ? kMaxTiles : tiles;
  a.steps = cdiv(cdiv(a.K, 32), kSteps) * kSteps;
  // few rows: us per call, split / tiles, at 5 states 4096 rows 6.4 / 28.6, 32768 29 / 34,
  // 65536 52 / 43; 20 states 16384 rows 30 / 44, 32768 54 / 45; 40 states 16384 rows 46 / 47;
  // 64 states 8192 rows 31 / 52, 16384 60 / 53.  Every group of 64 states is that work again:
  // 128 states 4096 rows 31 / 52, 8192 60 / 53; 192 states 4096 rows 49 / 53; 256 states 2048
  // rows 31 / 54, 4096 58 / 54; 512 states 1000 rows 32 / 56, 8192 223 / 57
  if ((long)cdiv(a.rows, 16) * mt * groups <= 12 * cu_count()) {
    switch (mt) {
      case 1: return launch_split<1>(a, groups);
      case 2: return launch_split<2>(a, groups);
      case 3: return launch_split<3>(a, groups);
      default: return launch_split<4>(a, groups);
    }
  }
  void *mem = nullptr;
  const int all = groups > 1 ? groups * kMaxTiles : tiles;
  if (int rc = g_head_ws.get((size_t)all * a.steps * 3 * 1024, &mem, "g4_bf16_head_rows")) return rc;
  a.parts = static_cast<u32x4 *>(mem);
  hipLaunchKernelGGL(head_parts_kernel, dim3(cdiv(all * a.steps * 64, 256)), dim3(256), 0, stream(), a,
                     all);
  G4_LAUNCH_CHECK("head_parts_kernel");
  switch (mt) {
    case 1: return launch_tiles<1, 2, 4, 4>(a, groups);
    case 2: return launch_tiles<2, 2, 8, 2>(a, groups);
    case 3: return launch_tiles<3, 2, 8, 2>(a, groups);
    default: return launch_tiles<4, 2, 8, 2>(a, groups);
  }
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_bf16_head_rows(const float *x, int n, const void *E, int rows, int in_dim, float *out,
                             size_t out_stride, float scale, float softcap) {
  if (n < 0 || n > kMaxStates || rows < 0 || rows > kMaxRows)
    return fail(G4_E_ARG, "g4_bf16_head_rows: n %d (<= %d), rows %d (<= %d)", n, kMaxStates, rows,
                kMaxRows);
  if (in_dim <= 0 || in_dim % 8 != 0 || in_dim > 4096)
    return fail(G4_E_ARG, "g4_bf16_head_rows: in_dim %d must be a positive multiple of 8 <= 4096",
                in_dim);
  if (out_stride < (size_t)rows || out_stride > (size_t(1) << 60) / (n > 0 ? n : 1))
    return fail(G4_E_ARG, "g4_bf16_head_rows: out_stride %zu for %d rows, n %d", out_stride, rows, n);
  if ((reinterpret_cast<uintptr_t>(E) & 15u) != 0)
    return fail(G4_E_ARG, "g4_bf16_head_rows: E must be 16-byte aligned");
  G4_CHECK_INIT();
  if (n == 0 || rows == 0) return ok();
  int rc = check_device_range(x, (size_t)n * in_dim * 4, "g4_bf16_head_rows x");
  if (!rc) rc = check_device_range(E, (size_t)rows * in_dim * 2, "g4_bf16_head_rows E");
  if (!rc)
    rc = check_device_range(out, ((size_t)(n - 1) * out_stride + rows) * 4, "g4_bf16_head_rows out");
  if (rc) return rc;
  const uint16_t *e = static_cast<const uint16_t *>(E);
  if (n == 1) {
    rc = launch_bf16_head(x, e, rows, in_dim, out, scale, softcap, nullptr);
  } else {
    HeadArgs a{};
    a.x = x;
    a.E = e;
    a.out = out;
    a.out_stride = out_stride;
    a.n = n;
    a.rows = rows;
    a.K = in_dim;
    a.scale = scale;
    a.softcap = softcap;
    rc = launch_head_rows(a);
  }
  return rc ? rc : ok();
}
