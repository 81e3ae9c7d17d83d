// The tied BF16 head for several hidden states:
//   out[j, r] = softcap * tanh((scale * sum_k x[j, k] * E[r, k]) / softcap)
//
// The table is read once for up to 64 states.  Numerics: the BF16 matrix form takes E as it
// is and a state as three BF16 parts, whose sum is the FP32 value (3 x 8 bits of its 24), so
// every product is exact and only the FP32 sums round.
#include "g4_internal.h"
#include "g4_ops.h"

namespace g4 {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxTiles = 4;  // 16-state tiles of a block
constexpr int kRowTiles = 4;  // 16-row tiles of E per wave
constexpr int kBlockRows = 4 * 16 * kRowTiles;

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

// States as parts in the order the matrix instructions read them: step s, part p of tile
// m holds, for lane (c, g), state 16 m + c, k = 32 s + 8 g .. + 7.  Zeros past n and K.
// (The parts are truncations: they have the value's sign and cannot overflow.  The first
// one holds what is not finite.)
__global__ __launch_bounds__(256) void head_parts_kernel(HeadArgs a, int tiles) {
  const int u = blockIdx.x * 256 + threadIdx.x, lane = u & 63, c = lane & 15, g = lane >> 4;
  const int step = (u >> 6) % a.steps, m = (u >> 6) / a.steps;
  if (m >= tiles) return;
  const int j = 16 * m + c, k = 32 * step + 8 * g;
  uint32_t w[3][4] = {};
  if (j < a.n && k < a.K) {
    const float *src = a.x + (size_t)j * a.K + k;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = src[e];
      const uint32_t b = __float_as_uint(v);
      uint32_t p[3] = {b & 0xffff0000u, 0u, 0u};
      if ((b & 0x7f800000u) != 0x7f800000u) {
        const float r = v - __uint_as_float(p[0]);
        p[1] = __float_as_uint(r) & 0xffff0000u;
        p[2] = __float_as_uint(r - __uint_as_float(p[1])) & 0xffff0000u;
      } else if (b & 0x7fffffu) {
        p[0] |= 0x400000u;  // a NaN stays one
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) w[i][e >> 1] |= e & 1 ? p[i] : p[i] >> 16;
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    a.parts[(((size_t)m * a.steps + step) * 3 + i) * 64 + lane] = (u32x4){w[i][0], w[i][1], w[i][2], w[i][3]};
}

// A block owns 256 rows of E, 64 per wave, and MT 16-state tiles.  D = E . X^T: lane (c, g)
// feeds row c of a row tile and state c, k 8 g .. + 7 of a step, and gets state c of rows
// 4 g .. + 3.  A stage is KS steps: the waves' rows go to registers, the states' parts to
// LDS (direct loads, two buffers), both issued one stage ahead.
template <int MT, int KS>
__global__ __launch_bounds__(256, 2) void head_rows_kernel(HeadArgs a) {
  constexpr int P = KS * MT * 3;  // 1 KB pieces of a stage
  __shared__ u32x4 xs[2][P * 64];
  typedef __attribute__((address_space(3))) void *lds_ptr;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int r0 = blockIdx.x * kBlockRows + w * (16 * kRowTiles);
  const int m0 = blockIdx.y * kMaxTiles;
  const int chunks = a.K / 8;
  const u32x4 *row[kRowTiles];
#pragma unroll
  for (int i = 0; i < kRowTiles; ++i) {
    const int r = r0 + 16 * i + c;
    row[i] = reinterpret_cast<const u32x4 *>(a.E + (size_t)(r < a.rows ? r : a.rows - 1) * a.K);
  }
  auto load_rows = [&](int stage, u32x4 (&e)[KS][kRowTiles]) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = (stage * KS + s) * 4 + g, at = k < chunks ? k : chunks - 1;
#pragma unroll
      for (int i = 0; i < kRowTiles; ++i) e[s][i] = __builtin_nontemporal_load(row[i] + at);
    }
  };
  auto load_states = [&](int stage) {
    constexpr int W = (P + 3) / 4;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int p = w + 4 * i < P ? w + 4 * i : P - 1;  // the last one again, same bytes
      const int m = p / (KS * 3), q = p - m * (KS * 3);
      __builtin_amdgcn_global_load_lds(
          (const void *)(a.parts + (((size_t)(m0 + m) * a.steps + stage * KS) * 3 + q) * 64 + lane),
          (lds_ptr)(xs[stage & 1] + p * 64), 16, 0, 0);
    }
  };
  f32x4 d[kRowTiles][MT];
#pragma unroll
  for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) d[i][m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int stages = a.steps / KS;
  auto stage = [&](int st, const u32x4 (&e)[KS][kRowTiles], u32x4 (&next)[KS][kRowTiles]) {
    // this stage has landed everywhere, and the other buffer is free
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (st + 1 < stages) {
      load_rows(st + 1, next);
      load_states(st + 1);
    }
    const u32x4 *x = xs[st & 1] + lane;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int p = 2; p >= 0; --p) {
          const bf16x8 b = __builtin_bit_cast(bf16x8, x[((m * KS + s) * 3 + p) * 64]);
#pragma unroll
          for (int i = 0; i < kRowTiles; ++i)
            d[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, e[s][i]), b,
                                                              d[i][m], 0, 0, 0);
        }
  };
  u32x4 e0[KS][kRowTiles], e1[KS][kRowTiles];
  load_rows(0, e0);
  load_states(0);
  for (int st = 0; st < stages; st += 2) {
    stage(st, e0, e1);
    if (st + 1 < stages) stage(st + 1, e1, e0);
  }
  const bool wide = ((reinterpret_cast<uintptr_t>(a.out) & 15) | (a.out_stride & 3)) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int j = 16 * (m0 + m) + c;
    if (j >= a.n) continue;
    float *o = a.out + (size_t)j * a.out_stride;
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i) {
      const int r = r0 + 16 * i + 4 * g;
      f32x4 v = d[i][m] * a.scale;
      if (a.softcap > 0.f)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = tanhf(v[k] / a.softcap) * a.softcap;
      if (wide && r + 3 < a.rows) {
        *reinterpret_cast<f32x4 *>(o + r) = v;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (r + k < a.rows) o[r + k] = v[k];
      }
    }
  }
}

Workspace g_head_ws;

int launch_head_rows(HeadArgs a) {
  const int tiles = cdiv(a.n, 16), ks = 2;
  a.steps = cdiv(cdiv(a.K, 32), ks) * ks;
  const int groups = cdiv(tiles, kMaxTiles), mt = groups > 1 ? kMaxTiles : tiles;
  void *mem = nullptr;
  const int all = groups > 1 ? groups * kMaxTiles : tiles;
  if (int rc = g_head_ws.get((size_t)all * a.steps * 3 * 1024, &mem, "g4_bf16_head_rows")) return rc;
  a.parts = static_cast<u32x4 *>(mem);
  hipLaunchKernelGGL(head_parts_kernel, dim3(cdiv(all * a.steps * 64, 256)), dim3(256), 0, stream(), a,
                     all);
  G4_LAUNCH_CHECK("head_parts_kernel");
  void (*kernel)(HeadArgs) = mt == 1   ? head_rows_kernel<1, 2>
                             : mt == 2 ? head_rows_kernel<2, 2>
                             : mt == 3 ? head_rows_kernel<3, 2>
                                       : head_rows_kernel<4, 2>;
  hipLaunchKernelGGL(kernel, dim3(cdiv(a.rows, kBlockRows), groups), dim3(256), 0, stream(), a);
  G4_LAUNCH_CHECK("head_rows_kernel");
  return G4_OK;
}

}  // namespace
}  // namespace g4

using namespace g4;

G4_API int g4_bf16_head_rows(const float *x, int n, const void *E, int rows, int in_dim, float *out,
                             size_t out_stride, float scale, float softcap) {
  if (n < 0 || rows < 0) return fail(G4_E_ARG, "g4_bf16_head_rows: n %d, rows %d", n, rows);
  if (in_dim <= 0 || in_dim % 8 != 0 || in_dim > 4096)
    return fail(G4_E_ARG, "g4_bf16_head_rows: in_dim %d must be a positive multiple of 8 <= 4096",
                in_dim);
  if (out_stride < (size_t)rows)
    return fail(G4_E_ARG, "g4_bf16_head_rows: out_stride %zu < rows %d", out_stride, rows);
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
