// Attention over a cache held in 4 bits, with the weight that each key got if asked for.
#include <math.h>

#include <type_traits>

#include "g4_gemv.h"
#include "g4_internal.h"
#include "g4_key_weights.h"
#include "g4_kv4.h"

namespace g4 {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t any_u16 __attribute__((may_alias));

constexpr float kLog2e = 1.4426950408889634f;
// How far (log 2) a score may pass its row's reference before the outputs are scaled again.  Weights
// are split into two FP16 values times 2^(15 - kSlack), so one is held to 2^-22 of it, or to 2^-38 of
// its row's largest if that is more.  (The attention over FP32 caches takes three BF16 parts of all four
// operands, 24 bits.  Here k and v are exact in one FP16 value and would not be in one of BF16, 11 bits of
// a nibble times a scale, so q and the weights are FP16 too: two values each, two products instead
// of six, and the error that is left is far below what 4 bits of k and v make.)
constexpr float kSlack = 2.f;
constexpr float kWeight = 1 << (15 - (int)kSlack);
constexpr int kStep = 32;                   // keys of a wave's step
constexpr int kMaxSplits = 512;

struct Kv4Args {
  const float *q;
  const uint32_t *k, *v;
  const uint16_t *ks, *vs;
  float *y;
  float *part;  // [splits][rows][hd], each split's outputs
  Scores s;     // score null: not kept
};

// Scales that are not plain: how many octaves of them one product takes, and how far (log 2) a key's
// largest contribution may pass the outputs' own exponent.
constexpr int kBand = 12, kRoom = 64;

// Scales are taken times 2^kLift.  Plain ones, from 2^-18 up to 2^7, then are normal FP16 numbers, and
// so are eight times they: BF16 bits of the least and how many there are.
constexpr int kLift = 4;
constexpr uint16_t kLeastScale = (127 - 14 - kLift) << 7, kPlainScales = 25 << 7;

// Eight values of a cache as FP16, in pairs (0, 4) (1, 5) (2, 6) (3, 7) of the word's nibbles or of
// two words' halves: a nibble n in the mantissa's upper four bits under the exponent of 16 is
// 16 + n, and (16 + n) s - 24 s = (n - 8) s is exact in one fused step: s has 8 bits, 24 s 10.
struct Scale {
  half2_t s, c;  // s and -24 s
};
__device__ __forceinline__ Scale scale_of(half2_t s) { return {s, s * (half2_t){(_Float16)-24.f, (_Float16)-24.f}}; }
__device__ __forceinline__ Scale scale_pair(float a, float b) {
  return scale_of(__builtin_convertvector((f32x2_t){a, b}, half2_t));
}
// (mask and exponent in registers, so that one instruction takes both)
struct Magic {
  uint32_t mask, exponent;
  __device__ __forceinline__ Magic() {
    asm("v_mov_b32 %0, 0x03c003c0" : "=v"(mask));
    asm("s_mov_b32 %0, 0x4c004c00" : "=s"(exponent));
  }
};
// The same for two BF16 scales as they are: FP16 bits by whole numbers, and how far they lie from the
// least plain one, kept as the largest seen.
__device__ __forceinline__ Scale plain_pair(uint32_t lo, uint32_t hi, ushort2_t &beyond) {
  const ushort2_t u = __builtin_bit_cast(ushort2_t, __builtin_amdgcn_perm(hi, lo, 0x05040100u));
  const ushort2_t d = u - (ushort2_t){kLeastScale, kLeastScale};
  beyond = __builtin_elementwise_max(beyond, d);
  constexpr uint16_t least = (kLeastScale - ((127 - kLift - 15) << 7)) << 3;
  return scale_of(__builtin_bit_cast(half2_t, (ushort2_t)(d * (ushort2_t){8, 8} + (ushort2_t){least, least})));
}
template <int T>
__device__ __forceinline__ uint32_t value_pair(uint32_t w, const Scale &x, const Magic &mg) {
  const uint32_t sh = T == 0 ? w << 6 : T == 1 ? w << 2 : T == 2 ? w >> 2 : w >> 6;
  const half2_t h = __builtin_bit_cast(half2_t, (sh & mg.mask) | mg.exponent);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(h, x.s, x.c));
}

// max over the lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float group_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Rows of q whose exponent a factor of FP32 holds with all its bits.
__device__ __forceinline__ bool usual_row(int e) { return e >= -120; }
// A BF16 scale's exponent, 127 more: 1 .. 254, 255 if it is no number; 0 for a scale of 0.  And the scale
// under another one: from 2^(6 - kBand) up to 2^6 if that is within kBand above it.
__device__ __forceinline__ int scale_exponent(uint32_t bits) { return bits & 0x7fffu ? max((int)(bits >> 7 & 255u), 1) : 0; }
__device__ __forceinline__ float scale_under(uint32_t bits, int top) { return ldexpf(bf16_to_f32(bits), 132 - top); }

// The kernel's arguments once more from memory, for the general way behind its loop: held in registers
// through it, they cost 4000 rows of 256 with a window of 512 66.3 us for 63.6.
__device__ __forceinline__ const Kv4Args &args_again() {
  uint64_t p = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const Kv4Args *)reinterpret_cast<const __attribute__((address_space(4))) Kv4Args *>(p);
}

// Dims that a wave works on (DW); the waves of a key group share the head dim.
template <int HD>
constexpr int kDims = HD > 256 ? 256 : HD;
template <int HD, int W, int DW = kDims<HD>>
constexpr int kGroups = W / (HD / DW);  // key groups of a block

// Eight weights times `up` as sums of two FP16 values.  PAIR: the lo part alone for lanes 8 .. 15 of each
// 16.
template <bool PAIR>
__device__ __forceinline__ void weight_parts(const float (&p)[8], float up, half8_t &h, half8_t &l) {
  u32x4 h4, l4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x2_t z = {p[2 * j] * up, p[2 * j + 1] * up};
    const half2_t y = __builtin_convertvector(z, half2_t);
    h4[j] = __builtin_bit_cast(uint32_t, y);
    l4[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(z - __builtin_convertvector(y, f32x2_t), half2_t));
    if (PAIR && (threadIdx.x & 8)) h4[j] = l4[j];
  }
  h = __builtin_bit_cast(half8_t, h4);
  l = __builtin_bit_cast(half8_t, l4);
}

// x of lane c ^ 8 of each 16
__device__ __forceinline__ float other_half(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));  // row_ror:8
}

// A block owns 16 RT rows of [qrows * heads, hd] and a run of 32-key steps, which its key groups
// take in turn; lane (c, g) of a wave works for row c throughout:
//   S^T = K . Q^T     keys 4 g .. + 3 of each half per lane; q in LDS as FP16 hi + lo; a group's
//                     waves add theirs through LDS, in order, so that they hold the same scores
//   softmax           running maximum and sum per row
//   O^T += V^T . P^T  the lane's weights are its operand as they are, FP16 hi + lo; a lane unpacks
//                     DW / 16 dims of 8 keys
// PAIR: 8 rows, lanes c and c + 8 both working for row c, with the hi part in the first and the lo
// part in the second one, so that one product does both.
// The values are used where they are unpacked, in the lanes that the matrix instructions want them:
// nothing of k or v passes through LDS.  A row's maximum is a reference that follows the scores with
// kSlack, so the outputs are hardly ever scaled again; a step's loads are under way during the one
// before it.
// A block that met a scale that is not plain (or a row of q below 2^-103) does its rows again in the
// general way, without PLAIN, in as many products as the step has bands of kBand octaves of scales: k's
// counted from each key's largest, v's from the step's, these with the weights of the keys in a band
// scaled for their largest; exponents are put back in FP32.  (With one exponent per row of the cache and
// of the outputs, a large value takes the bits of the row's small ones and of all other keys' weights,
// in all dims.)  One token over 16001 keys of 512, all scales plain / none: 13.4 / 19.5 us; both ways in
// one loop, 188 bytes of spills per lane.
// What bounds it: one token over 131072 keys of 512 (75.5 MB) 22.0 us without its join, 3.4 TB/s: 4 steps
// per wave, each about 600 vector instructions (three per pair of values unpacked: shift, mask and
// exponent, fused step) and the products between them, and as long again before and behind them
// (launch, q, the groups' sums, 8.4 MB of partial outputs).  Over 16001 keys a wave has one step:
// 9.1 us, a chain of latencies (by the clock in a block, as it came in: launch and arguments 1.2, q and the
// first k 1.8, the scores 1.1, softmax and outputs 1.9, the groups' sums and stores 1.9; what is left
// lies between two launches).
template <int HD, int RT, bool PAIR, int W, int DW>
struct AttendSmem {
  static constexpr int DQ = HD / DW, KG = kGroups<HD, W, DW>, R = PAIR ? 8 : 16 * RT;
  union {
    struct {
      u32x4 q[PAIR ? 1 : 2][RT][HD / 32][64];
      f32x4 sx[DQ > 1 ? 2 : 0][KG][DQ][RT][2][64];  // the waves' scores, two buffers
    } loop;
    float o[KG > 1 ? KG / 2 : 1][PAIR ? 8 : 16][HD + 4];
  };
  int xq[R];
  float2 wml[KG][R];
  int other[W];
};
template <int HD, int RT, bool PAIR, int W, int DW, bool PLAIN>
__device__ __forceinline__ void attend(const Kv4Args &a, int R0, int split, const Run &run, AttendSmem<HD, RT, PAIR, W, DW> &sm) {
  constexpr int DQ = HD / DW, KG = kGroups<HD, W, DW>;
  static_assert(!PAIR || RT == 1, "one tile");
  constexpr int KW = DW / 32;                  // words of a key per lane, and products
  constexpr int KS = DW >= 128 ? DW / 128 : 1; // scales of a key per lane
  constexpr int VD = DW / 16;                  // dims per lane, and output tiles
  constexpr int VW = VD >= 8 ? VD / 8 : 1;     // words of them (64: half a word)
  constexpr int R = PAIR ? 8 : 16 * RT;
  const Scores &S = a.s;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kg = w / DQ, dq = w % DQ, c = lane & 15, g = lane >> 4;
  const int cr = PAIR ? c & 7 : c;  // the lane's row of a tile
  const int pa = S.pos0 + R0 / S.heads, pb = S.pos0 + (min(R0 + R, S.rows) - 1) / S.heads;
  const int lo = run.lo, hi = run.hi, steps = run.steps, t0 = run.t0, t1 = run.t1;

  uint32_t kr[2][KW], ksr[2][KS], vr[8][VW], vsr[8];
  // Loads by an offset per lane from a step's first row; rows behind the last key give zeros, which
  // `look_*` makes 1 among the scales.
  const int row_k = c, row_v = 4 * g;
  const uint32_t at_k = row_k * (HD / 2) + dq * (DW / 2) + g * (DW >= 128 ? 16 : 8);
  const uint32_t at_ks = row_k * (HD / 16) + dq * (DW / 16) + (DW >= 128 ? g : g >> 1) * 2;
  const uint32_t at_v = row_v * (HD / 2) + dq * (DW / 2) + c * (DW / 32);
  const uint32_t at_vs = row_v * (HD / 16) + dq * (DW / 16) + c * DW / 512 * 2;
  auto rows_of = [&](const void *plane, int step, int bytes) {
    const int k0 = __builtin_amdgcn_readfirstlane(lo + min(step, steps - 1) * kStep);
    char *p = const_cast<char *>(static_cast<const char *>(plane)) + (size_t)k0 * bytes;
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, min(hi - k0, kStep) * bytes, 0x00020000);
  };
  auto load_k = [&](int step) {
    const auto p = rows_of(a.k, step, HD / 2), ps = rows_of(a.ks, step, HD / 16);
#pragma unroll
    for (int T = 0; T < 2; ++T) {
#pragma unroll
      for (int J = 0; J < KS; ++J) {
        if constexpr (DW >= 128) {
          const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(p, at_k + 64 * J + 16 * T * (HD / 2), 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) kr[T][4 * J + i] = x[i];
        } else {
          const u32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(p, at_k + 16 * T * (HD / 2), 0, 0);
          kr[T][0] = x[0];
          kr[T][1] = x[1];
        }
        ksr[T][J] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ps, at_ks + 8 * J + 16 * T * (HD / 16), 0, 0);
      }
    }
  };
  auto load_v = [&](int step) {
    const auto p = rows_of(a.v, step, HD / 2), ps = rows_of(a.vs, step, HD / 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t at = at_v + (16 * (j >> 2) + (j & 3)) * (HD / 2);
      if constexpr (DW == 256) {
        const u32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(p, at, 0, 0);
        vr[j][0] = x[0];
        vr[j][1] = x[1];
      } else if constexpr (DW == 128) {
        vr[j][0] = __builtin_amdgcn_raw_buffer_load_b32(p, at, 0, 0);
      } else {
        vr[j][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(p, at, 0, 0);
      }
      vsr[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ps, at_vs + (16 * (j >> 2) + (j & 3)) * (HD / 16), 0, 0);
    }
  };
  auto look_k = [&](int last) {
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int J = 0; J < KS; ++J) ksr[T][J] = 16 * T + row_k > last ? 0x3f80u : ksr[T][J];
  };
  auto look_v = [&](int last) {
#pragma unroll
    for (int j = 0; j < 8; ++j) vsr[j] = 16 * (j >> 2) + row_v + (j & 3) > last ? 0x3f80u : vsr[j];
  };
  // q: a thread takes 8 values of a row, whose largest gets the exponent 13.  Its loads go first, so that
  // it is worked on while the first k and v are under way (loads arrive in their order).
  {
    constexpr int TW = HD / 8, PASS = 64 * W / TW;
    constexpr int N = (R + PASS - 1) / PASS;
    const int wd = t % TW;
    f32x4 qx[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = min(R0 + min(t / TW + i * PASS, R - 1), S.rows - 1);
      const f32x4 *p = reinterpret_cast<const f32x4 *>(a.q + (size_t)row * HD + 8 * wd);
      qx[i][0] = p[0];
      qx[i][1] = p[1];
    }
    if constexpr (PLAIN) {
      asm volatile("" ::: "memory");
      load_k(t0 + kg);
      load_v(t0 + kg);
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int pass = 0; pass < N; ++pass) {
      const int r = t / TW + pass * PASS;
      const f32x4 x0 = qx[pass][0], x1 = qx[pass][1];
      int top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = max(top, max(__float_as_int(x0[i]) & 0x7fffffff, __float_as_int(x1[i]) & 0x7fffffff));
      top = team_max<TW>(top);
      const int e = top == 0 || top >= 0x7f800000 ? 0 : max((top >> 23) - 127, -126);
      if (r >= R) break;
      if (wd == 0) sm.xq[r] = e - 13 - kLift;
      u32x4 hi4, lo4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_t x = {ldexpf(x0[i], 13 - e), ldexpf(x1[i], 13 - e)};
        const half2_t h = __builtin_convertvector(x, half2_t);
        const half2_t l = __builtin_convertvector(x - __builtin_convertvector(h, f32x2_t), half2_t);
        hi4[i] = __builtin_bit_cast(uint32_t, h);
        lo4[i] = __builtin_bit_cast(uint32_t, l);
      }
      // the wave's lane (c, g) holds dims g DW / 4 .. of each 128, or of its 64
      const int n = DW >= 128 ? (wd >> 4) * 4 + (wd & 3) : (wd >> 3) * 2 + (wd & 1);
      const int at = DW >= 128 ? (wd >> 2) & 3 : (wd >> 1) & 3;
      sm.loop.q[0][r >> 4][n][(r & 15) + 16 * at] = hi4;
      sm.loop.q[PAIR ? 0 : 1][r >> 4][n][(r & 15) + 16 * at + (PAIR ? 8 : 0)] = lo4;
    }
  }
  __syncthreads();

  int pos[RT], xe[RT];
  int E[RT];  // outputs are held times 2^(15 + kLift - E)
  float xf[RT], m[RT], l[RT];
  ushort2_t beyond = {0, 0};  // the scales' largest distance from the least plain one
  f32x4 o[RT][VD];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    pos[r] = S.pos0 + min(R0 + 16 * r + cr, S.rows - 1) / S.heads;
    xe[r] = sm.xq[16 * r + cr];
    xf[r] = PLAIN ? ldexpf(kLog2e, xe[r]) : kLog2e;
    if (!usual_row(xe[r])) beyond = (ushort2_t){0xffff, 0xffff};
    m[r] = kNoScore;
    l[r] = 0.f;
    E[r] = (int)kSlack;
#pragma unroll
    for (int n = 0; n < VD; ++n) o[r][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  uint32_t none = 0;  // bit 4 r + v: register v of row tile r holds no numbers
  const Magic mg;
  const int turns = (t1 - t0 + KG - 1) / KG;
  if constexpr (PLAIN) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the waits in the loop then count its own loads
  for (int it = 0; it < turns; ++it) {
    const int step = t0 + kg + it * KG, key0 = lo + step * kStep;
    const bool mine = step < t1;
    const int last = hi - 1 - (lo + min(step, steps - 1) * kStep);  // row of the step
    if constexpr (!PLAIN) load_k(step);
    if (last < kStep - 1) look_k(last);
    // S^T = K . Q^T with the values' scales x
    auto scores = [&](const Scale (&x)[2][KS], f32x4 (&y)[RT][2]) {
      f32x4 sh[RT][2], sl[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < 2; ++T) sh[r][T] = sl[r][T] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int J = 0; J < KS; ++J) {
#pragma unroll
        for (int i = 0; i < KW / KS; ++i) {
          const int n = J * (KW / KS) + i;
          half8_t kv[2];
#pragma unroll
          for (int T = 0; T < 2; ++T) {
            const uint32_t wd = kr[T][n];
            kv[T] = __builtin_bit_cast(
                half8_t, (u32x4){value_pair<0>(wd, x[T][J], mg), value_pair<1>(wd, x[T][J], mg), value_pair<2>(wd, x[T][J], mg),
                                 value_pair<3>(wd, x[T][J], mg)});
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const half8_t qh = __builtin_bit_cast(half8_t, sm.loop.q[0][r][dq * KW + n][lane]);
#pragma unroll
            for (int T = 0; T < 2; ++T) sh[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv[T], qh, sh[r][T], 0, 0, 0);
            if constexpr (!PAIR) {
              const half8_t ql = __builtin_bit_cast(half8_t, sm.loop.q[1][r][dq * KW + n][lane]);
#pragma unroll
              for (int T = 0; T < 2; ++T)
                sl[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv[T], ql, sl[r][T], 0, 0, 0);
            }
          }
          if (i & 1) __builtin_amdgcn_sched_barrier(0);  // (else all is unpacked at once, and spilled)
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[r][T][i] = (sh[r][T][i] + (PAIR ? other_half(sh[r][T][i]) : sl[r][T][i])) * xf[r];
    };
    f32x4 s[RT][2];
    Scale x[2][KS];
    if constexpr (PLAIN) {
      ushort2_t far = {0, 0};
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int J = 0; J < KS; ++J) x[T][J] = plain_pair(ksr[T][J], ksr[T][J], far);
      if (mine) beyond = __builtin_elementwise_max(beyond, far);
      scores(x, s);
    } else {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < 2; ++T) s[r][T] = (f32x4){0.f, 0.f, 0.f, 0.f};
      uint32_t left = ~0u;  // scales of this lane that have yet to be taken
      for (;;) {  // 22 times at most: each takes kBand of 255 exponents of every key, and some scale
        int top[2];
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          top[T] = 0;
#pragma unroll
          for (int J = 0; J < KS; ++J)
            if (left >> (T * KS + J) & 1) top[T] = max(top[T], scale_exponent(ksr[T][J]));
          top[T] = max(top[T], __shfl_xor(top[T], 16, 64));
          top[T] = max(top[T], __shfl_xor(top[T], 32, 64));
        }
        if (!__any(max(top[0], top[1]) > 0)) break;
        // (each time anew, as v below)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < KW; ++i) asm volatile("" : "+v"(kr[T][i]));
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int J = 0; J < KS; ++J) {
            const bool in = (left >> (T * KS + J) & 1) && scale_exponent(ksr[T][J]) > max(top[T] - kBand, 0);
            if (in) left &= ~(1u << (T * KS + J));
            const float f = in ? scale_under(ksr[T][J], top[T]) : 0.f;
            x[T][J] = scale_pair(f, f);
          }
        f32x4 y[RT][2];
        scores(x, y);
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = __shfl(top[T], 4 * g + i, 64) - 132 + kLift;
            // (q's exponent and the key's at once: either alone may overflow)
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][T][i] += ldexpf(y[r][T][i], xe[r] + e);
          }
      }
    }
    if constexpr (PLAIN) load_k(step + KG);
    else load_v(step);
    if constexpr (DQ > 1) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < 2; ++T) sm.loop.sx[it & 1][kg][dq][r][T][lane] = s[r][T];
      __syncthreads();
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          s[r][T] = sm.loop.sx[it & 1][kg][0][r][T][lane];
#pragma unroll
          for (int d = 1; d < DQ; ++d) s[r][T] += sm.loop.sx[it & 1][kg][d][r][T][lane];
        }
    }

    // v: keys 4 g + i of each half, as the weights are held
    if (last < kStep - 1) look_v(last);
    Scale vx[4];
    uint32_t odd = 0;  // keys of which this lane's dims are no numbers
    if constexpr (PLAIN) {
      ushort2_t far = {0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) vx[j] = plain_pair(vsr[2 * j], vsr[2 * j + 1], far);
      if (mine) beyond = __builtin_elementwise_max(beyond, far);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((vsr[j] & 0x7fff) >= 0x7f80) {
          odd |= 1u << j;
          vsr[j] = 0;
        }
    }
    // whether every row sees every key of the step
    const bool inner = mine && key0 + kStep - 1 <= pa && (S.window == 0 || key0 > pb - S.window);
    half8_t ph[RT], pl[RT];
    uint32_t seen[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float x[8];
      seen[r] = 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[r][j >> 2][j & 3];
      if (!inner) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
          if (!mine || key > pos[r] || (S.window > 0 && key <= pos[r] - S.window)) {
            x[j] = -INFINITY;
            seen[r] &= ~(1u << j);
          }
        }
      }
      const int row = min(R0 + 16 * r + cr, S.rows - 1);
      if (S.score && mine && dq == 0) {
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          *reinterpret_cast<float4 *>(S.score + (size_t)row * S.stride + (key0 + 16 * T + 4 * g - S.first)) =
              make_float4(x[4 * T], x[4 * T + 1], x[4 * T + 2], x[4 * T + 3]);
        }
      }
      float tm = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      // (fmaxf drops a NaN score, whose weight is NaN.)
      tm = group_max(tm);
      const float mn = tm > m[r] + kSlack ? tm : m[r];
      const float corr = __builtin_amdgcn_exp2f(m[r] - mn);
      float p[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(x[j] - mn);
        sum += p[j];
        s[r][j >> 2][j & 3] = x[j] - mn;
      }
      l[r] = fmaf(l[r], corr, sum);
      if constexpr (PLAIN) weight_parts<PAIR>(p, kWeight, ph[r], pl[r]);
      m[r] = mn;
      if (__any(corr != 1.f)) {
#pragma unroll
        for (int n = 0; n < VD; ++n) o[r][n] *= corr;
      }
    }
    // O^T += V^T . P^T with the values' scales vs, or a factor of the products
    auto outputs = [&](const Scale (&vs)[4], const half8_t (&wh)[RT], const half8_t (&wl)[RT], auto scaled, const float (&factor)[RT]) {
#pragma unroll
      for (int i = 0; i < VW; ++i) {
#pragma unroll
        for (int h = 0; h < (VD >= 8 ? 2 : 1); ++h) {
          uint32_t d[4];  // the word's lower or upper four dims of two keys
#pragma unroll
          for (int j = 0; j < 4; ++j)
            d[j] = __builtin_amdgcn_perm(vr[2 * j + 1][i], vr[2 * j][i], h ? 0x07060302u : 0x05040100u);
          auto tile = [&](auto T) {
            constexpr int e = decltype(T)::value;
            const half8_t vv = __builtin_bit_cast(
                half8_t, (u32x4){value_pair<e>(d[0], vs[0], mg), value_pair<e>(d[1], vs[1], mg), value_pair<e>(d[2], vs[2], mg),
                                 value_pair<e>(d[3], vs[3], mg)});
            const int n = 8 * i + 4 * h + e;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              f32x4 y = scaled ? (f32x4){0.f, 0.f, 0.f, 0.f} : o[r][n];
              y = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, wh[r], y, 0, 0, 0);
              if constexpr (!PAIR) y = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, wl[r], y, 0, 0, 0);
              o[r][n] = scaled ? o[r][n] + y * factor[r] : y;
            }
          };
          tile(std::integral_constant<int, 0>());
          tile(std::integral_constant<int, 1>());
          tile(std::integral_constant<int, 2>());
          tile(std::integral_constant<int, 3>());
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    float factor[RT] = {};
    if constexpr (PLAIN) {
      outputs(vx, ph, pl, std::false_type(), factor);
    } else {
      uint32_t left = 0;  // keys of which this lane's dims have yet to be added
#pragma unroll
      for (int j = 0; j < 8; ++j) left |= (vsr[j] & 0x7fff ? 1u : 0u) << j;
      for (;;) {  // 22 times at most: each takes kBand of 254 exponents, and some key
        int top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (left >> j & 1) top = max(top, scale_exponent(vsr[j]));
        top = __builtin_amdgcn_readfirstlane(team_max<64>(top));
        if (top == 0) break;
        // (each time anew: unpacked before the loop, the codes alone would fill the registers)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < VW; ++i) asm volatile("" : "+v"(vr[j][i]));
        float f[8];
        uint32_t take = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = (left >> j & 1) && scale_exponent(vsr[j]) > top - kBand;
          take |= (in ? 1u : 0u) << j;
          f[j] = in ? scale_under(vsr[j], top) : 0.f;
        }
        left &= ~take;
        Scale vs[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[j] = scale_pair(f[2 * j], f[2 * j + 1]);
        uint32_t here = take;  // of any dims
#pragma unroll
        for (int i = 1; i < 16; i *= 2) here |= (uint32_t)__shfl_xor((int)here, i, 64);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          // these keys' weights times 2^(15 - F)
          float F = -1000.f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (here >> j & 1) F = fmaxf(F, s[r][j >> 2][j & 3]);
          F = ceilf(group_max(F));
          float z[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            z[j] = here >> j & 1 ? __builtin_amdgcn_exp2f(s[r][j >> 2][j & 3] - F) : 0.f;
          weight_parts<PAIR>(z, 32768.f, ph[r], pl[r]);
          const int E2 = max(E[r], (int)F + top - 123 - kRoom);
          if (__any(E2 != E[r])) {
            const float down = ldexpf(1.f, E[r] - E2);
#pragma unroll
            for (int n = 0; n < VD; ++n) o[r][n] *= down;
          }
          E[r] = E2;
          factor[r] = ldexpf(1.f, (int)F + top - 132 + kLift - E2);
        }
        outputs(vs, ph, pl, std::true_type(), factor);
      }
    }
    if (!PLAIN && __any(odd != 0)) {  // rows that see such a key: NaN in its dims
#pragma unroll
      for (int r = 0; r < RT; ++r)
        for (int i = 0; i < 16; ++i) {  // keys of lanes (., i / 4), dims of register i % 4
          const uint32_t bad = (uint32_t)__shfl((int)odd, 16 * (i >> 2) + 4 * g + (i & 3), 64);
          if (bad & (uint32_t)__shfl((int)seen[r], 16 * (i >> 2) + c, 64)) none |= 1u << (4 * r + (i & 3));
        }
    }
    if constexpr (PLAIN) load_v(step + KG);
  }

  // the key groups' sums through LDS, the upper half of the groups to the lower one
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    if (g == 0 && dq == 0) sm.wml[kg][16 * r + cr] = make_float2(m[r], l[r]);
  }
  if constexpr (PLAIN) {
    const bool other = __any(max(beyond[0], beyond[1]) >= kPlainScales);
    if (lane == 0) sm.other[w] = other;
  }
  __syncthreads();
  if constexpr (PLAIN) {
    int again = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) again |= sm.other[i];
    if (__builtin_amdgcn_readfirstlane(again)) {
      __syncthreads();
      const Kv4Args &b = args_again();
      attend<HD, RT, PAIR, W, DW, false>(b, R0, split, Run(b.s, R0, R, split, kStep), sm);
      return;
    }
  }
  const bool whole = S.splits == 1;
  float *out = whole ? a.y : a.part + (size_t)split * S.rows * HD;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float M = kNoScore, L = 0.f;
#pragma unroll
    for (int i = 0; i < KG; ++i) M = fmaxf(M, sm.wml[i][16 * r + cr].x);
#pragma unroll
    for (int i = 0; i < KG; ++i)
      L = fmaf(sm.wml[i][16 * r + cr].y, __builtin_amdgcn_exp2f(sm.wml[i][16 * r + cr].x - M), L);
    const int row = R0 + 16 * r + cr;
    if (S.ml && w == 0 && g == 0 && row < S.rows) S.ml[(size_t)row * S.splits + split] = make_float2(M, L);
    // (a split of which the row sees nothing: 0, not 0 / 0)
    float f = __builtin_amdgcn_exp2f(m[r] - M) / L;
    if (!whole && L == 0.f) f = 0.f;
    f = ldexpf(f, E[r] - 15 - kLift);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float fv = none >> (4 * r + v) & 1 ? __int_as_float(0x7fc00000) : f;
#pragma unroll
      for (int n = 0; n < VD; ++n) {
        if (PAIR) o[r][n][v] += other_half(o[r][n][v]);
        o[r][n][v] *= fv;
      }
    }
    // lane (c, g): tile n, register v holds dim (4 g + v) VD + n of the wave's
#pragma unroll
    for (int half = KG / 2; half >= 1; half /= 2) {
      float *at = &sm.o[kg & (half - 1)][cr][dq * DW + 4 * g * VD];
      if (kg >= half && kg < 2 * half && c == cr)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int n = 0; n < VD; n += 4)
            *reinterpret_cast<f32x4 *>(at + v * VD + n) =
                (f32x4){o[r][n][v], o[r][n + 1][v], o[r][n + 2][v], o[r][n + 3][v]};
      __syncthreads();
      if (kg < half)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int n = 0; n < VD; n += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(at + v * VD + n);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][n + e][v] += x[e];
          }
      if (half > 1 || r + 1 < RT) __syncthreads();
    }
    if (kg == 0 && c == cr && row < S.rows) {
      float *p = out + (size_t)row * HD + dq * DW + 4 * g * VD;
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int n = 0; n < VD; n += 4)
          *reinterpret_cast<f32x4 *>(p + v * VD + n) =
              (f32x4){o[r][n][v], o[r][n + 1][v], o[r][n + 2][v], o[r][n + 3][v]};
    }
  }
}

template <int HD, int RT, bool PAIR, int W, int DW = kDims<HD>>
__global__ __launch_bounds__(64 * W, 2) void attn_kv4_kernel(Kv4Args a) {
  __shared__ AttendSmem<HD, RT, PAIR, W, DW> sm;
  attend<HD, RT, PAIR, W, DW, true>(a, blockIdx.x * sm.R, blockIdx.y, Run(a.s, blockIdx.x * sm.R, sm.R, blockIdx.y, kStep), sm);
}

// Many rows of a cache whose scales all are plain, by the same mathematics: a block owns 16 RT rows and a
// run of 32-key steps; its W waves share the head dim both for the scores and for the outputs, so that
// each value of the cache is unpacked once for all rows.  The waves' partial scores go through LDS; wave
// w < RT adds those of rows 16 w .. + 15, in order, does their softmax and leaves the weights in LDS for
// all.  The next step's scores are formed before, so that one barrier per step makes both known.
// A block that met another scale (or a row of q below 2^-103) does its rows again in the general way, 16 at a
// time (a second launch for them cost all calls 2 to 3 us).
// 512 rows over 4608 keys of 512 (8 heads, 73 GFLOP with both parts of q and of the weights): 83.0 us
// without the join, 0.88 PFLOP/s, where a product of 8192^3 FP16 values runs at 1.08 (traced 92, until its
// 33.5 MB of partial outputs are in memory).  The matrix units are busy for 40% of the cycles, and a
// wave issues half of theirs while the other one of its SIMD waits; the rest are vector instructions (280
// per step of a wave that does softmax, 140 of the others), the 64 KB of partial scores through
// LDS and back, and the barrier.  Tried and slower, by passes of the whole call at the time: 8
// rows of softmax for each wave (105.7), softmax before the next step's scores (105.5), 32 rows per
// block (129), two blocks of 4 waves per CU (alike).
template <int HD, int RT, int W>
__global__ __launch_bounds__(64 * W, W == 4 ? 3 : 2) void attn_kv4_rows_kernel(Kv4Args a) {
  constexpr int DW = HD / W, R = 16 * RT, NT = 2, KEYS = 16 * NT;
  constexpr int KN = DW / 32;         // words of a key per lane, and products
  constexpr int VD = DW / 16;         // dims per lane, and output tiles
  static_assert(DW == 64, "32 bytes of a row per wave");
  // (two of each: what the step's readers may still look at, and the next)
  // (of 32 rows: spills that all calls feel, 102.7 us for 94.  So, HD 256 at three blocks per CU spills 9
  // registers, HD 512 of 64 rows one: outside the loop, but for one where a reference moves.)
  using General = AttendSmem<HD, 1, false, W, DW>;
  union Smem {
    struct {
      f32x4 sx[2][W][RT][NT][64];
      u32x4 sp[2][RT][2][64];
    };
    float rows[R][HD + 4];  // q and the outputs, on their way from and to whole lines of memory
    General general;
  };
  __shared__ Smem sm;
  __shared__ u32x4 sv[W][64];         // v's codes of a step
  __shared__ float sf[2][R];
  __shared__ int smoved[2][4];        // whether some row's reference moved
  static_assert(RT <= 4, "a flag per row tile");
  __shared__ int stop[W][R], sxq[R];  // q's largest, q's exponents
  const Scores &S = a.s;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int R0 = blockIdx.x * R, split = blockIdx.y;
  const int pa = S.pos0 + R0 / S.heads, pb = S.pos0 + (min(R0 + R, S.rows) - 1) / S.heads;
  const Run run(S, R0, R, split, KEYS);
  const int lo = run.lo, hi = run.hi, steps = run.steps, t0 = run.t0, t1 = run.t1;
  ushort2_t beyond = {0, 0};  // the scales' largest distance from the least plain one

  // A lane loads 16 bytes and a scale of a key, and of a v: lane (c, g) key 16 (g / 2) + c, bytes
  // 16 (g % 2) .. of the wave's 32, of which the lanes' halves then swap 8; as v's, lane l those of
  // slot l / 2 = 4 j + g that holds key 16 (j / 4) + 4 g + j % 4, by LDS to lanes (., g) as their
  // j-th; and the scale of slot 4 (c % 8) + g and of dims 32 (c / 8) ...  Rows behind the last key
  // give zeros, whose scales are made 1.
  u32x4 kr, vr;
  uint32_t ksr, vsr;
  const auto slot_row = [](int j, int gg) { return 16 * (j >> 2) + 4 * gg + (j & 3); };
  const int row_k = 16 * (g >> 1) + c, row_v = slot_row(lane >> 3, lane >> 1 & 3), row_vs = slot_row(c & 7, g);
  const uint32_t at_k = row_k * (HD / 2) + w * (DW / 2) + (g & 1) * 16;
  const uint32_t at_ks = row_k * (HD / 16) + w * (DW / 16) + (g & 1) * 2;
  const uint32_t at_v = row_v * (HD / 2) + w * (DW / 2) + (lane & 1) * 16;
  const uint32_t at_vs = row_vs * (HD / 16) + w * (DW / 16) + (c >> 3) * 2;
  auto rows_of = [&](const void *plane, int step, int bytes) {
    const int k0 = __builtin_amdgcn_readfirstlane(lo + min(step, steps - 1) * KEYS);
    char *p = const_cast<char *>(static_cast<const char *>(plane)) + (size_t)k0 * bytes;
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, min(hi - k0, KEYS) * bytes, 0x00020000);
  };
  auto load_k = [&](int step) {
    kr = __builtin_amdgcn_raw_buffer_load_b128(rows_of(a.k, step, HD / 2), at_k, 0, 0);
    ksr = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rows_of(a.ks, step, HD / 16), at_ks, 0, 0);
  };
  auto load_v = [&](int step) {
    vr = __builtin_amdgcn_raw_buffer_load_b128(rows_of(a.v, step, HD / 2), at_v, 0, 0);
    vsr = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rows_of(a.vs, step, HD / 16), at_vs, 0, 0);
  };
  auto last_row = [&](int step) { return hi - 1 - (lo + min(step, steps - 1) * KEYS); };
  load_k(t0);

  // q: lane (c, g) holds its row's dims 32 (g % 2) + 16 (g / 2) + 8 n .. + 7 of the wave's, as k's are
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
      int top = 0;
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(&sm.rows[16 * r + c][w * DW + 32 * (g & 1) + 16 * (g >> 1) + 8 * n]);
        x[r][n][0] = p[0];
        x[r][n][1] = p[1];
      }
#pragma unroll
      for (int n = 0; n < KN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = max(top, max(__float_as_int(x[r][n][0][i]) & 0x7fffffff, __float_as_int(x[r][n][1][i]) & 0x7fffffff));
      top = max(top, __shfl_xor(top, 16, 64));
      top = max(top, __shfl_xor(top, 32, 64));
      if (g == 0) stop[w][16 * r + c] = top;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      int top = 0;
#pragma unroll
      for (int d = 0; d < W; ++d) top = max(top, stop[d][16 * r + c]);
      const int e = top == 0 || top >= 0x7f800000 ? 0 : max((top >> 23) - 127, -126);
      if (w == 0 && g == 0) sxq[16 * r + c] = e - 13 - kLift;
      if (!usual_row(e - 13 - kLift)) beyond = (ushort2_t){0xffff, 0xffff};
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        u32x4 h4, l4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2_t z = {ldexpf(x[r][n][0][i], 13 - e), ldexpf(x[r][n][1][i], 13 - e)};
          const half2_t h = __builtin_convertvector(z, half2_t);
          h4[i] = __builtin_bit_cast(uint32_t, h);
          l4[i] = __builtin_bit_cast(
              uint32_t, __builtin_convertvector(z - __builtin_convertvector(h, f32x2_t), half2_t));
        }
        qh[r][n] = __builtin_bit_cast(half8_t, h4);
        ql[r][n] = __builtin_bit_cast(half8_t, l4);
      }
    }
  }
  const Magic mg;
  // partial scores of a step into LDS
  auto scores = [&](int step) {
    if (row_k > last_row(step)) ksr = 0x3f80u;
    Scale x[NT];
    uint32_t kw[NT][KN];
    f32x4 s[RT][NT];
    {
      const uint32_t both = __builtin_bit_cast(uint32_t, plain_pair(ksr, ksr, beyond).s);
      const auto y = __builtin_amdgcn_permlane32_swap(both, both, false, false);
#pragma unroll
      for (int T = 0; T < NT; ++T) x[T] = scale_of(__builtin_bit_cast(half2_t, (uint32_t)y[T]));
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const auto z = __builtin_amdgcn_permlane32_swap(kr[n], kr[n + 2], false, false);
#pragma unroll
        for (int T = 0; T < NT; ++T) kw[T][n] = z[T];
      }
    }
#pragma unroll
    for (int T = 0; T < NT; ++T)
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][T] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < KN; ++n)
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        const uint32_t wd = kw[T][n];
        const half8_t kv = __builtin_bit_cast(
            half8_t, (u32x4){value_pair<0>(wd, x[T], mg), value_pair<1>(wd, x[T], mg), value_pair<2>(wd, x[T], mg),
                             value_pair<3>(wd, x[T], mg)});
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, ql[r][n], s[r][T], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, qh[r][n], s[r][T], 0, 0, 0);
      }
    load_k(step + 1);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int T = 0; T < NT; ++T) sm.sx[(step - t0) & 1][w][r][T][lane] = s[r][T];
  };

  float m = kNoScore, l = 0.f;  // of row 16 w + c
  f32x4 o[RT][VD];              // outputs times 2^(15 + kLift - kSlack)
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < VD; ++n) o[r][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int my_row = R0 + 16 * min(w, RT - 1) + c, my_pos = S.pos0 + min(my_row, S.rows - 1) / S.heads;
  load_v(t0);
  __syncthreads();
  const float my_factor = ldexpf(kLog2e, sxq[16 * min(w, RT - 1) + c]);
  if (t0 < t1) scores(t0);
  asm volatile("" ::: "memory");  // (else loads move into the loop, with an address of 64 bits each)
  // Everything loaded so far has to be there: a wait in the loop counts the loads behind the one it
  // is for, and would count by the loop's entry, where k's are the last, in every turn.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
  for (int step = t0; step < t1; ++step) {
    const int key0 = lo + step * KEYS, at = (step - t0) & 1;
    // (formed by all waves first: behind the softmax, by those that do it, 105.5 us for 97.6)
    if (step + 1 < t1) scores(step + 1);
    if (w < RT) {
      // this wave's rows: the scores of all, in order
      float x[NT][4];
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        f32x4 y = sm.sx[at][0][w][T][lane];
#pragma unroll
        for (int d = 1; d < W; ++d) y += sm.sx[at][d][w][T][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[T][i] = y[i] * my_factor;
      }
      const bool inner = key0 + KEYS - 1 <= pa && (S.window == 0 || key0 > pb - S.window);
      if (!inner) {
#pragma unroll
        for (int T = 0; T < NT; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * T + 4 * g + i;
            if (key > my_pos || (S.window > 0 && key <= my_pos - S.window)) x[T][i] = -INFINITY;
          }
      }
      if (S.score) {
#pragma unroll
        for (int T = 0; T < NT; ++T)
          *reinterpret_cast<f32x4 *>(S.score + (size_t)min(my_row, S.rows - 1) * S.stride + (key0 + 16 * T + 4 * g - S.first)) =
              (f32x4){x[T][0], x[T][1], x[T][2], x[T][3]};
      }
      float tm = kNoScore;
#pragma unroll
      for (int T = 0; T < NT; ++T) tm = fmaxf(tm, fmaxf(fmaxf(x[T][0], x[T][1]), fmaxf(x[T][2], x[T][3])));
      // (fmaxf drops a NaN score, whose weight is NaN.)
      tm = group_max(tm);
      const float mn = tm > m + kSlack ? tm : m;
      const float corr = __builtin_amdgcn_exp2f(m - mn);
      float sum = 0.f;
      u32x4 h4, l4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int T = j >> 1, i = 2 * (j & 1);
        const float p0 = __builtin_amdgcn_exp2f(x[T][i] - mn), p1 = __builtin_amdgcn_exp2f(x[T][i + 1] - mn);
        sum += p0;
        sum += p1;
        const f32x2_t z = {p0 * kWeight, p1 * kWeight};
        const half2_t h = __builtin_convertvector(z, half2_t);
        h4[j] = __builtin_bit_cast(uint32_t, h);
        l4[j] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(z - __builtin_convertvector(h, f32x2_t), half2_t));
      }
      sm.sp[at][w][0][lane] = h4;
      sm.sp[at][w][1][lane] = l4;
      l = fmaf(l, corr, sum);
      if (g == 0) sf[at][16 * w + c] = corr;
      const bool moved = __any(corr != 1.f);
      if (lane == 0) smoved[at][w] = moved;
      m = mn;
    }
    if (row_vs > last_row(step)) vsr = 0x3f80u;
    Scale vx[4];
    {
      // keys j and j + 1 of even j's lane, then from there to all of its 8
      const uint32_t next = __builtin_amdgcn_update_dpp(0, (int)vsr, 0xB1, 0xf, 0xf, true);
      const int both = __builtin_bit_cast(int, plain_pair(vsr, next, beyond).s);
      auto of = [&](auto j) {
        constexpr int at = 0x150 + 2 * decltype(j)::value;  // row_newbcast
        int y = __builtin_amdgcn_update_dpp(0, both, at, 0xf, 0xf, true);
        y = __builtin_amdgcn_update_dpp(y, both, at + 8, 0xf, 0xc, false);
        vx[decltype(j)::value] = scale_of(__builtin_bit_cast(half2_t, y));
      };
      of(std::integral_constant<int, 0>());
      of(std::integral_constant<int, 1>());
      of(std::integral_constant<int, 2>());
      of(std::integral_constant<int, 3>());
    }
    sv[w][lane] = vr;
    load_v(step + 1);
    __syncthreads();
    int moved = 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) moved |= smoved[at][r];
    half8_t ph[RT], pl[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      ph[r] = __builtin_bit_cast(half8_t, sm.sp[at][r][0][lane]);
      pl[r] = __builtin_bit_cast(half8_t, sm.sp[at][r][1][lane]);
    }
    if (__builtin_amdgcn_readfirstlane(moved)) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float f = sf[at][16 * r + c];
#pragma unroll
        for (int n = 0; n < VD; ++n) o[r][n] *= f;
      }
    }
    {
      const any_u16 *codes = reinterpret_cast<const any_u16 *>(sv[w]) + lane;
      uint32_t d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        d[j] = __builtin_bit_cast(uint32_t, (ushort2_t){codes[128 * j], codes[128 * j + 64]});
      auto tile = [&](auto T) {
        constexpr int e = decltype(T)::value;
        const half8_t vv = __builtin_bit_cast(
            half8_t, (u32x4){value_pair<e>(d[0], vx[0], mg), value_pair<e>(d[1], vx[1], mg),
                             value_pair<e>(d[2], vx[2], mg), value_pair<e>(d[3], vx[3], mg)});
#pragma unroll
        for (int r = 0; r < RT; ++r) o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pl[r], o[r][e], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < RT; ++r) o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, ph[r], o[r][e], 0, 0, 0);
      };
      tile(std::integral_constant<int, 0>());
      tile(std::integral_constant<int, 1>());
      tile(std::integral_constant<int, 2>());
      tile(std::integral_constant<int, 3>());
    }
  }

  const bool odd = __any(max(beyond[0], beyond[1]) >= kPlainScales);
  __syncthreads();
  if (lane == 0) stop[w][0] = odd;
  __syncthreads();
  int again = 0;
#pragma unroll
  for (int d = 0; d < W; ++d) again |= stop[d][0];
  if (__builtin_amdgcn_readfirstlane(again)) {
    const Kv4Args &b = args_again();
    const Run all(b.s, R0, R, split, KEYS);
    for (int r = 0; r < R && R0 + r < b.s.rows; r += 16) {
      __syncthreads();
      attend<HD, 1, false, W, DW, false>(b, R0 + r, split, all, sm.general);
    }
    return;
  }
  const bool whole = S.splits == 1;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (S.ml && w < RT && g == 0 && my_row < S.rows) S.ml[(size_t)my_row * S.splits + split] = make_float2(m, l);
  // (a split of which the row sees nothing: 0, not 0 / 0)
  const float fin = !whole && l == 0.f ? 0.f : ldexpf(1.f / l, (int)kSlack - 15 - kLift);
  __syncthreads();  // (sf is read to the last step's end)
  if (w < RT && g == 0) sf[0][16 * w + c] = fin;
  __syncthreads();
  float *out = whole ? a.y : a.part + (size_t)split * S.rows * HD;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float f = sf[0][16 * r + c];
    // lane (c, g): tile n, register v holds dim (4 g + v) VD + n of the wave's
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int n = 0; n < VD; n += 4)
        *reinterpret_cast<f32x4 *>(&sm.rows[16 * r + c][w * DW + (4 * g + v) * VD + n]) =
            (f32x4){o[r][n][v], o[r][n + 1][v], o[r][n + 2][v], o[r][n + 3][v]} * f;
  }
  __syncthreads();
#pragma unroll 4
  for (int u = t; u < R * HD / 4; u += 64 * W) {
    const int row = u / (HD / 4), d = u % (HD / 4) * 4;
    if (R0 + row < S.rows)
      *reinterpret_cast<f32x4 *>(out + (size_t)(R0 + row) * HD + d) = *reinterpret_cast<const f32x4 *>(&sm.rows[row][d]);
  }
}

// The power of two that takes a sum of weights to 1 .. 2: outputs added under it stay in FP32's range
// wherever their mean does, and no bit of them changes otherwise.
__device__ __forceinline__ float to_one(float sum) { return ldexpf(1.f, 127 - (int)(__float_as_uint(sum) >> 23)); }

// Adds the key splits of a row: y = sum_s w_s y_s / sum_s w_s, w_s = 2^(m_s - M) l_s.  A block is
// one row's 32 dims; thread (j, u) adds splits j, j + 32, .. of 16-byte unit u in order, 8 of them
// under way together and before their weights are known.  8 rows of 512 splits of 512: 8.4 MB in 4.2 us.
template <int HD>
__device__ __forceinline__ void merge(const Kv4Args &a, int row, int part) {
  constexpr int U = 8, G = 256 / U, N = 8, PER = kMaxSplits / 256;
  const Scores &S = a.s;
  const int t = threadIdx.x, u = t % U, j = t / U;
  __shared__ float wt[kMaxSplits];
  __shared__ float wmax[4], wsum[4];
  __shared__ f32x4 sums[G][U];
  const f32x4 *p = reinterpret_cast<const f32x4 *>(a.part + (size_t)row * HD) + part * U + u;
  const size_t step = (size_t)S.rows * HD / 4;
  f32x4 x[N];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = p[min(s0 + G * i, S.splits - 1) * step];
  };
  float2 ml[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) ml[i] = S.ml[(size_t)row * S.splits + min(t + 256 * i, S.splits - 1)];
  load(j);
  float M = ml[0].x;
#pragma unroll
  for (int i = 1; i < PER; ++i) M = fmaxf(M, ml[i].x);
  M = team_max(64, M);
  if ((t & 63) == 0) wmax[t >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  float e = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float z = t + 256 * i < S.splits ? ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - M) : 0.f;
    wt[t + 256 * i] = z;
    e += z;
  }
  const float L = team_sum(64, e);
  if ((t & 63) == 0) wsum[t >> 6] = L;
  __syncthreads();
  const float sum = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]), one = to_one(sum);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = j; s0 < S.splits; s0 += G * N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (s0 + G * i < S.splits) y += wt[s0 + G * i] * one * x[i];
    if (s0 + G * N < S.splits) load(s0 + G * N);
  }
  sums[j][u] = y;
  __syncthreads();
  if (j > 0) return;
  y = sums[0][u];
#pragma unroll
  for (int i = 1; i < G; ++i) y += sums[i][u];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] /= sum * one;
  reinterpret_cast<f32x4 *>(a.y + (size_t)row * HD)[part * U + u] = y;
}

template <int HD>
__global__ __launch_bounds__(256) void attn_kv4_merge_kernel(Kv4Args a) { merge<HD>(a, blockIdx.x, blockIdx.y); }

// Few rows whose keys' weights are asked for: both need the first kernel's sums alone, so the same
// launch does the one and the other (one token of 32003 keys, when it came in: 17.3 us in all, with two
// launches 21.3).
template <int HD>
__global__ __launch_bounds__(256) void attn_kv4_merge_weights_kernel(Kv4Args a, SumArgs w) {
  const int merges = a.s.rows * (HD / 32), b = blockIdx.x;
  if (b < merges) merge<HD>(a, b / (HD / 32), b % (HD / 32));
  else add_weights(w, b - merges, 0);
}

// The same for up to 16 splits of many rows: a thread per 16-byte unit.  4096 rows of 4 splits of 512:
// 42 MB in 10.7 us, 3.9 TB/s.
template <int HD>
__device__ __forceinline__ void join(const Kv4Args &a, int block) {
  constexpr int MOST = 16;
  const Scores &S = a.s;
  const size_t unit = (size_t)block * 256 + threadIdx.x, units = (size_t)S.rows * (HD / 4);
  if (unit >= units) return;
  const float2 *ml = S.ml + unit / (HD / 4) * S.splits;
  const f32x4 *p = reinterpret_cast<const f32x4 *>(a.part) + unit;
  f32x4 x[MOST];
  float e[MOST];
  float M = kNoScore, L = 0.f;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    x[i] = p[min(i, S.splits - 1) * units];
    M = fmaxf(M, ml[min(i, S.splits - 1)].x);
  }
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const float2 z = ml[min(i, S.splits - 1)];
    e[i] = i < S.splits ? z.y * __builtin_amdgcn_exp2f(z.x - M) : 0.f;
    L += e[i];
  }
  const float one = to_one(L);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < MOST; ++i) y += e[i] * one * x[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] /= L * one;
  reinterpret_cast<f32x4 *>(a.y)[unit] = y;
}
template <int HD>
__global__ __launch_bounds__(256) void attn_kv4_join_kernel(Kv4Args a) { join<HD>(a, blockIdx.x); }

// And with the keys' weights, as for few rows: 1624 rows over 2403 keys, when it came
// in, 49.6 us in all, with two launches 51.7.
template <int HD>
__global__ __launch_bounds__(256) void attn_kv4_join_weights_kernel(Kv4Args a, SumArgs w, int joins, int tiles) {
  const int b = blockIdx.x;
  if (b < joins) join<HD>(a, b);
  else add_weights(w, (b - joins) % tiles, (b - joins) / tiles);
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

Workspace g_kv4_ws;

// The kernel for the call's rows: its rows per block, keys per step of all its waves, blocks per
// CU and threads.
struct Plan {
  void (*kernel)(Kv4Args);
  int rows, keys, per_cu, threads;
};
// Up to 16 rows, a wave working on DW dims: whether a block per CU (of more than 8 rows, whose splits
// cost more to join, per two) then has all keys at once.
template <int HD, int DW>
bool few_of(int rows, int keys, Plan &plan) {
  constexpr int KEYS = kStep * kGroups<HD, 4, DW>;
  if (rows <= 8) plan = {attn_kv4_kernel<HD, 1, true, 4, DW>, 8, KEYS, 2, 256};
  else plan = {attn_kv4_kernel<HD, 1, false, 4, DW>, 16, KEYS, 2, 256};
  return cdiv(keys, KEYS) <= (rows <= 8 ? cu_count() : cu_count() / 2);
}

// Few rows: less of a row per wave as long as there are CUs for the keys.  One token, us, with 64 / 128 /
// 256 dims per wave: 4000 keys of 512 - / 9.9 / 11.3, 8000 - / 11.8 / 11.8, 30000 - / 16.2 / 15.6 (125,
// 250 and 938 blocks of 128); 512 of 256 8.8 / 9.3 / 10.7, 4000 9.4 / 9.5 / 10.9, 16000 11.3 / 10.5 /
// 11.7, 60000 19.7 / 15.3 / 13.9; of 128, 4000 8.7 / 9.1.  Two tokens: 4000 of 512 - / 12.3 / 12.5, 8000
// - / 15.1 / 14.3.
// Many rows of 512 whose 64-row blocks would have up to 4 steps each on all CUs: blocks of 32, which
// start and end sooner.  us, 32 / 64 rows per block: 96 rows over 2000 keys (3 steps) 29.1 / 42.2, 128
// over 2000 and 32 over 8000 (4) 32.2 / 35.4 and 30.9 / 32.3, 160 over 2000 (5) 44.3 / 36.4, 512
// over 4608 (36) 129 / 95.  Rows of 256 have room for three blocks of 32 on a CU, or one of 64 in
// four waves: 512 over 4608 70.6 / 84.7 (48 rows, two blocks: 76.6), 20 over 3000 17.5 / 23.0.
template <int HD>
Plan plan_of(int rows, int keys) {
  if (rows <= 16) {
    Plan plan;
    if constexpr (HD == 512) {
      if (few_of<HD, 128>(rows, keys, plan)) return plan;
    } else if constexpr (HD == 256) {
      if (few_of<HD, 64>(rows, keys, plan) || few_of<HD, 128>(rows, keys, plan)) return plan;
    } else if constexpr (HD == 128) {
      if (few_of<HD, 64>(rows, keys, plan)) return plan;
    }
    few_of<HD, kDims<HD>>(rows, 0, plan);
    return plan;
  }
  if constexpr (HD == 512) {
    if ((int64_t)cdiv(rows, 64) * cdiv(keys, 32) <= 4 * cu_count())
      return {attn_kv4_rows_kernel<HD, 2, 8>, 32, 32, 1, 512};
    return {attn_kv4_rows_kernel<HD, 4, 8>, 64, 32, 1, 512};
  }
  else if constexpr (HD == 256) return {attn_kv4_rows_kernel<HD, 2, 4>, 32, 32, 3, 256};
  else return {attn_kv4_kernel<HD, 2, false, 4>, 32, kStep * kGroups<HD, 4>, 2, 256};
}

// What the rows of s, all at once, take.
struct Needs {
  Plan plan;
  int blocks, splits;
  size_t part, score, ml, sum;  // floats
  size_t bytes() const { return (part + score + ml + sum) * 4; }
};
template <int HD>
Needs needs_of(const Scores &s, bool weights) {
  const int keys = s.window > 0 ? min(s.end - s.first, s.window + 64) : s.end - s.first;  // of a block
  Needs n;
  n.plan = plan_of<HD>(s.rows, keys);
  n.blocks = cdiv(s.rows, n.plan.rows);
  // A block per CU, or as many as fit where each then has several turns: the join of their outputs
  // costs more than a shorter loop gains.  One token, us: 16001 keys of 512, 251 splits of one turn
  // 14.7, 126 of two 16.4; 32003 with weights 256 of two 20.9, 512 of one 24.9; 131072 512 of
  // four 29.1, 256 of eight 30.7.
  const int turns = cdiv(keys, n.plan.keys);
  n.splits = cu_count() / n.blocks;
  if (turns >= 4 * n.plan.per_cu * n.splits) n.splits = n.plan.per_cu * cu_count() / n.blocks;
  if (n.splits > turns) n.splits = turns;
  if (n.splits > kMaxSplits) n.splits = kMaxSplits;
  if (n.splits < 1) n.splits = 1;
  n.part = n.splits > 1 ? (size_t)n.splits * s.rows * HD : 0;
  n.ml = weights || n.splits > 1 ? (size_t)n.splits * s.rows * 2 : 0;
  n.score = weights ? s.rows * s.stride : 0;
  n.sum = weights ? weight_part_floats(s.rows, s.end - s.first) : 0;
  return n;
}

// The rows of a.s, all at once; `before` and `weights` of keys key0 .. keylen - 1.
template <int HD>
int launch_rows(Kv4Args a, void *mem, int key0, int keylen, const float *before, float *weights) {
  Scores &s = a.s;
  const Needs n = needs_of<HD>(s, weights != nullptr);
  const int splits = s.splits = n.splits;
  float *part = nullptr;
  if (n.bytes()) {
    a.part = static_cast<float *>(mem);
    s.score = weights ? a.part + n.part : nullptr;
    s.ml = reinterpret_cast<float2 *>(a.part + n.part + n.score);
    part = a.part + n.part + n.score + n.ml;
  }
  hipLaunchKernelGGL(n.plan.kernel, dim3(n.blocks, splits), dim3(n.plan.threads), 0, stream(), a);
  G4_LAUNCH_CHECK("attn_kv4_kernel");
  if (splits > 1 && weights && s.rows <= kGroup) {
    const SumArgs sums{s, key0, keylen, before, weights, nullptr};
    hipLaunchKernelGGL(attn_kv4_merge_weights_kernel<HD>, dim3(s.rows * (HD / 32) + cdiv(keylen - key0, 256)), dim3(256), 0,
                       stream(), a, sums);
    G4_LAUNCH_CHECK("attn_kv4_merge_weights_kernel");
    return G4_OK;
  }
  const int joins = (int)(((size_t)s.rows * (HD / 4) + 255) / 256);
  const bool join = splits > 1 && s.rows >= 64 && splits <= 16;
  if (join && weights) {
    const SumArgs sums{s, key0, keylen, before, weights, part};
    const int tiles = cdiv(s.end - s.first, 256);
    hipLaunchKernelGGL(attn_kv4_join_weights_kernel<HD>, dim3(joins + tiles * cdiv(s.rows, kGroup)), dim3(256), 0,
                       stream(), a, sums, joins, tiles);
    G4_LAUNCH_CHECK("attn_kv4_join_weights_kernel");
    return launch_weights_join(s, key0, keylen, part, before, weights);
  }
  if (splits > 1) {
    if (join)
      hipLaunchKernelGGL(attn_kv4_join_kernel<HD>, dim3(joins), dim3(256), 0, stream(), a);
    else
      hipLaunchKernelGGL(attn_kv4_merge_kernel<HD>, dim3(s.rows, HD / 32), dim3(256), 0, stream(), a);
    G4_LAUNCH_CHECK("attn_kv4_merge_kernel");
  }
  if (!weights) return G4_OK;
  return launch_weights(s, key0, keylen, part, before, weights);
}

// All rows of a call, in chunks whose scores are kept at once.
template <int HD>
int launch_chunks(const Kv4Args &call, int qrows, int heads, int keylen, int qpos0, int win, const float *before,
                  float *weights) {
  const int most = weights ? weighted_rows(qrows, heads, qpos0, win) : qrows;
  auto scores_at = [&](int r0) { return scores_of(qrows - r0 < most ? qrows - r0 : most, heads, qpos0 + r0, win); };
  size_t need = 0;  // of the chunk that takes most, before the first one
  for (int r0 = 0; r0 < qrows; r0 += most) {
    const size_t n = needs_of<HD>(scores_at(r0), weights != nullptr).bytes();
    if (n > need) need = n;
  }
  void *mem = nullptr;
  if (need)
    if (int rc = growing_scratch(g_kv4_ws, need, &mem, "g4_attention_kv4")) return rc;
  for (int r0 = 0; r0 < qrows; r0 += most) {
    Kv4Args a = call;
    a.q += (size_t)r0 * heads * HD;
    a.y += (size_t)r0 * heads * HD;
    a.s = scores_at(r0);
    // (later chunks add to the keys that they see)
    const int rc = r0 ? launch_rows<HD>(a, mem, a.s.first, a.s.end, weights, weights)
                      : launch_rows<HD>(a, mem, 0, keylen, before, weights);
    if (rc) return rc;
  }
  return G4_OK;
}

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
  const int head_dim = cache->head_dim;
  const size_t qn = (size_t)qrows * heads * head_dim * 4, wn = weights ? (size_t)keylen * 4 : 0;
  const size_t codes = (size_t)keylen * head_dim / 2, scales = codes / 8;
  auto in_cache = [&](const void *p, size_t n) {
    return overlap(p, n, cache->k, codes) || overlap(p, n, cache->v, codes) || overlap(p, n, cache->k_scales, scales) ||
           overlap(p, n, cache->v_scales, scales);
  };
  if (overlap(q, qn, y, qn) || overlap(q, qn, weights, wn) || overlap(y, qn, weights, wn) ||
      (before && overlap(y, qn, before, wn)) || in_cache(y, qn) || in_cache(weights, wn))
    return fail(G4_E_ARG, "%s: y or weights overlaps another argument", who);
  G4_CHECK_INIT();
  if (keylen == 0) return ok();
  int rc = check_kv4_memory(cache, keylen, true, true, "g4_attention_kv4 cache");
  if (!rc && qrows) rc = check_device_range(q, qn, "g4_attention_kv4 q");
  if (!rc && qrows) rc = check_device_range(y, qn, "g4_attention_kv4 y");
  if (!rc && weights) rc = check_device_range(weights, (size_t)keylen * 4, "g4_attention_kv4 weights");
  if (!rc && before) rc = check_device_range(before, (size_t)keylen * 4, "g4_attention_kv4 before");
  if (rc) return rc;
  const int win = sliding ? (window < keylen ? window : keylen) : 0;
  if (qrows == 0) {
    Scores s{};
    s.heads = 1;
    if (weights) rc = launch_weights(s, 0, keylen, nullptr, before, weights);
    return rc ? rc : ok();
  }
  Kv4Args a{};
  a.q = q;
  a.y = y;
  a.k = cache->k;
  a.v = cache->v;
  a.ks = cache->k_scales;
  a.vs = cache->v_scales;
  switch (head_dim) {
    case 64: rc = launch_chunks<64>(a, qrows, heads, keylen, qpos0, win, before, weights); break;
    case 128: rc = launch_chunks<128>(a, qrows, heads, keylen, qpos0, win, before, weights); break;
    case 256: rc = launch_chunks<256>(a, qrows, heads, keylen, qpos0, win, before, weights); break;
    default: rc = launch_chunks<512>(a, qrows, heads, keylen, qpos0, win, before, weights); break;
  }
  return rc ? rc : ok();
}
