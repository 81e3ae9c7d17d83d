// What the operators of long caches share.
#pragma once

#include <type_traits>

#include "g4_internal.h"

namespace g4 {

// Shape, alignment and rows at .. at + n - 1 of a cache; nothing of it needs the device.
int check_kv4(const g4_kv4 *c, int at, int n, const char *who);
// The memory of its first `rows` rows.
int check_kv4_memory(const g4_kv4 *c, size_t rows, bool k, bool v, const char *who);

// Scores of `rows` = query rows * heads, kept for the keys' weights: score[row][key - first], in
// units of log 2, and (maximum, sum of 2^(score - maximum)) of each row and key split.  Query row
// i sits at position pos0 + i; a key is seen at positions key .. key + window - 1 (window 0: all
// from key on).
// Kernels store whole steps of up to 32 keys: what score_stride adds to the keys is theirs.  Rows that
// pad a block are the last row again, scores and address.
struct Scores {
  float *score;
  float2 *ml;  // [rows][splits]
  size_t stride;
  int rows, heads, splits;
  int first, end, pos0, window;  // keys first .. end - 1 are seen by some row
};

// The keys that some of rows R0 .. R0 + n - 1 see, lo .. hi - 1, and a split's steps of
// `keys` of them.
struct Run {
  int lo, hi, steps, t0, t1;
  __device__ __forceinline__ Run(const Scores &S, int R0, int n, int split, int keys) {
    const int pa = S.pos0 + R0 / S.heads, pb = S.pos0 + (min(R0 + n, S.rows) - 1) / S.heads;
    lo = S.first;
    if (S.window > 0) lo += max(0, pa - S.window + 1 - S.first) & ~3;
    hi = pb + 1;
    steps = (hi - lo + keys - 1) / keys;
    const int per = (steps + S.splits - 1) / S.splits;
    t0 = split * per;
    t1 = min(t0 + per, steps);
  }
};

// Query rows at positions pos0 .. without their memory.
Scores scores_of(int qrows, int heads, int pos0, int window);
size_t score_stride(int keys);

// Scratch whose need follows a cache's length: a little more than there is asks for half as much again,
// so that a chat whose every token needs a few rows more allocates (and clears) it now and then, not
// at each of them.
int growing_scratch(Workspace &ws, size_t need, void **p, const char *who);

// weights[key] = before[key] + sum over the rows of 2^(score - max) / sum, for keys key0 .. keylen - 1;
// `part` holds weight_part_floats(rows, end - first).
size_t weight_part_floats(int rows, int keys);
int launch_weights(const Scores &s, int key0, int keylen, float *part, const float *before, float *weights);
// Its second launch alone, for more than 32 rows: the sums of each 32 rows are in `part`.
int launch_weights_join(const Scores &s, int key0, int keylen, float *part, const float *before, float *weights);

// Arguments that g4_attention_kv4 and g4_attention_weights have in common.
int check_weighted(int qrows, int heads, int keylen, int qpos0, int sliding, int window,
                   const float *before, const float *weights, const char *who);
// Query rows of a call whose scores are kept at once.
int weighted_rows(int qrows, int heads, int qpos0, int window);

// op over aligned teams of `team` lanes, 4 .. 64 and the same for all, known to each of them
template <class Op>
__device__ __forceinline__ float team_of(int team, float v, Op op) {
  auto dpp = [&](auto c) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(c)::value, 0xf, 0xf, true));
  };
  v = op(v, dpp(std::integral_constant<int, 0xB1>()));
  v = op(v, dpp(std::integral_constant<int, 0x4E>()));
  if (team >= 8) v = op(v, dpp(std::integral_constant<int, 0x141>()));
  if (team >= 16) v = op(v, dpp(std::integral_constant<int, 0x140>()));
  if (team >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if (team >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return v;
}
__device__ __forceinline__ float team_max(int team, float v) {
  return team_of(team, v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float team_sum(int team, float v) {
  return team_of(team, v, [](float a, float b) { return a + b; });
}

// max over aligned teams of 8, 16, 32 or 64 lanes
template <int TEAM>
__device__ __forceinline__ int team_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));
  if constexpr (TEAM >= 16) v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));
  if constexpr (TEAM >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((int)a[0], (int)a[1]);
  }
  if constexpr (TEAM >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((int)a[0], (int)a[1]);
  }
  return v;
}

// Whether two ranges of bytes have some in common; none where one is empty.
inline bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && (x < y ? y - x < na : x - y < nb);
}

}  // namespace g4
