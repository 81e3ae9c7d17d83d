// The tied BF16 head for several hidden states:
//   out[j, r] = softcap * tanh((scale * sum_k x[j, k] * E[r, k]) / softcap)
#include "g4_internal.h"
#include "g4_ops.h"

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
  for (int j = 0; j < n && !rc; ++j)
    rc = launch_bf16_head(x + (size_t)j * in_dim, static_cast<const uint16_t *>(E), rows, in_dim,
                          out + j * out_stride, scale, softcap, nullptr);
  return rc ? rc : ok();
}
