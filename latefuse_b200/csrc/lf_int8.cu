// The 8-bit projection on float rows, and the encoder's feed-forward half in 8-bit
// integers: runs of this library's entries over one caller-provided workspace, so that a
// binding makes one call (and one allocation) where the parts would take several.
#include "lf_common.cuh"
#include "lf_internal.h"

namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
int64_t row16(int64_t k) { return (k + 15) / 16 * 16; }

// m rows of k in 8-bit integers: q, then the scales
struct RowsAt {
  size_t q, scale, end;
  int64_t ld;
  RowsAt(size_t at, int64_t m, int64_t k) : ld(row16(k)) {
    q = at;
    scale = q + up256(size_t(m) * size_t(ld));
    end = scale + up256(size_t(m) * 4);
  }
};

bool sizes_ok(int dtype, int64_t m, int64_t a, int64_t b) {
  return (dtype == LF_DTYPE_F32 || dtype == LF_DTYPE_BF16 || dtype == LF_DTYPE_F16) && m >= 0 &&
         m <= INT32_MAX - 256 && a > 0 && a <= 131072 && b > 0 && b <= 131072;
}

}  // namespace

using namespace lf;

extern "C" {

size_t lf_linear_rows_int8_workspace_bytes(int64_t m, int k) {
  return sizes_ok(LF_DTYPE_F32, m, k, 1) && !linear_int8_takes_rows(m, k) ? RowsAt(0, m, k).end : 0;
}

int lf_linear_rows_int8(void* stream, int dtype, const void* x, int64_t ldx, const int8_t* w, int64_t ldw,
                        const float* w_scale, const void* bias, void* y, int64_t ldy, int64_t m, int n, int k, int act,
                        void* workspace, size_t workspace_bytes, int32_t* status) {
  if (!sizes_ok(dtype, m, k, 1))
    return set_error(LF_ERR_INVALID, "lf_linear_rows_int8: dtype %d, m %lld, k %d (k up to 131072)", dtype, (long long)m, k);
  if (m == 0) return LF_OK;
  if (linear_int8_takes_rows(m, k))
    return linear_int8_rows(stream, dtype, x, ldx, w, ldw, w_scale, bias, y, ldy, m, n, k, act, status);
  const RowsAt at(0, m, k);
  if (workspace == nullptr || workspace_bytes < at.end || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return set_error(LF_ERR_WORKSPACE, "lf_linear_rows_int8: %zu bytes of 256-byte aligned workspace needed, %zu given", at.end,
                     workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int8_t* q = reinterpret_cast<int8_t*>(ws + at.q);
  float* scale = reinterpret_cast<float*>(ws + at.scale);
  const int rc = lf_quantize_rows(stream, dtype, x, ldx, m, k, q, at.ld, scale);
  if (rc) return rc;
  return lf_linear_int8(stream, dtype, q, at.ld, scale, w, ldw, w_scale, bias, y, ldy, m, n, k, act, status);
}

size_t lf_ffn_int8_workspace_bytes(int dtype, int64_t m, int hidden, int inner) {
  if (!sizes_ok(dtype, m, hidden, inner)) return 0;
  const RowsAt first(0, m, hidden), second(first.end, m, inner);
  return second.end + up256(size_t(m) * size_t(row16(inner)) * (dtype == LF_DTYPE_F32 ? 4 : 2));
}

int lf_ffn_int8(void* stream, int dtype, const void* a, int64_t lda, const void* r, int64_t ldr, const void* gamma,
                const void* beta, float eps, const int8_t* up, int64_t ld_up, const float* up_scale,
                const void* up_bias, const int8_t* down, int64_t ld_down, const float* down_scale,
                const void* down_bias, int64_t m, int hidden, int inner, int act, void* h, int64_t ldh, void* o,
                int64_t ldo, void* workspace, size_t workspace_bytes, int32_t* status) {
  if (!sizes_ok(dtype, m, hidden, inner))
    return set_error(LF_ERR_INVALID, "lf_ffn_int8: dtype %d, m %lld, hidden %d, inner %d", dtype, (long long)m, hidden, inner);
  if (m == 0) return LF_OK;
  const size_t need = lf_ffn_int8_workspace_bytes(dtype, m, hidden, inner);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return set_error(LF_ERR_WORKSPACE, "lf_ffn_int8: %zu bytes of 256-byte aligned workspace needed, %zu given", need,
                     workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const RowsAt first(0, m, hidden), second(first.end, m, inner);
  int8_t *q1 = reinterpret_cast<int8_t*>(ws + first.q), *q2 = reinterpret_cast<int8_t*>(ws + second.q);
  float *s1 = reinterpret_cast<float*>(ws + first.scale), *s2 = reinterpret_cast<float*>(ws + second.scale);
  void* mid = ws + second.end;
  const int64_t ld_mid = row16(inner);
  int rc = lf_add_layernorm_int8(stream, dtype, a, lda, r, ldr, gamma, beta, eps, m, hidden, h, ldh, q1, first.ld, s1);
  if (rc) return rc;
  rc = lf_linear_int8(stream, dtype, q1, first.ld, s1, up, ld_up, up_scale, up_bias, mid, ld_mid, m, inner, hidden, act, status);
  if (rc) return rc;
  if (linear_int8_takes_rows(m, inner))
    return linear_int8_rows(stream, dtype, mid, ld_mid, down, ld_down, down_scale, down_bias, o, ldo, m, hidden, inner,
                            LF_ACT_NONE, status);
  rc = lf_quantize_rows(stream, dtype, mid, ld_mid, m, inner, q2, second.ld, s2);
  if (rc) return rc;
  return lf_linear_int8(stream, dtype, q2, second.ld, s2, down, ld_down, down_scale, down_bias, o, ldo, m, hidden, inner,
                        LF_ACT_NONE, status);
}

}  // extern "C"
