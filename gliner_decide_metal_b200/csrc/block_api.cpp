// C entries of the block operators over packed rows (include/gdc.h): argument checks, all of
// them before the first CUDA call, and dispatch to the launchers.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kernels/kernels.h"

namespace gdc {
namespace {

constexpr int64_t kMaxRows = int64_t(1) << 30;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1) == 0; }

gdc_status check_elem(const char* what, gdc_dtype dtype, Elem* t) {
  if (dtype != GDC_FLOAT16 && dtype != GDC_BFLOAT16)
    return set_error(GDC_ERR_UNSUPPORTED, "%s: dtype %d is neither GDC_FLOAT16 nor GDC_BFLOAT16", what, int(dtype));
  *t = dtype == GDC_FLOAT16 ? Elem::kF16 : Elem::kBF16;
  return GDC_OK;
}

gdc_status check_attention_sizes(int32_t batch, int64_t q_rows, int64_t k_rows, int32_t heads, int32_t kv_heads,
                                 int32_t head_dim) {
  if (batch < 0 || batch > (1 << 20) || q_rows < 0 || q_rows > kMaxRows || k_rows < 0 || k_rows > kMaxRows)
    return set_error(GDC_ERR_INVALID_INPUT, "packed attention: batch in [0, 2^20] and rows in [0, 2^30] required");
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return set_error(GDC_ERR_INVALID_INPUT, "packed attention: heads %d must be a positive multiple of kv_heads %d", heads,
                     kv_heads);
  if (heads / kv_heads > 128 || heads > 4096)
    return set_error(GDC_ERR_UNSUPPORTED, "packed attention: at most 128 heads a key head and 4096 heads (got %d / %d)",
                     heads, kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(GDC_ERR_UNSUPPORTED, "packed attention: head_dim %d is neither 64 nor 128", head_dim);
  return GDC_OK;
}

}  // namespace
}  // namespace gdc

using namespace gdc;

extern "C" {

gdc_status gdc_packed_attention_workspace(int32_t batch, int64_t q_rows, int64_t k_rows, int32_t heads, int32_t kv_heads,
                                          int32_t head_dim, size_t* bytes) {
  clear_error();
  if (!bytes) return set_error(GDC_ERR_NULL_POINTER, "gdc_packed_attention_workspace: null argument");
  GDC_TRY(check_attention_sizes(batch, q_rows, k_rows, heads, kv_heads, head_dim));
  *bytes = packed_attention_workspace(batch, q_rows, k_rows, heads, kv_heads, head_dim);
  return GDC_OK;
}

gdc_status gdc_packed_attention(gdc_dtype dtype, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                int64_t ldv, void* out, int64_t ldo, const int32_t* q_off, const int32_t* k_off,
                                int32_t batch, int64_t q_rows, int64_t k_rows, int32_t heads, int32_t kv_heads,
                                int32_t head_dim, int32_t causal, float scale, void* workspace, size_t workspace_bytes,
                                void* stream) {
  clear_error();
  Elem t = Elem::kF16;
  GDC_TRY(check_elem("gdc_packed_attention", dtype, &t));
  GDC_TRY(check_attention_sizes(batch, q_rows, k_rows, heads, kv_heads, head_dim));
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_packed_attention: scale must be positive and finite");
  if (batch == 0 || q_rows == 0) return GDC_OK;
  if (!q || !out || !q_off || (k_rows > 0 && (!k || !v)))
    return set_error(GDC_ERR_NULL_POINTER, "gdc_packed_attention: null argument");
  if (k_rows == 0) {  // k and v are not read, whatever they are
    k = v = nullptr;
    ldk = ldv = 0;
  }
  const int64_t qw = int64_t(heads) * head_dim, kw = int64_t(kv_heads) * head_dim;
  if (ldq < qw || ldo < qw || (k_rows > 0 && (ldk < kw || ldv < kw)))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_packed_attention: a row pitch is below the row's width");
  if (ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8 || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return set_error(GDC_ERR_INVALID_INPUT,
                     "gdc_packed_attention: pointers must be 16-byte aligned and pitches multiples of 8");
  if (!aligned4(q_off) || !aligned4(k_off))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_packed_attention: offsets must be aligned to their type");
  if (std::max(std::max(ldq, ldo), std::max(ldk, ldv)) > (int64_t(1) << 31))
    return set_error(GDC_ERR_UNSUPPORTED, "gdc_packed_attention: row pitch above 2^31");
  const size_t need = packed_attention_workspace(batch, q_rows, k_rows, heads, kv_heads, head_dim);
  if (need > 0 && !workspace) return set_error(GDC_ERR_NULL_POINTER, "gdc_packed_attention: null workspace");
  if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_packed_attention: workspace of %zu bytes, 256-byte aligned, required", need);
  int* err = nullptr;
  GDC_TRY(device_error_word(&err));
  const PackedAttentionArgs a{q, k, v, out, ldq, ldk, ldv, ldo, q_off, k_off ? k_off : q_off, batch, q_rows, k_rows,
                              heads, kv_heads, head_dim, causal != 0, scale, static_cast<uint8_t*>(workspace)};
  return launch_packed_attention(t, a, static_cast<cudaStream_t>(stream), err);
}

gdc_status gdc_linear_residual(gdc_dtype dtype, const void* a, int64_t lda, const void* w, int64_t ldw, const void* bias,
                               const void* residual, int64_t ldr, void* out, int64_t ldo, int64_t M,
                               const int32_t* rows_dev, int32_t N, int32_t K, int32_t act, void* stream) {
  clear_error();
  Elem t = Elem::kF16;
  GDC_TRY(check_elem("gdc_linear_residual", dtype, &t));
  if (M < 0 || M > kMaxRows || N <= 0 || K <= 0 || N > (1 << 30) || K > (1 << 30))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: M=%lld in [0, 2^30], N=%d and K=%d in [1, 2^30] required",
                     (long long)M, N, K);
  if (act < 0 || act > kActSilu) return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: unknown activation %d", act);
  if (M == 0) return GDC_OK;
  if (!a || !w || !out) return set_error(GDC_ERR_NULL_POINTER, "gdc_linear_residual: null argument");
  if (!residual) ldr = 0;  // the pitch of a tensor that is not there says nothing
  if (lda < K || ldw < K || ldo < N || (residual && ldr < N))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: a row pitch is below the row's width");
  if (lda % 8 || ldw % 8 || !aligned16(a) || !aligned16(w))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: a and w must be 16-byte aligned, their pitches multiples of 8");
  if (!aligned2(bias) || !aligned2(residual) || !aligned2(out) || !aligned4(rows_dev))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: bias, residual, out and rows_dev must be aligned to their type");
  if (std::max(std::max(lda, ldw), std::max(ldo, ldr)) > (int64_t(1) << 31))
    return set_error(GDC_ERR_UNSUPPORTED, "gdc_linear_residual: row pitch above 2^31");
  if (residual == out && ldr != ldo && M > 1)
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_linear_residual: a residual that is out needs its pitch");
  int* err = nullptr;
  GDC_TRY(device_error_word(&err));
  const LinearResidualArgs args{a, w, bias, residual, out, lda, ldw, ldr, ldo, M, rows_dev, N, K, act};
  return launch_linear_residual(t, args, static_cast<cudaStream_t>(stream), err);
}

gdc_status gdc_gated_residual_norm(gdc_dtype dtype, const void* y, int64_t ldy, const void* x, int64_t ldx,
                                   int32_t post_norm, const void* post_weight, const void* post_bias, const void* gate,
                                   int64_t gate_rows, const int32_t* gate_index, float scale, int32_t pre_norm,
                                   const void* pre_weight, const void* pre_bias, void* x_out, int64_t ldxo, void* n_out,
                                   int64_t ldno, int64_t rows, const int32_t* rows_dev, int32_t cols, float eps,
                                   void* stream) {
  clear_error();
  Elem t = Elem::kF16;
  GDC_TRY(check_elem("gdc_gated_residual_norm", dtype, &t));
  if (rows < 0 || rows > kMaxRows || cols < 1 || cols > 16384)
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: rows in [0, 2^30] and cols in [1, 16384] required");
  if (post_norm < 0 || post_norm > 2 || pre_norm < 0 || pre_norm > 2)
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: unknown norm %d / %d", post_norm, pre_norm);
  if (!std::isfinite(scale) || !(eps >= 0.f) || !std::isfinite(eps))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: scale and eps must be finite, eps not negative");
  if (rows == 0) return GDC_OK;
  if (!x || (!x_out && y) || (!x_out && !n_out))
    return set_error(GDC_ERR_NULL_POINTER, "gdc_gated_residual_norm: null argument");
  if ((pre_norm != 0) != (n_out != nullptr))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: n_out goes with a pre_norm");
  if ((gate && gate_rows < 1) || (gate && !gate_index && gate_rows != 1 && gate_rows < rows) || (!gate && gate_index) ||
      gate_rows > kMaxRows)
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: gate_rows %lld does not fit", (long long)gate_rows);
  if (!y) ldy = 0;  // the pitch of a tensor that is not there says nothing
  if (!x_out) ldxo = 0;
  if (!n_out) ldno = 0;
  if (!y && (gate || post_norm != 0))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: a gate or post_norm needs y");
  if ((y && ldy < cols) || ldx < cols || (x_out && ldxo < cols) || (n_out && ldno < cols))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: a row pitch is below cols");
  const void* all[] = {y, x, post_weight, post_bias, gate, pre_weight, pre_bias, x_out, n_out};
  for (const void* p : all)
    if (!aligned2(p) || !aligned4(rows_dev) || !aligned4(gate_index))
      return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: pointers must be aligned to their type");
  if (std::max(std::max(ldy, ldx), std::max(ldxo, ldno)) > (int64_t(1) << 31))
    return set_error(GDC_ERR_UNSUPPORTED, "gdc_gated_residual_norm: row pitch above 2^31");
  if (rows > 1 && ((x_out == x && ldxo != ldx) || (n_out && n_out == y && ldno != ldy)))
    return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: an output that is an input needs its pitch");
  if (x_out && x_out == n_out) return set_error(GDC_ERR_INVALID_INPUT, "gdc_gated_residual_norm: x_out and n_out are the same");
  int* err = nullptr;
  GDC_TRY(device_error_word(&err));
  const GatedNormArgs a{y, x, post_norm != 0 ? post_weight : nullptr, post_norm != 0 ? post_bias : nullptr, gate,
                        pre_norm != 0 ? pre_weight : nullptr, pre_norm != 0 ? pre_bias : nullptr, x_out, n_out, ldy, ldx,
                        ldxo, ldno, rows, gate_rows, gate_index, rows_dev, post_norm, pre_norm, cols, scale, eps};
  return launch_gated_residual_norm(t, a, static_cast<cudaStream_t>(stream), err);
}

}  // extern "C"
