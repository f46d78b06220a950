// dion_lm.hip -- MI355X (gfx950) training operators around the Dion optimizer: the C entry points
// of include/dion_lm.h (argument checks) over the kernels of the lm_*.hpp files.
#include "lm_common.hpp"
#include "lm_dropout.hpp"
#include "lm_norm.hpp"
#include "lm_gemm.hpp"
#include "lm_xent.hpp"

#ifndef DION_LM_BUILD_ID
#define DION_LM_BUILD_ID "unknown"
#endif

namespace {

int check_p(const char* what, double p, const DionRng* rng) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(DION_E_INVALID, "%s: p = %g is not in 0 .. 1", what, p);
  if (p > 0.0 && rng == nullptr) return fail(DION_E_INVALID, "%s: p > 0 without rng", what);
  return DION_OK;
}

int check_norm(const DionNormDesc* d) {
  if (d == nullptr) return fail(DION_E_INVALID, "null descriptor");
  if (d->rows < 0 || d->rows > 0x7FFFFFFF || d->cols < 1)
    return fail(DION_E_INVALID, "rows = %lld, cols = %d", static_cast<long long>(d->rows), d->cols);
  if (d->cols > rms::kMaxCols) return fail(DION_E_UNSUPPORTED, "cols = %d > %d", d->cols, rms::kMaxCols);
  if (!is_float_dtype(d->dtype) || !is_float_dtype(d->w_dtype))
    return fail(DION_E_UNSUPPORTED, "dtype %d, weight dtype %d", d->dtype, d->w_dtype);
  return DION_OK;
}

void norm_args(const DionNormDesc* d, const DionRng* rng, NormArgs* a) {
  memset(a, 0, sizeof(*a));
  a->rows = d->rows;
  a->cols = d->cols;
  a->w_bf16 = d->w_dtype == DION_DTYPE_BF16;
  a->eps = d->eps;
  a->drop = drop_args(d->p, rng);
  a->dropping = d->p > 0.0;
}

int check_xent(const DionXentDesc* d, int op) {
  if (d == nullptr) return fail(DION_E_INVALID, "null descriptor");
  if (op != DION_XENT_FORWARD && op != DION_XENT_BACKWARD) return fail(DION_E_INVALID, "op %d", op);
  if (d->tokens < 0 || d->hidden < 1 || d->vocab < 1)
    return fail(DION_E_INVALID, "tokens = %lld, hidden = %d, vocab = %d", static_cast<long long>(d->tokens), d->hidden,
                d->vocab);
  // byte offsets within a tile of 256 rows are 31 bits
  if (d->tokens > (1 << 24) || d->hidden > (1 << 20) || d->vocab > (1 << 21) || d->ld_weight > (1 << 21))
    return fail(DION_E_UNSUPPORTED, "tokens = %lld, hidden = %d, vocab = %d, ld_weight = %lld",
                static_cast<long long>(d->tokens), d->hidden, d->vocab, static_cast<long long>(d->ld_weight));
  if (!is_float_dtype(d->dtype) || (op == DION_XENT_BACKWARD && !is_float_dtype(d->gw_dtype)))
    return fail(DION_E_UNSUPPORTED, "dtype %d, grad_weight dtype %d", d->dtype, d->gw_dtype);
  if (d->piece_bytes < 0) return fail(DION_E_INVALID, "piece_bytes < 0");
  if (d->ld_hidden < d->hidden || d->ld_weight < d->hidden)
    return fail(DION_E_INVALID, "ld_hidden = %lld, ld_weight = %lld", static_cast<long long>(d->ld_hidden),
                static_cast<long long>(d->ld_weight));
  if (d->vocab_start < 0 || d->vocab_total < d->vocab || d->vocab_start > d->vocab_total - d->vocab)
    return fail(DION_E_INVALID, "words %lld .. + %d of %lld", static_cast<long long>(d->vocab_start), d->vocab,
                static_cast<long long>(d->vocab_total));
  return DION_OK;
}

int check_xent_call(const DionXentDesc* d, int op, const void* hidden, const void* weight, const void* target,
                    const void* ws, size_t ws_bytes) {
  if (hidden == nullptr || weight == nullptr || target == nullptr) return fail(DION_E_INVALID, "null tensor");
  if (d->dtype == DION_DTYPE_BF16 && !d->pack_weight && !aligned16(weight) && d->hidden % 8 == 0 && d->ld_weight % 8 == 0)
    return fail(DION_E_INVALID, "weight is not 16-byte aligned: set pack_weight");
  const size_t need = xent::make_plan(d, op).total;
  if (ws == nullptr || ws_bytes < need || !aligned16(ws))
    return fail(DION_E_WORKSPACE, "needs %zu workspace bytes, 16-byte aligned", need);
  return DION_OK;
}

}  // namespace

extern "C" {

int dion_lm_abi_version(void) { return DION_LM_ABI_VERSION; }
const char* dion_lm_build_id(void) { return DION_LM_BUILD_ID; }
const char* dion_lm_last_error(void) { return g_err; }

int dion_dropout_add(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ld_x, const void* residual,
                     int64_t ld_residual, void* out, int64_t ld_out, double p, const DionRng* rng,
                     dion_stream_t stream) {
  if (rows < 0 || cols < 0) return fail(DION_E_INVALID, "rows or cols < 0");
  if (!is_float_dtype(dtype)) return fail(DION_E_UNSUPPORTED, "dtype %d", dtype);
  const int rc = check_p("dropout_add", p, rng);
  if (rc != DION_OK) return rc;
  if (rows == 0 || cols == 0) return DION_OK;
  if (x == nullptr || out == nullptr) return fail(DION_E_INVALID, "null tensor");
  if (rows > INT64_MAX / 8 / cols) return fail(DION_E_UNSUPPORTED, "rows * cols overflows");
  if (rows == 1) ld_x = ld_out = ld_residual = cols;
  if (ld_x < cols || ld_out < cols || (residual && ld_residual < cols)) return fail(DION_E_INVALID, "row stride < cols");
  DropoutArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x;
  a.residual = residual;
  a.out = out;
  a.ldx = ld_x;
  a.ldr = ld_residual;
  a.ldo = ld_out;
  a.rows = rows;
  a.cols = cols;
  a.drop = drop_args(p, rng);
  if (dtype == DION_DTYPE_F32)
    return residual ? dropout::launch<float, true>(a, stream) : dropout::launch<float, false>(a, stream);
  return residual ? dropout::launch<bf16, true>(a, stream) : dropout::launch<bf16, false>(a, stream);
}

int dion_rms_norm_add(const DionNormDesc* d, const void* x, const void* residual, const void* weight, void* h, void* y,
                      float* scale, float* rstd, const DionRng* rng, dion_stream_t stream) {
  int rc = check_norm(d);
  if (rc == DION_OK) rc = check_p("rms_norm_add", d->p, rng);
  if (rc != DION_OK) return rc;
  const bool quant = d->y_dtype == DION_DTYPE_E4M3;
  if (!quant && d->y_dtype != d->dtype) return fail(DION_E_UNSUPPORTED, "y dtype %d", d->y_dtype);
  if (quant && (d->scale_block < (d->cols < 8 ? d->cols : 8) || d->scale_block > d->cols))
    return fail(DION_E_INVALID, "scale_block = %d of %d columns: 8 at least", d->scale_block, d->cols);
  if (d->rows == 0) return DION_OK;
  if (x == nullptr || weight == nullptr || y == nullptr || rstd == nullptr || (quant && scale == nullptr))
    return fail(DION_E_INVALID, "null tensor");
  if (h == nullptr && (residual != nullptr || d->p > 0.0)) return fail(DION_E_INVALID, "h is another tensor than x here");
  if (d->ld_x < d->cols || d->ld_y < d->cols || (residual && d->ld_residual < d->cols) || (h && d->ld_h < d->cols))
    return fail(DION_E_INVALID, "row stride < cols");
  NormArgs a;
  norm_args(d, rng, &a);
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.h = h;
  a.y = y;
  a.scale = scale;
  a.rstd_out = rstd;
  a.ldx = d->ld_x;
  a.ldr = d->ld_residual;
  a.ldh = d->ld_h;
  a.ldy = d->ld_y;
  if (quant) {
    a.sblock = d->scale_block;
    a.sblocks = static_cast<int>(ceil_div(d->cols, d->scale_block));
  }
  const bool f32 = d->dtype == DION_DTYPE_F32;
  if (!quant) return f32 ? rms::forward<float, Q8_NONE>(a, stream) : rms::forward<bf16, Q8_NONE>(a, stream);
  const bool lanes = a.sblock >= 8 && a.sblock <= 512 && (a.sblock & (a.sblock - 1)) == 0;
  if (lanes) return f32 ? rms::forward<float, Q8_LANES>(a, stream) : rms::forward<bf16, Q8_LANES>(a, stream);
  return f32 ? rms::forward<float, Q8_ANY>(a, stream) : rms::forward<bf16, Q8_ANY>(a, stream);
}

int dion_rms_norm_add_workspace_bytes(const DionNormDesc* d, size_t* bytes) {
  const int rc = check_norm(d);
  if (rc != DION_OK) return rc;
  if (bytes == nullptr) return fail(DION_E_INVALID, "null bytes");
  *bytes = rms::ws_bytes(d);
  return DION_OK;
}

int dion_rms_norm_add_backward(const DionNormDesc* d, const void* grad_y, const void* h, const void* weight,
                               const float* rstd, const void* grad_h, void* grad_x, void* grad_residual,
                               void* grad_weight, const DionRng* rng, void* ws, size_t ws_bytes, dion_stream_t stream) {
  int rc = check_norm(d);
  if (rc == DION_OK) rc = check_p("rms_norm_add_backward", d->p, rng);
  if (rc != DION_OK) return rc;
  if (grad_weight && !is_float_dtype(d->gw_dtype)) return fail(DION_E_UNSUPPORTED, "grad_weight dtype %d", d->gw_dtype);
  if (!grad_x && !grad_residual && !grad_weight) return DION_OK;
  if (d->rows > 0 && (grad_y == nullptr || h == nullptr || weight == nullptr || rstd == nullptr))
    return fail(DION_E_INVALID, "null tensor");
  if (weight == nullptr) return fail(DION_E_INVALID, "null weight");
  if (d->ld_grad_y < d->cols || d->ld_h < d->cols || (grad_h && d->ld_grad_h < d->cols) ||
      (grad_x && d->ld_grad_x < d->cols) || (grad_residual && d->ld_grad_residual < d->cols))
    return fail(DION_E_INVALID, "row stride < cols");
  if (grad_weight && (ws == nullptr || ws_bytes < rms::ws_bytes(d) || !aligned16(ws)))
    return fail(DION_E_WORKSPACE, "needs %zu workspace bytes, 16-byte aligned", rms::ws_bytes(d));
  NormArgs a;
  norm_args(d, rng, &a);
  a.gy = grad_y;
  a.h_in = h;
  a.weight = weight;
  a.rstd = rstd;
  a.gh = grad_h;
  a.gx = grad_x;
  a.gr = grad_residual;
  a.gw = grad_weight;
  a.gw_bf16 = d->gw_dtype == DION_DTYPE_BF16;
  a.accumulate = d->accumulate;
  a.part = grad_weight ? static_cast<float*>(ws) : nullptr;
  a.ldgy = d->ld_grad_y;
  a.ldh = d->ld_h;
  a.ldgh = d->ld_grad_h;
  a.ldgx = d->ld_grad_x;
  a.ldgr = d->ld_grad_residual;
  if (d->dtype == DION_DTYPE_F32) return rms::backward<float>(a, stream);
  return rms::backward<bf16>(a, stream);
}

int dion_xent_workspace_bytes(const DionXentDesc* d, int op, size_t* bytes) {
  const int rc = check_xent(d, op);
  if (rc != DION_OK) return rc;
  if (bytes == nullptr) return fail(DION_E_INVALID, "null bytes");
  *bytes = d->tokens == 0 ? 0 : xent::make_plan(d, op).total;
  return DION_OK;
}

int dion_xent_forward(const DionXentDesc* d, const void* hidden, const void* weight, const int64_t* target, float* loss,
                      float* lse, float* tlogit, void* ws, size_t ws_bytes, dion_stream_t stream) {
  int rc = check_xent(d, DION_XENT_FORWARD);
  if (rc != DION_OK) return rc;
  if (d->tokens == 0) return DION_OK;
  rc = check_xent_call(d, DION_XENT_FORWARD, hidden, weight, target, ws, ws_bytes);
  if (rc != DION_OK) return rc;
  if (lse == nullptr) return fail(DION_E_INVALID, "null lse");
  return xent::forward(d, hidden, weight, target, loss, lse, tlogit, static_cast<char*>(ws), stream);
}

int dion_xent_backward(const DionXentDesc* d, const void* hidden, const void* weight, const int64_t* target,
                       const float* lse, const float* grad_loss, void* grad_hidden, void* grad_weight, void* ws,
                       size_t ws_bytes, dion_stream_t stream) {
  int rc = check_xent(d, DION_XENT_BACKWARD);
  if (rc != DION_OK) return rc;
  if (grad_hidden == nullptr && grad_weight == nullptr) return DION_OK;
  if (d->tokens == 0) return fail(DION_E_INVALID, "no tokens: there is no gradient to add");
  rc = check_xent_call(d, DION_XENT_BACKWARD, hidden, weight, target, ws, ws_bytes);
  if (rc != DION_OK) return rc;
  if (lse == nullptr || grad_loss == nullptr) return fail(DION_E_INVALID, "null lse or grad_loss");
  if ((grad_hidden && d->ld_grad_hidden < d->hidden) || (grad_weight && d->ld_grad_weight < d->hidden))
    return fail(DION_E_INVALID, "row stride of a gradient < hidden");
  return xent::backward(d, hidden, weight, target, lse, grad_loss, grad_hidden, grad_weight, static_cast<char*>(ws),
                        stream);
}

}  // extern "C"
