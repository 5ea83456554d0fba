// C ABI of the products with weights in 8 bits: argument checks, host staging.
#include "f8.h"

#include <algorithm>

using fa::set_error;
using namespace fa::slots;

namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 27, kMaxCols = (int64_t)1 << 24;
constexpr int64_t kMaxLd = (int64_t)1 << 30;  // offsets in bytes stay within 63 bits

int check_matrix(fa_ctx* ctx, const char* op, const fa_f8_matrix* w, bool buffers = true) {
  if (!w) return set_error(ctx, FA_ERR_ARG, "%s: matrix is NULL", op);
  if (w->n < 0 || w->n >= kMaxRows || w->k < 0 || w->k >= kMaxCols)
    return set_error(ctx, FA_ERR_ARG, "%s: matrix [%lld x %lld] outside [0..2^27) x [0..2^24)", op, (long long)w->n,
                     (long long)w->k);
  if (!buffers || w->n == 0 || w->k == 0) return FA_OK;
  if (!w->codes || !w->scales) return set_error(ctx, FA_ERR_ARG, "%s: NULL matrix buffer", op);
  if ((reinterpret_cast<uintptr_t>(w->codes) & 15) || (reinterpret_cast<uintptr_t>(w->scales) & 3))
    return set_error(ctx, FA_ERR_ARG, "%s: the matrix's codes must be 16-byte and its scales 4-byte aligned", op);
  return FA_OK;
}

int check_dtype(fa_ctx* ctx, const char* op, int dtype) {
  if (dtype != FA_DT_F32 && dtype != FA_DT_BF16) return set_error(ctx, FA_ERR_ARG, "%s: unknown dtype %d", op, dtype);
  return FA_OK;
}

int check_ld(fa_ctx* ctx, const char* op, int64_t rows, int64_t cols, int64_t ld) {
  if (rows > 0 && (ld < cols || ld > kMaxLd))
    return set_error(ctx, FA_ERR_ARG, "%s: leading dimension %lld of rows of %lld", op, (long long)ld, (long long)cols);
  return FA_OK;
}

fa::F8View view_of(const fa_f8_matrix* w) {
  return {static_cast<uint8_t*>(w->codes), static_cast<uint8_t*>(w->scales), w->n, w->k, fa::f8_kp(w->k)};
}

size_t elem(int dtype) { return dtype == FA_DT_F32 ? 4 : 2; }
size_t span(int64_t rows, int64_t cols, int64_t ld, int dtype) {
  return rows > 0 ? (size_t)((rows - 1) * ld + cols) * elem(dtype) : 0;
}

int convert_check(fa_ctx* ctx, const char* op, const fa_f8_matrix* w, int dtype, const void* x, int64_t ldx) {
  int rc;
  if ((rc = check_matrix(ctx, op, w)) || (rc = check_dtype(ctx, op, dtype)) ||
      (rc = check_ld(ctx, op, w->n, w->k, ldx)))
    return rc;
  if (w->n > 0 && w->k > 0 && !x) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", op);
  if (!ctx) return set_error(ctx, FA_ERR_ARG, "%s: ctx is NULL", op);
  return FA_OK;
}

bool nothing(const fa_f8_matrix* w) { return w->n == 0 || w->k == 0; }

int product_check(fa_ctx* ctx, int64_t m, int a_dtype, const void* a, int64_t lda, const fa_f8_matrix* w,
                  const fa_epilogue* e, int c_dtype, const void* c, int64_t ldc) {
  const char* op = "MatMulF8";
  int rc;
  if ((rc = check_matrix(ctx, op, w)) || (rc = check_dtype(ctx, op, a_dtype)) || (rc = check_dtype(ctx, op, c_dtype)))
    return rc;
  if (m < 0 || m >= kMaxRows) return set_error(ctx, FA_ERR_ARG, "%s: %lld rows outside [0..2^27)", op, (long long)m);
  if ((rc = check_ld(ctx, op, m, w->k, lda)) || (rc = check_ld(ctx, op, m, w->n, ldc))) return rc;
  if (e && (e->act < FA_ACT_NONE || e->act > FA_ACT_TANH))
    return set_error(ctx, FA_ERR_ARG, "%s: unknown activation %d", op, e->act);
  if (e && e->mul && (rc = check_ld(ctx, "MatMulF8: Mul", m, w->n, e->ldm))) return rc;
  if (e && e->residual && (rc = check_ld(ctx, "MatMulF8: Residual", m, w->n, e->ldr))) return rc;
  if (fa::f8_grid(m, w->n) >= (int64_t)1 << 24)
    return set_error(ctx, FA_ERR_ARG, "%s: [%lld x %lld] is more than one call takes", op, (long long)m,
                     (long long)w->n);
  if (m > 0 && w->n > 0 && ((w->k > 0 && !a) || !c)) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", op);
  if (!ctx) return set_error(ctx, FA_ERR_ARG, "%s: ctx is NULL", op);
  return FA_OK;
}

fa::F8GemmArgs args_of(int64_t m, int a_dtype, const void* a, int64_t lda, const fa_f8_matrix* w,
                       const fa_epilogue* e, int c_dtype, void* c, int64_t ldc) {
  fa::F8GemmArgs g = {m, a_dtype, a, lda, view_of(w), {}, c_dtype, c, ldc};
  if (e) g.e = *e;
  return g;
}

}  // namespace

extern "C" {

size_t fa_f8_codes_bytes(int64_t n, int64_t k) {
  if (n < 0 || n >= kMaxRows || k < 0 || k >= kMaxCols) return 0;
  return (size_t)n * fa::f8_kp(k);
}

size_t fa_f8_scales_bytes(int64_t n, int64_t k) {
  if (n < 0 || n >= kMaxRows || k < 0 || k >= kMaxCols) return 0;
  return (size_t)n * fa::f8_ks(k);
}

int fa_f8_write_dev(fa_ctx* ctx, const fa_f8_matrix* w, int dtype, const void* x, int64_t ldx) {
  const int rc = convert_check(ctx, "F8Write", w, dtype, x, ldx);
  if (rc || nothing(w)) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  return fa::launch_f8_write(ctx, view_of(w), dtype, x, ldx, ctx->stream);
}

int fa_f8_write(fa_ctx* ctx, const fa_f8_matrix* w, int dtype, const void* x, int64_t ldx) {
  int rc = convert_check(ctx, "F8Write", w, dtype, x, ldx);
  if (rc || nothing(w)) return rc;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "F8Write"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  void* dx;
  if ((rc = fa::stage_h2d(ctx, S_X, x, span(w->n, w->k, ldx, dtype), &dx))) return rc;
  if ((rc = fa::launch_f8_write(ctx, view_of(w), dtype, dx, ldx, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

int fa_f8_read_dev(fa_ctx* ctx, const fa_f8_matrix* w, int dtype, void* out, int64_t ldo) {
  const int rc = convert_check(ctx, "F8Read", w, dtype, out, ldo);
  if (rc || nothing(w)) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  return fa::launch_f8_read(ctx, view_of(w), dtype, out, ldo, ctx->stream);
}

int fa_f8_read(fa_ctx* ctx, const fa_f8_matrix* w, int dtype, void* out, int64_t ldo) {
  int rc = convert_check(ctx, "F8Read", w, dtype, out, ldo);
  if (rc || nothing(w)) return rc;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "F8Read"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  const size_t row = (size_t)w->k * elem(dtype);
  if ((rc = ctx->slot(S_OUT).ensure(ctx, row * w->n))) return rc;
  if ((rc = fa::launch_f8_read(ctx, view_of(w), dtype, ctx->slot(S_OUT).ptr, w->k, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipMemcpy2DAsync(out, (size_t)ldo * elem(dtype), ctx->slot(S_OUT).ptr, row, row, (size_t)w->n,
                                     hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

int fa_matmul_f8_work(int64_t m, const fa_f8_matrix* w, size_t* bytes) {
  if (!bytes) return set_error(nullptr, FA_ERR_ARG, "MatMulF8: bytes is NULL");
  *bytes = 0;
  const int rc = check_matrix(nullptr, "MatMulF8", w, false);
  if (rc) return rc;
  if (m < 0 || m >= kMaxRows) return set_error(nullptr, FA_ERR_ARG, "MatMulF8: %lld rows outside [0..2^27)", (long long)m);
  if (m > 0 && w->n > 0) *bytes = fa::f8_scratch(m, w->n, w->k);
  return FA_OK;
}

int fa_matmul_f8_dev(fa_ctx* ctx, int64_t m, int a_dtype, const void* a, int64_t lda, const fa_f8_matrix* w,
                     const fa_epilogue* e, int c_dtype, void* c, int64_t ldc, void* work, size_t work_bytes) {
  int rc = product_check(ctx, m, a_dtype, a, lda, w, e, c_dtype, c, ldc);
  if (rc || m == 0 || w->n == 0) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  const size_t need = fa::f8_scratch(m, w->n, w->k);
  if (work) {
    if (work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15))
      return set_error(ctx, FA_ERR_ARG, "MatMulF8: work of %zu bytes, 16-byte aligned, is needed (%zu given)", need,
                       work_bytes);
  } else if (need) {
    if ((rc = fa::refuse_capture(ctx, ctx->stream, "MatMulF8", "fa_matmul_f8_work"))) return rc;
    if ((rc = ctx->slot(S_F8).ensure(ctx, need))) return rc;
    work = ctx->slot(S_F8).ptr;
  }
  return fa::launch_f8_gemm(ctx, args_of(m, a_dtype, a, lda, w, e, c_dtype, c, ldc), work, ctx->stream);
}

int fa_matmul_f8(fa_ctx* ctx, int64_t m, int a_dtype, const void* a, int64_t lda, const fa_f8_matrix* w,
                 const fa_epilogue* e, int c_dtype, void* c, int64_t ldc) {
  int rc = product_check(ctx, m, a_dtype, a, lda, w, e, c_dtype, c, ldc);
  if (rc || m == 0 || w->n == 0) return rc;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "MatMulF8"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  const int64_t n = w->n;
  void *da = nullptr, *p = nullptr;
  if ((rc = fa::stage_h2d(ctx, S_A, a, span(m, w->k, lda, a_dtype), &da))) return rc;
  const size_t row = (size_t)n * elem(c_dtype);
  if ((rc = ctx->slot(S_C).ensure(ctx, row * m)) || (rc = ctx->slot(S_F8).ensure(ctx, fa::f8_scratch(m, n, w->k))))
    return rc;
  fa::F8GemmArgs g = args_of(m, a_dtype, da, lda, w, e, c_dtype, ctx->slot(S_C).ptr, n);
  if (e) {
    if (e->bias) { if ((rc = fa::stage_h2d(ctx, S_BIAS, e->bias, (size_t)n * 4, &p))) return rc; g.e.bias = (const float*)p; }
    if (e->row_scale) { if ((rc = fa::stage_h2d(ctx, S_ROWSCALE, e->row_scale, (size_t)m * 4, &p))) return rc; g.e.row_scale = (const float*)p; }
    if (e->mul) { if ((rc = fa::stage_h2d(ctx, S_MUL, e->mul, span(m, n, e->ldm, FA_DT_F32), &p))) return rc; g.e.mul = (const float*)p; }
    if (e->residual) { if ((rc = fa::stage_h2d(ctx, S_RES, e->residual, span(m, n, e->ldr, FA_DT_F32), &p))) return rc; g.e.residual = (const float*)p; }
  }
  if ((rc = fa::launch_f8_gemm(ctx, g, ctx->slot(S_F8).ptr, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipMemcpy2DAsync(c, (size_t)ldc * elem(c_dtype), ctx->slot(S_C).ptr, row, row, (size_t)m,
                                     hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

}  // extern "C"
