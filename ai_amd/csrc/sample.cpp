// C ABI of sampling: argument checks, host staging.
#include "sample.h"

#include <cmath>

using fa::set_error;
using namespace fa::slots;

namespace {

constexpr const char* kOp = "Sample";
constexpr int64_t kMaxRows = (int64_t)1 << 20, kMaxVocab = (int64_t)1 << 24, kMaxLd = (int64_t)1 << 40;

int check_sizes(fa_ctx* ctx, int64_t rows, int64_t vocab) {
  if (rows < 0 || rows >= kMaxRows) return set_error(ctx, FA_ERR_ARG, "%s: %lld rows outside [0..2^20)", kOp, (long long)rows);
  if (vocab < 1 || vocab > kMaxVocab)
    return set_error(ctx, FA_ERR_ARG, "%s: a vocabulary of %lld outside 1..2^24", kOp, (long long)vocab);
  if (fa::sample_grid(rows, vocab) >= (int64_t)1 << 23)
    return set_error(ctx, FA_ERR_ARG, "%s: %lld rows of %lld are more than one call takes", kOp, (long long)rows,
                     (long long)vocab);
  return FA_OK;
}

int check(fa_ctx* ctx, int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld, const float* u,
          const int32_t* ids) {
  int rc;
  if ((rc = check_sizes(ctx, rows, vocab))) return rc;
  if (dtype != FA_DT_F32 && dtype != FA_DT_BF16) return set_error(ctx, FA_ERR_ARG, "%s: unknown dtype %d", kOp, dtype);
  if (rows > 0 && (ld < vocab || ld > kMaxLd))
    return set_error(ctx, FA_ERR_ARG, "%s: leading dimension %lld of rows of %lld", kOp, (long long)ld, (long long)vocab);
  if (rows > 0 && (!logits || !u || !ids)) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", kOp);
  if (!ctx) return set_error(ctx, FA_ERR_ARG, "%s: ctx is NULL", kOp);
  return FA_OK;
}

// Settings and numbers on the host: the ones that the kernels would answer with -1 are errors.
int check_values(fa_ctx* ctx, int64_t rows, const fa_sampling& s, const float* u) {
  for (int64_t r = 0; r < rows; r++) {
    if (s.temperature && !(s.temperature[r] >= 0 && std::isfinite(s.temperature[r])))
      return set_error(ctx, FA_ERR_ARG, "%s: row %lld has temperature %g", kOp, (long long)r, s.temperature[r]);
    if (s.top_p && !(s.top_p[r] >= 0 && s.top_p[r] <= 1))
      return set_error(ctx, FA_ERR_ARG, "%s: row %lld has top_p %g outside 0..1", kOp, (long long)r, s.top_p[r]);
    if (s.min_p && !(s.min_p[r] >= 0 && s.min_p[r] <= 1))
      return set_error(ctx, FA_ERR_ARG, "%s: row %lld has min_p %g outside 0..1", kOp, (long long)r, s.min_p[r]);
    if (!(u[r] >= 0 && u[r] < 1))
      return set_error(ctx, FA_ERR_ARG, "%s: row %lld has the number %g outside [0, 1)", kOp, (long long)r, u[r]);
  }
  return FA_OK;
}

}  // namespace

extern "C" {

int fa_sample_work(int64_t rows, int64_t vocab, size_t* bytes) {
  if (!bytes) return set_error(nullptr, FA_ERR_ARG, "%s: bytes is NULL", kOp);
  *bytes = 0;
  const int rc = check_sizes(nullptr, rows, vocab);
  if (rc || rows == 0) return rc;
  *bytes = fa::sample_scratch(rows, vocab, true);
  return FA_OK;
}

int fa_sample_dev(fa_ctx* ctx, int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld,
                  const fa_sampling* s, const float* u, int32_t* ids, float* logp, void* work, size_t work_bytes) {
  int rc = check(ctx, rows, vocab, dtype, logits, ld, u, ids);
  if (rc || rows == 0) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  const fa_sampling h = s ? *s : fa_sampling{};
  const size_t need = fa::sample_scratch(rows, vocab, fa::sample_filters(h));
  if (work) {
    if (work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15))
      return set_error(ctx, FA_ERR_ARG, "%s: work of %zu bytes, 16-byte aligned, is needed (%zu given)", kOp, need,
                       work_bytes);
  } else if (need) {
    if ((rc = fa::refuse_capture(ctx, ctx->stream, kOp, "fa_sample_work"))) return rc;
    if ((rc = ctx->slot(S_SAMPLE).ensure(ctx, need))) return rc;
    work = ctx->slot(S_SAMPLE).ptr;
  }
  const fa::SampleArgs a = {rows, vocab, dtype, logits, ld, h, u, ids, logp};
  return fa::launch_sample(ctx, a, work, ctx->stream);
}

int fa_sample(fa_ctx* ctx, int64_t rows, int64_t vocab, int dtype, const void* logits, int64_t ld,
              const fa_sampling* s, const float* u, int32_t* ids, float* logp) {
  int rc = check(ctx, rows, vocab, dtype, logits, ld, u, ids);
  if (rc || rows == 0) return rc;
  const fa_sampling h = s ? *s : fa_sampling{};
  if ((rc = check_values(ctx, rows, h, u))) return rc;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, kOp))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  void* dl;
  const size_t elem = dtype == FA_DT_F32 ? 4 : 2;
  if ((rc = fa::stage_h2d(ctx, S_X, logits, (size_t)((rows - 1) * ld + vocab) * elem, &dl))) return rc;
  // temperature, top_k, top_p, min_p and u, a row's results after them
  fa::DevBuf& in = ctx->slot(S_SAMPLE_IN);
  if ((rc = in.ensure(ctx, (size_t)rows * 4 * 7))) return rc;
  float* d = in.as<float>();
  const void* from[5] = {h.temperature, h.top_k, h.top_p, h.min_p, u};
  const void* at[5];
  for (int i = 0; i < 5; i++) {
    at[i] = from[i] ? d + i * rows : nullptr;
    if (from[i])
      FA_HIP_CHECK(ctx, hipMemcpyAsync(d + i * rows, from[i], (size_t)rows * 4, hipMemcpyHostToDevice, ctx->stream));
  }
  if ((rc = ctx->slot(S_SAMPLE).ensure(ctx, fa::sample_scratch(rows, vocab, fa::sample_filters(h))))) return rc;
  fa::SampleArgs a = {rows, vocab, dtype, dl, ld, {}, (const float*)at[4], (int32_t*)(d + 5 * rows), d + 6 * rows};
  a.s = {(const float*)at[0], (const int32_t*)at[1], (const float*)at[2], (const float*)at[3]};
  if ((rc = fa::launch_sample(ctx, a, ctx->slot(S_SAMPLE).ptr, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipMemcpyAsync(ids, a.ids, (size_t)rows * 4, hipMemcpyDeviceToHost, ctx->stream));
  if (logp) FA_HIP_CHECK(ctx, hipMemcpyAsync(logp, a.logp, (size_t)rows * 4, hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

}  // extern "C"
