// C ABI of the key/value cache in 8 bits: argument checks, host staging.
#include "kvcache.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

using fa::set_error;
using namespace fa::slots;

namespace {

constexpr int64_t kMaxGrid = 0x7FFFFFFF;
constexpr int32_t kMaxTable = (1 << 25) - 1;  // positions stay below 2^31

int check_cache_sizes(fa_ctx* ctx, const char* op, const fa_kv_cache* c) {
  if (!c) return set_error(ctx, FA_ERR_ARG, "%s: cache is NULL", op);
  if (c->blocks < 0) return set_error(ctx, FA_ERR_ARG, "%s: %d blocks", op, c->blocks);
  if (c->kv_heads < 1 || c->kv_heads > 65535)
    return set_error(ctx, FA_ERR_ARG, "%s: %d key/value heads outside 1..65535", op, c->kv_heads);
  if (c->head_dim < 1 || c->head_dim > fa::kKvMaxDim)
    return set_error(ctx, FA_ERR_ARG, "%s: head dimension %d outside 1..%d", op, c->head_dim, fa::kKvMaxDim);
  return FA_OK;
}

int check_cache(fa_ctx* ctx, const char* op, const fa_kv_cache* c) {
  const int rc = check_cache_sizes(ctx, op, c);
  if (rc) return rc;
  if (c->blocks > 0 && (!c->codes || !c->scales)) return set_error(ctx, FA_ERR_ARG, "%s: NULL cache buffer", op);
  if ((reinterpret_cast<uintptr_t>(c->codes) & 15) || (reinterpret_cast<uintptr_t>(c->scales) & 7))
    return set_error(ctx, FA_ERR_ARG, "%s: the cache's codes must be 16-byte and its scales 8-byte aligned", op);
  return FA_OK;
}

int check_batch(fa_ctx* ctx, const char* op, const fa_kv_batch* b, int dtype) {
  if (!b) return set_error(ctx, FA_ERR_ARG, "%s: batch is NULL", op);
  if (b->nseq < 0 || b->rows < 0 || b->table_stride < 0)
    return set_error(ctx, FA_ERR_ARG, "%s: negative size (%d sequences, %lld rows, table rows of %d)", op, b->nseq,
                     (long long)b->rows, b->table_stride);
  if (b->table_stride > kMaxTable)
    return set_error(ctx, FA_ERR_ARG, "%s: table rows of %d entries, at most %d", op, b->table_stride, kMaxTable);
  if (dtype != FA_DT_F32 && dtype != FA_DT_BF16) return set_error(ctx, FA_ERR_ARG, "%s: unknown dtype %d", op, dtype);
  if (b->nseq > 0 && (!b->lengths || !b->cu_rows || (b->table_stride > 0 && !b->tables)))
    return set_error(ctx, FA_ERR_ARG, "%s: NULL batch array", op);
  return FA_OK;
}

// Rows of a batch, units of work and int32 row indexes in the kernels.
int check_sizes(fa_ctx* ctx, const char* op, const fa_kv_batch* b, int64_t heads) {
  if (b->rows > kMaxGrid / heads || b->rows * heads + (int64_t)b->nseq * std::max<int64_t>(heads, 2) > kMaxGrid)
    return set_error(ctx, FA_ERR_ARG, "%s: %lld rows of %d sequences with %lld heads are more than one call takes", op,
                     (long long)b->rows, b->nseq, (long long)heads);
  return FA_OK;
}

// Workgroups of a launch (of 256 threads, which are counted in 32 bits).
int check_grid(fa_ctx* ctx, const char* op, int64_t workgroups) {
  if (workgroups >= (int64_t)1 << 24)
    return set_error(ctx, FA_ERR_ARG, "%s: %lld workgroups are more than one call takes", op, (long long)workgroups);
  return FA_OK;
}

enum class Use { Write, Read, Attend };

// The host entry points see the batch: everything that the kernels would
// have to leave out is an error here.
int check_host_batch(fa_ctx* ctx, const char* op, const fa_kv_cache* c, const fa_kv_batch* b, Use use,
                     int32_t window = 0) try {
  if (b->nseq == 0) return FA_OK;
  if (b->cu_rows[0] != 0) return set_error(ctx, FA_ERR_ARG, "%s: cu_rows starts at %d, not 0", op, b->cu_rows[0]);
  for (int i = 0; i < b->nseq; i++)
    if (b->cu_rows[i + 1] < b->cu_rows[i])
      return set_error(ctx, FA_ERR_ARG, "%s: cu_rows falls from %d to %d at sequence %d", op, b->cu_rows[i],
                       b->cu_rows[i + 1], i);
  if (b->cu_rows[b->nseq] > b->rows)
    return set_error(ctx, FA_ERR_ARG, "%s: cu_rows ends at %d of %lld rows", op, b->cu_rows[b->nseq],
                     (long long)b->rows);
  std::vector<int32_t> written;
  for (int i = 0; i < b->nseq; i++) {
    const int64_t n = b->cu_rows[i + 1] - b->cu_rows[i], len = b->lengths[i];
    if (len < n) return set_error(ctx, FA_ERR_ARG, "%s: sequence %d has %lld tokens but %lld rows", op, i,
                                  (long long)len, (long long)n);
    if (n == 0) continue;
    const int64_t used = (len + FA_KV_BLOCK - 1) / FA_KV_BLOCK;
    if (used > b->table_stride)
      return set_error(ctx, FA_ERR_ARG, "%s: sequence %d of %lld tokens needs %lld table entries, has %d", op, i,
                       (long long)len, (long long)used, b->table_stride);
    const int64_t from = use != Use::Attend ? len - n : window ? std::max<int64_t>(0, len - n - window + 1) : 0;
    const int64_t first = from / FA_KV_BLOCK;
    for (int64_t p = first; p < used; p++) {
      const int32_t id = b->tables[(int64_t)i * b->table_stride + p];
      if (id < 0 || id >= c->blocks)
        return set_error(ctx, FA_ERR_ARG, "%s: sequence %d's block %lld is %d, outside 0..%d", op, i, (long long)p, id,
                         c->blocks - 1);
      if (use == Use::Write) written.push_back(id);
    }
  }
  std::sort(written.begin(), written.end());
  const auto twice = std::adjacent_find(written.begin(), written.end());
  if (twice != written.end())
    return set_error(ctx, FA_ERR_ARG, "%s: block %d would be written twice", op, *twice);
  return FA_OK;
} catch (const std::bad_alloc&) {
  return set_error(ctx, FA_ERR_OOM, "%s: no host memory to check the batch", op);
}

fa::KvArgs args_of(const fa_kv_cache* c, const fa_kv_batch* b) {
  fa::KvArgs a;
  a.codes = static_cast<uint8_t*>(c->codes);
  a.scales = c->scales;
  a.blocks = c->blocks;
  a.hkv = c->kv_heads;
  a.nc = fa::kv_slices(c->head_dim);
  a.D = c->head_dim;
  a.tables = b->tables;
  a.tstride = b->table_stride;
  a.lengths = b->lengths;
  a.cu = b->cu_rows;
  a.nseq = b->nseq;
  a.rows = b->rows;
  return a;
}

// The batch's arrays in device scratch; dev.tables etc. point there.
int stage_batch(fa_ctx* ctx, const fa_kv_batch* b, fa_kv_batch* dev) {
  const size_t nt = (size_t)b->nseq * b->table_stride, n = (size_t)b->nseq;
  fa::DevBuf& buf = ctx->slot(S_KV);
  const int rc = buf.ensure(ctx, (nt + 2 * n + 1) * 4);
  if (rc) return rc;
  int32_t* d = static_cast<int32_t*>(buf.ptr);
  if (nt) FA_HIP_CHECK(ctx, hipMemcpyAsync(d, b->tables, nt * 4, hipMemcpyHostToDevice, ctx->stream));
  FA_HIP_CHECK(ctx, hipMemcpyAsync(d + nt, b->lengths, n * 4, hipMemcpyHostToDevice, ctx->stream));
  FA_HIP_CHECK(ctx, hipMemcpyAsync(d + nt + n, b->cu_rows, (n + 1) * 4, hipMemcpyHostToDevice, ctx->stream));
  *dev = *b;
  dev->tables = d;
  dev->lengths = d + nt;
  dev->cu_rows = d + nt + n;
  return FA_OK;
}

size_t elem(int dtype) { return dtype == FA_DT_F32 ? 4 : 2; }

// Bytes from a strided operand's first element to its last row's end.
size_t span(int64_t rows, int64_t heads, int64_t st, int64_t sh, int64_t D, int dtype) {
  return (size_t)((rows - 1) * st + (heads - 1) * sh + D) * elem(dtype);
}

int check_strides(fa_ctx* ctx, const char* op, int64_t rows, int64_t heads, int64_t st, int64_t sh) {
  if (st < 0 || sh < 0) return set_error(ctx, FA_ERR_ARG, "%s: negative stride", op);
  constexpr int64_t most = (int64_t)1 << 58;  // elements: offsets in bytes stay within 63 bits
  if (st > most / std::max<int64_t>(rows, 1) || sh > most / heads)
    return set_error(ctx, FA_ERR_ARG, "%s: strides of %lld and %lld elements are too large", op, (long long)st,
                     (long long)sh);
  return FA_OK;
}

int attn_args(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* q, int64_t q_st,
              int64_t q_sh, int32_t heads, int causal, int32_t window, float scale, void* out, fa::KvAttnArgs* a) {
  const char* op = "KVAttention";
  int rc;
  if ((rc = check_cache(ctx, op, cache)) || (rc = check_batch(ctx, op, batch, dtype))) return rc;
  if (heads < 1 || heads % cache->kv_heads != 0 || heads > 65535)
    return set_error(ctx, FA_ERR_ARG, "%s: %d query heads on %d key/value heads", op, heads, cache->kv_heads);
  if (window < 0) return set_error(ctx, FA_ERR_ARG, "%s: window %d", op, window);
  if (!(std::fabs(scale) <= 0x1p126f)) return set_error(ctx, FA_ERR_ARG, "%s: scale is not finite, or over 2^126", op);
  if ((rc = check_strides(ctx, op, batch->rows, heads, q_st, q_sh)) || (rc = check_sizes(ctx, op, batch, heads)))
    return rc;
  if (batch->rows > 0 && batch->nseq > 0 && (!q || !out)) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", op);
  a->c = args_of(cache, batch);
  a->dtype = dtype;
  a->q = q;
  a->q_st = q_st;
  a->q_sh = q_sh;
  a->H = heads;
  a->causal = causal != 0;
  a->window = window;
  a->scale = scale;
  a->out = out;
  return check_grid(ctx, op, fa::kv_attention_grid(*a));
}

int write_check(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* k,
                int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh) {
  const char* op = "KVWrite";
  int rc;
  if ((rc = check_cache(ctx, op, cache)) || (rc = check_batch(ctx, op, batch, dtype)) ||
      (rc = check_strides(ctx, op, batch->rows, cache->kv_heads, k_st, k_sh)) ||
      (rc = check_strides(ctx, op, batch->rows, cache->kv_heads, v_st, v_sh)) ||
      (rc = check_sizes(ctx, op, batch, cache->kv_heads)) || (rc = check_grid(ctx, op, fa::kv_grid(args_of(cache, batch)))))
    return rc;
  if (batch->rows > 0 && batch->nseq > 0 && (!k || !v)) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", op);
  return FA_OK;
}

int read_check(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* k,
               const void* v) {
  const char* op = "KVRead";
  int rc;
  if ((rc = check_cache(ctx, op, cache)) || (rc = check_batch(ctx, op, batch, dtype)) ||
      (rc = check_sizes(ctx, op, batch, cache->kv_heads)) || (rc = check_grid(ctx, op, fa::kv_grid(args_of(cache, batch)))))
    return rc;
  if (batch->rows > 0 && batch->nseq > 0 && (!k || !v)) return set_error(ctx, FA_ERR_ARG, "%s: NULL buffer", op);
  return FA_OK;
}

int need_ctx(fa_ctx* ctx, const char* op) {
  return ctx ? FA_OK : set_error(ctx, FA_ERR_ARG, "%s: ctx is NULL", op);
}

// The context's scratch for attention, its counters zero.
int own_parts(fa_ctx* ctx, size_t need, void** work) {
  fa::DevBuf& buf = ctx->slot(S_KV_PARTS);
  const bool grows = buf.bytes < need;
  int rc = buf.ensure(ctx, need);
  if (rc) return rc;
  *work = buf.ptr;
  return grows ? fa::launch_zero(ctx, buf.ptr, fa::kKvCountBytes, ctx->stream) : FA_OK;
}

bool nothing(const fa_kv_batch* b) { return b->rows == 0 || b->nseq == 0; }

}  // namespace

extern "C" {

size_t fa_kv_codes_bytes(int32_t blocks, int32_t kv_heads, int32_t head_dim) {
  if (blocks < 0 || kv_heads < 1 || kv_heads > 65535 || head_dim < 1 || head_dim > fa::kKvMaxDim) return 0;
  return (size_t)blocks * kv_heads * 2 * FA_KV_BLOCK * 64 * fa::kv_slices(head_dim);
}

int fa_kv_write_dev(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* k,
                    int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh) {
  int rc = write_check(ctx, cache, batch, dtype, k, k_st, k_sh, v, v_st, v_sh);
  if (rc || (rc = need_ctx(ctx, "KVWrite")) || nothing(batch)) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  return fa::launch_kv_write(ctx, args_of(cache, batch), dtype, k, k_st, k_sh, v, v_st, v_sh, ctx->stream);
}

int fa_kv_write(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* k,
                int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh) {
  int rc = write_check(ctx, cache, batch, dtype, k, k_st, k_sh, v, v_st, v_sh);
  if (rc || (rc = check_host_batch(ctx, "KVWrite", cache, batch, Use::Write)) || (rc = need_ctx(ctx, "KVWrite")) ||
      nothing(batch))
    return rc;
  const int64_t rows = batch->cu_rows[batch->nseq];
  if (rows == 0) return FA_OK;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "KVWrite"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  fa_kv_batch dev;
  void *dk, *dv;
  if ((rc = stage_batch(ctx, batch, &dev))) return rc;
  if ((rc = fa::stage_h2d(ctx, S_K, k, span(rows, cache->kv_heads, k_st, k_sh, cache->head_dim, dtype), &dk))) return rc;
  if ((rc = fa::stage_h2d(ctx, S_V, v, span(rows, cache->kv_heads, v_st, v_sh, cache->head_dim, dtype), &dv))) return rc;
  if ((rc = fa::launch_kv_write(ctx, args_of(cache, &dev), dtype, dk, k_st, k_sh, dv, v_st, v_sh, ctx->stream)))
    return rc;
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

int fa_kv_read_dev(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, void* k, void* v) {
  int rc = read_check(ctx, cache, batch, dtype, k, v);
  if (rc || (rc = need_ctx(ctx, "KVRead")) || nothing(batch)) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  return fa::launch_kv_read(ctx, args_of(cache, batch), dtype, k, v, ctx->stream);
}

int fa_kv_read(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, void* k, void* v) {
  int rc = read_check(ctx, cache, batch, dtype, k, v);
  if (rc || (rc = check_host_batch(ctx, "KVRead", cache, batch, Use::Read)) || (rc = need_ctx(ctx, "KVRead")) ||
      nothing(batch))
    return rc;
  const int64_t rows = batch->cu_rows[batch->nseq];
  if (rows == 0) return FA_OK;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "KVRead"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  fa_kv_batch dev;
  if ((rc = stage_batch(ctx, batch, &dev))) return rc;
  const size_t bytes = (size_t)rows * cache->kv_heads * cache->head_dim * elem(dtype);
  if ((rc = ctx->slot(S_K).ensure(ctx, bytes)) || (rc = ctx->slot(S_V).ensure(ctx, bytes))) return rc;
  void *dk = ctx->slot(S_K).ptr, *dv = ctx->slot(S_V).ptr;
  if ((rc = fa::launch_kv_read(ctx, args_of(cache, &dev), dtype, dk, dv, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipMemcpyAsync(k, dk, bytes, hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipMemcpyAsync(v, dv, bytes, hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

int fa_kv_attention_work(const fa_kv_cache* cache, const fa_kv_batch* batch, int32_t heads, size_t* bytes) {
  if (!bytes) return set_error(nullptr, FA_ERR_ARG, "KVAttention: bytes is NULL");
  *bytes = 0;
  int rc;
  if ((rc = check_cache_sizes(nullptr, "KVAttention", cache))) return rc;
  if (!batch || batch->nseq < 0 || batch->rows < 0 || batch->table_stride < 0 || batch->table_stride > kMaxTable)
    return set_error(nullptr, FA_ERR_ARG, "KVAttention: batch is NULL or has a negative size or too long table rows");
  if (heads < 1 || heads % cache->kv_heads != 0 || heads > 65535)
    return set_error(nullptr, FA_ERR_ARG, "KVAttention: %d query heads on %d key/value heads", heads, cache->kv_heads);
  if ((rc = check_sizes(nullptr, "KVAttention", batch, heads))) return rc;
  fa::KvAttnArgs a = {};
  a.c = args_of(cache, batch);
  a.H = heads;
  if (!nothing(batch)) *bytes = fa::kv_attention_scratch_any(a);
  return FA_OK;
}

int fa_kv_attention_dev(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* q,
                        int64_t q_st, int64_t q_sh, int32_t heads, int causal, int32_t window, float scale, void* out,
                        void* work, size_t work_bytes) {
  fa::KvAttnArgs a;
  int rc = attn_args(ctx, cache, batch, dtype, q, q_st, q_sh, heads, causal, window, scale, out, &a);
  if (rc || (rc = need_ctx(ctx, "KVAttention")) || nothing(batch)) return rc;
  const size_t need = fa::kv_attention_scratch(a);
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  if (work) {
    if (work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15))
      return set_error(ctx, FA_ERR_ARG, "KVAttention: work of %zu bytes, 16-byte aligned, is needed (%zu given)", need,
                       work_bytes);
    if (need && (rc = fa::launch_zero(ctx, work, fa::kKvCountBytes, ctx->stream))) return rc;
  } else if (need) {
    if ((rc = fa::refuse_capture(ctx, ctx->stream, "KVAttention without work"))) return rc;
    if ((rc = own_parts(ctx, need, &work))) return rc;
  }
  return fa::launch_kv_attention(ctx, a, work, ctx->stream);
}

int fa_kv_attention(fa_ctx* ctx, const fa_kv_cache* cache, const fa_kv_batch* batch, int dtype, const void* q,
                    int64_t q_st, int64_t q_sh, int32_t heads, int causal, int32_t window, float scale, void* out) {
  fa::KvAttnArgs a;
  int rc = attn_args(ctx, cache, batch, dtype, q, q_st, q_sh, heads, causal, window, scale, out, &a);
  if (rc || (rc = check_host_batch(ctx, "KVAttention", cache, batch, Use::Attend, window)) ||
      (rc = need_ctx(ctx, "KVAttention")) || nothing(batch))
    return rc;
  const int64_t rows = batch->cu_rows[batch->nseq];
  if (rows == 0) return FA_OK;
  if ((rc = fa::refuse_capture(ctx, ctx->stream, "KVAttention"))) return rc;
  FA_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  fa_kv_batch dev;
  if ((rc = stage_batch(ctx, batch, &dev))) return rc;
  dev.rows = rows;
  void* dq;
  if ((rc = fa::stage_h2d(ctx, S_Q, q, span(rows, heads, q_st, q_sh, cache->head_dim, dtype), &dq))) return rc;
  const size_t bytes = (size_t)rows * heads * cache->head_dim * elem(dtype);
  if ((rc = ctx->slot(S_OUT).ensure(ctx, bytes))) return rc;
  a.c = args_of(cache, &dev);
  a.q = dq;
  a.out = ctx->slot(S_OUT).ptr;
  const size_t need = fa::kv_attention_scratch(a);
  void* work = nullptr;
  if (need && (rc = own_parts(ctx, need, &work))) return rc;
  if ((rc = fa::launch_kv_attention(ctx, a, work, ctx->stream))) return rc;
  FA_HIP_CHECK(ctx, hipMemcpyAsync(out, a.out, bytes, hipMemcpyDeviceToHost, ctx->stream));
  FA_HIP_CHECK(ctx, hipStreamSynchronize(ctx->stream));
  return FA_OK;
}

}  // extern "C"
