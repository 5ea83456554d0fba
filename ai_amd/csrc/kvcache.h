// The key/value cache in 8 bits: what its translation units share.
#pragma once

#include "fa_internal.h"

namespace fa {

constexpr int kKvBlock = FA_KV_BLOCK;  // tokens of a block, and of a scale
constexpr int kKvMaxDim = 512;
// Scale exponents. Above: the largest a finite float32 needs. Below: a
// block whose largest magnitude is under 448 * 2^-80 (4e-22) keeps the
// scale 2^-80, so that a scale times a softmax weight stays far from
// float32's subnormals in attention.
constexpr int kKvMinExp = -80, kKvMaxExp = 120;

// Head dims as stored: whole slices of 64.
inline int kv_slices(int head_dim) { return (head_dim + 63) / 64; }

// A batch on the device (fa_kv_batch) with its cache, by value to a kernel.
struct KvArgs {
  uint8_t* codes;   // [blocks][hkv][2][64 * 64 * nc]
  float* scales;    // [blocks][hkv][2]
  int32_t blocks, hkv, nc, D;
  const int32_t* tables;
  int32_t tstride;
  const int32_t* lengths;
  const int32_t* cu;
  int32_t nseq;
  int64_t rows;
};

int launch_kv_write(fa_ctx* ctx, const KvArgs& a, int dtype, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                    int64_t v_st, int64_t v_sh, hipStream_t s);
int64_t kv_grid(const KvArgs& a);  // workgroups of both along a grid's x
int launch_kv_read(fa_ctx* ctx, const KvArgs& a, int dtype, void* k, void* v, hipStream_t s);

struct KvAttnArgs {
  KvArgs c;
  int dtype;
  const void* q;
  int64_t q_st, q_sh;
  int32_t H;
  int32_t causal, window;
  float scale;
  void* out;  // [rows][H][D]
};
// Scratch that a call needs (partial results of a split token axis); 0: none.
// It begins with kKvCountBytes of counters that are zero between calls (the last word is no counter).
constexpr size_t kKvCountBytes = 16384;
size_t kv_attention_scratch(const KvAttnArgs& a);
size_t kv_attention_scratch_any(KvAttnArgs a);  // enough for either type, any window, causal or not
int64_t kv_attention_grid(const KvAttnArgs& a);  // workgroups along a grid's x
int launch_kv_attention(fa_ctx* ctx, const KvAttnArgs& a, void* scratch, hipStream_t s);

#ifdef __HIPCC__
// ---- device side ------------------------------------------------------------

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float kvf4 __attribute__((ext_vector_type(4)));

// Rows and length of sequence b, made safe: whatever the arrays hold, the
// rows are inside [0, rows) and the length is not negative.
struct KvSeq {
  int64_t row0;
  int32_t n;    // new tokens: rows row0 .. row0 + n - 1
  int32_t len;  // tokens of the sequence, the new ones last
};
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int b) {
  KvSeq s;
  const int64_t r0 = a.cu[b], r1 = a.cu[b + 1];
  s.row0 = r0 < 0 ? 0 : r0 > a.rows ? a.rows : r0;
  const int64_t e = r1 < s.row0 ? s.row0 : r1 > a.rows ? a.rows : r1;
  s.n = (int32_t)(e - s.row0);
  const int32_t l = a.lengths[b];
  s.len = l < 0 ? 0 : l;
  return s;
}

// The block of slot p of sequence b, or -1 where the table has none (a slot
// past its row, an entry outside the pool).
__device__ __forceinline__ int kv_block(const KvArgs& a, int b, int64_t slot) {
  if (slot < 0 || slot >= a.tstride) return -1;
  const int id = a.tables[(int64_t)b * a.tstride + slot];
  return id >= 0 && id < a.blocks ? id : -1;
}

__device__ __forceinline__ int64_t kv_part_bytes(const KvArgs& a) { return (int64_t)4096 * a.nc; }
__device__ __forceinline__ uint8_t* kv_part(const KvArgs& a, int block, int h, int part) {
  return a.codes + (((int64_t)block * a.hkv + h) * 2 + part) * kv_part_bytes(a);
}

// The sequence that unit u belongs to: the largest b in [0, nseq) with
// base(cu[b], b) <= u (base does not fall), found by the 64 lanes of a wave
// together, and its rows and length. Up to 64 sequences: one round of loads
// for all of it. Any array contents end the search in range.
struct KvFound {
  int b;
  int32_t cu0;
  KvSeq s;
};
__device__ __forceinline__ int64_t lane64(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ KvSeq lane_seq(const KvSeq& s, int lane) {
  return {lane64(s.row0, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.len, lane)};
}
template <typename F>
__device__ __forceinline__ KvFound kv_find(const KvArgs& a, int64_t u, F base) {
  const int lane = threadIdx.x & 63;
  if (a.nseq <= 64) {
    const int i = min(lane, a.nseq - 1);
    const int32_t c = a.cu[i];
    const KvSeq s = kv_seq(a, i);
    const uint64_t m = __ballot(lane < a.nseq && base(c, lane) <= u);
    const int b = __builtin_amdgcn_readfirstlane(max(1, (int)__popcll(m)) - 1);
    return {b, __builtin_amdgcn_readlane(c, b), lane_seq(s, b)};
  }
  int lo = 0, n = a.nseq;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int off = lane * step;
    const bool at = off < n && base(a.cu[lo + min(off, n - 1)], lo + off) <= u;
    const uint64_t m = __ballot(at);
    const int c = max(1, (int)__popcll(m));
    const int skip = (c - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  return {b, a.cu[b], kv_seq(a, b)};
}
#endif

}  // namespace fa
