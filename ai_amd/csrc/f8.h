// Products with weights held in 8 bits: what their translation units share.
#pragma once

#include "e4m3.h"
#include "fa_internal.h"

namespace fa {

constexpr int kF8Block = FA_F8_BLOCK;  // columns of a scale

inline int64_t f8_kp(int64_t k) { return (k + kF8Block - 1) / kF8Block * kF8Block; }
inline int64_t f8_ks(int64_t k) { return (f8_kp(k) / kF8Block + 3) / 4 * 4; }

// A matrix [n x k] in 8 bits on the device (fa_f8_matrix).
struct F8View {
  uint8_t* codes;   // [n][stride], kp of them used
  uint8_t* scales;  // [n][ks]
  int64_t n, k, stride;
};
// zeros words from `zero` on are set to 0 on the way.
int launch_f8_write(fa_ctx* ctx, const F8View& w, int dtype, const void* x, int64_t ldx, hipStream_t s,
                    uint32_t* zero = nullptr, int zeros = 0);
int launch_f8_read(fa_ctx* ctx, const F8View& w, int dtype, void* out, int64_t ldo, hipStream_t s);

struct F8GemmArgs {
  int64_t m;
  int a_dtype;
  const void* a;
  int64_t lda;
  F8View w;
  fa_epilogue e;  // arrays on the device
  int c_dtype;
  void* c;
  int64_t ldc;
};
// Scratch of a product of m rows: A in 8 bits, sums of a split K.
size_t f8_scratch(int64_t m, int64_t n, int64_t k);
int64_t f8_grid(int64_t m, int64_t n);
int launch_f8_gemm(fa_ctx* ctx, const F8GemmArgs& g, void* work, hipStream_t s);

}  // namespace fa
