// Sampling: what its translation units share.
#pragma once

#include "fa_internal.h"

namespace fa {

struct SampleArgs {
  int64_t rows, vocab;
  int dtype;
  const void* logits;
  int64_t ld;
  fa_sampling s;  // arrays on the device
  const float* u;
  int32_t* ids;
  float* logp;  // may be null
};
size_t sample_scratch(int64_t rows, int64_t vocab);
int64_t sample_grid(int64_t rows, int64_t vocab);  // workgroups of a launch
int launch_sample(fa_ctx* ctx, const SampleArgs& a, void* work, hipStream_t s);

}  // namespace fa
