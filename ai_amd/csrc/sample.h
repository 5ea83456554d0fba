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
// Whether tokens may be dropped from any row.
inline bool sample_filters(const fa_sampling& s) { return s.top_k || s.top_p || s.min_p; }
size_t sample_scratch(int64_t rows, int64_t vocab, bool filtered);
int64_t sample_grid(int64_t rows, int64_t vocab);  // workgroups of a launch
int launch_sample(fa_ctx* ctx, const SampleArgs& a, void* work, hipStream_t s);

}  // namespace fa
