// The next token of each row of logits: temperature, top-k, top-p and min-p, drawn
// with a given number.
//
// A row's tokens have one order: by logit, falling, then by id. As an unsigned
// number it is the logit's bits, made to rise with the value, over the id's
// complement; every filter keeps the tokens down to some number of that order, so
// that all of them together are one bound, found bit by bit from the top by
// counting (top-k) or weighing (top-p) what lies at or above a candidate. Weights
// and sums are float64: the shares of a vocabulary's tokens go down to 1e-6 and
// less, and sums in float32 would move the bounds by whole tokens.
#include "device_math.h"
#include "sample.h"

namespace fa {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// Rises with the value; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l != l ? -__builtin_inff() : l + 0.f);
  return b ^ ((int32_t)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of_key(uint32_t k) {
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kNone = 0x007FFFFFu;  // key_of(-inf)

// Sum over the workgroup, the same in every thread, in a fixed order.
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int i = 1; i < kWaves; i++) t += red[i];
  return t;
}

// One workgroup draws one row's token.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ double red[kWaves];
  __shared__ long long cnt[kWaves];
  __shared__ double run[kThreads];
  __shared__ int found;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, V = (int)a.vocab;
  const T* l = (const T*)a.logits + row * a.ld;
  const float temp = a.s.temperature ? a.s.temperature[row] : 1.f, u = a.u[row];
  const float top_p = a.s.top_p ? a.s.top_p[row] : 1.f, min_p = a.s.min_p ? a.s.min_p[row] : 0.f;
  const int top_k = a.s.top_k ? a.s.top_k[row] : 0;
  const bool sound = temp >= 0.f && temp < __builtin_inff() && top_p >= 0.f && top_p <= 1.f && min_p >= 0.f &&
                     min_p <= 1.f && u >= 0.f && u < 1.f;
  auto order = [&](int i) { return (uint64_t)key_of(value_of(l[i])) << 32 | (uint32_t)~i; };
  // the first of the order
  uint64_t top = 0;
  for (int i = tid; i < V; i += kThreads) top = max(top, order(i));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint64_t)__shfl_xor((unsigned long long)top, o, 64));
  if ((tid & 63) == 0) cnt[tid >> 6] = (long long)top;
  __syncthreads();
  for (int i = 0; i < kWaves; i++) top = max(top, (uint64_t)cnt[i]);
  const uint32_t top_key = (uint32_t)(top >> 32);
  const int top_id = (int)~(uint32_t)top;
  if (!sound || top_key <= kNone || temp == 0.f) {
    if (tid == 0) {
      const bool none = !sound || top_key <= kNone;
      a.ids[row] = none ? -1 : top_id;
      if (a.logp) a.logp[row] = none ? __builtin_nanf("") : 0.f;
    }
    return;
  }
  const double M = (double)value_of_key(top_key), T_ = (double)temp;
  // exp((l - M) / T); of infinite ones, each 1
  auto weight = [&](uint32_t key) { return key == top_key ? 1.0 : exp(((double)value_of_key(key) - M) / T_); };
  uint64_t bound = 0;  // tokens at or above it in the order stay
  if (top_k > 0 && top_k < V) {
    for (int bit = 63; bit >= 0; bit--) {
      const uint64_t c = bound | 1ull << bit;
      long long n = 0;
      for (int i = tid; i < V; i += kThreads) n += order(i) >= c;
      if (block_sum(n, cnt) >= top_k) bound = c;
    }
  }
  if (top_p < 1.f) {
    auto mass = [&](uint64_t c) {
      double m = 0;
      for (int i = tid; i < V; i += kThreads) {
        const uint64_t o = order(i);
        if (o >= c) m += weight((uint32_t)(o >> 32));
      }
      return block_sum(m, red);
    };
    const double want = (double)top_p * mass(bound);
    uint64_t b = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const uint64_t c = b | 1ull << bit;
      if (c <= bound || (c <= top && mass(c) >= want)) b = c;
    }
    bound = max(bound, min(b, top));
  }
  // the draw: each thread weighs a run of ids, the one whose run passes the aim walks it
  const int per = (V + kThreads - 1) / kThreads, i0 = min(V, tid * per), i1 = min(V, i0 + per);
  auto share = [&](int i) {
    const uint64_t o = order(i);
    if (o < bound) return 0.0;
    const double w = weight((uint32_t)(o >> 32));
    return w >= (double)min_p ? w : 0.0;
  };
  double mine = 0;
  for (int i = i0; i < i1; i++) mine += share(i);
  run[tid] = mine;
  if (tid == 0) found = kThreads;
  __syncthreads();
  double before = 0, total = 0;
  for (int t = 0; t < kThreads; t++) {
    if (t == tid) before = total;
    total += run[t];
  }
  const double aim = (double)u * total;
  if (mine > 0 && before + mine > aim) atomicMin(&found, tid);
  __syncthreads();
  int who = found;
  if (who == kThreads) {  // (rounding: the last run of any weight)
    for (int t = 0; t < kThreads; t++)
      if (run[t] > 0) who = t;
  }
  if (tid == who) {
    double at = before;
    int id = -1;
    double w_id = 0;
    for (int i = i0; i < i1; i++) {
      const double w = share(i);
      if (w > 0) {
        id = i;
        w_id = w;
        at += w;
        if (at > aim) break;
      }
    }
    a.ids[row] = id;
    if (a.logp) a.logp[row] = (float)log(w_id / total);
  }
}

}  // namespace

size_t sample_scratch(int64_t rows, int64_t vocab) { return 0; }

int launch_sample(fa_ctx* ctx, const SampleArgs& a, void* work, hipStream_t s) {
  if (a.dtype == FA_DT_F32) sample_kernel<float><<<(unsigned)a.rows, kThreads, 0, s>>>(a);
  else sample_kernel<uint16_t><<<(unsigned)a.rows, kThreads, 0, s>>>(a);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

}  // namespace fa
