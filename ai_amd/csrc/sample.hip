// The next token of each row of logits: temperature, top-k, top-p and min-p, drawn
// with a given number.
//
// A row's tokens have one order: by logit, falling, then by id. As an unsigned
// number (larger first) it is the logit's bits, made to rise with the value, over
// the id's complement. top-k and top-p keep the tokens down to some number of that
// order, min-p those down to some weight, so that what stays is a run of the order
// from its start. Weights and sums are float64 or exact integers: the shares of a
// vocabulary's tokens go down to 1e-6 and less, and sums in float32 would move the
// bounds by whole tokens. Integer sums do not depend on the order in which
// atomics arrive, so a call's results are the same every time.
//
// The logits are read once, by workgroups that each hold a slice of a row in
// registers; a second, partial reading finds the few tokens near the bounds:
//   scan    a slice's first token of the order, and the weight of all of it, or
//           (where a filter is set) a histogram of counts and weights by l / T in
//           steps of 1/32, further down of 1, on grids that all slices share.
//   join    adds up a row's histograms, which gives the steps in which its bounds lie.
//   gather  slices that have tokens there list them.
//   finish  finds the bounds among the listed tokens, weighs what stays of every
//           slice, takes the slice that the number falls into and walks it.
#include <algorithm>

#include "device_math.h"
#include "sample.h"

namespace fa {
namespace {

constexpr int kScan = 512;     // threads of scan and gather
constexpr int kFinish = 512;   // of finish
constexpr int kFine = 768;     // bins of one step of 1/32: weights down to e^-24
constexpr int kBins = 1024;    // and bins of 32 steps below: down to e^-280, the last holds the rest
constexpr int kMaxSlices = 1024;
constexpr int kSub = 2048;     // bins of a selection's pass
constexpr int kCached = 8192;  // listed tokens that finish keeps in LDS

// ---- a row's layout in the scratch ------------------------------------------------

struct Slice {
  uint64_t top;   // its first token of the order
  double mass;    // the weight of all of it, relative to the first token
  int32_t bins;   // bins in use
};

// Bins in which a row's bounds may lie. Tokens in listed bins are looked at one by one.
struct Cut {
  float most;         // the row's largest logit
  int k_bin;          // the bin of the top_k-th token (kBins: no limit)
  int k_rank;         // its rank there, from 1
  int p_lo, p_hi;     // bins of top_p's bound (kBins: none)
  int m_lo, m_hi;     // of min_p's
  double step;        // the grid's step of most
  double above_k, above_p;  // weights of the bins before k_bin, before p_lo
  double all;         // of all bins
  __device__ __forceinline__ bool listed(int b) const {
    return b == k_bin || (b >= p_lo && b <= p_hi) || (b >= m_lo && b <= m_hi);
  }
};

struct Plan {
  int per, slices;  // tokens of a slice (a power of two), slices of a row
  int room;         // tokens that a slice may list: all of its own
  int vec;          // rows aligned for 16-byte loads
  Slice* slice;     // [rows][slices]
  Cut* cut;         // [rows]
  double* mass;     // [rows][slices][kBins] weights of the bins up to each, relative to the slice's first token
  uint32_t* count;  // likewise tokens (without top-k: bins with tokens)
  uint32_t* listed; // [rows][slices]
  uint16_t* list;   // [rows][slices * room]
};

// ---- order, weights, bins --------------------------------------------------------------

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
__device__ __forceinline__ uint64_t order_of(float l, int id) { return (uint64_t)key_of(l) << 32 | (uint32_t)~id; }
__device__ __forceinline__ int id_of(uint64_t o) { return (int)~(uint32_t)o; }
__device__ __forceinline__ float logit_of(uint64_t o) { return value_of_key((uint32_t)(o >> 32)); }

// 2^scale e^x, x <= 0: x = n ln 2 + r, |r| <= 0.347, ln 2 in two parts, e^r by its
// series to r^13 (the next term is 4e-18).
__device__ __forceinline__ double exp_scaled(double x, int scale) {
  const double y = fmax(x, -800.0), n = rint(y * 1.4426950408889634);
  double r = fma(-n, 0.6931471805599453, y);
  r = fma(-n, 2.3190468138462996e-17, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n + scale);
}

// A row's settings.
struct Row {
  float temp, top_p, min_p, u;
  int top_k;
  bool sound, greedy, cut;  // cut: a filter may drop tokens
  double inv;               // 1 / T
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
  Row r;
  r.temp = a.s.temperature ? a.s.temperature[row] : 1.f;
  r.top_p = a.s.top_p ? a.s.top_p[row] : 1.f;
  r.min_p = a.s.min_p ? a.s.min_p[row] : 0.f;
  r.top_k = a.s.top_k ? a.s.top_k[row] : 0;
  r.u = a.u[row];
  r.sound = r.temp >= 0.f && r.temp < __builtin_inff() && r.top_p >= 0.f && r.top_p <= 1.f && r.min_p >= 0.f &&
            r.min_p <= 1.f && r.u >= 0.f && r.u < 1.f;
  r.greedy = r.temp == 0.f;
  if (r.top_k <= 0 || r.top_k > a.vocab) r.top_k = (int)a.vocab;
  r.cut = r.top_k < a.vocab || r.top_p < 1.f || r.min_p > 0.f;
  r.inv = 1.0 / (double)r.temp;
  return r;
}

// Weight of l beside the largest logit, times 2^scale; of infinite ones, each 1.
__device__ __forceinline__ double weight(float l, float most, double inv, int scale = 0) {
  return l == most ? ldexp(1.0, scale) : exp_scaled(((double)l - (double)most) * inv, scale);
}

// The grid: t = 32 l / T, its steps whole numbers; 32 of them make a wide step.
// Where the largest logit is infinite, only infinite ones count, at 0.
__device__ __forceinline__ double grid_of(float l, double inv) { return l == __builtin_inff() ? 0.0 : (double)l * (32.0 * inv); }
__device__ __forceinline__ bool counts(float l, float most) {
  return most == __builtin_inff() ? l == most : l > -__builtin_inff();
}
// The bin of step `at` below the top step: by steps up to kFine of them, then by wide ones.
__device__ __forceinline__ int bin_of_step(double at, double top) {
  const double down = top - at;
  if (down < (double)kFine) return (int)down;
  const double wide = floor(top * 0.03125) - floor(at * 0.03125);  // at least kFine / 32
  return (int)fmin(wide + (double)(kFine - kFine / 32), (double)(kBins - 1));
}
// The lowest step of bin b of those counted from `top`.
__device__ __forceinline__ double last_step(int b, double top) {
  return b < kFine ? top - (double)b : (floor(top * 0.03125) - (double)(b - (kFine - kFine / 32))) * 32.0;
}
__device__ __forceinline__ int bin_of(float l, double inv, double top) { return bin_of_step(floor(grid_of(l, inv)), top); }
// From here on unequal logits are 2^16 steps and more apart, and t is taken as it is.
constexpr double kFar = 0x1p40;
// Weight in the middle of bin b of steps counted from `top`, beside the logit l. The
// distance takes l's place on the grid unrounded: 2^39 steps from zero its rounding is 2e-6
// of the weight.
__device__ __forceinline__ double middle(int b, double top, float l, double inv) {
  const double t = grid_of(l, inv);
  if (!(fabs(t) < kFar)) return b == 0 && top == floor(t) ? 1.0 : 0.0;
  double at = top - (double)b + 0.5;
  if (b >= kFine) at = (floor(top * 0.03125) - (double)(b - (kFine - kFine / 32))) * 32.0 + 16.0;
  return exp_scaled(fma(l == __builtin_inff() ? 0.0 : -(double)l, 32.0 * inv, at) * 0.03125, 0);
}
// Weights in bin b are below 2^-bin_exp(b): (b - 1) / 32 below the first, or a wide step less than wide steps.
__device__ __forceinline__ int bin_exp(int b) {
  if (b < kFine) return b > 1 ? (int)((float)(b - 1) * 0.04508f) : 0;
  return (int)((float)(b - (kFine - kFine / 32) - 1) * 1.4426f);
}
// A number below 2^51 as an integer, to nearest.
__device__ __forceinline__ uint64_t to_int(double x) {
  return (uint64_t)__double_as_longlong(x + 0x1p52) - (uint64_t)0x4330000000000000ull;
}
constexpr int kUnit = 48;  // a bin's weights are held in units of 2^-48 of its middle: 2^14 of them fit
// Sums are right to 1e-13: weights to 2^-48, a thousand additions (of more than 2^19 listed
// tokens to 2^-37, but for weights of 1, which are whole numbers). Two that the definition
// has equal (of equal logits, whose weights are 1) may differ by that much either way, so
// a sum reaches a bound from this much below it on, and exceeds it from this much above.
constexpr double kNear = 1e-12;

// ---- a workgroup's sums and scans, in a fixed order -----------------------------------------

template <int NT, typename V, typename F>
__device__ __forceinline__ V block_join(V v, V* red, F join) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; i++) t = join(t, red[i]);
  return t;
}
struct Add {
  template <typename V>
  __device__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  template <typename V>
  __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct Min {
  template <typename V>
  __device__ V operator()(V a, V b) const { return a < b ? a : b; }
};
// The sum of the threads before this one; *total: of all.
template <int NT, typename V>
__device__ __forceinline__ V block_scan(V v, V* red, V* total) {
  V x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(x, o, 64);
    if ((int)(threadIdx.x & 63) >= o) x = x + y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = x;
  __syncthreads();
  V before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    if (i == (int)(threadIdx.x >> 6)) before = all;
    all = all + red[i];
  }
  *total = all;
  const V mine = __shfl_up(x, 1, 64);
  return (threadIdx.x & 63) ? before + mine : before;
}

// ---- a slice in registers ------------------------------------------------------------------------

// Thread t holds, 16 bytes at a time, W neighbouring tokens from (i * kScan + t) * W.
template <typename T, int E>
struct Held {
  static constexpr int W = 16 / sizeof(T);
  float v[E];
  static __device__ __forceinline__ int at(int e) { return ((e / W) * kScan + (int)threadIdx.x) * W + e % W; }
  // n: tokens of the slice; those past it are -inf
  __device__ __forceinline__ void load(const T* l, int n, bool vec) {
#pragma unroll
    for (int e = 0; e < E; e += W) {
      const int i = at(e);
      if (vec && i + W <= n) {
        const uint4 x = *reinterpret_cast<const uint4*>(l + i);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < W; j++)
          v[e + j] = W == 4 ? __uint_as_float(w[j & 3])
                            : __uint_as_float(j & 1 ? w[(j >> 1) & 3] & 0xFFFF0000u : w[(j >> 1) & 3] << 16);
      } else {
#pragma unroll
        for (int j = 0; j < W; j++) v[e + j] = i + j < n ? value_of(l[i + j]) : -__builtin_inff();
      }
    }
  }
};

// Bound by its arithmetic where rows are many: an exponential in float64 and two
// additions in LDS a token (256 rows of 262144 in float32 124 us, 2.2 TB/s, where the
// bytes take 53; without filters nothing is added in LDS). One such row: 9 us, latencies.
template <typename T, int E>
__global__ __launch_bounds__(kScan) void scan_kernel(SampleArgs a, Plan p) {
  __shared__ uint64_t red[kScan / 64];
  __shared__ double redd[kScan / 64];
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  const int64_t row = blockIdx.x / p.slices;
  const int s = (int)(blockIdx.x - row * p.slices), first = s * p.per, tid = threadIdx.x;
  const Row r = row_of(a, row);
  Slice* out = p.slice + row * p.slices + s;
  if (!r.sound) return;
  Held<T, E> h;
  h.load((const T*)a.logits + row * a.ld + first, min(p.per, (int)a.vocab - first), p.vec);
#pragma unroll
  for (int i = 0; i < kBins / kScan; i++) mass[i * kScan + tid] = 0, count[i * kScan + tid] = 0;
  float most = -__builtin_inff();
#pragma unroll
  for (int e = 0; e < E; e++) most = fmaxf(most, h.v[e]);
  most = block_join<kScan>(most, (float*)red, Max());
  if (most == -__builtin_inff()) {
    if (tid == 0) *out = {0, 0.0, 0};
    return;
  }
  int id = 0x7FFFFFFF;  // the lowest of those equal to it
#pragma unroll
  for (int e = 0; e < E; e++)
    if (h.v[e] == most) id = min(id, first + Held<T, E>::at(e));
  const uint64_t top = order_of(most, block_join<kScan>(id, (int*)redd, Min()));
  if (r.greedy) {
    if (tid == 0) *out = {top, 0.0, 0};
    return;
  }
  if (!r.cut) {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++)
      if (counts(h.v[e], most)) sum += weight(h.v[e], most, r.inv);
    sum = block_join<kScan>(sum, redd, Add());
    if (tid == 0) *out = {top, sum, 0};
    return;
  }
  const double c = 32.0 * r.inv, step = floor(grid_of(most, r.inv)), near = fabs(step) < kFar ? 1.0 : 0.0;
  const bool counted = r.top_k < a.vocab;
#pragma unroll
  for (int e = 0; e < E; e++) {
#pragma clang fp contract(off)  // (t - floor(t) is exact, and the rounding of t is added by itself)
    const float v = h.v[e];
    if (!counts(v, most)) continue;
    const double t = grid_of(v, r.inv), whole = floor(t), down = step - whole;
    int b;
    uint64_t w;
    if (down < (double)kFine) {
      b = (int)down;
      const double rest = v == __builtin_inff() ? 0.0 : fma((double)v, c, -t);
      // 2^48 e^d to d^6, |d| <= 1/64: the next term is 5e-17
      const double d = near != 0 ? ((t - whole) - 0.5 + rest) * 0.03125 : 0.0;
      double x = 1.0 / 720.0;
      x = fma(x, d, 1.0 / 120.0);
      x = fma(x, d, 1.0 / 24.0);
      x = fma(x, d, 1.0 / 6.0);
      x = fma(x, d, 0.5);
      x = fma(x, d, 1.0);
      x = fma(x, d, 1.0);
      w = to_int(x * 0x1p48);
    } else {
      // 4e-11 of the slice's first weight and less: seven digits of them are enough
      b = bin_of_step(whole, step);
      const float d = (float)(t * 0.03125 - floor(t * 0.03125)) - 0.5f;
      w = b == kBins - 1 ? 0 : to_int((double)__builtin_amdgcn_exp2f(d * 1.4426950408889634f) * 0x1p48);
    }
    atomicAdd((unsigned long long*)&mass[b], (unsigned long long)w);
    if (counted) atomicAdd(&count[b], 1u);
  }
  __syncthreads();
  // running sums over the bins (two neighbours a thread); without top-k, whether there are tokens in a bin is all that is asked
  static_assert(kBins == 2 * kScan, "two bins a thread");
  uint64_t w[2];
  double m[2];
  uint32_t n[2];
  int last = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int b = 2 * tid + i;
    w[i] = mass[b];
    n[i] = counted ? count[b] : w[i] != 0;
    m[i] = w[i] ? ldexp((double)w[i], -kUnit) * middle(b, step, most, r.inv) : 0.0;
    if (n[i]) last = b + 1;
  }
  last = block_join<kScan>(last, (int*)red, Max());
  double all_m;
  uint32_t all_n;
  const double m0 = block_scan<kScan>(m[0] + m[1], redd, &all_m);
  const uint32_t n0 = block_scan<kScan>(n[0] + n[1], (uint32_t*)red, &all_n);
  const int64_t at = (row * p.slices + s) * kBins + 2 * tid;
  if (2 * tid < last) {
    *reinterpret_cast<double2*>(p.mass + at) = make_double2(m0 + m[0], m0 + m[0] + m[1]);
    *reinterpret_cast<uint2*>(p.count + at) = make_uint2(n0 + n[0], n0 + n[0] + n[1]);
  }
  if (tid == 0) *out = {top, all_m, last};
}

// ---- a row's histograms joined ----------------------------------------------------------------------

// The row's bin of a slice's bin b: the slice's steps are counted from `own`, the row's from `top`.
__device__ __forceinline__ int row_bin(int b, double own, double top) {
  if (b < kFine) return bin_of_step(own - (double)b, top);
  const double wide = floor(top * 0.03125) - floor(own * 0.03125);
  return (int)fmin((double)b + wide, (double)(kBins - 1));
}
template <int NT>
__device__ __forceinline__ uint64_t row_top(const Plan& p, int64_t row, uint64_t* red) {
  uint64_t top = 0;
  for (int s = threadIdx.x; s < p.slices; s += NT) top = max(top, p.slice[row * p.slices + s].top);
  return block_join<NT>(top, red, Max());
}

// One workgroup a row, a thread a bin: what the slices have down to the last step of
// each. Slices are taken kChunk at a time, their heads first, and the sums of kAtOnce
// slices are under way at once. A chain of loads and scans in one workgroup: 10 us for 8
// slices, 12 for 32, 15 for 256 rows of 32.
constexpr int kChunk = 64, kAtOnce = 16;
__global__ __launch_bounds__(kBins) void join_kernel(SampleArgs a, Plan p) {
  constexpr int NT = kBins;
  __shared__ double sums[kBins], scale[kChunk];
  __shared__ uint64_t red[NT / 64], counts_to[kBins];
  __shared__ int found[4], bins[kChunk], below[kChunk], wide_below[kChunk];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const Row r = row_of(a, row);
  if (!r.sound || r.greedy || !r.cut) return;
  const Slice* slice = p.slice + row * p.slices;
  const float most = logit_of(row_top<NT>(p, row, red));
  if (!(most > -__builtin_inff())) return;
  Cut c;
  c.most = most;
  c.step = floor(grid_of(most, r.inv));
  c.k_bin = c.p_lo = c.m_lo = kBins;
  c.p_hi = c.m_hi = -1;
  c.k_rank = 0;
  c.above_k = c.above_p = 0;
  const int down = (int)fmin(c.step - last_step(tid, c.step), 0x1p24);  // steps to the last of this bin
  double m = 0;
  uint64_t n = 0;
  for (int s0 = 0; s0 < p.slices; s0 += kChunk) {
    __syncthreads();
    if (tid < kChunk) {
      bins[tid] = below[tid] = wide_below[tid] = 0;
      scale[tid] = 0;
      if (s0 + tid < p.slices) {
        const Slice x = slice[s0 + tid];
        const float l = logit_of(x.top);
        if (x.bins && counts(l, most)) {
          // the slice's first step below the row's, in steps and in wide ones
          const double own = floor(grid_of(l, r.inv));
          below[tid] = (int)fmin(c.step - own, 0x1p25);
          wide_below[tid] = (int)fmin(floor(c.step * 0.03125) - floor(own * 0.03125), 0x1p20);
          scale[tid] = weight(l, most, r.inv);
          bins[tid] = x.bins;
        }
      }
    }
    __syncthreads();
    const int64_t at = (row * p.slices + s0) * kBins;
    const int many = min(kChunk, p.slices - s0);
    for (int s = 0; s < many; s += kAtOnce) {
      double mass[kAtOnce];
      uint32_t count[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) {
        const int q = min(s + i, kChunk - 1), d = down - below[q];  // (of slices past the last: no bins)
        int j = d < kFine ? d : tid - wide_below[q];
        if (tid == kBins - 1) j = kBins - 1;
        const bool in = bins[q] > 0 && j >= 0;
        const int64_t from = at + min(s + i, many - 1) * kBins + (in ? min(j, bins[q] - 1) : 0);
        mass[i] = p.mass[from];
        count[i] = p.count[from];
        if (!in) mass[i] = 0, count[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) m = fma(mass[i], scale[min(s + i, kChunk - 1)], m), n += count[i];
    }
  }
  sums[tid] = m;
  counts_to[tid] = n;
  if (tid < 4) found[tid] = tid == 1 ? 0 : kBins;
  __syncthreads();
  const double before = tid ? sums[tid - 1] : 0.0;
  const uint64_t n_before = tid ? counts_to[tid - 1] : 0, tokens = counts_to[kBins - 1];
  c.all = sums[kBins - 1];
  // top-k: the bin of the top_k-th token, if there are more
  const uint64_t k = (uint64_t)r.top_k;
  if (k < (uint64_t)a.vocab && n_before < k && n >= k && tokens > k) {
    found[0] = tid;
    found[1] = (int)(k - n_before);
  }
  __syncthreads();
  c.k_bin = found[0];
  c.k_rank = found[1];
  double k_least = c.all, k_most = c.all;  // weight of the top_k tokens
  if (c.k_bin < kBins) {
    c.above_k = k_least = c.k_bin ? sums[c.k_bin - 1] : 0.0;
    k_most = sums[c.k_bin];
  }
  // top-p: the aim is taken kNear lower from other sums, a margin of that keeps to either side
  if (r.top_p < 1.f) {
    const double least = (double)r.top_p * k_least * (1 - 2 * kNear), want = (double)r.top_p * k_most * (1 + kNear);
    if (before < least && m >= least) atomicMin(&found[2], tid);
    if (before < want && m >= want) atomicMin(&found[3], tid);
    __syncthreads();
    const int end = min(c.k_bin, kBins - 1);
    c.p_lo = least > 0 ? min(found[2], end) : 0;
    c.p_hi = want > 0 ? min(found[3], end) : 0;
    c.above_p = c.p_lo ? sums[c.p_lo - 1] : 0.0;
  }
  // min-p: l >= most + T ln(min_p), in the step of that bound or the next
  if (r.min_p > 0.f) {
    const double down = most == __builtin_inff() ? 0.0 : -32.0 * log((double)r.min_p);
    c.m_lo = max(0, bin_of_step(c.step - floor(down), c.step) - 1);
    c.m_hi = bin_of_step(c.step - floor(down) - 2.0, c.step) + 1;
  }
  if (tid == 0) p.cut[row] = c;
}

// Slices without such tokens are left after their head. 256 rows of 262144 in float32 66 us,
// 4.1 TB/s; one 7.
template <typename T, int E>
__global__ __launch_bounds__(kScan) void gather_kernel(SampleArgs a, Plan p) {
  __shared__ uint32_t n_listed;
  const int64_t row = blockIdx.x / p.slices;
  const int s = (int)(blockIdx.x - row * p.slices), first = s * p.per, tid = threadIdx.x;
  const Row r = row_of(a, row);
  const Slice x = p.slice[row * p.slices + s];  // (of a row without histograms: not used)
  if (!r.sound || r.greedy || !r.cut) return;
  if (x.bins == 0) {
    if (tid == 0) p.listed[row * p.slices + s] = 0;
    return;
  }
  const Cut c = p.cut[row];
  const float most = c.most;
  const float own = logit_of(x.top);
  const double step = floor(grid_of(own, r.inv));
  const int64_t at = (row * p.slices + s) * kBins;
  // does the slice have tokens in listed bins?
  bool any = false;
  if (counts(own, most))
    for (int b = tid; b < x.bins; b += kScan)
      if (c.listed(row_bin(b, step, c.step))) any |= p.count[at + b] != (b ? p.count[at + b - 1] : 0);
  if (tid == 0) n_listed = 0;
  if (__syncthreads_or(any)) {
    Held<T, E> h;
    h.load((const T*)a.logits + row * a.ld + first, min(p.per, (int)a.vocab - first), p.vec);
    uint16_t* list = p.list + (row * p.slices + s) * p.room;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const bool in = counts(h.v[e], most) && c.listed(bin_of(h.v[e], r.inv, c.step));
      const uint64_t mask = __ballot(in);
      if (mask == 0) continue;  // (uniform in the wave)
      uint32_t base = 0;
      if ((tid & 63) == 0) base = atomicAdd(&n_listed, (uint32_t)__popcll(mask));
      base = __builtin_amdgcn_readfirstlane(base);
      if (in) list[base + __popcll(mask & ((1ull << (tid & 63)) - 1))] = (uint16_t)Held<T, E>::at(e);
    }
    __syncthreads();
  }
  if (tid == 0) p.listed[row * p.slices + s] = n_listed;
}

// ---- finish -----------------------------------------------------------------------------------------

struct FinishMem {
  double redd[kFinish / 64];
  uint64_t red[kFinish / 64];
  uint64_t token[kCached];         // the row's listed tokens, if they fit
  uint64_t sub_mass[kSub];
  uint32_t sub_count[kSub];
  uint32_t start[kMaxSlices + 1];  // of a slice's listed tokens among the row's
  uint64_t part[kMaxSlices];       // weight of the listed tokens of each slice that stay
  int found;
  double found_before;
  uint64_t one, pass[3];
};

constexpr int kAhead = 4;
// The listed tokens of a row, each given to f as its number in the order.
template <typename T, typename F>
__device__ __forceinline__ void each_in_memory(const SampleArgs& a, const Plan& p, int64_t row, const FinishMem& mem, F f) {
  const T* l = (const T*)a.logits + row * a.ld;
  for (int s = threadIdx.x >> 6; s < p.slices; s += kFinish / 64) {
    const uint32_t from = mem.start[s], m = mem.start[s + 1] - from;
    const uint16_t* list = p.list + (row * p.slices + s) * p.room;
    for (uint32_t i = threadIdx.x & 63; i < m; i += 64 * kAhead) {  // several under way at once
      int id[kAhead];
      T v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; j++) id[j] = s * p.per + list[min(i + 64 * j, m - 1)];
#pragma unroll
      for (int j = 0; j < kAhead; j++) v[j] = l[id[j]];
#pragma unroll
      for (int j = 0; j < kAhead; j++)
        if (i + 64 * j < m) f(order_of(value_of(v[j]), id[j]), from + i + 64 * j);
    }
  }
}
template <typename T, typename F>
__device__ __forceinline__ void each_listed(const SampleArgs& a, const Plan& p, int64_t row, const FinishMem& mem,
                                            uint32_t n, F f) {
  if (n > kCached) {
    each_in_memory<T>(a, p, row, mem, [&](uint64_t o, uint32_t) { f(o); });
    return;
  }
  for (uint32_t i = threadIdx.x; i < n; i += kFinish) f(mem.token[i]);
}

// Of the listed tokens from hi down to lo, the one down to which there are `rank`
// (by count), or down to which weights and `above` make `want`. Weights count in
// units of 2^-unit. The last of them if there are not so many.
template <typename T, bool MASS>
__device__ uint64_t select_token(const SampleArgs& a, const Plan& p, int64_t row, FinishMem& mem, uint32_t n, uint64_t lo,
                                 uint64_t hi, float most, double inv, int unit, uint64_t rank, double above, double want) {
  constexpr int W = kSub / kFinish;  // bins of a thread
  const int tid = threadIdx.x;
  uint64_t before = 0, count_before = 0;  // integer weight and tokens above hi
  want = fmax(want * (1 - kNear), above + ldexp(1.0, -unit));  // (top_p = 0: the first token all the same)
  while (lo < hi) {
    const int shift = max(0, 64 - (int)__builtin_clzll(hi - lo) - 11);
    for (int i = tid; i < kSub; i += kFinish) {
      mem.sub_count[i] = 0;
      if (MASS) mem.sub_mass[i] = 0;
    }
    if (tid == 0) mem.found = -1;
    __syncthreads();
    each_listed<T>(a, p, row, mem, n, [&](uint64_t o) {
      if (o < lo || o > hi) return;
      const int i = (int)((hi - o) >> shift);
      atomicAdd(&mem.sub_count[i], 1u);
      if (MASS) atomicAdd((unsigned long long*)&mem.sub_mass[i], to_int(weight(logit_of(o), most, inv, unit)));
    });
    __syncthreads();
    uint64_t c[W], w[W], cs = 0, ws = 0, all;
#pragma unroll
    for (int i = 0; i < W; i++) {
      c[i] = mem.sub_count[W * tid + i];
      w[i] = MASS ? mem.sub_mass[W * tid + i] : 0;
      cs += c[i];
      ws += w[i];
    }
    uint64_t cb = block_scan<kFinish>(cs, mem.red, &all);
    uint64_t wb = MASS ? block_scan<kFinish>(ws, mem.red, &all) : 0;
    auto reached = [&](uint64_t count, uint64_t mass) {
      return MASS ? above + ldexp((double)(before + mass), -unit) >= want : count_before + count >= rank;
    };
    const int last_used = block_join<kFinish>(cs ? tid : -1, (int*)mem.redd, Max());
    // the one thread before whose tokens the aim is not reached and with them is, or the last of any
    const bool open = !reached(cb, wb) || count_before + cb == 0;
    if (cs && open && (reached(cb + cs, wb + ws) || tid == last_used)) {
      int pick = -1;
#pragma unroll
      for (int i = 0; i < W; i++) {
        if (pick >= 0 || c[i] == 0) continue;
        bool more = false;  // tokens of this thread after bin i
#pragma unroll
        for (int j = 0; j < W; j++) more |= j > i && c[j] != 0;
        if (reached(cb + c[i], wb + w[i]) || !more) {
          pick = W * tid + i;
          mem.found = pick;
          mem.pass[0] = cb;
          mem.pass[1] = wb;
          mem.pass[2] = c[i];
        }
        cb += c[i];
        wb += w[i];
      }
    }
    __syncthreads();
    const int pick = mem.found;
    count_before += mem.pass[0];
    before += mem.pass[1];
    const bool single = mem.pass[2] == 1;
    hi -= (uint64_t)pick << shift;
    const uint64_t width = 1ull << shift;
    if (hi - lo >= width) lo = hi - width + 1;
    if (single && lo < hi) {
      each_listed<T>(a, p, row, mem, n, [&](uint64_t o) {
        if (o >= lo && o <= hi) mem.one = o;
      });
      __syncthreads();
      hi = lo = mem.one;
    }
    __syncthreads();
  }
  return hi;
}

// One workgroup a row, bound by its own chain: two selections, each of passes over the
// listed tokens, the slices' weights, the walk. One row of 262144 22 us, 64 of 32000 31, 256
// of 262144 92 (rows of more than kCached listed tokens read them from memory in every
// pass, and the slowest row is the launch's time); 37 of 49999 without filters 12.
template <typename T, int E>
__global__ __launch_bounds__(kFinish) void finish_kernel(SampleArgs a, Plan p) {
  __shared__ FinishMem mem;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const Row r = row_of(a, row);
  uint64_t top = 0;
  if (r.sound) top = row_top<kFinish>(p, row, mem.red);
  const float most = logit_of(top);
  const bool none = !r.sound || !(most > -__builtin_inff());
  if (none || r.greedy) {
    if (tid == 0) {
      a.ids[row] = none ? -1 : id_of(top);
      if (a.logp) a.logp[row] = none ? __builtin_nanf("") : 0.f;
    }
    return;
  }
  const Slice* slice = p.slice + row * p.slices;
  const T* l = (const T*)a.logits + row * a.ld;
  uint64_t bound = 0;  // tokens at or above it stay (but for min_p)
  int whole = kBins;   // bins before it stay whole, listed tokens of the others are asked
  int unit = 0;        // mem.part counts 2^-unit
  double step = 0;
  if (r.cut) {
    const Cut c = p.cut[row];
    step = c.step;
    // where each slice's listed tokens go
    uint32_t n = 0;
    for (int s0 = 0; s0 < p.slices; s0 += kFinish) {
      const int s = s0 + tid;
      const uint32_t mine = s < p.slices ? p.listed[row * p.slices + s] : 0;
      uint32_t all;
      const uint32_t start = block_scan<kFinish>(mine, (uint32_t*)mem.red, &all);
      if (s < p.slices) mem.start[s] = n + start, mem.part[s] = 0;
      n += all;
    }
    if (tid == 0) mem.start[p.slices] = n;
    __syncthreads();
    auto bin = [&](uint64_t o) { return bin_of(logit_of(o), r.inv, step); };
    uint64_t k_hi = 0, k_lo = ~0ull, p_hi = 0, p_lo = ~0ull;
    each_in_memory<T>(a, p, row, mem, [&](uint64_t o, uint32_t i) {
      if (n <= kCached) mem.token[i] = o;
      const int b = bin(o);
      if (b == c.k_bin) k_hi = max(k_hi, o), k_lo = min(k_lo, o);
      if (b >= c.p_lo && b <= c.p_hi) p_hi = max(p_hi, o), p_lo = min(p_lo, o);
    });
    __syncthreads();
    // integer weights: n of them, each below 2^bits, stay below 2^62
    const int bits = min(49, 61 - (32 - __builtin_clz(n | 1)));
    double k_mass = c.all;
    if (c.k_bin < kBins) {
      k_hi = block_join<kFinish>(k_hi, mem.red, Max());
      k_lo = block_join<kFinish>(k_lo, mem.red, Min());
      bound = select_token<T, false>(a, p, row, mem, n, k_lo, k_hi, most, r.inv, 0, (uint64_t)c.k_rank, 0, 0);
      whole = c.k_bin;
      if (r.top_p < 1.f) {
        uint64_t sum = 0;
        const int u = bits + bin_exp(c.k_bin);
        each_listed<T>(a, p, row, mem, n, [&](uint64_t o) {
          if (o >= bound && o <= k_hi) sum += to_int(weight(logit_of(o), most, r.inv, u));
        });
        sum = block_join<kFinish>(sum, mem.red, Add());
        k_mass = c.above_k + ldexp((double)sum, -u);
      }
    }
    if (r.top_p < 1.f) {
      p_hi = block_join<kFinish>(p_hi, mem.red, Max());
      p_lo = max(bound, block_join<kFinish>(p_lo, mem.red, Min()));
      if (p_lo <= p_hi) {
        bound = select_token<T, true>(a, p, row, mem, n, p_lo, p_hi, most, r.inv, bits + bin_exp(c.p_lo), 0, c.above_p,
                                      (double)r.top_p * k_mass);
        whole = min(whole, bin(bound));
      }
    }
    whole = min(whole, c.m_lo);
    unit = bits + bin_exp(whole);
    auto stays = [&](uint64_t o) -> uint64_t {
      if (o < bound || bin(o) < whole) return 0;
      const double w = weight(logit_of(o), most, r.inv);
      return w >= (double)r.min_p ? to_int(ldexp(w, unit)) : 0;
    };
    if (n <= kCached) {
      for (int s = wave; s < p.slices; s += kFinish / 64) {
        const uint32_t from = mem.start[s], to = mem.start[s + 1];
        if (from == to) continue;
        uint64_t sum = 0;
        for (uint32_t i = from + lane; i < to; i += 64) sum += stays(mem.token[i]);
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k, 64);
        if (lane == 0) mem.part[s] = sum;
      }
    } else {
      each_in_memory<T>(a, p, row, mem, [&](uint64_t o, uint32_t) {
        const uint64_t w = stays(o);
        if (w) atomicAdd((unsigned long long*)&mem.part[id_of(o) / p.per], (unsigned long long)w);
      });
    }
    __syncthreads();
  }
  // the slice that the number falls into
  double total = 0;
  auto keep = [&](int s) {
    if (s >= p.slices) return 0.0;
    const Slice x = slice[s];
    const float first = logit_of(x.top);
    if (!counts(first, most) || x.top < bound) return 0.0;
    const double w = weight(first, most, r.inv);
    if (w < (double)r.min_p) return 0.0;
    double m = x.mass;
    if (r.cut) {
      const double own = floor(grid_of(first, r.inv)), to = last_step(whole - 1, step);
      if (whole < kBins) {
        m = 0;
        if (whole > 0 && x.bins > 0 && to <= own)
          m = p.mass[(row * p.slices + s) * kBins + min(bin_of_step(to, own), x.bins - 1)];
      }
      m = m * w + ldexp((double)mem.part[s], -unit);
    } else {
      m *= w;
    }
    return fmax(w, m);  // (a slice whose first token stays has some weight, however small)
  };
  double mine[kMaxSlices / kFinish], at[kMaxSlices / kFinish];
#pragma unroll
  for (int i = 0; i < kMaxSlices / kFinish; i++) {
    mine[i] = at[i] = 0;
    if (i * kFinish >= p.slices) continue;
    mine[i] = keep(i * kFinish + tid);
    double all;
    at[i] = total + block_scan<kFinish>(mine[i], mem.redd, &all);
    total += all;
  }
  const double aim = (double)r.u * total * (1 + kNear);  // (equal to a running sum: not exceeded by it)
  // the first slice whose end is past it: one thread's answer, also where the sums before two
  // neighbours, which come from different trees of additions, overlap or leave a gap
  int s = kMaxSlices, last = -1;
#pragma unroll
  for (int i = 0; i < kMaxSlices / kFinish; i++) {
    if (!(mine[i] > 0)) continue;
    if (at[i] + mine[i] > aim) s = min(s, i * kFinish + tid);
    last = i * kFinish + tid;
  }
  s = block_join<kFinish>(s, (int*)mem.redd, Min());
  if (s == kMaxSlices) s = block_join<kFinish>(last, (int*)mem.redd, Max());  // (rounding: the last slice of any weight)
#pragma unroll
  for (int i = 0; i < kMaxSlices / kFinish; i++)
    if (s == i * kFinish + tid) mem.found_before = at[i];
  __syncthreads();
  // the walk: each wave weighs a run of the slice's ids, the one that the number falls into goes along it
  const double rest = aim - mem.found_before;
  const int first = s * p.per + wave * 64 * E + lane, end = (int)a.vocab;
  auto share = [&](float v, int id) {
    if (id >= end || !counts(v, most) || order_of(v, id) < bound) return 0.0;
    const double w = weight(v, most, r.inv);
    return w >= (double)r.min_p ? w : 0.0;
  };
  double run = 0;
#pragma unroll 1
  for (int e = 0; e < E; e += kAhead) {
    float v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) v[i] = value_of(l[min(first + (e + i) * 64, end - 1)]);
#pragma unroll
    for (int i = 0; i < kAhead; i++) run += share(v[i], first + (e + i) * 64);
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) run += __shfl_xor(run, k, 64);
  __syncthreads();
  if (lane == 0) mem.redd[wave] = run;
  __syncthreads();
  int who = -1;
  double before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kFinish / 64; i++) {
    const double x = mem.redd[i];
    if (x > 0 && (who < 0 || sum <= rest)) who = i, before = sum;  // (the last of any weight, should none reach it)
    sum += x;
  }
  if (wave != who) return;
  int id = -1;
  float x = most;
  bool done = false;
#pragma unroll 1
  for (int e = 0; e < E && !done; e += kAhead) {
    float v[kAhead];
    double w[kAhead], upto[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) v[i] = value_of(l[min(first + (e + i) * 64, end - 1)]);
#pragma unroll
    for (int i = 0; i < kAhead; i++) upto[i] = w[i] = share(v[i], first + (e + i) * 64);
#pragma unroll
    for (int k = 1; k < 64; k <<= 1)
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const double y = __shfl_up(upto[i], k, 64);
        if (lane >= k) upto[i] += y;
      }
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      const uint64_t any = __ballot(w[i] > 0), past = __ballot(w[i] > 0 && before + upto[i] > rest);
      if (any && !done) {
        const int pick = past ? __ffsll((unsigned long long)past) - 1 : 63 - __builtin_clzll(any);
        id = __builtin_amdgcn_readlane(first + (e + i) * 64, pick);
        x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[i]), pick));
      }
      done |= past != 0;
      before += __shfl(upto[i], 63, 64);
    }
  }
  if (lane == 0) {
    a.ids[row] = id;
    if (a.logp) a.logp[row] = (float)((x == most ? 0.0 : ((double)x - (double)most) * r.inv) - log(total));
  }
}

// ---- the division of rows ----------------------------------------------------------------------------

int per_of(int64_t rows, int64_t vocab) {
  // few workgroups: shorter slices, but not so many that joining them takes longer (64 of a
  // row: 17 us, 32: 9); a row has no more than kMaxSlices
  const auto slices = [&](int e) { return (vocab + e * kScan - 1) / (e * kScan); };
  if (slices(8) <= 16 && (rows * slices(8) <= 1024 || slices(8) == 1)) return 8 * kScan;
  return slices(16) <= kMaxSlices ? 16 * kScan : 32 * kScan;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// What rows without filters use comes first, and is all that they need.
size_t lay_out(int64_t rows, int64_t vocab, bool filtered, char* work, Plan* p) {
  const int per = per_of(rows, vocab);
  const int64_t slices = (vocab + per - 1) / per, all = rows * slices;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return work ? work + here : nullptr;
  };
  const int room = (int)std::min<int64_t>(per, vocab);
  Plan q = {per, (int)slices, room, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  q.slice = (Slice*)take(all * sizeof(Slice));
  if (filtered) {
    q.cut = (Cut*)take(rows * sizeof(Cut));
    q.mass = (double*)take(all * kBins * 8);
    q.count = (uint32_t*)take(all * kBins * 4);
    q.listed = (uint32_t*)take(all * 4);
    q.list = (uint16_t*)take(all * room * 2);
  }
  if (p) *p = q;
  return at;
}

template <typename T, int E>
void launch_e(const SampleArgs& a, const Plan& p, hipStream_t s) {
  const unsigned grid = (unsigned)(a.rows * p.slices);
  scan_kernel<T, E><<<grid, kScan, 0, s>>>(a, p);
  if (sample_filters(a.s)) {
    join_kernel<<<(unsigned)a.rows, kBins, 0, s>>>(a, p);
    gather_kernel<T, E><<<grid, kScan, 0, s>>>(a, p);
  }
  finish_kernel<T, E * kScan / kFinish><<<(unsigned)a.rows, kFinish, 0, s>>>(a, p);
}

template <typename T>
void launch_t(const SampleArgs& a, Plan p, hipStream_t s) {
  p.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld * sizeof(T) % 16 == 0;
  if (p.per == 8 * kScan) launch_e<T, 8>(a, p, s);
  else if (p.per == 16 * kScan) launch_e<T, 16>(a, p, s);
  else launch_e<T, 32>(a, p, s);
}

}  // namespace

size_t sample_scratch(int64_t rows, int64_t vocab, bool filtered) {
  return lay_out(rows, vocab, filtered, nullptr, nullptr);
}

int64_t sample_grid(int64_t rows, int64_t vocab) {
  const int per = per_of(rows, vocab);
  return rows * ((vocab + per - 1) / per);
}

int launch_sample(fa_ctx* ctx, const SampleArgs& a, void* work, hipStream_t s) {
  Plan p;
  lay_out(a.rows, a.vocab, sample_filters(a.s), static_cast<char*>(work), &p);
  if (a.dtype == FA_DT_F32) launch_t<float>(a, p, s);
  else launch_t<uint16_t>(a, p, s);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

}  // namespace fa
