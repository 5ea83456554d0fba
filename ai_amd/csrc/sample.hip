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
//           (where a filter is set) a histogram of counts and weights by z = l / T
//           in steps of 1/8, on a grid that all slices share.
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
constexpr int kFinish = 1024;  // of finish
constexpr int kBins = 512;     // steps of 1/8: weights down to e^-64, the last bin holds the rest
constexpr int kMaxSlices = 1024;
constexpr int kSub = 2048;     // bins of a selection's pass
constexpr int kCached = 4096;  // listed tokens that finish keeps in LDS

// ---- a row's layout in the scratch ------------------------------------------------

struct Slice {
  uint64_t top;    // its first token of the order
  double mass;     // weights of all its tokens, relative to the first
  uint32_t count;  // tokens that can be drawn
  int32_t bins;    // bins in use
};

// Bins in which a row's bounds may lie. Tokens in listed bins are looked at one by one.
struct Cut {
  float most;         // the row's largest logit
  int k_bin;          // the bin of the top_k-th token (kBins: no limit)
  int k_rank;         // its rank there, from 1
  int p_lo, p_hi;     // bins of top_p's bound (kBins: none)
  int m_lo, m_hi;     // of min_p's
  double step;        // of most
  double above_k, above_p;  // weights of the bins before k_bin, before p_lo
  double all;         // of all bins
  __device__ __forceinline__ bool listed(int b) const {
    return b == k_bin || (b >= p_lo && b <= p_hi) || (b >= m_lo && b <= m_hi);
  }
};

struct Plan {
  int per, slices;  // tokens of a slice (a power of two), slices of a row
  int vec;          // rows aligned for 16-byte loads
  Slice* slice;     // [rows][slices]
  Cut* cut;         // [rows]
  uint64_t* mass;   // [rows][slices][kBins]
  uint32_t* count;  // likewise
  uint32_t* listed; // [rows][slices]
  uint16_t* list;   // [rows][slices * per]
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
// Steps of 1/8 from the grid's step of `most` down to that of l.
__device__ __forceinline__ int bin_of(float l, float most, double inv, double most_step) {
  if (l == most) return 0;
  return (int)fmin(most_step - floor((double)l * 8.0 * inv), (double)(kBins - 1));
}
__device__ __forceinline__ double step_of(float l, double inv) { return floor((double)l * 8.0 * inv); }
// Weights in bin b are below 2^-bin_exp(b): l / T is more than (b - 1) / 8 below.
__device__ __forceinline__ int bin_exp(int b) { return b > 1 ? (int)((float)(b - 1) * 0.18033f) : 0; }
// A number below 2^51 as an integer, to nearest.
__device__ __forceinline__ uint64_t to_int(double x) {
  return (uint64_t)__double_as_longlong(x + 0x1p52) - (uint64_t)0x4330000000000000ull;
}

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
  mass[tid] = 0;
  count[tid] = 0;
  uint64_t top = 0;
#pragma unroll
  for (int e = 0; e < E; e++) top = max(top, order_of(h.v[e], first + Held<T, E>::at(e)));
  top = block_join<kScan>(top, red, Max());
  const float most = logit_of(top);
  if (r.greedy || most == -__builtin_inff()) {
    if (tid == 0) *out = {top, 0.0, 0, 0};
    return;
  }
  if (!r.cut) {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++)
      if (h.v[e] > -__builtin_inff()) sum += weight(h.v[e], most, r.inv);
    sum = block_join<kScan>(sum, redd, Add());
    if (tid == 0) *out = {top, sum, 0, 0};
    return;
  }
  const double step = step_of(most, r.inv);
  uint64_t last = 0, valid = 0;
#pragma unroll
  for (int e = 0; e < E; e++)
    if (h.v[e] > -__builtin_inff()) {
      const int b = bin_of(h.v[e], most, r.inv, step);
      // up to 2^14 tokens of less than 2^49 each
      atomicAdd((unsigned long long*)&mass[b], to_int(weight(h.v[e], most, r.inv, 48 + bin_exp(b))));
      atomicAdd(&count[b], 1u);
      valid++;
    }
  __syncthreads();
  const uint64_t m = mass[tid];
  const uint32_t c = count[tid];
  if (c) last = tid + 1;
  last = block_join<kScan>(last, red, Max());
  valid = block_join<kScan>(valid, red, Add());
  const double all = block_join<kScan>(ldexp((double)m, -48 - bin_exp(tid)), redd, Add());
  const int64_t at = (row * p.slices + s) * kBins + tid;
  if (tid < (int)last) {
    p.mass[at] = m;
    p.count[at] = c;
  }
  if (tid == 0) *out = {top, all, (uint32_t)valid, (int32_t)last};
}

// ---- a row's histograms joined ----------------------------------------------------------------------

// Bins that a slice whose first token has logit l lies below the row's.
__device__ __forceinline__ int slice_offset(float l, float most, double step, double inv) {
  if (l == most) return 0;
  if (l == -__builtin_inff()) return kBins;
  return (int)fmin(step - step_of(l, inv), (double)kBins);
}

template <int NT>
__device__ __forceinline__ uint64_t row_top(const Plan& p, int64_t row, uint64_t* red) {
  uint64_t top = 0;
  for (int s = threadIdx.x; s < p.slices; s += NT) top = max(top, p.slice[row * p.slices + s].top);
  return block_join<NT>(top, red, Max());
}

// One workgroup a row, a thread a bin. Slices are taken kChunk at a time: their
// heads first, then all their bins, so that loads do not wait for one another.
constexpr int kChunk = 64;
__global__ __launch_bounds__(kBins) void join_kernel(SampleArgs a, Plan p) {
  constexpr int NT = kBins;
  __shared__ double redd[NT / 64], sums[kBins], scale[kChunk];
  __shared__ uint64_t red[NT / 64];
  __shared__ int found[4], offset[kChunk], bins[kChunk];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const Row r = row_of(a, row);
  if (!r.sound || r.greedy || !r.cut) return;
  const Slice* slice = p.slice + row * p.slices;
  const float most = logit_of(row_top<NT>(p, row, red));
  if (most == -__builtin_inff()) return;
  Cut c;
  c.most = most;
  c.step = step_of(most, r.inv);
  c.k_bin = c.p_lo = c.m_lo = kBins;
  c.p_hi = c.m_hi = -1;
  c.k_rank = 0;
  c.above_k = c.above_p = 0;
  double m = 0, far_m = 0;
  uint64_t n = 0, far_n = 0;
  for (int s0 = 0; s0 < p.slices; s0 += kChunk) {
    const int many = min(kChunk, p.slices - s0);
    __syncthreads();
    if (tid < many) {
      const Slice x = slice[s0 + tid];
      const float l = logit_of(x.top);
      int off = kBins, used = 0;
      double w = 0;
      if (x.bins) {
        off = slice_offset(l, most, c.step, r.inv);
        w = weight(l, most, r.inv);
        if (off >= kBins - 1) far_m += x.mass * w, far_n += x.count;  // all of it past the row's last bin
        else used = x.bins;
      }
      offset[tid] = off;
      bins[tid] = used;
      scale[tid] = w;
    }
    __syncthreads();
    const int64_t at = (row * p.slices + s0) * kBins;
#pragma unroll 8
    for (int s = 0; s < many; s++) {
      const int j = tid - offset[s];
      const bool in = tid < kBins - 1 && j >= 0 && j < bins[s];
      const int64_t i = at + (int64_t)s * kBins + (in ? j : 0);
      const uint64_t mass = p.mass[i];
      const uint32_t count = p.count[i];
      if (in) m += ldexp((double)mass, -48 - bin_exp(j)) * scale[s], n += count;
    }
    for (int s = 0; s < many; s++)
      for (int i = kBins - 1 - offset[s] + tid; i < bins[s]; i += NT) {  // past the row's last bin
        far_m += ldexp((double)p.mass[at + (int64_t)s * kBins + i], -48 - bin_exp(i)) * scale[s];
        far_n += p.count[at + (int64_t)s * kBins + i];
      }
  }
  far_m = block_join<NT>(far_m, redd, Add());
  far_n = block_join<NT>(far_n, red, Add());
  if (tid == kBins - 1) m = far_m, n = far_n;
  uint64_t tokens;
  const double before = block_scan<NT>(m, redd, &c.all);
  const uint64_t n_before = block_scan<NT>(n, red, &tokens);
  sums[tid] = before;
  if (tid < 4) found[tid] = tid == 1 ? 0 : kBins;
  __syncthreads();
  // top-k: the bin of the top_k-th token, if there are more
  const uint64_t k = (uint64_t)r.top_k;
  if (n_before < k && n_before + n >= k && tokens > k) {
    found[0] = tid;
    found[1] = (int)(k - n_before);
  }
  __syncthreads();
  c.k_bin = found[0];
  c.k_rank = found[1];
  double k_least = c.all, k_most = c.all;  // weight of the top_k tokens
  if (c.k_bin < kBins) {
    c.above_k = k_least = sums[c.k_bin];
    k_most = c.k_bin + 1 < kBins ? sums[c.k_bin + 1] : c.all;
  }
  // top-p: sums of bins are right to 1e-14 or so, the margin of 1e-12 keeps to either side
  if (r.top_p < 1.f) {
    const double least = (double)r.top_p * k_least * (1 - 1e-12), want = (double)r.top_p * k_most * (1 + 1e-12);
    if (n > 0) {
      if (before + m >= least) atomicMin(&found[2], tid);
      if (before + m >= want) atomicMin(&found[3], tid);
    }
    __syncthreads();
    c.p_lo = min(found[2], min(c.k_bin, kBins - 1));
    c.p_hi = min(found[3], min(c.k_bin, kBins - 1));
    c.above_p = sums[c.p_lo];
  }
  // min-p: l >= most + T ln(min_p), in the step of that bound or the next
  if (r.min_p > 0.f) {
    const int b = most == __builtin_inff() ? 0 : (int)fmin(-8.0 * log((double)r.min_p), (double)kBins);
    c.m_lo = max(0, b - 1);
    c.m_hi = b + 2;
  }
  if (tid == 0) p.cut[row] = c;
}

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
  const int off = slice_offset(logit_of(x.top), most, c.step, r.inv);
  const int64_t at = (row * p.slices + s) * kBins;
  // does the slice have tokens in listed bins?
  bool any = off >= kBins - 1 && c.listed(kBins - 1);
  if (off < kBins - 1 && tid < x.bins) any = p.count[at + tid] && c.listed(min(tid + off, kBins - 1));
  if (tid == 0) n_listed = 0;
  if (__syncthreads_or(any)) {
    Held<T, E> h;
    h.load((const T*)a.logits + row * a.ld + first, min(p.per, (int)a.vocab - first), p.vec);
    uint16_t* list = p.list + (row * p.slices + s) * p.per;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const bool in = h.v[e] > -__builtin_inff() && c.listed(bin_of(h.v[e], most, r.inv, c.step));
      const uint64_t mask = __ballot(in);
      if (mask == 0) continue;
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
  int found[4];
  uint64_t token[kCached];   // the row's listed tokens, if they fit
  uint64_t sub_mass[kSub];
  uint32_t sub_count[kSub];
  uint32_t start[kMaxSlices + 1];  // of a slice's listed tokens among the row's
  double keep[kMaxSlices];   // weight that stays of each slice
  uint64_t part[kMaxSlices]; // of its listed tokens
  int pick;
  uint64_t one;
  uint64_t pass[3];
};

// The listed tokens of a row, each given to f as its number in the order.
template <typename T, typename F>
__device__ __forceinline__ void each_listed(const SampleArgs& a, const Plan& p, int64_t row, const FinishMem& mem,
                                            uint32_t n, F f) {
  if (n <= kCached) {
    for (uint32_t i = threadIdx.x; i < n; i += kFinish) f(mem.token[i], i);
    return;
  }
  const T* l = (const T*)a.logits + row * a.ld;
  for (int s = threadIdx.x >> 6; s < p.slices; s += kFinish / 64) {
    const uint32_t from = mem.start[s], m = mem.start[s + 1] - from;
    const uint16_t* list = p.list + (row * p.slices + s) * p.per;
    for (uint32_t i = threadIdx.x & 63; i < m; i += 64) {
      const int id = s * p.per + list[i];
      f(order_of(value_of(l[id]), id), from + i);
    }
  }
}

// Of the listed tokens that `in` takes, the one down to which there are `rank`
// (by count), or down to which weights and `above` make `want`. Weights count in
// units of 2^-unit. The last of them if there are not so many.
template <typename T, bool MASS, typename IN>
__device__ uint64_t select_token(const SampleArgs& a, const Plan& p, int64_t row, FinishMem& mem, uint32_t n, IN in,
                                 float most, double inv, int unit, uint64_t rank, double above, double want) {
  const int tid = threadIdx.x;
  uint64_t hi = 0, lo = ~0ull;
  each_listed<T>(a, p, row, mem, n, [&](uint64_t o, uint32_t) {
    if (in(o)) hi = max(hi, o), lo = min(lo, o);
  });
  hi = block_join<kFinish>(hi, mem.red, Max());
  lo = block_join<kFinish>(lo, mem.red, Min());
  uint64_t before = 0, count_before = 0;  // integer weight and tokens above hi
  while (lo < hi) {
    const int shift = max(0, 64 - (int)__builtin_clzll(hi - lo) - 11);
    for (int i = tid; i < kSub; i += kFinish) mem.sub_mass[i] = 0, mem.sub_count[i] = 0;
    __syncthreads();
    each_listed<T>(a, p, row, mem, n, [&](uint64_t o, uint32_t) {
      if (o < lo || o > hi || !in(o)) return;
      const int i = (int)((hi - o) >> shift);
      atomicAdd(&mem.sub_count[i], 1u);
      if (MASS) atomicAdd((unsigned long long*)&mem.sub_mass[i], to_int(weight(logit_of(o), most, inv, unit)));
    });
    __syncthreads();
    // each thread two bins
    const uint64_t m0 = mem.sub_mass[2 * tid], m1 = mem.sub_mass[2 * tid + 1];
    const uint64_t c0 = mem.sub_count[2 * tid], c1 = mem.sub_count[2 * tid + 1];
    uint64_t all;
    uint64_t cb = block_scan<kFinish>(c0 + c1, mem.red, &all);
    uint64_t mb = MASS ? block_scan<kFinish>(m0 + m1, mem.red, &all) : 0;
    if (tid == 0) mem.found[0] = kSub, mem.found[1] = -1;
    __syncthreads();
    auto reached = [&](uint64_t count, uint64_t mass) {
      return MASS ? above + ldexp((double)(before + mass), -unit) >= want : count_before + count >= rank;
    };
    if (c0) atomicMax(&mem.found[1], 2 * tid);
    if (c1) atomicMax(&mem.found[1], 2 * tid + 1);
    if (c0 && reached(cb + c0, mb + m0)) atomicMin(&mem.found[0], 2 * tid);
    else if (c1 && reached(cb + c0 + c1, mb + m0 + m1)) atomicMin(&mem.found[0], 2 * tid + 1);
    __syncthreads();
    const int pick = mem.found[0] < kSub ? mem.found[0] : mem.found[1];
    if (pick >> 1 == tid) {
      mem.pass[0] = pick & 1 ? cb + c0 : cb;
      mem.pass[1] = pick & 1 ? mb + m0 : mb;
      mem.pass[2] = pick & 1 ? c1 : c0;
    }
    __syncthreads();
    count_before += mem.pass[0];
    before += mem.pass[1];
    const bool single = mem.pass[2] == 1;
    hi -= (uint64_t)pick << shift;
    const uint64_t width = 1ull << shift;
    if (hi - lo >= width) lo = hi - width + 1;
    if (single && lo < hi) {
      each_listed<T>(a, p, row, mem, n, [&](uint64_t o, uint32_t) {
        if (o >= lo && o <= hi && in(o)) mem.one = o;
      });
      __syncthreads();
      hi = lo = mem.one;
    }
    __syncthreads();
  }
  return hi;
}

template <typename T>
__global__ __launch_bounds__(kFinish) void finish_kernel(SampleArgs a, Plan p) {
  __shared__ FinishMem mem;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const Row r = row_of(a, row);
  uint64_t top = 0;
  if (r.sound) top = row_top<kFinish>(p, row, mem.red);
  const float most = logit_of(top);
  const bool none = !r.sound || most == -__builtin_inff();
  if (none || r.greedy) {
    if (tid == 0) {
      a.ids[row] = none ? -1 : id_of(top);
      if (a.logp) a.logp[row] = none ? __builtin_nanf("") : 0.f;
    }
    return;
  }
  const Slice* slice = p.slice + row * p.slices;
  const T* l = (const T*)a.logits + row * a.ld;
  uint64_t bound = 0;     // tokens at or above it stay (but for min_p)
  int whole = kBins;      // bins before it stay whole, listed tokens of the others are asked
  if (r.cut) {
    const Cut c = p.cut[row];
    const uint32_t mine = tid < p.slices ? p.listed[row * p.slices + tid] : 0;
    uint32_t n;
    const uint32_t start = block_scan<kFinish>(mine, (uint32_t*)mem.red, &n);
    if (tid < p.slices) mem.start[tid] = start, mem.part[tid] = 0;
    if (tid == 0) mem.start[p.slices] = n;
    __syncthreads();
    if (n <= kCached) {
      for (int s = wave; s < p.slices; s += kFinish / 64) {
        const uint32_t from = mem.start[s], m = mem.start[s + 1] - from;
        const uint16_t* list = p.list + (row * p.slices + s) * p.per;
        for (uint32_t i = lane; i < m; i += 64) {
          const int id = s * p.per + list[i];
          mem.token[from + i] = order_of(value_of(l[id]), id);
        }
      }
      __syncthreads();
    }
    auto bin = [&](uint64_t o) { return bin_of(logit_of(o), most, r.inv, c.step); };
    // integer weights: n of them, each below 2^(bits + 1), stay below 2^63
    const int bits = min(49, 61 - (32 - __builtin_clz(n | 1)));
    double k_mass = c.all;
    if (c.k_bin < kBins) {
      const int b = c.k_bin;
      bound = select_token<T, false>(a, p, row, mem, n, [&](uint64_t o) { return bin(o) == b; }, most, r.inv, 0,
                                     (uint64_t)c.k_rank, 0, 0);
      uint64_t sum = 0;
      const int unit = bits + bin_exp(b);
      each_listed<T>(a, p, row, mem, n, [&](uint64_t o, uint32_t) {
        if (o >= bound && bin(o) == b) sum += to_int(weight(logit_of(o), most, r.inv, unit));
      });
      sum = block_join<kFinish>(sum, mem.red, Add());
      k_mass = c.above_k + ldexp((double)sum, -unit);
      whole = b;
    }
    if (r.top_p < 1.f) {
      const uint64_t o_k = bound;
      const int unit = bits + bin_exp(c.p_lo);
      const uint64_t o_p = select_token<T, true>(
          a, p, row, mem, n, [&](uint64_t o) { const int b = bin(o); return o >= o_k && b >= c.p_lo && b <= c.p_hi; }, most,
          r.inv, unit, 0, c.above_p, (double)r.top_p * k_mass);
      bound = max(bound, o_p);
      whole = min(whole, bin(o_p));
    }
    whole = min(whole, c.m_lo);
    // what stays of each slice: its whole bins, then its listed tokens
    for (int s = wave; s < p.slices; s += kFinish / 64) {
      const Slice x = slice[s];
      const int off = slice_offset(logit_of(x.top), most, c.step, r.inv);
      const int64_t at = (row * p.slices + s) * kBins;
      double m = 0;
      for (int i = lane; i < x.bins && min(i + off, kBins - 1) < whole; i += 64)
        m += ldexp((double)p.mass[at + i], -48 - bin_exp(i));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
      if (lane == 0) mem.keep[s] = m * weight(logit_of(x.top), most, r.inv);
    }
    const int unit = bits + bin_exp(whole);
    each_listed<T>(a, p, row, mem, n, [&](uint64_t o, uint32_t) {
      if (o < bound || bin(o) < whole) return;
      const double w = weight(logit_of(o), most, r.inv);
      if (w >= (double)r.min_p)
        atomicAdd((unsigned long long*)&mem.part[id_of(o) / p.per], to_int(ldexp(w, unit)));
    });
    __syncthreads();
    for (int s = tid; s < p.slices; s += kFinish) mem.keep[s] += ldexp((double)mem.part[s], -unit);
  } else {
    for (int s = tid; s < p.slices; s += kFinish) {
      const float first = logit_of(slice[s].top);
      mem.keep[s] = first == -__builtin_inff() ? 0.0 : slice[s].mass * weight(first, most, r.inv);
    }
  }
  // a slice whose first token stays has some weight, however small
  __syncthreads();
  double mine = 0;
  if (tid < p.slices) {
    mine = mem.keep[tid];
    const uint64_t o = slice[tid].top;
    if (logit_of(o) > -__builtin_inff() && o >= bound) {
      const double w = weight(logit_of(o), most, r.inv);
      if (w >= (double)r.min_p) mine = fmax(mine, w);
      else mine = 0;
    } else {
      mine = 0;
    }
  }
  double total;
  const double before = block_scan<kFinish>(mine, mem.redd, &total);
  const double aim = (double)r.u * total;
  if (tid == 0) mem.found[0] = kMaxSlices, mem.found[1] = 0;
  __syncthreads();
  if (mine > 0) {
    atomicMax(&mem.found[1], tid);
    if (before + mine > aim) atomicMin(&mem.found[0], tid);
  }
  __syncthreads();
  const int s = mem.found[0] < kMaxSlices ? mem.found[0] : mem.found[1];
  if (tid == s) mem.keep[0] = before;
  __syncthreads();
  // the walk: each thread a run of the slice's ids
  const double rest = aim - mem.keep[0];
  const int first = s * p.per, end = min((int)a.vocab, first + p.per), each = p.per / kFinish;
  const int i0 = min(end, first + tid * each), i1 = min(end, i0 + each);
  auto share = [&](int i) {
    const float v = value_of(l[i]);
    const uint64_t o = order_of(v, i);
    if (o < bound || !(v > -__builtin_inff())) return 0.0;
    const double w = weight(v, most, r.inv);
    return w >= (double)r.min_p ? w : 0.0;
  };
  double run = 0;
  for (int i = i0; i < i1; i++) run += share(i);
  double unused;
  const double at0 = block_scan<kFinish>(run, mem.redd, &unused);
  __syncthreads();
  if (tid == 0) mem.found[0] = kFinish, mem.found[1] = 0;
  __syncthreads();
  if (run > 0) {
    atomicMax(&mem.found[1], tid);
    if (at0 + run > rest) atomicMin(&mem.found[0], tid);
  }
  __syncthreads();
  if (tid == (mem.found[0] < kFinish ? mem.found[0] : mem.found[1])) {
    double at = at0;
    int id = -1;
    for (int i = i0; i < i1; i++) {
      const double w = share(i);
      if (w > 0) {
        id = i;
        at += w;
        if (at > rest) break;
      }
    }
    a.ids[row] = id;
    const float v = value_of(l[max(id, 0)]);
    if (a.logp) a.logp[row] = (float)((v == most ? 0.0 : ((double)v - (double)most) * r.inv) - log(total));
  }
}

// ---- the division of rows ----------------------------------------------------------------------------

int per_of(int64_t rows, int64_t vocab) {
  // few workgroups: shorter slices; a row has no more than kMaxSlices
  if (vocab > (int64_t)kMaxSlices * 16 * kScan) return 32 * kScan;
  return rows * ((vocab + 16 * kScan - 1) / (16 * kScan)) < 256 && vocab <= (int64_t)kMaxSlices * 8 * kScan ? 8 * kScan
                                                                                                             : 16 * kScan;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

size_t lay_out(int64_t rows, int64_t vocab, char* work, Plan* p) {
  const int per = per_of(rows, vocab);
  const int64_t slices = (vocab + per - 1) / per, all = rows * slices;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return work ? work + here : nullptr;
  };
  Plan q = {per, (int)slices, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  q.slice = (Slice*)take(all * sizeof(Slice));
  q.cut = (Cut*)take(rows * sizeof(Cut));
  q.mass = (uint64_t*)take(all * kBins * 8);
  q.count = (uint32_t*)take(all * kBins * 4);
  q.listed = (uint32_t*)take(all * 4);
  q.list = (uint16_t*)take(all * per * 2);
  if (p) *p = q;
  return at;
}

template <typename T, int E>
void launch_e(const SampleArgs& a, const Plan& p, hipStream_t s) {
  const unsigned grid = (unsigned)(a.rows * p.slices);
  scan_kernel<T, E><<<grid, kScan, 0, s>>>(a, p);
  if (a.s.top_k || a.s.top_p || a.s.min_p) {
    join_kernel<<<(unsigned)a.rows, kBins, 0, s>>>(a, p);
    gather_kernel<T, E><<<grid, kScan, 0, s>>>(a, p);
  }
  finish_kernel<T><<<(unsigned)a.rows, kFinish, 0, s>>>(a, p);
}

template <typename T>
void launch_t(const SampleArgs& a, Plan p, hipStream_t s) {
  p.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld * sizeof(T) % 16 == 0;
  if (p.per == 8 * kScan) launch_e<T, 8>(a, p, s);
  else if (p.per == 16 * kScan) launch_e<T, 16>(a, p, s);
  else launch_e<T, 32>(a, p, s);
}

}  // namespace

size_t sample_scratch(int64_t rows, int64_t vocab) { return lay_out(rows, vocab, nullptr, nullptr); }

int64_t sample_grid(int64_t rows, int64_t vocab) {
  const int per = per_of(rows, vocab);
  return rows * ((vocab + per - 1) / per);
}

int launch_sample(fa_ctx* ctx, const SampleArgs& a, void* work, hipStream_t s) {
  Plan p;
  lay_out(a.rows, a.vocab, static_cast<char*>(work), &p);
  if (a.dtype == FA_DT_F32) launch_t<float>(a, p, s);
  else launch_t<uint16_t>(a, p, s);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

}  // namespace fa
