// The key/value cache in 8 bits: tokens quantised into it and read back.
//
// A block holds 64 tokens of every key/value head: e4m3 codes and, for the
// keys and for the values of each head, one scale 2^e (value = code * scale).
// A power of two makes every product with it exact, and e4m3 has the same
// relative step at every scale, so nothing is lost against a free scale but a
// part of one of its 15 binades.
//
// Layout of a head's part (64 x Dp bytes, Dp = head_dim in whole slices of
// 64), made for the attention kernel's matrix operands, 16 bytes a lane and a
// KB a wave's load:
//   keys    [slice of 64 dims][token][64 dims]
//   values  [dim][64 tokens], token 16 a + 4 b + c at place 16 b + 4 a + c:
//           lane group b of a wave holds tokens 4 b .. 4 b + 3 of each 16 in
//           the layout in which it gets their scores, so weights meet values
//           without leaving their registers.
#include <algorithm>
#include <atomic>

#include "device_math.h"
#include "kvcache.h"

namespace fa {
namespace {

// Units of work of the writer and the reader: the (sequence, block slot)
// pairs that a batch's rows touch. Few rows: one unit per row, used by the
// first row of a slot. Many: sequence b's units start at cu[b] / 64 + 2 b,
// which leaves room for every slot that n rows can touch (n / 64 + 2).
struct KvUnit {
  int b;
  int64_t slot;      // may be negative or past the table (no block then)
  int64_t row;       // first row of the unit
  int32_t place, n;  // its place in the block, and the rows of the unit
  bool ok;
};

int64_t kv_units(int64_t rows, int nseq, bool* by_row) {
  const int64_t many = rows / 64 + 2 * (int64_t)nseq;
  *by_row = rows <= many;
  return *by_row ? rows : many;
}

__device__ __forceinline__ KvUnit kv_unit(const KvArgs& a, int64_t u, bool by_row) {
  KvUnit r;
  int64_t slot;
  if (by_row) {
    const KvFound f = kv_find(a, u, [](int32_t c, int) { return (int64_t)c; });
    const KvSeq s = f.s;
    r.b = f.b;
    const int64_t start = (int64_t)s.len - s.n, pos = start + (u - s.row0);
    slot = pos >> 6;
    r.ok = u >= s.row0 && u < s.row0 + s.n && (u == s.row0 || (pos & 63) == 0);
    r.row = u;
    r.place = (int32_t)(pos & 63);
    r.n = (int32_t)min((int64_t)(64 - r.place), s.row0 + s.n - u);
  } else {
    auto base = [](int32_t c, int b) { return ((int64_t)c >> 6) + 2 * b; };
    const KvFound f = kv_find(a, u, base);
    const KvSeq s = f.s;
    r.b = f.b;
    const int64_t start = (int64_t)s.len - s.n, end = s.len;
    slot = (start >> 6) + (u - base(f.cu0, f.b));
    const int64_t p0 = max(start, slot * 64), p1 = min(end, slot * 64 + 64);
    r.ok = slot >= (start >> 6) && p0 < p1;
    r.row = s.row0 + (p0 - start);
    r.place = (int32_t)(p0 & 63);
    r.n = (int32_t)(p1 - p0);
  }
  r.slot = slot;
  return r;
}

// Each code times 2^sh (sh <= 0), rounded to a code again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const f32x4 v = unpack4(w);
  return pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
}

// The exponent of a stored scale (whatever the bits, a valid one).
__device__ __forceinline__ int stored_exp(float s) {
  const int e = (int)((__float_as_uint(s) >> 23) & 255u) - 127;
  return min(max(e, kMinExp), kMaxExp);
}
// A thread's share of a 64 x 64 slice: the tokens 16 a + 4 b + 0..3 and dims
// 4 dq + 0..3, with dq = tid & 15, a = (tid >> 4) & 3, b = tid >> 6. A
// wave's loads cover 256 (float32) or 128 (bf16) bytes of each of four
// rows, and its words of a value row fall into different LDS banks.
//
// One workgroup writes one (block, head, keys or values): all its new values
// in registers, one reduction for the scale, one store. Bytes are read and
// written once. Prompts (16 of up to 2048 tokens, 8 heads of 128 dims in bf16) take
// 35 us, where the bytes take 28 at a large copy's rate (43 with each load widened, and so
// waited for, before the next; over head dims of 32 to 512 in either type that order of
// loads is 1.0 to 1.3 times as fast for prompts and chunks, and costs one token up to 0.13
// of 4 us). Slices that a head does not have are jumped over as a
// whole (64 single tokens of 320 dims 7.7 -> 7.4 us). Single tokens are bound by the
// chain of dependent loads (sequence, block, row) and the write-back of the 128 lines
// that one token's values touch in a head (64 sequences, one float32 token each,
// written 7.1 us).
// at(row): a row's values. vec: fours of them are aligned.
template <typename T, int NCM, typename F>
__device__ __forceinline__ void write_block(const KvArgs& a, const KvUnit& u, int id, int h, int part, bool vec, F at) {
  __shared__ float red[4];
  __shared__ uint32_t tile[64 * 17];
  const int tid = threadIdx.x, dq = tid & 15, ta = (tid >> 4) & 3, tb = tid >> 6;
  const int t0 = ta * 16 + tb * 4;
  const int end = u.place + u.n;
  f32x4 x[NCM][4];
  float big = 0.f;
  Raw4<T> raw[NCM][4];  // (all loads under way before the first is widened)
#pragma unroll
  for (int c = 0; c < NCM; c++)
    if (c < a.nc)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i, d = c * 64 + dq * 4;
        raw[c][i] = Raw4<T>{};
        if (vec && t >= u.place && t < end && d + 4 <= a.D) raw[c][i] = raw4(at(u.row + (t - u.place)) + d);
      }
#pragma unroll
  for (int c = 0; c < NCM; c++)
    if (c < a.nc)
#pragma unroll
      for (int i = 0; i < 4; i++) x[c][i] = widen(raw[c][i]);
  if (!vec || a.D % 4 != 0)
#pragma unroll
    for (int c = 0; c < NCM; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i, d = c * 64 + dq * 4;
        if (t >= u.place && t < end && !(vec && d + 4 <= a.D))
          x[c][i] = load4(at(u.row + (t - u.place)), d, a.D, false);
      }
#pragma unroll
  for (int c = 0; c < NCM; c++)
    if (c < a.nc)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float y = x[c][i][j];
          join_max(y, big);  // not finite: stored as NaN
          x[c][i][j] = y;
        }
  uint8_t* dst = kv_part(a, id, h, part);
  const bool whole = u.place == 0 && end == 64;
  float* scale = a.scales + ((int64_t)id * a.hkv + h) * 2 + part;
  const bool keep = u.place > 0;  // tokens below the first new one stay
  const int e_old = keep ? stored_exp(*scale) : kMinExp;
  big = wave_max(big);
  if ((tid & 63) == 0) red[tid >> 6] = big;
  __syncthreads();
  big = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int e_new = scale_exp(big);
  const int e = max(e_new, e_old);
  const bool grow = keep && e > e_old;
  const float inv = exp2_int(-e), shrink = exp2_int(max(e_old - e, -126));
  if (e == kMaxExp) {  // 256 * 2^120 and above would be read back as infinite
#pragma unroll
    for (int c = 0; c < NCM; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (c < a.nc) x[c][i][j] = clamp_top(x[c][i][j]);
  }
  if (tid == 0) *scale = exp2_int(e);  // (every thread read the old one before the maximum was joined)
  if (part == 1 && u.n <= 8 && !grow) {
    // few values: their bytes alone (one token of 64 sequences, 8 heads of
    // 128 dims: 7.1 us, and 8.3 with the value rows read and written whole)
#pragma unroll
    for (int c = 0; c < NCM; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i;
        if (c < a.nc && t >= u.place && t < end) {
          const uint32_t w = pack4(x[c][i][0] * inv, x[c][i][1] * inv, x[c][i][2] * inv, x[c][i][3] * inv);
          uint8_t* to = dst + (int64_t)(c * 64 + dq * 4) * 64 + tb * 16 + ta * 4 + i;
#pragma unroll
          for (int j = 0; j < 4; j++) to[j * 64] = (uint8_t)(w >> (8 * j));
        }
      }
    return;
  }
#pragma unroll
  for (int c = 0; c < NCM; c++) {
    if (c >= a.nc) continue;
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i;
        uint32_t* w = reinterpret_cast<uint32_t*>(dst + c * 4096 + t * 64 + dq * 4);
        if (t >= u.place && t < end) *w = pack4(x[c][i][0] * inv, x[c][i][1] * inv, x[c][i][2] * inv, x[c][i][3] * inv);
        else if (grow && t < u.place) *w = rescale4(*w, shrink);
      }
    } else {
      // four tokens of one dim to a word, the slice's words through LDS so
      // that whole value rows are stored
      if (c) __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; j++)
        tile[(dq * 4 + j) * 17 + tb * 4 + ta] =
            pack4(x[c][0][j] * inv, x[c][1][j] * inv, x[c][2][j] * inv, x[c][3][j] * inv);
      __syncthreads();
      // this thread: dim row tid / 4, words 4 (tid % 4) .. + 3 = tokens 4 b + 0..3 of each 16, b = tid % 4
      const int row = tid >> 2, b = tid & 3;
      uint4* w = reinterpret_cast<uint4*>(dst + (int64_t)(c * 64 + row) * 64 + b * 16);
      uint32_t nw[4];
#pragma unroll
      for (int q = 0; q < 4; q++) nw[q] = tile[row * 17 + b * 4 + q];
      if (!whole) {
        const uint4 o4 = *w;
        const uint32_t old[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint32_t fresh = 0, below = 0;  // byte masks: new tokens, kept ones
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int t = q * 16 + b * 4 + i;
            if (t >= u.place && t < end) fresh |= 0xFFu << (8 * i);
            else if (t < u.place) below |= 0xFFu << (8 * i);
          }
          uint32_t o = old[q];
          if (grow) o = (rescale4(o, shrink) & below) | (o & ~below);
          nw[q] = (nw[q] & fresh) | (o & ~fresh);
        }
      }
      *w = make_uint4(nw[0], nw[1], nw[2], nw[3]);
    }
  }
}

// (eight waves a SIMD for heads of up to 64 dims, where the compiler's own choice of
// registers leaves six or seven: prompts of 32 dims in float32 19.9 -> 18.2 us)
template <typename T, int NCM>
__global__ __launch_bounds__(256, NCM == 1 ? 8 : 1) void kv_write_kernel(KvArgs a, const T* __restrict__ k, int64_t k_st, int64_t k_sh,
                                                       const T* __restrict__ v, int64_t v_st, int64_t v_sh,
                                                       bool by_row, bool vec) {
  const KvUnit u = kv_unit(a, blockIdx.x, by_row);
  if (!u.ok) return;
  const int id = kv_block(a, u.b, u.slot);
  if (id < 0) return;
  const int h = blockIdx.y, part = blockIdx.z;
  const T* src = part ? v : k;
  const int64_t st = part ? v_st : k_st, sh = part ? v_sh : k_sh;
  write_block<T, NCM>(a, u, id, h, part, vec, [&](int64_t row) { return src + row * st + h * sh; });
}

// ---- rotary positions on the way ---------------------------------------------------

// Cosine and sine of an angle in float64, rounded to float32 as fa_rope's tables. a -
// n pi / 2 with pi / 2 in two parts (the products exact in the fma), then the series of
// both to a^15 and a^16: the next terms are below 2^-53 of a sine and 2^-58 of a cosine, so
// that the rounding to float32 is float64's but where that lies within 2^-52 of the middle
// of two numbers (to a^11 and a^12: 322 of 40 million other than the library's, now none).
// |a| < 2^31; WIDE: any angle.
template <bool WIDE>
__device__ __forceinline__ float2 cos_sin(double a) {
  if (WIDE) {
    double s, c;
    sincos(a, &s, &c);
    return make_float2((float)c, (float)s);
  }
  const double n = rint(a * 0.63661977236758134);
  double r = fma(-n, 1.5707963267948966, a);
  r = fma(-n, 6.123233995736766e-17, r);
  const double x = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  c = fma(c, x, -1.0 / 87178291200.0);
  s = fma(s, x, 1.0 / 6227020800.0);
  c = fma(c, x, 1.0 / 479001600.0);
  s = fma(s, x, -1.0 / 39916800.0);
  c = fma(c, x, -1.0 / 3628800.0);
  s = fma(s, x, 1.0 / 362880.0);
  c = fma(c, x, 1.0 / 40320.0);
  s = fma(s, x, -1.0 / 5040.0);
  c = fma(c, x, -1.0 / 720.0);
  s = fma(s, x, 1.0 / 120.0);
  c = fma(c, x, 1.0 / 24.0);
  s = fma(s, x, -1.0 / 6.0);
  c = fma(c, x, -0.5);
  s = fma(s * x, r, r);
  c = fma(c, x, 1.0);
  const int q = (int)n;
  const float fs = (float)s, fc = (float)c;
  const float u = q & 1 ? fs : fc, v = q & 1 ? fc : fs;
  return make_float2((q + 1) & 2 ? -u : u, q & 2 ? -v : v);
}

// x_i cos - x_{i + half} sin of a pair and x_{i + half} cos + x_i sin. EXACT: products
// of float32 are exact in float64, so that each is rounded once there and once to
// float32; otherwise one product is rounded to float32 and then the sum.
template <bool EXACT>
__device__ __forceinline__ void turn(float& lo, float& hi, float2 cs) {
  if (EXACT) {
    const double x = (double)lo, y = (double)hi, c = (double)cs.x, s = (double)cs.y;
    lo = (float)(x * c - y * s);
    hi = (float)(y * c + x * s);
  } else {
    const float x = lo, y = hi;
    lo = fmaf(x, cs.x, -(y * cs.y));
    hi = fmaf(y, cs.x, x * cs.y);
  }
}

// Rows i0 .. i1 - 1 of a unit, heads h0 .. h1 - 1 of src, turned into put(i, h, d,
// end, four values): dims d .. end - 1, four at most. A thread holds the cosines and
// sines of four pairs of a row and goes through heads with them, HEADS at once, the
// next loads under way; a pair is read and written by one thread, so the target may be
// the source. Rows fill the threads first, then heads. WHOLE: fours of values are
// aligned, and whole.
template <typename T, bool WIDE, bool EXACT, int HEADS, bool WHOLE, typename F>
__device__ __forceinline__ void turn_rows(const KvArgs& a, const KvRopeArgs& r, const KvUnit& u, int64_t first,
                                          const T* src, int64_t st, int64_t sh, int i0, int i1, int h0, int h1, F put) {
  // slots of a row's head: fours of pairs, then fours of the dims that stay (at most 129)
  const int pairs = (r.half + 3) / 4, slots = pairs + (a.D - 2 * r.half + 3) / 4;
  const int items = 256 / slots, at_once = min(items, i1 - i0), runs = items / at_once;
  const int item = (int)threadIdx.x / slots, slot = (int)threadIdx.x - item * slots;
  if (item >= at_once * runs) return;
  const int run = item % runs;
  const bool rest = slot >= pairs;
  // this thread's dims d .. end - 1 and d2 .. end2 - 1; the same where nothing turns
  const int d = rest ? 2 * r.half + (slot - pairs) * 4 : slot * 4, end = rest ? a.D : r.half;
  const int d2 = rest ? d : d + r.half, end2 = rest ? a.D : 2 * r.half;
  double inv[4];
#pragma unroll
  for (int j = 0; j < 4; j++) inv[j] = r.inv[min(d + j, r.half - 1)];
  Raw4<T> x[HEADS], y[HEADS];
  auto fetch = [&](int i, int h) {
    const T* p = src + (u.row + i) * st;
#pragma unroll
    for (int k = 0; k < HEADS; k++) {
      const T* from = p + min(h + k * runs, h1 - 1) * sh;
      x[k] = raw4(from + d);
      y[k] = raw4(from + d2);
    }
  };
  int i = i0 + item / runs, h = h0 + run;
  if (h >= h1) return;
  if (WHOLE && i < i1) fetch(i, h);
  float2 cs[4];
  while (i < i1) {
    if (h == h0 + run) {
      const double pos = (double)(r.positions ? (int64_t)r.positions[u.row + i] : first + i);
#pragma unroll
      for (int j = 0; j < 4; j++) cs[j] = cos_sin<WIDE>(pos * inv[j]);
    }
    f32x4 lo[HEADS], hi[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; k++) {
      if (WHOLE) {
        lo[k] = widen(x[k]);
        hi[k] = widen(y[k]);
      } else {
        const T* from = src + (u.row + i) * st + min(h + k * runs, h1 - 1) * sh;
        lo[k] = load4(from, d, end, false);
        hi[k] = load4(from, d2, end2, false);
      }
    }
    const int at = i, head = h;
    h += runs * HEADS;
    if (h >= h1) {
      h = h0 + run;
      i += at_once;
    }
    if (WHOLE && i < i1) fetch(i, h);
#pragma unroll
    for (int k = 0; k < HEADS; k++) {
      if (head + k * runs >= h1) break;
      if (!rest)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float l = lo[k][j], g = hi[k][j];
          turn<EXACT>(l, g, cs[j]);
          lo[k][j] = l;
          hi[k][j] = g;
        }
      put(at, head + k * runs, d, end, lo[k]);
      put(at, head + k * runs, d2, end2, hi[k]);
    }
  }
}

// Jobs of a unit along the grid's y: key heads, value heads, then q_parts parts of the
// rows (one pass of the threads each) by groups of q_heads query heads. Keys are turned
// into float32 in LDS, each pair by one thread, and stored from there as the writer's.
//
// Bound by memory: prompts (16 of up to 2048 tokens, 32 query and 8 key/value heads of
// 128 dims in bf16) take 129 us, 4.0 TB/s, where a large copy's rate gives 102. With 16
// query and 4 key/value heads of 256 dims 154 us of 102, 230 of 195 in float32; 8 and 2
// of 512 dims 233 of 102 and 287 of 195: every workgroup is held to the keys' LDS (68 KB
// at 256 dims, two on a CU; 132 at 512, one). Chunks of 512
// in float32, half of each head turning: 13 us of 8. Single tokens wait for the chain
// sequence, block, row, store: 64 sequences 8.2 us, one 7.0. What it took, in us of the
// prompts: keys turned where the writer loads them, each pair twice, and queries by a
// thread per four dims 326; cosines shared by heads and pairs turned once, but loads
// waited for one by one 212; cosines' factors and all loads of a thread under way
// before the first is used 161; the next heads' loads too, 16 heads a job 138 (8 heads
// 146: more cosines; 32 leave too few workgroups: the queries alone by 13% slower);
// all of a value job's loads under way too 129.
template <typename T, int NCM, bool WIDE>
__global__ __launch_bounds__(256, NCM <= 2 ? 4 : 2) void kv_write_rope_kernel(KvArgs a, KvRopeArgs r, int q_parts,
                                                                              int q_heads, bool by_row, bool vec,
                                                                              bool whole, bool whole_q) {
  extern __shared__ float keys[];  // [token of the unit][dim], rows of whole fours + 4
  const KvUnit u = kv_unit(a, blockIdx.x, by_row);
  if (!u.ok) return;
  const int64_t first = u.slot * 64 + u.place;
  int job = blockIdx.y;
  if (job >= 2 * a.hkv) {
    job -= 2 * a.hkv;
    const int part = job % q_parts, group = job / q_parts, n = (64 + q_parts - 1) / q_parts;
    const int i0 = part * n, i1 = q_parts == 1 ? u.n : min(u.n, i0 + n);
    if (i0 >= i1) return;
    const int h0 = group * q_heads, h1 = min(r.H, h0 + q_heads);
    auto put = [&](bool v4, int i, int h, int d, int end, f32x4 x) {
      store4((T*)r.q_out + ((u.row + i) * r.H + h) * a.D, d, end, v4, x);
    };
    if (whole_q)
      turn_rows<T, WIDE, false, 4, true>(a, r, u, first, (const T*)r.q, r.q_st, r.q_sh, i0, i1, h0, h1,
                                         [&](int i, int h, int d, int end, f32x4 x) { put(true, i, h, d, end, x); });
    else
      turn_rows<T, WIDE, false, 1, false>(a, r, u, first, (const T*)r.q, r.q_st, r.q_sh, i0, i1, h0, h1,
                                          [&](int i, int h, int d, int end, f32x4 x) { put(false, i, h, d, end, x); });
    return;
  }
  const int id = kv_block(a, u.b, u.slot);
  if (id < 0) return;
  const int h = job % a.hkv;
  if (job >= a.hkv) {
    write_block<T, NCM>(a, u, id, h, 1, vec, [&](int64_t row) { return (const T*)r.v + row * r.v_st + h * r.v_sh; });
    return;
  }
  const int stride = (a.D + 3) / 4 * 4 + 4;
  if (whole)
    turn_rows<T, WIDE, true, 1, true>(a, r, u, first, (const T*)r.k, r.k_st, r.k_sh, 0, u.n, h, h + 1,
                                      [&](int i, int, int d, int, f32x4 x) { *(f32x4*)(keys + i * stride + d) = x; });
  else
    turn_rows<T, WIDE, true, 1, false>(
        a, r, u, first, (const T*)r.k, r.k_st, r.k_sh, 0, u.n, h, h + 1,
        [&](int i, int, int d, int end, f32x4 x) { store4(keys + i * stride, d, end, false, x); });
  __syncthreads();
  write_block<float, NCM>(a, u, id, h, 0, true, [&](int64_t row) { return keys + (row - u.row) * stride; });
}

// One workgroup reads back one (block, head, keys or values): the thread
// layout of the writer, a slice of values transposed through LDS. A code
// times a power of two has four bits, exact in either type. Rows without a
// block (a bad table entry, a position below zero) become NaN. Bound by its
// bytes: 32 sequences of up to 2000 tokens to float32, 43 us, 4.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, T* __restrict__ k, T* __restrict__ v, bool by_row,
                                                      bool vec) {
  __shared__ uint32_t tile[64 * 17];
  const KvUnit u = kv_unit(a, blockIdx.x, by_row);
  if (!u.ok) return;
  const int id = kv_block(a, u.b, u.slot);
  const int h = blockIdx.y, part = blockIdx.z;
  const int tid = threadIdx.x, dq = tid & 15, ta = (tid >> 4) & 3, tb = tid >> 6;
  const int t0 = ta * 16 + tb * 4;
  T* dst = part ? v : k;
  const int end = u.place + u.n;
  const float scale = id < 0 ? __builtin_nanf("") : a.scales[((int64_t)id * a.hkv + h) * 2 + part];
  const uint8_t* src = id < 0 ? nullptr : kv_part(a, id, h, part);
  for (int c = 0; c < a.nc; c++) {
    f32x4 x[4];
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i;
        uint32_t w = 0;
        if (src && t >= u.place && t < end) w = *reinterpret_cast<const uint32_t*>(src + c * 4096 + t * 64 + dq * 4);
        x[i] = unpack4(w);
      }
    } else {
      uint4 w = make_uint4(0, 0, 0, 0);
      const int row = tid >> 2, b = tid & 3;
      if (src) w = *reinterpret_cast<const uint4*>(src + (int64_t)(c * 64 + row) * 64 + b * 16);
      if (c) __syncthreads();
      uint32_t* to = tile + row * 17 + b * 4;
      to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f32x4 y = unpack4(tile[(dq * 4 + j) * 17 + tb * 4 + ta]);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i][j] = y[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int t = t0 + i;
      if (t >= u.place && t < end)
        store4(dst + ((u.row + (t - u.place)) * a.hkv + h) * a.D, c * 64 + dq * 4, a.D, vec, x[i] * scale);
    }
  }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T>
int write_t(fa_ctx* ctx, const KvArgs& a, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
            int64_t v_sh, hipStream_t s) {
  bool by_row;
  const int64_t units = kv_units(a.rows, a.nseq, &by_row);
  const bool vec = aligned(k, 4 * sizeof(T)) && aligned(v, 4 * sizeof(T)) && (k_st | k_sh | v_st | v_sh) % 4 == 0;
  const dim3 grid((unsigned)units, (unsigned)a.hkv, 2);
  const T *kt = (const T*)k, *vt = (const T*)v;
#define FA_KV_W(N) kv_write_kernel<T, N><<<grid, 256, 0, s>>>(a, kt, k_st, k_sh, vt, v_st, v_sh, by_row, vec)
  if (a.nc <= 1) FA_KV_W(1);
  else if (a.nc <= 2) FA_KV_W(2);
  else if (a.nc <= 4) FA_KV_W(4);
  else FA_KV_W(8);
#undef FA_KV_W
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

template <typename T, int NCM, bool WIDE>
int write_rope_nc(fa_ctx* ctx, const KvArgs& a, const KvRopeArgs& r, hipStream_t s) {
  bool by_row;
  const int64_t units = kv_units(a.rows, a.nseq, &by_row);
  const size_t al = 4 * sizeof(T);
  const bool vec = aligned(r.k, al) && aligned(r.v, al) && (r.k_st | r.k_sh | r.v_st | r.v_sh) % 4 == 0;
  const bool vec_q = r.q && aligned(r.q, al) && aligned(r.q_out, al) && (r.q_st | r.q_sh) % 4 == 0;
  const bool fours = a.D % 4 == 0 && r.half % 4 == 0;
  const int slots = (r.half + 3) / 4 + (a.D - 2 * r.half + 3) / 4;
  const int q_parts = by_row ? 1 : (64 + 256 / slots - 1) / (256 / slots);
  int q_heads = 16;  // (a grid's y holds 65535)
  while (2 * a.hkv + (int64_t)q_parts * ((r.H + q_heads - 1) / q_heads) > 65535) q_heads *= 2;
  const size_t lds = (size_t)64 * ((a.D + 3) / 4 * 4 + 4) * sizeof(float);
  auto kernel = kv_write_rope_kernel<T, NCM, WIDE>;
  static std::atomic<uint64_t> ready{0};  // devices that know of more than 64 KB, the first 64
  const uint64_t bit = ctx->device < 64 ? uint64_t(1) << ctx->device : 0;
  if (lds > 48 * 1024 && !(ready.load() & bit)) {
    FA_HIP_CHECK(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                          64 * (2 * kKvMaxPairs + 4) * (int)sizeof(float)));
    ready.fetch_or(bit);
  }
  const unsigned jobs = (unsigned)(2 * a.hkv + q_parts * ((r.H + q_heads - 1) / q_heads));
  kernel<<<dim3((unsigned)units, jobs), 256, lds, s>>>(a, r, q_parts, q_heads, by_row, vec, vec && fours,
                                                       vec_q && fours);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

template <typename T>
int write_rope_t(fa_ctx* ctx, const KvArgs& a, const KvRopeArgs& r, hipStream_t s) {
  // bases below 1 alone turn by more than the position, which is below 2^31
  const double most = std::max(r.inv[0], r.inv[r.half - 1]);
  return most > 1      ? write_rope_nc<T, 8, true>(ctx, a, r, s)
         : a.nc <= 1   ? write_rope_nc<T, 1, false>(ctx, a, r, s)
         : a.nc <= 2   ? write_rope_nc<T, 2, false>(ctx, a, r, s)
         : a.nc <= 4   ? write_rope_nc<T, 4, false>(ctx, a, r, s)
                       : write_rope_nc<T, 8, false>(ctx, a, r, s);
}

}  // namespace

int launch_kv_write_rope(fa_ctx* ctx, const KvArgs& a, int dtype, const KvRopeArgs& r, hipStream_t s) {
  return dtype == FA_DT_F32 ? write_rope_t<float>(ctx, a, r, s) : write_rope_t<uint16_t>(ctx, a, r, s);
}

int64_t kv_grid(const KvArgs& a) {
  bool by_row;
  return kv_units(a.rows, a.nseq, &by_row);
}

int launch_kv_write(fa_ctx* ctx, const KvArgs& a, int dtype, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                    int64_t v_st, int64_t v_sh, hipStream_t s) {
  return dtype == FA_DT_F32 ? write_t<float>(ctx, a, k, k_st, k_sh, v, v_st, v_sh, s)
                            : write_t<uint16_t>(ctx, a, k, k_st, k_sh, v, v_st, v_sh, s);
}

int launch_kv_read(fa_ctx* ctx, const KvArgs& a, int dtype, void* k, void* v, hipStream_t s) {
  bool by_row;
  const int64_t units = kv_units(a.rows, a.nseq, &by_row);
  const dim3 grid((unsigned)units, (unsigned)a.hkv, 2);
  const size_t al = dtype == FA_DT_F32 ? 16 : 8;
  const bool vec = a.D % 4 == 0 && aligned(k, al) && aligned(v, al);
  if (dtype == FA_DT_F32) kv_read_kernel<float><<<grid, 256, 0, s>>>(a, (float*)k, (float*)v, by_row, vec);
  else kv_read_kernel<uint16_t><<<grid, 256, 0, s>>>(a, (uint16_t*)k, (uint16_t*)v, by_row, vec);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

}  // namespace fa
