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
// 42 us after other work, 33 one after another, where the bytes take 28 at a large
// copy's rate (in float32 41 one after another, of 46): each of 6288 workgroups waits
// for its sequence, its block and its rows in turn, then reduces and stores with
// nothing of the next under way. Single tokens are bound by that chain and the
// write-back of the 128 lines that one token's values touch in a head (64 sequences,
// one float32 token each, written 7.1 us).
// load(row, d): four values of the part from dim d on in row `row`, zeros past D.
template <int NCM, typename F>
__device__ __forceinline__ void write_block(const KvArgs& a, const KvUnit& u, int id, int h, int part, F load) {
  __shared__ float red[4];
  __shared__ uint32_t tile[64 * 17];
  const int tid = threadIdx.x, dq = tid & 15, ta = (tid >> 4) & 3, tb = tid >> 6;
  const int t0 = ta * 16 + tb * 4;
  const int end = u.place + u.n;
  f32x4 x[NCM][4];
  float big = 0.f;
#pragma unroll
  for (int c = 0; c < NCM; c++)
    if (c < a.nc)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = t0 + i;
        x[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (t >= u.place && t < end) x[c][i] = load(u.row + (t - u.place), c * 64 + dq * 4);
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

template <typename T, int NCM>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a, const T* __restrict__ k, int64_t k_st, int64_t k_sh,
                                                       const T* __restrict__ v, int64_t v_st, int64_t v_sh,
                                                       bool by_row, bool vec) {
  const KvUnit u = kv_unit(a, blockIdx.x, by_row);
  if (!u.ok) return;
  const int id = kv_block(a, u.b, u.slot);
  if (id < 0) return;
  const int h = blockIdx.y, part = blockIdx.z;
  const T* src = part ? v : k;
  const int64_t st = part ? v_st : k_st, sh = part ? v_sh : k_sh;
  write_block<NCM>(a, u, id, h, part, [&](int64_t row, int d) { return load4(src + row * st + h * sh, d, a.D, vec); });
}

// Four values of a head from dim d on, turned: dim i < half of the first 2 *
// half becomes x_i cos - x_{i + half} sin, dim i + half x_{i + half} cos + x_i
// sin, the angle position * inv_i in float64, cos and sin rounded to float32 (as
// fa_rope's tables), the products exact in float64.
template <typename T>
__device__ __forceinline__ f32x4 load_turned(const KvRopeArgs& r, const T* p, int64_t position, int d, int D, bool vec) {
  f32x4 x = load4(p, d, D, vec);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int i = d + j;
    if (i >= 2 * r.half) continue;
    const bool up = i >= r.half;
    const int pair = up ? i - r.half : i;
    double sn, cs;
    sincos((double)position * r.inv[pair], &sn, &cs);
    const double c = (double)(float)cs, s = (double)(float)sn;
    const double other = (double)to_f32(p[up ? pair : i + r.half]);
    x[j] = (float)((double)x[j] * c + (up ? other : -other) * s);
  }
  return x;
}

template <typename T, int NCM>
__global__ __launch_bounds__(256) void kv_write_rope_kernel(KvArgs a, KvRopeArgs r, bool by_row, bool vec) {
  const KvUnit u = kv_unit(a, blockIdx.x, by_row);
  if (!u.ok) return;
  const int64_t first = u.slot * 64 + u.place;  // position of the unit's first row in its sequence
  auto position = [&](int64_t row) { return r.positions ? (int64_t)r.positions[row] : first + (row - u.row); };
  const int job = blockIdx.y;
  if (job < 2 * a.hkv) {
    const int id = kv_block(a, u.b, u.slot);
    if (id < 0) return;
    const int h = job >> 1, part = job & 1;
    write_block<NCM>(a, u, id, h, part, [&](int64_t row, int d) {
      if (part) return load4((const T*)r.v + row * r.v_st + h * r.v_sh, d, a.D, vec);
      return load_turned(r, (const T*)r.k + row * r.k_st + h * r.k_sh, position(row), d, a.D, vec);
    });
    return;
  }
  // queries: a thread turns whole pairs, so that q_out may be q
  const int h = job - 2 * a.hkv;
  const int pairs = (r.half + 3) / 4, words = pairs + (a.D - 2 * r.half + 3) / 4;
  const bool vec2 = vec && r.half % 4 == 0, vec_out = vec && a.D % 4 == 0;
  for (int i = threadIdx.x; i < u.n * words; i += 256) {
    const int64_t row = u.row + i / words;
    const int w = i % words;
    const T* p = (const T*)r.q + row * r.q_st + h * r.q_sh;
    T* o = (T*)r.q_out + (row * r.H + h) * a.D;
    if (w >= pairs) {
      const int d = 2 * r.half + (w - pairs) * 4;
      store4(o, d, a.D, vec_out && r.half % 2 == 0, load4(p, d, a.D, vec && r.half % 2 == 0));
      continue;
    }
    f32x4 lo = load4(p, w * 4, r.half, vec), hi = load4(p + r.half, w * 4, r.half, vec2);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      double sn, cs;
      sincos((double)position(row) * r.inv[min(w * 4 + j, r.half - 1)], &sn, &cs);
      const double c = (double)(float)cs, s = (double)(float)sn, x = (double)lo[j], y = (double)hi[j];
      lo[j] = (float)(x * c - y * s);
      hi[j] = (float)(y * c + x * s);
    }
    store4(o, w * 4, r.half, vec_out, lo);
    store4(o + r.half, w * 4, r.half, vec_out && vec2, hi);
  }
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

template <typename T>
int write_rope_t(fa_ctx* ctx, const KvArgs& a, const KvRopeArgs& r, hipStream_t s) {
  bool by_row;
  const int64_t units = kv_units(a.rows, a.nseq, &by_row);
  const size_t al = 4 * sizeof(T);
  const bool vec = aligned(r.k, al) && aligned(r.v, al) && (r.k_st | r.k_sh | r.v_st | r.v_sh) % 4 == 0 &&
                   (!r.q || (aligned(r.q, al) && aligned(r.q_out, al) && (r.q_st | r.q_sh) % 4 == 0));
  const dim3 grid((unsigned)units, (unsigned)(2 * a.hkv + r.H));
  if (a.nc <= 1) kv_write_rope_kernel<T, 1><<<grid, 256, 0, s>>>(a, r, by_row, vec);
  else if (a.nc <= 2) kv_write_rope_kernel<T, 2><<<grid, 256, 0, s>>>(a, r, by_row, vec);
  else if (a.nc <= 4) kv_write_rope_kernel<T, 4><<<grid, 256, 0, s>>>(a, r, by_row, vec);
  else kv_write_rope_kernel<T, 8><<<grid, 256, 0, s>>>(a, r, by_row, vec);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
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
