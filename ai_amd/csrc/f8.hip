// Products with weights in 8 bits: C = epilogue(A^ . W^T) with A^ and W rows of
// e4m3 codes and one power of two for each 128 columns of a row.
//
// bf16 results come from the 8-bit matrix units, which take the two scales of a
// block with the product (32x32x64: half a block of a row is one operand). They cut
// each product of a group of eight to a multiple of 2^-13 of the power of two below
// the group's largest before they add it: 1.5e-5 of the result's 2-norm (normal
// operands; 5e-5 with long tails), where rounding to bf16 adds 1.7e-3. float32
// results need the sums that lose nothing: a code times its scale is exact in bf16,
// so they come from the bf16 units, whose products are exact and sums float32.
#include <algorithm>
#include <type_traits>

#include "f8.h"
#include "gemm_common.h"

namespace fa {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// 16 lanes take a block of 128 columns, eight values a lane, a wave 4 U neighbouring
// blocks, all their loads under way at once. The lanes of a row's last block also
// write the scale bytes that pad the row.
template <typename T, int U>
__global__ __launch_bounds__(256) void f8_write_kernel(F8View w, const T* __restrict__ x, int64_t ldx, int kb, int ks,
                                                       bool vec, uint32_t* zero, int zeros) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < zeros; i += gridDim.x * 256) zero[i] = 0;
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int64_t first = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (4 * U);
  const int64_t blocks = w.n * kb, row0 = blocks >> 32 ? first / kb : (uint32_t)first / (uint32_t)kb;
  const uint32_t b0 = (uint32_t)(first - row0 * kb);
  f32x4 v[U][2];
  int64_t row[U];
  int b[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t at = b0 + u * 4 + (lane >> 4);
    row[u] = row0 + at / (uint32_t)kb;
    b[u] = (int)(at % (uint32_t)kb);
    const bool in = first + u * 4 + (lane >> 4) < blocks;
    const T* from = x + min(row[u], w.n - 1) * ldx;
    const int d = b[u] * kF8Block + l * 8, k = in ? (int)w.k : 0;
    if constexpr (sizeof(T) == 2) {
      if (vec && d + 8 <= k) {
        const uint4 q = *reinterpret_cast<const uint4*>(from + d);
        v[u][0] = f32x4{__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xFFFF0000u), __uint_as_float(q.y << 16),
                        __uint_as_float(q.y & 0xFFFF0000u)};
        v[u][1] = f32x4{__uint_as_float(q.z << 16), __uint_as_float(q.z & 0xFFFF0000u), __uint_as_float(q.w << 16),
                        __uint_as_float(q.w & 0xFFFF0000u)};
        continue;
      }
    }
    v[u][0] = load4(from, d, k, vec && sizeof(T) == 4);
    v[u][1] = load4(from, d + 4, k, vec && sizeof(T) == 4);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float y = v[u][j >> 2][j & 3];
      join_max(y, big);
      v[u][j >> 2][j & 3] = y;
    }
    // over the 16 lanes: rotations of a row of lanes
    big = fmaxf(big, dpp_f32<0x128>(big));
    big = fmaxf(big, dpp_f32<0x124>(big));
    big = fmaxf(big, dpp_f32<0x122>(big));
    big = fmaxf(big, dpp_f32<0x121>(big));
    const int e = scale_exp(big);
    if (e == kMaxExp) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[u][j >> 2][j & 3] = clamp_top(v[u][j >> 2][j & 3]);
    }
    const float inv = exp2_int(-e);
    if (first + u * 4 + (lane >> 4) >= blocks) continue;
    *reinterpret_cast<uint2*>(w.codes + row[u] * w.stride + b[u] * kF8Block + l * 8) =
        make_uint2(pack4(v[u][0][0] * inv, v[u][0][1] * inv, v[u][0][2] * inv, v[u][0][3] * inv),
                   pack4(v[u][1][0] * inv, v[u][1][1] * inv, v[u][1][2] * inv, v[u][1][3] * inv));
    if (l == 0) w.scales[row[u] * ks + b[u]] = (uint8_t)(e + 127);
    if (b[u] == kb - 1 && kb + l < ks) w.scales[row[u] * ks + kb + l] = 127;
  }
}

// Bound by memory, a word of four codes a thread: 8192 x 8192 to float32 68 us, 4.9 TB/s, to
// bf16 38.
template <typename T>
__global__ __launch_bounds__(256) void f8_read_kernel(F8View w, T* __restrict__ out, int64_t ldo, int kb, int ks,
                                                      bool vec) {
  const int64_t words = w.n * kb * 32;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / (kb * 32);
    const int word = (int)(i - row * (kb * 32));
    const f32x4 v = unpack4(*reinterpret_cast<const uint32_t*>(w.codes + row * w.stride + word * 4));
    const float s = exp2_int((int)w.scales[row * ks + (word >> 5)] - 127);
    store4(out + row * ldo, word * 4, (int)w.k, vec, v * s);
  }
}

struct GemmParams {
  int64_t m, n, k;
  int kb, ks;   // blocks of a row, its scale bytes
  int64_t a_st;  // bytes from a row of A's codes to the next
  const uint8_t *a, *as, *w, *ws;  // codes and scale bytes
  fa_epilogue e;
  int vec_bias, vec_mul, vec_residual, vec_c;  // aligned for four values at a time
  int64_t ldc;
  int split;                       // waves that share a row's blocks (few rows)
  int parts, per;                  // parts of K, each of `per` blocks (a multiple of 4) or what is left
  float* part;                     // [tile][part][BM * BN], in the order of the threads that hold them
  uint32_t* count;                 // [tile] parts that are there
};

// Two codes times a power of two, exact in bf16.
__device__ __forceinline__ uint32_t widen2(uint32_t w, float s, bool hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false);
  return __builtin_bit_cast(uint32_t, r);
}
// Eight codes as an operand of the bf16 units.
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, float s) {
  const uint4 r = make_uint4(widen2(lo, s, false), widen2(lo, s, true), widen2(hi, s, false), widen2(hi, s, true));
  return __builtin_bit_cast(bf16x8, r);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }  // 2^(byte - 127)

// Bias, row scale and activation of four neighbouring values.
__device__ __forceinline__ f32x4 before_mul(const GemmParams& p, f32x4 v, int64_t row, int col) {
  if (p.e.bias) v = v + load4(p.e.bias, col, (int)p.n, p.vec_bias);
  if (p.e.row_scale) v = v * p.e.row_scale[min(row, p.m - 1)];
  if (p.e.act == FA_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = fmaxf(v[j], 0.f);
  } else if (p.e.act != FA_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = v[j];
      v[j] = p.e.act == FA_ACT_GELU ? gelu_tanh_ref(x) : tanh_ref(x);
    }
  }
  return v;
}

// R rows of C, four neighbouring values of each, through the rest of the epilogue:
// what it reads of all of them under way at once. Rows and columns past C are left out.
template <int R, typename T>
__device__ __forceinline__ void put4(const GemmParams& p, T* c, const int64_t (&row)[R], int64_t col, f32x4 (&v)[R]) {
  const int n = (int)p.n, at = (int)col;
  if (p.e.mul) {
    f32x4 x[R];
#pragma unroll
    for (int i = 0; i < R; i++) x[i] = load4(p.e.mul + min(row[i], p.m - 1) * p.e.ldm, at, n, p.vec_mul);
#pragma unroll
    for (int i = 0; i < R; i++) v[i] = v[i] * x[i];
  }
  if (p.e.residual) {
    f32x4 x[R];
#pragma unroll
    for (int i = 0; i < R; i++) x[i] = load4(p.e.residual + min(row[i], p.m - 1) * p.e.ldr, at, n, p.vec_residual);
#pragma unroll
    for (int i = 0; i < R; i++) v[i] = v[i] + x[i];
  }
#pragma unroll
  for (int i = 0; i < R; i++)
    if (row[i] < p.m) store4(c + row[i] * p.ldc, at, n, p.vec_c, v[i]);
}

// ---- few rows -----------------------------------------------------------------------

// Up to 16 rows. A wave computes 16 columns of C over every split-th block of 128, on
// the bf16 units (whose operands, codes times powers of two, are exact: the time goes
// into reading W, not into products); the waves of a column group add up through LDS, in
// their order. Both operands come straight from memory in the units' order, four blocks
// under way: a lane (row r of 16, g of 4) holds bytes 16 g .. and 64 + 16 g .. of its
// row's block, so that four lanes read 64 bytes together. 16 x 4096 x 4096 takes 9.7 us (and
// the launch before it, which quantises A, 3.0): each wave's four blocks are one round of
// loads, so what is left is that round (16 rows an instruction, a byte for each scale),
// widening both operands and the join; which of them was not taken apart.
constexpr int kFewWaves = 8, kFewDeep = 4;
template <typename TC>
__device__ __forceinline__ void f8_few(const GemmParams& p, TC* c) {
  __shared__ f32x4 part[kFewWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int group = wave / p.split, ks = wave % p.split;  // split divides kFewWaves
  const int64_t n0 = ((int64_t)blockIdx.x * (kFewWaves / p.split) + group) * 16;
  const int64_t n_row = min(n0 + r, p.n - 1), m_row = min((int64_t)r, p.m - 1);
  const uint8_t *w = p.w + n_row * p.kb * kF8Block + g * 16, *ws = p.ws + n_row * p.ks;
  const uint8_t *a = p.a + m_row * p.a_st + g * 16, *as = p.as + m_row * p.ks;
  struct Block {
    uint4 lo, hi;
    uint32_t s;
  };
  auto get = [](const uint8_t* codes, const uint8_t* scales, int b) {
    const uint8_t* q = codes + (int64_t)b * kF8Block;
    return Block{*reinterpret_cast<const uint4*>(q), *reinterpret_cast<const uint4*>(q + 64), scales[b]};
  };
  auto widen = [](const Block& x, bf16x8 (&o)[4]) {
    const float s = scale_of(x.s);
    o[0] = widen8(x.lo.x, x.lo.y, s);
    o[1] = widen8(x.lo.z, x.lo.w, s);
    o[2] = widen8(x.hi.x, x.hi.y, s);
    o[3] = widen8(x.hi.z, x.hi.w, s);
  };
  f32x4 acc = {};
  Block cw[kFewDeep], ca[kFewDeep];
#pragma unroll
  for (int d = 0; d < kFewDeep; d++)
    if (ks + d * p.split < p.kb) {
      cw[d] = get(w, ws, ks + d * p.split);
      ca[d] = get(a, as, ks + d * p.split);
    }
  for (int b0 = ks; b0 < p.kb; b0 += kFewDeep * p.split) {
#pragma unroll
    for (int d = 0; d < kFewDeep; d++) {
      const int b = b0 + d * p.split, next = b + kFewDeep * p.split;
      if (b >= p.kb) break;  // (uniform in the wave)
      bf16x8 x[4], y[4];
      widen(cw[d], x);
      widen(ca[d], y);
      if (next < p.kb) {
        cw[d] = get(w, ws, next);
        ca[d] = get(a, as, next);
      }
#pragma unroll
      for (int q = 0; q < 4; q++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[q], y[q], acc, 0, 0, 0);
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  // lane: row r of A, columns 4 g .. + 3
  const int64_t col = n0 + g * 4;
  if (ks != 0 || col >= p.n) return;
  f32x4 one[1] = {part[wave][lane]};
  for (int s = 1; s < p.split; s++) one[0] = one[0] + part[wave + s][lane];
  const int64_t row[1] = {r};
  one[0] = before_mul(p, one[0], r, (int)col);
  put4(p, c, row, col, one);
}

template <typename TC>
__global__ __launch_bounds__(kFewWaves * 64) void f8_few_kernel(GemmParams p, TC* c) {
  f8_few(p, c);
}

// ---- tiles ---------------------------------------------------------------------------------

// Workgroup barrier after the wave's LDS reads are done and its direct loads to LDS have
// landed but for the LEFT last ones.
template <int LEFT = 0>
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | (LEFT >> 4) << 14);  // (the other counters to 0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Order of a half block's READS reads of operands, LOADS loads to LDS and PRODUCTS
// products (0: left to the compiler): the reads in turn with products, so that they
// arrive under them, the loads among the first half of these (at the next meeting
// every load has to have landed).
template <int READS, int LOADS, int PRODUCTS>
__device__ __forceinline__ void mix() {
  constexpr int R = PRODUCTS ? (READS + PRODUCTS - 1) / PRODUCTS : 0, L = PRODUCTS ? (2 * LOADS + PRODUCTS - 1) / PRODUCTS : 0;
#pragma unroll
  for (int i = 0; i < PRODUCTS; i++) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if (i * R < READS) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    if (i * L < LOADS) __builtin_amdgcn_sched_group_barrier(0x20, L, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// Leaves a thread's sums of a part of K beside the other parts' of the tile. The
// workgroup that comes last (true) adds them up, in their order: the result does not
// depend on which one that is. last: a word of LDS.
template <int SIZE>
__device__ __forceinline__ bool join(const GemmParams& p, f32x16& x, int tile, int part, int* last) {
  float* to = p.part + ((int64_t)tile * p.parts + part) * SIZE + threadIdx.x * 2;
#pragma unroll
  for (int q = 0; q < 8; q++) put2(to + q * 512, x[2 * q], x[2 * q + 1]);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's are where every workgroup finds them
  __syncthreads();
  if (threadIdx.x == 0)
    *last = __hip_atomic_fetch_add(p.count + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)p.parts - 1;
  __syncthreads();
  if (!*last) return false;
  const float* from = p.part + (int64_t)tile * p.parts * SIZE + threadIdx.x * 2;
  x = f32x16{};
  for (int s = 0; s < p.parts; s++, from += SIZE) {
    float2 y[8];
#pragma unroll
    for (int q = 0; q < 8; q++) y[q] = get2(from + q * 512);
#pragma unroll
    for (int q = 0; q < 8; q++) {
      x[2 * q] += y[q].x;
      x[2 * q + 1] += y[q].y;
    }
  }
  return true;
}

// Four waves, WM of them one below the other, each with its part of the tile in 32 x 32
// products. A block of both operands (128 bytes of each row) goes straight from memory
// to LDS, D blocks held: at the middle of a block the waves have read all of it, meet
// once, and start the loads of the block D on into its place. Rows lie 128 bytes
// apart, their 16-byte pieces permuted by the row (piece j at j ^ (row & 7)), so that
// eight lanes reading the same piece of eight rows use all banks. Operands of the
// next half block are read while the products of this one run. F8: on the 8-bit units.
//
// Large tiles are bound by products and two blocks are enough: 8192 x 8192 x 8192 with a
// residual takes 545 to 560 us, 2.0 PFLOP/s (its products alone at 2.76), without it 509,
// 4096^3 76 (quantising A among each: 38 of 8192^3). Small ones
// wait for memory, a latency for each D - 1 blocks: 128 x 4096 x 4096 22 us with two
// blocks, 13 with four. 1 x 262144 x 768 in float32 takes 45 us, 4.6 TB/s; 16 x 16384 x
// 4096 16 us, 4.1 TB/s. float32 results, whose operands every wave widens for itself:
// 8192^3 991 us, 1.1 PFLOP/s, 4096^3 146.
template <int BM, int BN, int WM, int D, bool F8, typename TC>
__device__ __forceinline__ void f8_tile(const GemmParams& p, TC* c, int tiles_m, int tiles_n) {
  constexpr int WN = 4 / WM, MW = BM / WM, NW = BN / WN;  // waves each way, their parts of the tile
  constexpr int FM = MW / 32, FN = NW / 32, NA = BM * 8 / 256, NB = BN * 8 / 256;
  constexpr bool kJoins = FM * FN == 1;  // K may be split
  constexpr int kStage = (BM + BN) * kF8Block;
  __shared__ __attribute__((aligned(16))) uint8_t S0[kStage], S1[kStage], S2[D > 2 ? kStage : 16],
      S3[D > 2 ? kStage : 16];  // (arrays of their own: reads of one need not wait for loads to another)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int64_t kp = (int64_t)p.kb * kF8Block;
  // Tiles of an XCD's run are taken in groups of 4 tile rows, down the columns: the
  // ones that run together share their rows of A and of W in its L2.
  int tm, tn, tile, part = 0;
  {
    if (kJoins && p.parts > 1) {
      tile = blockIdx.x % (tiles_m * tiles_n);
      part = blockIdx.x / (tiles_m * tiles_n);
    } else {
      tile = xcd_tile(tiles_m, tiles_n);
    }
    constexpr int G = 4;
    const int group = tile / (G * tiles_n), rows = min(G, tiles_m - group * G), at = tile - group * G * tiles_n;
    tm = group * G + at % rows;
    tn = at / rows;
  }
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  // the tile's first rows (the same for the workgroup), and a thread's pieces from there
  const int first_block = part * p.per, kb = min(p.kb - first_block, p.per);
  const int64_t skip = (int64_t)first_block * kF8Block;
  const uint8_t *a0 = p.a + m0 * p.a_st + skip, *b0 = p.w + n0 * kp + skip;
  uint32_t ga[NA], gb[NB];
  {
    const int row = tid >> 3, piece = (tid & 7) ^ (row & 7);
    const int rows_a = (int)min(p.m - m0, (int64_t)BM) - 1, rows_b = (int)min(p.n - n0, (int64_t)BN) - 1;
#pragma unroll
    for (int i = 0; i < NA; i++) ga[i] = (uint32_t)min(i * 32 + row, rows_a) * (uint32_t)p.a_st + piece * 16;
#pragma unroll
    for (int i = 0; i < NB; i++) gb[i] = (uint32_t)min(i * 32 + row, rows_b) * (uint32_t)kp + piece * 16;
  }
  auto stage = [&](uint8_t* s, int b) {
    const uint8_t *a = a0 + (int64_t)b * kF8Block, *w = b0 + (int64_t)b * kF8Block;
#pragma unroll
    for (int i = 0; i < NA; i++)
      __builtin_amdgcn_global_load_lds(a + ga[i], (__attribute__((address_space(3))) void*)(s + (i * 256 + wave * 64) * 16), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < NB; i++)
      __builtin_amdgcn_global_load_lds(
          w + gb[i], (__attribute__((address_space(3))) void*)(s + BM * kF8Block + (i * 256 + wave * 64) * 16), 16, 0, 0);
  };
  // operands: row lane % 32, bytes 32 (lane / 32) .. + 31 of each half block
  const int row = lane & 31, half = lane >> 5;
  const int a_at = (wm * MW + row) * kF8Block, b_at = BM * kF8Block + (wn * NW + row) * kF8Block;
  int piece[2][2];
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int j = 0; j < 2; j++) piece[h][j] = ((h * 4 + half * 2 + j) ^ (row & 7)) * 16;
  struct Ops {
    i32x8 a[FM], b[FN];
  };
  auto two = [&](const uint8_t* s, int h) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(s + piece[h][0]), y = *reinterpret_cast<const i32x4*>(s + piece[h][1]);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read = [&](const uint8_t* s, int h, Ops& o) {
#pragma unroll
    for (int f = 0; f < FN; f++) o.b[f] = two(s + b_at + f * 32 * kF8Block, h);
#pragma unroll
    for (int f = 0; f < FM; f++) o.a[f] = two(s + a_at + f * 32 * kF8Block, h);
  };
  // scale bytes of four blocks at a time
  const uint8_t *as0 = p.as + m0 * p.ks + first_block, *bs0 = p.ws + n0 * p.ks + first_block;
  uint32_t sa[FM], sb[FN];
#pragma unroll
  for (int f = 0; f < FM; f++)
    sa[f] = (uint32_t)min((int64_t)(wm * MW + f * 32 + row), p.m - 1 - m0) * (uint32_t)p.ks;
#pragma unroll
  for (int f = 0; f < FN; f++)
    sb[f] = (uint32_t)min((int64_t)(wn * NW + f * 32 + row), p.n - 1 - n0) * (uint32_t)p.ks;
  uint32_t xa[FM], xb[FN], na[FM], nb[FN];
  auto scales = [&](int b) {  // (rows of scale bytes are whole groups of four)
    const int at = min(b, p.ks - 4 - first_block);
#pragma unroll
    for (int f = 0; f < FM; f++) na[f] = *reinterpret_cast<const uint32_t*>(as0 + at + sa[f]);
#pragma unroll
    for (int f = 0; f < FN; f++) nb[f] = *reinterpret_cast<const uint32_t*>(bs0 + at + sb[f]);
  };
  f32x16 acc[FM][FN] = {};
  auto multiply = [&](const Ops& o, auto sel) {
    constexpr int SEL = decltype(sel)::value;  // the block's byte of the scales
    if constexpr (F8) {
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(o.a[i], o.b[j], acc[i][j], 0, 0, SEL, (int)xa[i], SEL, (int)xb[j]);
    } else {
      float ea[FM], eb[FN];
#pragma unroll
      for (int i = 0; i < FM; i++) ea[i] = scale_of(xa[i] >> (8 * SEL) & 255);
#pragma unroll
      for (int j = 0; j < FN; j++) eb[j] = scale_of(xb[j] >> (8 * SEL) & 255);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        bf16x8 x[FM], y[FN];
#pragma unroll
        for (int i = 0; i < FM; i++) x[i] = widen8((uint32_t)o.a[i][2 * q], (uint32_t)o.a[i][2 * q + 1], ea[i]);
#pragma unroll
        for (int j = 0; j < FN; j++) y[j] = widen8((uint32_t)o.b[j][2 * q], (uint32_t)o.b[j][2 * q + 1], eb[j]);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[i], y[j], acc[i][j], 0, 0, 0);
      }
    }
  };
  Ops X, Y;
  // Block b, in s (its first half in X already); the next one is in `next`. Past the
  // last block the last is loaded again and not used: no branch in the loop.
  static_assert(D == 2 || D == 4, "a group of four blocks goes through the places evenly");
  uint8_t *const s2 = D > 2 ? S2 : S0, *const s3 = D > 2 ? S3 : S1;
  auto block = [&](uint8_t* s, uint8_t* next, int b, auto sel) {
    read(s, 1, Y);
    multiply(X, sel);
    mix<2 * (FM + FN), 0, F8 ? FM * FN : 0>();
    tile_barrier<(D - 2) * (NA + NB)>();
    stage(s, min(b + D, kb - 1));
    read(next, 0, X);
    multiply(Y, sel);
    mix<2 * (FM + FN), NA + NB, F8 ? FM * FN : 0>();
  };
  using std::integral_constant;
  if (kb > 0) {
    scales(0);
    stage(S0, 0);
    stage(S1, min(1, kb - 1));
    if constexpr (D > 2) {
      stage(S2, min(2, kb - 1));
      stage(S3, min(3, kb - 1));
    }
    tile_barrier<(D - 1) * (NA + NB)>();
    read(S0, 0, X);
    int b = 0;
    for (; b + 4 <= kb; b += 4) {
#pragma unroll
      for (int f = 0; f < FM; f++) xa[f] = na[f];
#pragma unroll
      for (int f = 0; f < FN; f++) xb[f] = nb[f];
      scales(b + 4);
      block(S0, S1, b, integral_constant<int, 0>());
      block(S1, s2, b + 1, integral_constant<int, 1>());
      block(s2, s3, b + 2, integral_constant<int, 2>());
      block(s3, S0, b + 3, integral_constant<int, 3>());
    }
#pragma unroll
    for (int f = 0; f < FM; f++) xa[f] = na[f];
#pragma unroll
    for (int f = 0; f < FN; f++) xb[f] = nb[f];
    if (b < kb) block(S0, S1, b, integral_constant<int, 0>());
    if (b + 1 < kb) block(S1, s2, b + 1, integral_constant<int, 1>());
    if (b + 2 < kb) block(s2, s3, b + 2, integral_constant<int, 2>());
    tile_barrier();  // (the loads that are not used)
  }
  if constexpr (kJoins) {
    static_assert(2 * 32 * (NW + 8) * 4 + 16 <= kStage, "a word that the epilogue leaves");
    if (p.parts > 1 && !join<BM * BN>(p, acc[0][0], tile, part, reinterpret_cast<int*>(S0 + kStage - 16))) return;
  }
  // Through LDS, 32 rows of the wave at a time, so that rows of C are written whole. One
  // copy of what follows the writes: jumping over code that is not needed costs
  // as much as running it.
  constexpr int kRow = NW + 8;  // (lanes 32 apart, four rows on, write to the other half of the banks)
  static_assert(2 * 32 * kRow * 4 <= kStage, "the waves' rows fit");
  float* mine = reinterpret_cast<float*>(wave < 2 ? S0 : S1) + (wave & 1) * 32 * kRow;
  constexpr int kLanes = NW / 4, kRows = 64 / kLanes, R = 32 / kRows < 8 ? 32 / kRows : 8;  // lanes of a row, rows at once, of those under way
  const int tr = lane / kLanes, tc = lane % kLanes * 4;
  const int64_t col = n0 + wn * NW + tc;
  auto spread = [&](const f32x16 (&x)[FN]) {
#pragma unroll
    for (int j = 0; j < FN; j++)
#pragma unroll
      for (int q = 0; q < 16; q++) mine[((q >> 2) * 8 + half * 4 + (q & 3)) * kRow + j * 32 + row] = x[j][q];
  };
#pragma unroll 1
  for (int i = 0; i < FM; i++) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);  // (a wave's own rows: its LDS accesses keep their order)
    if (i == 0) spread(acc[0]);
    if constexpr (FM > 1) { if (i == 1) spread(acc[1]); }
    if constexpr (FM > 2) { if (i == 2) spread(acc[2]); }
    if constexpr (FM > 3) { if (i == 3) spread(acc[3]); }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (col >= p.n) continue;
    const int64_t first = m0 + wm * MW + i * 32 + tr;
    if (p.e.bias || p.e.row_scale || p.e.act != FA_ACT_NONE) {
#pragma unroll 1
      for (int t = 0; t < 32; t += kRows) {
        f32x4* at = reinterpret_cast<f32x4*>(mine + (t + tr) * kRow + tc);
        *at = before_mul(p, *at, first + t, (int)col);
      }
    }
#pragma unroll 1
    for (int t = 0; t < 32; t += kRows * R) {
      int64_t at[R];
      f32x4 v[R];
#pragma unroll
      for (int k = 0; k < R; k++) {
        at[k] = first + t + k * kRows;
        v[k] = *reinterpret_cast<const f32x4*>(mine + (t + k * kRows + tr) * kRow + tc);
      }
      put4(p, c, at, col, v);
    }
  }
}

// (A kernel whose own body holds arrays of dependent bounds in lambdas loses its host stub.)
template <int BM, int BN, int WM, int D, bool F8, typename TC>
__global__ __launch_bounds__(256, (BM + BN) * D > 512 ? 1 : 2) void f8_tile_kernel(GemmParams p, TC* c, int tiles_m,
                                                                                 int tiles_n) {
  f8_tile<BM, BN, WM, D, F8, TC>(p, c, tiles_m, tiles_n);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace

int launch_f8_write(fa_ctx* ctx, const F8View& w, int dtype, const void* x, int64_t ldx, hipStream_t s, uint32_t* zero,
                    int zeros) {
  const int kb = (int)(f8_kp(w.k) / kF8Block), ks = (int)f8_ks(w.k);
  // few blocks: one to 16 lanes, so that they spread over the card
  const int64_t blocks = w.n * kb, per = blocks > 65536 ? 64 : 16, units = (blocks + per - 1) / per;
  if (units >= (int64_t)1 << 24)
    return set_error(ctx, FA_ERR_ARG, "F8Write: [%lld x %lld] is more than one call takes", (long long)w.n, (long long)w.k);
  const unsigned grid = (unsigned)units;
  if (dtype == FA_DT_F32) {
    const float* f = (const float*)x;
    const bool vec = ldx % 4 == 0 && aligned(x, 16);
    if (per == 64) f8_write_kernel<float, 4><<<grid, 256, 0, s>>>(w, f, ldx, kb, ks, vec, zero, zeros);
    else f8_write_kernel<float, 1><<<grid, 256, 0, s>>>(w, f, ldx, kb, ks, vec, zero, zeros);
  } else {
    const uint16_t* h = (const uint16_t*)x;
    const bool vec = ldx % 8 == 0 && aligned(x, 16);
    if (per == 64) f8_write_kernel<uint16_t, 4><<<grid, 256, 0, s>>>(w, h, ldx, kb, ks, vec, zero, zeros);
    else f8_write_kernel<uint16_t, 1><<<grid, 256, 0, s>>>(w, h, ldx, kb, ks, vec, zero, zeros);
  }
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

int launch_f8_read(fa_ctx* ctx, const F8View& w, int dtype, void* out, int64_t ldo, hipStream_t s) {
  const int kb = (int)(f8_kp(w.k) / kF8Block), ks = (int)f8_ks(w.k);
  const unsigned grid = (unsigned)std::min<int64_t>((w.n * kb * 32 + 255) / 256, 1 << 20);
  const bool vec = ldo % 4 == 0;
  if (dtype == FA_DT_F32)
    f8_read_kernel<float><<<grid, 256, 0, s>>>(w, (float*)out, ldo, kb, ks, vec && aligned(out, 16));
  else
    f8_read_kernel<uint16_t><<<grid, 256, 0, s>>>(w, (uint16_t*)out, ldo, kb, ks, vec && aligned(out, 8));
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

// Rows of A's codes a multiple of 2 KB apart would lie in few of the L2's channels:
// a block more between them (8192 x 8192 x 8192 504 -> 496 us).
int64_t a_stride(int64_t k) { return f8_kp(k) + (f8_kp(k) % 2048 == 0 ? kF8Block : 0); }

namespace {

// Tiles of a product, and the parts that K is split into. us, measured on both sides:
// - Up to 16 rows and 2^24 weights, whose reading takes about a launch's time, on the bf16
//   units whatever the result's type. Of these the kernel for few rows while its workgroups of 16
//   columns are at most two for each CU and a wave has at most six blocks, else tiles of 32
//   x 128: 16 x 4096 x 4096 10.9 and 11.2, 1 x 4096 x 4096 8.7 and 10.8, 1 x 2048 x 2048 7.2
//   and 9.3; 16 x 8192 x 1024 7.2 and 7.7, 16 x 9000 x 1024 8.4 and 7.8, 16 x 16384 x 1024
//   10.5 and 8.0; 1 x 1024 x 6144 9.7 and 11.1 (16 rows 12.4 and 11.5), 1 x 512 x 8192 11.5
//   and 11.6 (16 rows 15.9 and 12.1), 16 x 1024 x 16384 26.7 and 14.7. Above 2^24 weights:
//   16 x 5000 x 4096 16.2 and 11.8, 1 x 4096 x 8192 12.8 and 14.9, 16 rows 16.7 and 15.5, 1 x
//   32768 x 1024 14.4 and 9.9.
// - Tiles of 128 and of 256 (bf16) where they fill the card; of 128 with four blocks held,
//   for bf16, where they are at most one for each CU, and that for 3 of 4: 512 x 8192 x
//   8192 61 and 47, 896 x 4096 x 4096 in tiles of 64 40, so 29, but 512 x 4096 x 4096 (128
//   tiles) 23 and 26, and in float32, bound by widening, 384 x 8192 x 8192 67 and 68.
//   Below, tiles of 64, and of 32 x 128 up to 32 rows: 32 x 262144 x 768 57 and 63 in
//   tiles of 64, 1 x 262144 x 768 46 and 56 (two of either fit in a CU's LDS).
// - Where these do not fill the card either, K in up to 8 parts of 8 blocks or more, which
//   pays for joining them: 128 x 1152 x 16384 in float32 46 whole, 21 in parts; 32 x 4096 x
//   4096 15.5 and 12.6; 512 x 512 x 4096 17.5 and 15.7, parts of 4 blocks there 18, 32 x
//   1152 x 16384 42 whole, 17 in 8 parts, 19 in 16, 28 in twice the card's workgroups.
constexpr int kCUs = 256;  // of the card
struct Plan {
  int tile;   // 256, 128, 64, 32 (x 128); 0: few rows
  bool deep;  // four blocks held of tiles of 128
  bool exact;  // on the bf16 units
  int parts, per;
  int64_t tiles;
};
Plan plan_of(int64_t m, int64_t n, int64_t k, bool bf16) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
  const int kb = (int)(f8_kp(k) / kF8Block);
  const bool few = m <= 16 && n * kb <= 131072;
  Plan p = {0, false, few || !bf16, 1, kb, 0};
  if (few && n <= 8192 && kb <= 48) return p;
  const int64_t large = m > 64 ? tiles(128, 128) : 0;
  if (large >= kCUs || (bf16 && large * 4 >= kCUs * 3)) {
    p.tile = bf16 && m > 128 && tiles(256, 256) >= kCUs ? 256 : 128;
    p.deep = bf16 && large <= kCUs;
    return p;
  }
  p.tile = m > 32 ? 64 : 32;
  p.tiles = m > 32 ? tiles(64, 64) : tiles(32, 128);
  const int64_t most = std::min<int64_t>(kCUs / p.tiles, std::min(kb / 8, 8));
  if (most > 1) {
    p.per = (int)((kb + most - 1) / most + 3) / 4 * 4;
    p.parts = (kb + p.per - 1) / p.per;
  }
  return p;
}

}  // namespace

size_t f8_scratch(int64_t m, int64_t n, int64_t k) {
  const Plan p = plan_of(m, n, k, false);
  const size_t joined = p.parts > 1 ? align256((size_t)p.tiles * 4) + (size_t)p.tiles * p.parts * 4096 * 4 : 0;
  return align256((size_t)m * a_stride(k)) + align256((size_t)m * f8_ks(k)) + joined;
}

int64_t f8_grid(int64_t m, int64_t n) { return ((m + 15) / 16) * ((n + 63) / 64); }

namespace {

template <int BM, int BN, int WM, int D, typename TC, bool F8 = sizeof(TC) == 2>
void launch_tiles(const GemmParams& p, TC* c, hipStream_t s) {
  const int tm = (int)((p.m + BM - 1) / BM), tn = (int)((p.n + BN - 1) / BN);
  f8_tile_kernel<BM, BN, WM, D, F8, TC><<<(unsigned)(tm * tn * p.parts), 256, 0, s>>>(p, c, tm, tn);
}

template <typename TC>
void launch_gemm_t(const GemmParams& p, TC* c, const Plan& plan, hipStream_t s) {
  const int tile = plan.tile;
  if (tile == 256) {
    launch_tiles<256, 256, 2, 2>(p, (uint16_t*)c, s);
  } else if (plan.deep) {
    launch_tiles<128, 128, 2, 4>(p, (uint16_t*)c, s);
  } else if (tile == 128) {
    launch_tiles<128, 128, 2, 2>(p, c, s);
  } else if (tile == 64) {
    launch_tiles<64, 64, 2, 4>(p, c, s);
  } else if (tile == 32) {
    if (plan.exact) launch_tiles<32, 128, 1, 4, TC, false>(p, c, s);
    else launch_tiles<32, 128, 1, 4>(p, c, s);
  } else {
    GemmParams q = p;
    q.split = kFewWaves;
    while (q.split > std::max(1, p.kb)) q.split /= 2;
    const int columns = 16 * kFewWaves / q.split;
    f8_few_kernel<<<(unsigned)((p.n + columns - 1) / columns), kFewWaves * 64, 0, s>>>(q, c);
  }
}

}  // namespace

int launch_f8_gemm(fa_ctx* ctx, const F8GemmArgs& g, void* work, hipStream_t s) {
  const int64_t k = g.w.k;
  const Plan plan = plan_of(g.m, g.w.n, k, g.c_dtype != FA_DT_F32);
  F8View a = {nullptr, nullptr, g.m, k, a_stride(k)};
  GemmParams p = {};
  p.parts = plan.parts;
  p.per = plan.per;
  if (k > 0) {
    a.codes = static_cast<uint8_t*>(work);
    a.scales = a.codes + align256((size_t)g.m * a.stride);
    if (p.parts > 1) {
      p.count = reinterpret_cast<uint32_t*>(a.scales + align256((size_t)g.m * f8_ks(k)));
      p.part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.count) + align256((size_t)plan.tiles * 4));
    }
    const int rc = launch_f8_write(ctx, a, g.a_dtype, g.a, g.lda, s, p.count, p.parts > 1 ? (int)plan.tiles : 0);
    if (rc) return rc;
  }
  p.m = g.m;
  p.n = g.w.n;
  p.k = k;
  p.kb = (int)(f8_kp(k) / kF8Block);
  p.ks = (int)f8_ks(k);
  p.a = a.codes;
  p.a_st = a.stride;
  p.as = a.scales;
  p.w = g.w.codes;
  p.ws = g.w.scales;
  p.e = g.e;
  p.vec_bias = aligned(g.e.bias, 16);
  p.vec_mul = g.e.ldm % 4 == 0 && aligned(g.e.mul, 16);
  p.vec_residual = g.e.ldr % 4 == 0 && aligned(g.e.residual, 16);
  p.vec_c = g.ldc % 4 == 0 && aligned(g.c, g.c_dtype == FA_DT_F32 ? 16 : 8);
  p.ldc = g.ldc;
  if (g.c_dtype == FA_DT_F32) launch_gemm_t(p, (float*)g.c, plan, s);
  else launch_gemm_t(p, (uint16_t*)g.c, plan, s);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

}  // namespace fa
