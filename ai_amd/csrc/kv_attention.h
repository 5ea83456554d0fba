// What the attention kernels over the key/value cache share: the arguments,
// the division of a batch into work items, operand helpers.
#pragma once

#include "device_math.h"
#include "kvcache.h"

namespace fa {

constexpr int kTileRows = 16;   // query rows of a work item of the kernel for few rows,
constexpr int kPairRows = 32;   // of its form for some more,
constexpr int kWideRows = 128;  // and of the kernel for many

constexpr int kMinChunk = 4;    // blocks of a split part, at least (one per wave)
constexpr int kRound = 64;      // blocks of a part up to which one part for each CU is aimed at
constexpr int kTarget = 1024;   // else parts aimed at: two rounds of two workgroups on each of 256 CUs
constexpr float kWideGain = 20.f;  // blocks (plan_item)
// Weights are multiplied by the value scale 2^e and this, so that sums of 2^20
// times float32's largest values stay finite; the result is multiplied back.
constexpr float kWeightScale = 0x1p-24f;
// The least of these factors under which float32 holds scaled weights down to 2^-62.
constexpr float kLeastFactor = 0x1p-64f;
// The largest sum of a lane's weights in a block, relative to its row's reference.
constexpr float kMostWeight = 0x1p8f;

// The word of the counters in which the kernel for many rows leaves the blocks
// of a part for the launch that joins its parts: they come from sums and a
// threshold in float32, and two kernels need not be compiled to the same
// rounding. (Few rows count in words below 3080: kTarget and 2 kTarget items + 8.)
constexpr int kPlanWord = kKvCountBytes / 4 - 1;

// The work of one call: tiles of `tile` rows of a sequence's n * G, for
// each key/value head, over the blocks they see; in a planned call the blocks
// are cut into parts of about equal size over the whole batch.
struct AttnArgs {
  KvArgs c;
  const void* q;
  int64_t q_st, q_sh;
  int32_t H, G;
  int32_t causal, window;
  float scale2;  // scale * log2 e
  void* out;
  float* part;    // planned: [parts][tile][Dp] sums, then [parts][tile][2] maximum, sum
  uint32_t* count;  // planned: per part 0 of a tile, how many of its parts are done; [kPlanWord]
  int64_t parts;  // parts that the scratch holds
  int32_t tile;   // query rows of a work item
  int32_t target, least, cap;  // planned: parts aimed at, blocks of a part at least
  int32_t span;   // blocks that a tile sees at most, by its window
  float once;     // planned, with cap: workgroups aimed at in one round of short parts
  float places, uneven;  // planned: workgroups on the card at once, where a rule decides whether to split (see there)
  int32_t vec, out_vec;  // rows of q / out aligned for one load / store
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Tokens that the rows of new tokens t0 .. t1 (positions len - n + t) see at
// all: [lo, hi).
__device__ __forceinline__ void seen_range(const AttnArgs& a, const KvSeq& s, int t0, int t1, int* lo, int* hi) {
  const int64_t p0 = (int64_t)s.len - s.n + t0, p1 = (int64_t)s.len - s.n + t1;
  int64_t l = a.window ? p0 - a.window + 1 : 0;
  int64_t h = a.causal ? p1 + 1 : a.window ? p1 + a.window : s.len;
  l = max(l, (int64_t)0);
  h = min(h, (int64_t)s.len);
  *lo = (int)l;
  *hi = (int)max(h, l);
}

// The most blocks that a tile of sequence s sees.
__device__ __forceinline__ int seen_blocks(const AttnArgs& a, const KvSeq& s) {
  if (s.n == 0) return 0;
  int lo, hi;
  seen_range(a, s, 0, s.n - 1, &lo, &hi);
  hi = (int)min((int64_t)hi, (int64_t)a.c.tstride * 64);
  return hi <= lo ? 0 : min(((hi + 63) >> 6) - (lo >> 6), a.span);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
// Inclusive sums over the lanes: within rows of 16 by row shifts, then the
// last lane of a row added to the rows after it (row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// What lane % 64 = b - b0 knows of sequence b: its tiles and the blocks that one of them sees at most.
struct Seen {
  int tiles, blocks;
  KvSeq s;
};
__device__ __forceinline__ Seen seen_by(const AttnArgs& a, int b) {
  if (b >= a.c.nseq) return {0, 0, {0, 0, 0}};
  const KvSeq s = kv_seq(a.c, b);
  return {ceil_div(s.n * a.G, a.tile), seen_blocks(a, s), s};
}

struct Item {
  int b, tile, h, chunk, chunks;
  int64_t first;  // planned: the part of chunk 0
  int len;        // planned: blocks of a part
  bool ok;
  KvSeq s;  // the sequence's rows and length
};

// A part has the batch's blocks over a.target, a.least at least; but up to
// a.cap blocks, as many as leave one part for each CU: a part's beginning (its
// lengths, its table entries, its first codes, each load after the one before)
// takes as long as some ten blocks, and every part is written and read once
// more. One sequence of 131072 tokens, 32 heads on 8 of 128 dims: 57 us in 256
// parts, 63 in 512, 80 in 1024. Longer parts leave less to balance uneven
// sequences with: those are cut by the target. With a.places (many rows, a card
// not far from full) parts are made only where the longest tile's blocks times
// the free share of the card are kWideGain or more: a tile counts whole, or less
// by a.uneven of the part of its sequence that is new, whose tiles see less.
__device__ __forceinline__ int part_blocks(const AttnArgs& a, const Seen& first) {
  const int lane = threadIdx.x & 63;
  float total = 0.f, tiles = 0.f, longest = 0.f, busy = 0.f;
  auto count = [&](const Seen& x) {
    const float t = (float)x.tiles, b = (float)x.blocks;
    total += t * b;
    tiles += t;
    longest = fmaxf(longest, b);
    busy += t * (1.f - a.uneven * (float)x.s.n / (float)max(x.s.len, 1));
  };
  count(first);
  for (int b0 = 64; b0 < a.c.nseq; b0 += 64) count(seen_by(a, b0 + lane));
  total = wave_sum(total) * (float)a.c.hkv;
  tiles = wave_sum(tiles) * (float)a.c.hkv;
  const float round = total / fmaxf(a.once - tiles, a.once * 0.5f);
  int chunk = max(max((int)ceilf(fminf(total / (float)a.target, 1e9f)), a.least),
                  (int)ceilf(fminf(round, (float)a.cap)));
  if (a.places > 0.f) {
    busy = wave_sum(busy) * (float)a.c.hkv;
    if (!(wave_max(longest) * (a.places - busy) >= kWideGain * a.places)) chunk = 1 << 30;
  }
  return chunk;
}

// Parts are numbered by sequence, tile, head, chunk. The item of part w, or
// (w < 0) the first part of the tile and head that are asked for, with parts of
// `len` blocks as the kernel that wrote them had it. Every wave
// finds its own from the lengths, one load for up to 64 sequences (float32
// sums in a fixed order: the same in every wave of a kernel).
__device__ __forceinline__ Item plan_item(const AttnArgs& a, int64_t w, int want_b, int want_tile, int want_h,
                                          int len = 0) {
  const int lane = threadIdx.x & 63;
  const Seen first = seen_by(a, lane);
  const int chunk = w < 0 ? len : part_blocks(a, first);
  Item r = {0, 0, 0, 0, 1, 0, chunk, false, {0, 0, 0}};
  int64_t before = 0;
  for (int b0 = 0; b0 < a.c.nseq; b0 += 64) {
    const Seen x = b0 ? seen_by(a, b0 + lane) : first;
    const int cb = max(1, ceil_div(x.blocks, chunk));
    const int cnt = x.tiles * a.c.hkv * cb;
    const int incl = wave_scan(cnt);
    const bool mine = w >= 0 ? w < before + incl : b0 + lane == want_b;
    const uint64_t m = __ballot(mine && b0 + lane < a.c.nseq);
    if (m) {
      const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)m) - 1);
      const int tiles = __builtin_amdgcn_readlane(x.tiles, src);
      r.b = b0 + src;
      r.s = lane_seq(x.s, src);
      r.chunks = __builtin_amdgcn_readlane(cb, src);
      const int64_t base = before + __builtin_amdgcn_readlane(incl - cnt, src);
      if (w >= 0) {
        const int i = (int)(w - base), th = i / r.chunks;
        r.chunk = i - th * r.chunks;
        r.tile = th / a.c.hkv;
        r.h = th - r.tile * a.c.hkv;
      } else {
        r.tile = want_tile;
        r.h = want_h;
      }
      r.first = base + ((int64_t)r.tile * a.c.hkv + r.h) * r.chunks;
      // (row starts that are not in order number more parts than there are: those have no place)
      r.ok = r.tile >= 0 && r.tile < tiles && r.chunk >= 0 && r.h >= 0 && r.first >= 0 &&
             r.first + r.chunks <= a.parts;
      break;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return r;
}

// Unplanned: the slots of sequence b's tiles of `rows` rows start at cu[b] * G / rows + b.
__device__ __forceinline__ Item direct_item(const AttnArgs& a, int64_t slot, int h, int rows) {
  Item r = {0, 0, h, 0, 1, 0, 0, false, {0, 0, 0}};
  const int G = a.G;
  auto base = [&](int32_t c, int b) { return (int64_t)((uint32_t)c * (uint32_t)G / (uint32_t)rows) + b; };
  const KvFound f = kv_find(a.c, slot, base);
  r.b = f.b;
  r.s = f.s;
  const int64_t t = slot - base(f.cu0, f.b);
  r.ok = t >= 0 && t * rows < (int64_t)f.s.n * G;
  r.tile = (int)t;
  return r;
}

// The blocks of a run of table slots, first, first + step, ..: lane i of the
// wave holds the i-th of 64 at a time, so that a step of the main loop takes
// one from a register and does not wait for a load (and with it for every
// load issued before).
struct Blocks {
  int first, step, end, held;  // held: the index that lane 0 has
  int id;
  __device__ __forceinline__ void fill(const AttnArgs& a, int b, int i) {
    held = i;
    const int64_t slot = (int64_t)first + (int64_t)(i + (int)(threadIdx.x & 63)) * step;
    id = slot < end ? kv_block(a.c, b, slot) : -1;
  }
  __device__ __forceinline__ Blocks(const AttnArgs& a, int b, int first_, int step_, int end_)
      : first(first_), step(step_), end(end_) {
    fill(a, b, 0);
  }
  // The i-th block, -1 past the end; i does not fall by more than 1 from call to call.
  __device__ __forceinline__ int at(const AttnArgs& a, int b, int i) {
    if (i >= held + 64) fill(a, b, i);
    return __builtin_amdgcn_readlane(id, i - held);
  }
};

// The larger of two where neither is NaN (else the other or either), without
// the quieting of inputs that fmaxf has to do.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_amdgcn_fmed3f(a, b, __builtin_inff());
}

// Eight codes (two dwords) as a bf16 operand.
__device__ __forceinline__ bf16x8 widen(uint32_t a, uint32_t b) {
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false);
  const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false);
  const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

__device__ __forceinline__ kvf4 mfma(bf16x8 a, bf16x8 b, kvf4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The bf16 terms of eight float32 values as operands: all 24 bits in three
// (TERMS 3), 17 in two (TERMS 2: the value rounded to nearest and what that
// leaves, rounded again), or rounded to nearest (TERMS 1).
template <int TERMS>
__device__ __forceinline__ void terms_of(const float (&v)[8], bf16x8 (&t)[TERMS]) {
  if constexpr (TERMS == 1) {
#pragma unroll
    for (int i = 0; i < 8; i++) t[0][i] = (__bf16)v[i];
  } else if constexpr (TERMS == 2) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      t[0][i] = (__bf16)v[i];
      t[1][i] = (__bf16)(v[i] - (float)t[0][i]);
    }
  } else {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Split3 x = split3(v[2 * i]), y = split3(v[2 * i + 1]);
      w[0][i] = pack_hi16(x.h, y.h);
      w[1][i] = pack_hi16(x.m, y.m);
      w[2][i] = pack_hi16(x.l, y.l);
    }
#pragma unroll
    for (int k = 0; k < 3; k++) t[k] = __builtin_bit_cast(bf16x8, make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]));
  }
}

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, int d, int D, bool vec, float (&v)[8]) {
  if (vec && d + 8 <= D) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + d), y = *reinterpret_cast<const f32x4*>(p + d + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = x[i], v[4 + i] = y[i];
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(p + d);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = d + i < D ? ld(p + d + i) : 0.f;
  }
}

// Maximum over the four lane groups of a row (lanes 16 apart).
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, lane_xor16(v));
  return fmaxf(v, lane_xor32(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += lane_xor16(v);
  return v + lane_xor32(v);
}

// Bytes that are a NaN code, as 0x80 each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// Many rows (kv_attention_tile.hip): a.tile rows a work item.
int kv_tiles_per_cu(int nc, int dtype);
int launch_kv_tiles_attn(fa_ctx* ctx, const AttnArgs& a, int dtype, int64_t slots, hipStream_t s);

}  // namespace fa
