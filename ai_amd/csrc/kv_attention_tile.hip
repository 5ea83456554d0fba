// Attention over the 8-bit key/value cache for many query rows (prompts and
// chunks of them).
#include <atomic>

#include "kv_attention.h"

namespace fa {
namespace {

// bf16 pairs of a dword that are NaN: as ones, or dropped.
__device__ __forceinline__ uint32_t nan_ones(uint32_t w) {
  return ((w & 0x7FFFu) > 0x7F80u ? 0x3F80u : 0u) | ((w & 0x7FFF0000u) > 0x7F800000u ? 0x3F800000u : 0u);
}
__device__ __forceinline__ uint32_t nan_drop(uint32_t w) {
  return ((w & 0x7FFFu) > 0x7F80u ? 0u : w & 0xFFFFu) | ((w & 0x7FFF0000u) > 0x7F800000u ? 0u : w & 0xFFFF0000u);
}

// Order of N operand reads from LDS and the M products that use each: the
// reads kAhead products early (left to itself the compiler waits for each
// pair of reads just before its products: 740 against 721 us for a prompt of
// 8192 tokens, 308 against 296 for 4 chunks of 512, 32 heads on 8 of 128 dims).
constexpr int kAhead = 4;
template <int N, int M>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = 0; i < (N - kAhead) / 2; i++) {
    __builtin_amdgcn_sched_group_barrier(0x8, 2 * M, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, M * kAhead, 0);
}

// The w-th of `slots` whole tiles. Up to 64 sequences: those whose tiles see
// most go first, by eighths of the most (finding the exact order takes longer),
// and of one the later tiles, which see more if it is causal, so that the last
// tiles to start are short: 4 chunks of 512 tokens on 2979 .. 8704, 32 heads on 8
// of 128 dims in bf16, take 296 us from the longest down, 323 from the shortest
// up. Under kSortBlocks in their order; more sequences from the last to the first.
constexpr int kSortBlocks = 16;
__device__ __forceinline__ Item whole_item(const AttnArgs& a, int w, int slots, int h) {
  if (a.c.nseq > 64) return direct_item(a, (int64_t)slots - 1 - w, h, kWideRows);
  const Seen x = seen_by(a, threadIdx.x & 63);
  const int longest = __builtin_amdgcn_readfirstlane((int)wave_max((float)x.blocks));
  const int eighth = longest < kSortBlocks ? 0 : min(7, (int)((float)x.blocks * 8.f / (float)longest));
  int before = 0;
  uint64_t m = 0;
  for (int c = longest < kSortBlocks ? 0 : 7; c >= 0 && !m; c--) {
    const int t = eighth == c ? x.tiles : 0;
    if (!__ballot(t != 0)) continue;
    const int incl = wave_scan(t);
    const int at = before + incl - t;  // of this class, the lane's first
    m = __ballot(w >= at && w < at + t);
    if (m) before = at;
    else before += __builtin_amdgcn_readlane(incl, 63);
  }
  Item r = {0, 0, h, 0, 1, 0, 0, false, {0, 0, 0}};
  if (!m) return r;
  const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)m) - 1);
  r.b = src;
  r.s = lane_seq(x.s, src);
  r.tile = __builtin_amdgcn_readlane(x.tiles, src) - 1 - (w - __builtin_amdgcn_readlane(before, src));
  r.ok = true;
  return r;
}

// Workgroups that a CU holds, by their registers.
constexpr int per_cu(int nc, int terms) { return nc <= (terms == 1 ? 2 : 1) ? 2 : 1; }

typedef float kvf16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ kvf16 mfma32(bf16x8 a, bf16x8 b, kvf16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A workgroup of four waves takes 128 query rows of one key/value head, a wave
// 32 of them, all over the same blocks: a block's codes are loaded two blocks
// ahead into registers, widened once for all the waves into LDS one block
// ahead (two buffers, one barrier a block), in the order in which a wave reads
// them as operands (1 KB in a row: no bank conflicts). The products are
// transposed as in the kernel for few rows, on the 32x32x16 MFMA: it leaves
// lane l (row l % 32, half l / 32) the scores of tokens 8 i + 4 half + 0..3.
// 128 rows: a block's widening is shared by four waves (a wave alone would
// convert 2 * 64 * D codes for 32 rows, as many instructions as its softmax),
// and two such workgroups fit a CU (bf16, up to 128 dims).
//
// A prompt of 8192 tokens, 32 heads on 8 of 128 dims in bf16: 712 to 727 us, with
// two terms of the weights 1.13 to 1.16 PFLOP/s of products, where a large matrix
// product reaches 1.26. Bound by the card's power (1.84 GHz, matrix units busy 0.52
// of the time beside softmax and widening: a tenth fewer vector instructions took as long).
//
// Terms as in the kernel for few rows: which of the two a call takes changes no
// operand's bits.
template <typename T, int TERMS, int NC>
__global__ __launch_bounds__(256, per_cu(NC, TERMS)) void kv_attn_tile_kernel(AttnArgs a) {
  constexpr int W = 4, kThreads = W * 64, kRows = W * 32;
  constexpr int KS = NC * 4;            // steps of 16 dims
  constexpr int WT = TERMS == 3 ? 3 : 2;  // terms of a weight; TERMS: of a query
  constexpr int DT = NC * 2;            // tiles of 32 dims
  constexpr int kFrag = NC * 512;       // operands of a block's keys; as many of its values
  constexpr int kVals = (NC + 1) / 2;   // a thread's value loads of 2 x 16 codes; NC key loads of 16
  extern __shared__ __align__(16) uint4 tile_lds[];  // [2 buffers][keys, values][kFrag]
  __shared__ uint32_t nan_flag[2][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const bool planned = a.part != nullptr;
  // Heads alternate, so that a head's tiles run on the same XCDs where there
  // are 8 heads or a multiple.
  const Item it = planned ? plan_item(a, (int64_t)gridDim.x - 1 - blockIdx.x, 0, 0, 0)
                          : whole_item(a, blockIdx.x / a.c.hkv, gridDim.x / a.c.hkv, blockIdx.x % a.c.hkv);
  if (planned && blockIdx.x == 0 && tid == 0) a.count[kPlanWord] = it.len;
  if (!it.ok) return;
  const KvSeq s = it.s;
  const int rows = s.n * a.G, r0 = it.tile * kRows;
  const int valid = min(kRows, rows - r0);
  const bool too_long = (int64_t)s.len > (int64_t)a.c.tstride * 64;

  int lo, hi;  // what some row of the workgroup sees
  seen_range(a, s, r0 / a.G, (r0 + valid - 1) / a.G, &lo, &hi);
  if (too_long) hi = lo;
  int pg0 = lo >> 6, pg1 = hi <= lo ? pg0 : (hi + 63) >> 6;
  {
    const int np = pg1 - pg0;
    const int c0 = (int)((int64_t)np * it.chunk / it.chunks), c1 = (int)((int64_t)np * (it.chunk + 1) / it.chunks);
    pg1 = pg0 + c1;
    pg0 += c0;
  }
  int galo, gahi;  // what all of them see
  {
    int l0, h0, l1, h1;
    seen_range(a, s, r0 / a.G, r0 / a.G, &l0, &h0);
    seen_range(a, s, (r0 + valid - 1) / a.G, (r0 + valid - 1) / a.G, &l1, &h1);
    galo = max(l0, l1);
    gahi = min(h0, h1);
  }
  // this wave's rows: what one of them sees, what all of them see, each lane's
  const int w0 = r0 + wave * 32, wvalid = min(32, rows - w0);
  int wlo = 0, whi = 0, alo = 0, ahi = 0, rlo, rhi;
  if (wvalid > 0) {
    const int ta = w0 / a.G, tb = (w0 + wvalid - 1) / a.G;
    int l0, h0, l1, h1;
    seen_range(a, s, ta, tb, &wlo, &whi);
    seen_range(a, s, ta, ta, &l0, &h0);
    seen_range(a, s, tb, tb, &l1, &h1);
    alo = max(l0, l1);
    ahi = min(h0, h1);
  }
  const int r = w0 + col;
  const bool on = r < rows;
  const int tok = min(r, rows - 1) / a.G, head = it.h * a.G + (on ? r - tok * a.G : 0);
  seen_range(a, s, tok, tok, &rlo, &rhi);

  // Loads and widening of one block by the whole workgroup. A thread's loads:
  // 16 dims of a token (NC times), and the tokens 4 b .. 4 b + 3 and 4 b + 8 ..
  // 4 b + 11 of each 16 of a dim (b 0 or 1): an operand's eight from each 16.
  uint4 kraw[NC], vraw[kVals][2];
  uint32_t kat[NC], kto[NC], vat[kVals], vto[kVals];  // where from (16 bytes) in the part, where to in the buffer
  bool von[kVals];
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int x = tid + i * kThreads, t = x & 63, g = x >> 6;  // g: 16 dims, four to a slice
    kat[i] = (g >> 2) * 256 + t * 4 + (g & 3);
    kto[i] = (g * 2 + (t >> 5)) * 64 + (t & 31);
  }
#pragma unroll
  for (int i = 0; i < kVals; i++) {
    const int x = tid + i * kThreads, d = x % (64 * NC), b = x / (64 * NC);
    von[i] = (128 * NC) % kThreads == 0 || b < 2;
    vat[i] = d * 4 + b;
    vto[i] = kFrag + (d >> 5) * 64 + b * 32 + (d & 31);
  }
  Blocks blocks(a, it.b, pg0, 1, pg1);
  auto load = [&](int id) {
    if (id >= 0) {
      const uint4* kp = reinterpret_cast<const uint4*>(kv_part(a.c, id, it.h, 0));
      const uint4* vp = reinterpret_cast<const uint4*>(kv_part(a.c, id, it.h, 1));
#pragma unroll
      for (int i = 0; i < NC; i++) kraw[i] = kp[kat[i]];
#pragma unroll
      for (int i = 0; i < kVals; i++)
        if (von[i]) {
          vraw[i][0] = vp[vat[i]];
          vraw[i][1] = vp[vat[i] + 2];
        }
    } else {  // no such block: keys that are NaN
#pragma unroll
      for (int i = 0; i < NC; i++) kraw[i] = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
#pragma unroll
      for (int i = 0; i < kVals; i++) vraw[i][0] = vraw[i][1] = make_uint4(0, 0, 0, 0);
    }
  };
  auto stage = [&](int buf, int p) {
    uint4* to = tile_lds + buf * 2 * kFrag;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      to[kto[i]] = __builtin_bit_cast(uint4, widen(kraw[i].x, kraw[i].y));
      to[kto[i] + 32] = __builtin_bit_cast(uint4, widen(kraw[i].z, kraw[i].w));
    }
    const int j0 = p * 64;
    if (j0 < galo || j0 + 64 > gahi) {
      // tokens that no row of the workgroup sees: zero values, whatever is
      // there; NaN among the others is looked for
      uint32_t nan = 0;
#pragma unroll
      for (int i = 0; i < kVals; i++)
        if (von[i]) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            uint32_t w[4] = {vraw[i][u].x, vraw[i][u].y, vraw[i][u].z, vraw[i][u].w};
            const int b = (int)(vat[i] & 3) + 2 * u;
#pragma unroll
            for (int q = 0; q < 4; q++) {
#pragma unroll
              for (int c = 0; c < 4; c++) {
                const int j = j0 + q * 16 + b * 4 + c;
                if (j < lo || j >= hi) w[q] &= ~(0xFFu << (8 * c));
              }
              nan |= nan_bytes(w[q]);
            }
            vraw[i][u] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      const bool any = __ballot(nan != 0) != 0;
      if (lane == 0) nan_flag[buf][wave] = any;
    }
#pragma unroll
    for (int i = 0; i < kVals; i++)
      if (von[i]) {
        to[vto[i]] = __builtin_bit_cast(uint4, widen(vraw[i][0].x, vraw[i][1].x));
        to[vto[i] + DT * 64] = __builtin_bit_cast(uint4, widen(vraw[i][0].y, vraw[i][1].y));
        to[vto[i] + 2 * DT * 64] = __builtin_bit_cast(uint4, widen(vraw[i][0].z, vraw[i][1].z));
        to[vto[i] + 3 * DT * 64] = __builtin_bit_cast(uint4, widen(vraw[i][0].w, vraw[i][1].w));
      }
  };
  // a block's two scales, loaded with its codes
  auto scales = [&](int id) {
    return id >= 0 ? *reinterpret_cast<const float2*>(a.c.scales + ((int64_t)id * a.c.hkv + it.h) * 2)
                   : make_float2(1.f, 1.f);
  };
  float2 ksv = make_float2(1.f, 1.f), ksv1 = ksv;
  if (pg0 < pg1) {
    const int id = blocks.at(a, it.b, 0);
    ksv = scales(id);
    load(id);
  }

  // queries as operands, in registers; a negative scale turns their sign
  bf16x8 qf[KS][TERMS];
  {
    const float sign = a.scale2 < 0.f ? -1.f : 1.f;
    const T* p = (const T*)a.q + (s.row0 + tok) * a.q_st + head * a.q_sh;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (on) load8(p, k * 16 + half * 8, a.c.D, a.vec, v);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= sign;
      terms_of<TERMS>(v, qf[k]);
    }
  }

  kvf16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; i++)
#pragma unroll
    for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  uint64_t nan_sum[2] = {0, 0};  // sums that are NaN: bit 16 (i % 4) + j of word i / 4

  if (pg0 < pg1) {
    stage(0, pg0);
    if (pg0 + 1 < pg1) {
      const int id = blocks.at(a, it.b, 1);
      ksv1 = scales(id);
      load(id);
    }
  }
  __syncthreads();

  for (int p = pg0; p < pg1; p++) {
    const int buf = (p - pg0) & 1;
    const int j0 = p * 64;
    float2 ksv2 = ksv1;
    const bool here = j0 < whi && j0 + 64 > wlo;  // some row of the wave sees some token
    const uint4* kf = tile_lds + buf * 2 * kFrag;
    uint4* vf = tile_lds + buf * 2 * kFrag + kFrag;
    if (j0 < galo || j0 + 64 > gahi) {
      uint32_t nan = 0;
#pragma unroll
      for (int w = 0; w < W; w++) nan |= nan_flag[buf][w];
      if (__builtin_amdgcn_readfirstlane(nan)) {
        // as in the kernel for few rows: NaN values that some rows see and
        // others do not, counted by a product of their own, then dropped;
        // the sums become NaN at the end
#pragma unroll 1
        for (int i = 0; i < DT; i++) {
          kvf16 cnt;
#pragma unroll
          for (int j = 0; j < 16; j++) cnt[j] = 0.f;
#pragma unroll 1
          for (int k = 0; k < 4; k++) {
            bf16x8 see;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const int t = j0 + k * 16 + (e >> 2) * 8 + half * 4 + (e & 3);
              see[e] = (__bf16)(t >= rlo && t < rhi ? 1.f : 0.f);
            }
            const uint4 v = vf[(k * DT + i) * 64 + lane];
            cnt = mfma32(__builtin_bit_cast(bf16x8, make_uint4(nan_ones(v.x), nan_ones(v.y), nan_ones(v.z),
                                                               nan_ones(v.w))), see, cnt);
          }
          uint64_t bits = 0;
#pragma unroll
          for (int j = 0; j < 16; j++) bits |= (uint64_t)(cnt[j] > 0.f) << j;
          nan_sum[0] |= i < 4 ? bits << (16 * i) : 0;
          if (NC > 2) nan_sum[1] |= i < 4 ? 0 : bits << (16 * (i & 3));
        }
        __syncthreads();
        for (int i = tid; i < kFrag; i += kThreads) {
          const uint4 v = vf[i];
          vf[i] = make_uint4(nan_drop(v.x), nan_drop(v.y), nan_drop(v.z), nan_drop(v.w));
        }
        __syncthreads();
      }
    }
    kvf16 sc[2];
    if (here) {
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
#pragma unroll
        for (int j = 0; j < 16; j++) sc[tt][j] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const bf16x8 k0 = __builtin_bit_cast(bf16x8, kf[k * 128 + lane]);
        const bf16x8 k1 = __builtin_bit_cast(bf16x8, kf[k * 128 + 64 + lane]);
#pragma unroll
        for (int x = 0; x < TERMS; x++) {
          sc[0] = mfma32(k0, qf[k][x], sc[0]);
          sc[1] = mfma32(k1, qf[k][x], sc[1]);
        }
      }
      reads_ahead<KS * 2, TERMS>();
    }
    if (p + 1 < pg1) {
      stage(buf ^ 1, p + 1);
      if (p + 2 < pg1) {
        const int id = blocks.at(a, it.b, p + 2 - pg0);
        ksv2 = scales(id);
        load(id);
      }
    }
    if (here) {
      // (not zero: a hidden score is -inf times it; the smallest float, under
      // which a product with any other score is 2^-21 at most)
      const float mul = fmaxf(fabsf(a.scale2) * ksv.x, 0x1p-149f);
      const float f = ksv.y * kWeightScale;
      if (j0 < alo || j0 + 64 > ahi) {
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
#pragma unroll
          for (int j = 0; j < 16; j++) {
            const int t = j0 + tt * 32 + (j >> 2) * 8 + half * 4 + (j & 3);
            sc[tt][j] = t >= rlo && t < rhi ? sc[tt][j] : -__builtin_inff();
          }
      }
      // bf16: the value scale enters the exponent (down to kLeastFactor:
      // below it, weights that count in the row's sum would be lost), and the
      // sum of the scaled weights is scaled back once a block
      const float fe = TERMS == 1 ? (float)((int)(__float_as_uint(fmaxf(f, kLeastFactor)) >> 23) - 127) : 0.f;
      float part;
      bf16x8 pt[4][WT];
      auto weights = [&]() {
        const float mu = (m == -__builtin_inff() ? 0.f : m) - fe;
        part = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float y = __builtin_amdgcn_exp2f(fmaf(sc[k >> 1][(k & 1) * 8 + i], mul, -mu));
            part += y;
            x[i] = TERMS == 1 ? y : y * f;
          }
          terms_of<WT>(x, pt[k]);
        }
        part *= TERMS == 1 ? __builtin_amdgcn_exp2f(-fe) : 1.f;
      };
      weights();
      // The reference m of a row's weights is its maximum over the blocks up
      // to the one where it was last set, and any reference is as exact as
      // the maximum while no weight is over kMostWeight: no maximum is taken
      // but in a row's first block and where the sum says that one is.
      if (__ballot(part > kMostWeight || m == -__builtin_inff())) {
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 32; i++) top = larger(top, sc[i >> 4][i & 15]);
        top = larger(top, lane_xor32(top)) * mul;
        const float mn = fmaxf(m, top);
        const float alpha = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < DT; i++) acc[i] *= alpha;
        m = mn;
        weights();
      }
      l += part;
      if (TERMS == 1 && f < kLeastFactor) {  // (rare: values all zero, or none over 2^-31)
        const float rest = f * (1.f / kLeastFactor);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int x = 0; x < WT; x++)
#pragma unroll
            for (int i = 0; i < 8; i++) pt[k][x][i] = (__bf16)((float)pt[k][x][i] * rest);
      }
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < DT; i += 2) {
          const bf16x8 v0 = __builtin_bit_cast(bf16x8, vf[(k * DT + i) * 64 + lane]);
          const bf16x8 v1 = __builtin_bit_cast(bf16x8, vf[(k * DT + i + 1) * 64 + lane]);
#pragma unroll
          for (int x = 0; x < WT; x++) {
            acc[i] = mfma32(v0, pt[k][x], acc[i]);
            acc[i + 1] = mfma32(v1, pt[k][x], acc[i + 1]);
          }
        }
      reads_ahead<4 * DT, WT>();
    }
    __syncthreads();
    ksv = ksv1;
    ksv1 = ksv2;
  }

  const float L = l + lane_xor32(l);
  if (__ballot((nan_sum[0] | nan_sum[1]) != 0)) {
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (nan_sum[i >> 2] >> (16 * (i & 3) + j) & 1) acc[i][j] = __builtin_nanf("");
  }
  if (!on) return;
  const int Dp = a.c.nc * 64;
  if (it.chunks > 1) {
    const int64_t slot = (it.first + it.chunk) * kRows + (r - r0);
    float* dst = a.part + slot * Dp;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *reinterpret_cast<kvf4*>(dst + i * 32 + q * 8 + half * 4) =
            kvf4{acc[i][q * 4], acc[i][q * 4 + 1], acc[i][q * 4 + 2], acc[i][q * 4 + 3]};
    if (half == 0) {
      float* stat = a.part + a.parts * kRows * Dp + slot * 2;
      stat[0] = m;
      stat[1] = L;
    }
    return;
  }
  const float fin = too_long ? __builtin_nanf("") : (1.f / kWeightScale) / L;
  const bool empty = rhi <= rlo && !too_long;
  T* dst = (T*)a.out + ((s.row0 + tok) * a.H + head) * (int64_t)a.c.D;
#pragma unroll
  for (int i = 0; i < DT; i++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int d = i * 32 + q * 8 + half * 4;
      kvf4 o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = empty ? 0.f : acc[i][q * 4 + j] * fin;
      if (a.out_vec && d + 4 <= a.c.D) {
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<kvf4*>(dst + d) = o;
        } else {
          const bf16x2 x = {(__bf16)o[0], (__bf16)o[1]}, y = {(__bf16)o[2], (__bf16)o[3]};
          *reinterpret_cast<uint2*>(dst + d) =
              make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (d + j < a.c.D) st(dst + d + j, o[j]);
      }
    }
}

template <typename T, int TERMS, int NC>
int tile_launch(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  const size_t lds = (size_t)2 * 2 * NC * 512 * 16;
  static std::atomic<uint64_t> ready{0};  // devices that know of it, the first 64
  const uint64_t bit = ctx->device < 64 ? uint64_t(1) << ctx->device : 0;
  if (!(ready.load() & bit)) {
    FA_HIP_CHECK(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kv_attn_tile_kernel<T, TERMS, NC>),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    ready.fetch_or(bit);
  }
  const dim3 grid((unsigned)(a.part ? a.parts : a.c.hkv * slots));
  kv_attn_tile_kernel<T, TERMS, NC><<<grid, 256, lds, s>>>(a);
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

template <typename T, int TERMS>
int tiles_t(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  if (a.c.nc == 1) return tile_launch<T, TERMS, 1>(ctx, a, slots, s);
  if (a.c.nc == 2) return tile_launch<T, TERMS, 2>(ctx, a, slots, s);
  if (a.c.nc == 3) return tile_launch<T, TERMS, 3>(ctx, a, slots, s);
  return tile_launch<T, TERMS, 4>(ctx, a, slots, s);
}

}  // namespace

int kv_tiles_per_cu(int nc, int dtype) { return per_cu(nc, dtype == FA_DT_F32 ? 3 : 1); }

int launch_kv_tiles_attn(fa_ctx* ctx, const AttnArgs& a, int dtype, int64_t slots, hipStream_t s) {
  return dtype == FA_DT_F32 ? tiles_t<float, 3>(ctx, a, slots, s) : tiles_t<uint16_t, 1>(ctx, a, slots, s);
}

}  // namespace fa
