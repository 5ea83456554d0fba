// Attention of new tokens over the 8-bit key/value cache:
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
// over the tokens j that query i sees, one pass over the cached blocks with
// the running maximum and sum of the softmax.
//
// A query row is (new token, query head of the key/value head's group):
// heads that share keys share a tile. Scores are computed transposed, S^T =
// K . Q^T, and so is the output, O^T = V^T . P^T: the MFMA leaves a lane the
// scores of its row against the tokens whose values it needs next as an
// operand (the value layout is permuted to that order), so weights stay in
// registers. Codes become bf16 exactly; a block's key scale multiplies its
// scores, its value scale its weights (both powers of two).
//
// float32 queries, and the weights for them, enter as three exact bf16 terms
// (24 bits, the whole range of float32), bf16 queries as they are and their
// weights rounded to bf16, as many bits as the outputs keep. Scores,
// statistics and sums are float32.
#include <algorithm>

#include "kv_attention.h"

namespace fa {
namespace {

// One work item: 16 query rows of one key/value head over a run of blocks.
// Lane l: row l % 16, group l / 16. NC: slices of 64 dims (at most; nc in use).
// Its blocks go to the W waves in turn. A wave loads a block's keys
// while it turns the block before into weights and sums, and its values likewise, as registers
// allow: the loads of one block (D = 128: 16 KB) are always under way.
template <typename T, int TERMS, int NC, int W>
__global__ __launch_bounds__(W * 64, W == 4 && NC <= 2 ? 2 : 1) void kv_attn_kernel(AttnArgs a) {
  // registers: what is loaded a block ahead (2: keys and values, 1: keys)
  constexpr int AHEAD = NC > 4 ? 0 : NC <= 2 || W == 4 ? 2 : TERMS == 1 || NC == 3 ? 1 : 0;
  constexpr int kWaves = W, kThreads = W * 64;
  constexpr int kMergeDims = W == 4 ? 128 : 64;      // dims that the waves' results are merged at a time
  constexpr int kLane = kMergeDims / (W * 4);        // and a thread's of them, W * 4 threads a row
  const int nc = NC <= 4 ? NC : a.c.nc;
  constexpr int kQ = TERMS * NC * 2 * 64;           // operands of 16 bytes
  constexpr int kM = kWaves * kTileRows * (kMergeDims + 4);  // floats
  __shared__ __align__(16) char lds[kQ * 16 > kM * 4 ? kQ * 16 : kM * 4];
  __shared__ float stat[kWaves][kTileRows][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, grp = lane >> 4;
  const bool planned = a.part != nullptr;
  const Item it = planned ? plan_item(a, blockIdx.x, 0, 0, 0) : direct_item(a, blockIdx.x, blockIdx.y);
  if (!it.ok) return;
  const KvSeq s = kv_seq(a.c, it.b);
  const int rows = s.n * a.G, r0 = it.tile * kTileRows;
  const int valid = min(kTileRows, rows - r0);
  T* out = (T*)a.out;
  const bool too_long = (int64_t)s.len > (int64_t)a.c.tstride * 64;  // tokens without a table entry: NaN, not a guess

  // what the tile sees, and this lane's row of it
  int lo, hi;
  const int ta = r0 / a.G, tb = (r0 + valid - 1) / a.G;
  seen_range(a, s, ta, tb, &lo, &hi);
  if (too_long) hi = lo;
  const int t = min(r0 + row, rows - 1) / a.G;
  int rlo, rhi, alo, ahi;  // the row's range, and what every row of the tile sees
  seen_range(a, s, t, t, &rlo, &rhi);
  {
    int l0, h0, l1, h1;
    seen_range(a, s, ta, ta, &l0, &h0);
    seen_range(a, s, tb, tb, &l1, &h1);
    alo = max(l0, l1);
    ahi = min(h0, h1);
  }
  int pg0 = lo >> 6, pg1 = hi <= lo ? pg0 : (hi + 63) >> 6;
  {
    const int np = pg1 - pg0;
    const int c0 = (int)((int64_t)np * it.chunk / it.chunks), c1 = (int)((int64_t)np * (it.chunk + 1) / it.chunks);
    pg1 = pg0 + c1;
    pg0 += c0;
  }

  // a block's codes, 16 bytes a lane: kr[slice * 4 + tile of 16 tokens], vr[tile of 16 dims]
  uint4 kr[AHEAD >= 1 ? NC * 4 : 1], vr[AHEAD == 2 ? NC * 4 : 1];
  auto part = [&](int id, int which) {
    return reinterpret_cast<const uint4*>(kv_part(a.c, id, it.h, which)) + row * 4 + grp;
  };
  auto key = [&](const uint4* p, int i) {  // no such block: keys that are NaN
    return p && (NC <= 4 || i < nc * 4) ? p[(i >> 2) * 256 + (i & 3) * 64]
                                        : make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
  };
  auto value = [&](const uint4* p, int i) {
    return p && (NC <= 4 || i < nc * 4) ? p[i * 64] : make_uint4(0, 0, 0, 0);
  };
  auto load_k = [&](int id) {
    if constexpr (AHEAD >= 1) {
      const uint4* p = id >= 0 ? part(id, 0) : nullptr;
#pragma unroll
      for (int i = 0; i < NC * 4; i++) kr[i] = key(p, i);
    }
  };
  auto load_v = [&](int id) {
    if constexpr (AHEAD == 2) {
      const uint4* p = id >= 0 ? part(id, 1) : nullptr;
#pragma unroll
      for (int i = 0; i < NC * 4; i++) vr[i] = value(p, i);
    }
  };
  auto scales = [&](int id) {
    return id >= 0 ? *reinterpret_cast<const float2*>(a.c.scales + ((int64_t)id * a.c.hkv + it.h) * 2)
                   : make_float2(1.f, 1.f);
  };
  Blocks blocks(a, it.b, pg0 + wave, kWaves, pg1);
  int id = blocks.at(a, it.b, 0), turn = 0;
  float2 ksv = make_float2(1.f, 1.f);
  if (pg0 + wave < pg1) {
    ksv = scales(id);
    load_k(id);
    load_v(id);
  }

  // the tile's queries as operands in LDS: [term][slice of 32 dims][lane]
  uint4* qf = reinterpret_cast<uint4*>(lds);
  for (int i = tid; i < nc * 2 * 64; i += kThreads) {
    const int ks = i >> 6, l = i & 63, r = r0 + (l & 15);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const int tok = r / a.G, head = it.h * a.G + (r - tok * a.G);
      const T* p = (const T*)a.q + (s.row0 + tok) * a.q_st + head * a.q_sh;
      load8(p, (ks >> 1) * 64 + (l >> 4) * 16 + (ks & 1) * 8, a.c.D, a.vec, v);
    }
    bf16x8 tm[TERMS];
    terms_of<TERMS>(v, tm);
#pragma unroll
    for (int k = 0; k < TERMS; k++) qf[(k * NC * 2 + ks) * 64 + l] = __builtin_bit_cast(uint4, tm[k]);
  }
  __syncthreads();

  kvf4 acc[NC * 4];
#pragma unroll
  for (int i = 0; i < NC * 4; i++) acc[i] = kvf4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;

  for (int p = pg0 + wave; p < pg1; p += kWaves) {
    const int id1 = blocks.at(a, it.b, ++turn);
    const float ks = ksv.x, vs = ksv.y;
    const int j0 = p * 64;
    const uint4* kp = id >= 0 ? part(id, 0) : nullptr;
    const uint4* vp = id >= 0 ? part(id, 1) : nullptr;

    // S^T: four tiles of 16 tokens
    kvf4 sc4[4];
#pragma unroll
    for (int tt = 0; tt < 4; tt++) sc4[tt] = kvf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; c++) {
      if (NC > 4 && c >= nc) continue;
      uint4 kc[4];
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
        if constexpr (AHEAD >= 1) kc[tt] = kr[c * 4 + tt];
        else kc[tt] = key(kp, c * 4 + tt);
      }
#pragma unroll
      for (int k = 0; k < TERMS; k++) {
        const bf16x8 q0 = __builtin_bit_cast(bf16x8, qf[(k * NC * 2 + c * 2) * 64 + lane]);
        const bf16x8 q1 = __builtin_bit_cast(bf16x8, qf[(k * NC * 2 + c * 2 + 1) * 64 + lane]);
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
          sc4[tt] = mfma(widen(kc[tt].x, kc[tt].y), q0, sc4[tt]);
          sc4[tt] = mfma(widen(kc[tt].z, kc[tt].w), q1, sc4[tt]);
        }
      }
    }
    const bool more = p + kWaves < pg1;
    if (more) {
      ksv = scales(id1);
      load_k(id1);
    }
    const float mul = a.scale2 * ks;
    const bool edge = j0 < alo || j0 + 64 > ahi;  // some row does not see some token
    float top = -__builtin_inff();
#pragma unroll
    for (int tt = 0; tt < 4; tt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float x = sc4[tt][i] * mul;
        if (edge) {
          const int j = j0 + tt * 16 + grp * 4 + i;
          x = j >= rlo && j < rhi ? x : -__builtin_inff();
        }
        sc4[tt][i] = x;
        top = fmaxf(top, x);
      }
    const float mn = fmaxf(m, row_max(top));
    const float mu = mn == -__builtin_inff() ? 0.f : mn;  // a row that has seen nothing yet: weights 0, not NaN
    const float alpha = __builtin_amdgcn_exp2f(m - mu);
    if (__ballot(mn != m)) {
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NC * 4; i++) {
        acc[i] *= alpha;
      }
    }
    m = mn;
    // weights and their operands: two steps of 32 tokens
    const float f = vs * kWeightScale;
    bf16x8 pt[2][TERMS];
#pragma unroll
    for (int st2 = 0; st2 < 2; st2++) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float x = __builtin_amdgcn_exp2f(sc4[st2 * 2 + (i >> 2)][i & 3] - mu);
        l += x;
        w[i] = x * f;
      }
      terms_of<TERMS>(w, pt[st2]);
    }
    // Tokens that no row of the tile sees may hold anything (a length ends
    // inside the block): their value codes become zero. Tokens that some rows
    // see and others do not may be NaN: a zero weight times NaN would reach
    // the others, so NaN codes go aside and are counted by a product of their
    // own against the rows that see them.
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    if (edge) {
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
        keep[tt] = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int j = j0 + tt * 16 + grp * 4 + i;
          if (j >= lo && j < hi) keep[tt] |= 0xFFu << (8 * i);
        }
      }
    }
    bf16x8 see[2];
    const bool mixed = edge && ta != tb;
    if (mixed) {
#pragma unroll
      for (int st2 = 0; st2 < 2; st2++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int j = j0 + (st2 * 2 + (i >> 2)) * 16 + grp * 4 + (i & 3);
          see[st2][i] = (__bf16)(j >= rlo && j < rhi ? 1.f : 0.f);
        }
    }
#pragma unroll
    for (int dt = 0; dt < NC * 4; dt++) {
      if (NC > 4 && dt >= nc * 4) continue;
      uint4 v;
      if constexpr (AHEAD == 2) v = vr[dt];
      else v = value(vp, dt);
      if (edge) {
        v.x &= keep[0]; v.y &= keep[1]; v.z &= keep[2]; v.w &= keep[3];
        const uint4 nb = make_uint4(nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w));
        if (mixed && __ballot((nb.x | nb.y | nb.z | nb.w) != 0)) {
          // 0x80 of a NaN byte -> 0x38, the code of one
          auto one = [](uint32_t b) { return (b >> 7) * 0x38u; };
          kvf4 cnt = {0.f, 0.f, 0.f, 0.f};
          cnt = mfma(widen(one(nb.x), one(nb.y)), see[0], cnt);
          cnt = mfma(widen(one(nb.z), one(nb.w)), see[1], cnt);
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (cnt[i] > 0.f) acc[dt][i] = __builtin_nanf("");
          auto drop = [](uint32_t w, uint32_t b) { return w & ~((b >> 7) * 0xFFu); };
          v = make_uint4(drop(v.x, nb.x), drop(v.y, nb.y), drop(v.z, nb.z), drop(v.w, nb.w));
        }
      }
      const bf16x8 v0 = widen(v.x, v.y), v1 = widen(v.z, v.w);
#pragma unroll
      for (int k = 0; k < TERMS; k++) {
        acc[dt] = mfma(v0, pt[0][k], acc[dt]);
        acc[dt] = mfma(v1, pt[1][k], acc[dt]);
      }
    }
    if (more) load_v(id1);
    id = id1;
  }

  // merge the waves: maxima and sums, then the outputs kMergeDims at a time
  l = row_sum(l);
  if (grp == 0) {
    stat[wave][row][0] = m;
    stat[wave][row][1] = l;
  }
  __syncthreads();
  float M = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < kWaves; w++) M = fmaxf(M, stat[w][row][0]);
  const float Mu = M == -__builtin_inff() ? 0.f : M;
  const float mine = __builtin_amdgcn_exp2f(m - Mu);
  // the output rows: W * 4 threads a row, each kLane dims of every kMergeDims
  const int orow = tid / (W * 4), oat = (tid % (W * 4)) * kLane;
  float oM = -__builtin_inff(), L = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; w++) oM = fmaxf(oM, stat[w][orow][0]);
  const float oMu = oM == -__builtin_inff() ? 0.f : oM;
#pragma unroll
  for (int w = 0; w < kWaves; w++) L += stat[w][orow][1] * __builtin_amdgcn_exp2f(stat[w][orow][0] - oMu);
  const bool split = it.chunks > 1;
  const int Dp = nc * 64;
  const int otok = (r0 + orow) / a.G, ohead = it.h * a.G + (r0 + orow) - otok * a.G;
  float fin = 1.f;
  if (!split) {
    int l0, h0;
    seen_range(a, s, min(otok, s.n - 1), min(otok, s.n - 1), &l0, &h0);
    fin = too_long ? __builtin_nanf("") : h0 <= l0 ? 0.f : (1.f / kWeightScale) / L;
  }
  const bool empty = !split && fin == 0.f;
  float* buf = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int c = 0; c < (NC * 64 + kMergeDims - 1) / kMergeDims; c++) {
    if (NC > 4 && c * kMergeDims >= nc * 64) continue;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < kMergeDims / 16; dt++) {
      if (c * (kMergeDims / 16) + dt < NC * 4)
        *reinterpret_cast<kvf4*>(buf + (wave * kTileRows + row) * (kMergeDims + 4) + dt * 16 + grp * 4) =
            acc[c * (kMergeDims / 16) + dt] * mine;
    }
    __syncthreads();
    const int d = c * kMergeDims + oat;
    if (orow < valid && d < Dp) {
      float o[kLane];
#pragma unroll
      for (int i = 0; i < kLane; i++) o[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++)
#pragma unroll
        for (int i = 0; i < kLane; i++) o[i] += buf[(w * kTileRows + orow) * (kMergeDims + 4) + oat + i];
      if (split) {
        float* to = a.part + ((it.first + it.chunk) * kTileRows + orow) * Dp + d;
#pragma unroll
        for (int i = 0; i < kLane; i++) to[i] = o[i];
      } else {
        T* to = out + ((s.row0 + otok) * a.H + ohead) * (int64_t)a.c.D;
#pragma unroll
        for (int i = 0; i < kLane; i++)
          if (d + i < a.c.D) st(to + d + i, empty ? 0.f : o[i] * fin);
      }
    }
  }
  if (split && oat == 0 && orow < valid) {
    float* to = a.part + a.parts * kTileRows * Dp + ((it.first + it.chunk) * kTileRows + orow) * 2;
    to[0] = oM;
    to[1] = L;
  }
}

// Joins the parts of a planned call's split tiles: one workgroup for each
// row and head; 16 nc lanes by four dims, the rest of the workgroup by parts.
template <typename T>
__global__ __launch_bounds__(256) void kv_merge_kernel(AttnArgs a) {
  __shared__ float w[kTarget + 1];
  __shared__ float red[4], red2[4];
  __shared__ float sum[256 * 4];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y, h = head / a.G;
  const int32_t* cu = a.c.cu;
  const int b = kv_find(a.c.nseq, row, [&](int i) { return (int64_t)cu[i]; });
  const KvSeq s = kv_seq(a.c, b);
  const int64_t tok = row - s.row0;
  if (tok < 0 || tok >= s.n) return;
  const int r = (int)tok * a.G + (head - h * a.G), tile = r / a.tile, tr = r - tile * a.tile;
  const Item it = plan_item(a, -1, b, tile, h);
  if (!it.ok || it.chunks <= 1) return;
  const int Dp = a.c.nc * 64, n = it.chunks;
  const float* stat = a.part + a.parts * a.tile * Dp + (it.first * a.tile + tr) * 2;
  float M = -__builtin_inff();
  for (int i = tid; i < n; i += 256) M = fmaxf(M, stat[(int64_t)i * a.tile * 2]);
  M = wave_max(M);
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float Mu = M == -__builtin_inff() ? 0.f : M;
  float L = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float f = __builtin_amdgcn_exp2f(stat[(int64_t)i * a.tile * 2] - Mu);
    w[i] = f;
    L += f * stat[(int64_t)i * a.tile * 2 + 1];
  }
  L = wave_sum(L);
  if ((tid & 63) == 0) red2[tid >> 6] = L;
  __syncthreads();
  L = (red2[0] + red2[1]) + (red2[2] + red2[3]);
  const int lanes = a.c.nc * 16, groups = 256 / lanes, g = tid / lanes, ln = tid - g * lanes;
  kvf4 o = {0.f, 0.f, 0.f, 0.f};
  if (g < groups) {
    const float* src = a.part + (it.first * a.tile + tr) * Dp + ln * 4;
#pragma unroll 8
    for (int i = g; i < n; i += groups)
      o += *reinterpret_cast<const kvf4*>(src + (int64_t)i * a.tile * Dp) * w[i];
  }
  *reinterpret_cast<kvf4*>(sum + tid * 4) = o;
  __syncthreads();
  if (g != 0) return;
  for (int i = 1; i < groups; i++) o += *reinterpret_cast<const kvf4*>(sum + (i * lanes + ln) * 4);
  int l0, h0;
  seen_range(a, s, (int)tok, (int)tok, &l0, &h0);
  const bool too_long = (int64_t)s.len > (int64_t)a.c.tstride * 64;
  const float fin = too_long ? __builtin_nanf("") : (1.f / kWeightScale) / L;
  T* to = (T*)a.out + (row * a.H + head) * (int64_t)a.c.D;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (ln * 4 + i < a.c.D) st(to + ln * 4 + i, h0 <= l0 ? 0.f : o[i] * fin);
}

// Tiles of many rows are split only where they are fewer than this: joining
// the parts of every row costs more than a partly filled card.
constexpr int kWideItems = 200;

// How a call runs, from its sizes alone.
struct Shape {
  int tile;        // rows of a work item
  int64_t slots;   // tiles, at most
  int64_t parts;   // parts of a split token axis, at most; 0: not split
};

Shape shape_of(const KvAttnArgs& a) {
  Shape r;
  const int64_t all = a.c.rows * (a.H / a.c.hkv);
  r.tile = kv_tile_rows(a.c.nc, all, a.c.nseq);
  r.slots = all / r.tile + a.c.nseq;
  const int64_t items = r.slots * a.c.hkv;
  // enough tiles without, or no sequence that could be cut
  if (items >= (r.tile == kTileRows ? kTarget : kWideItems) || a.c.tstride <= kWhole) {
    r.parts = 0;
  } else {
    const int64_t most = (a.c.tstride + kMinChunk - 1) / kMinChunk;
    r.parts = std::min((int64_t)kTarget + items, items * most);
  }
  return r;
}

template <typename T, int TERMS>
int rows16_t(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  const dim3 grid = a.part ? dim3((unsigned)a.parts) : dim3((unsigned)slots, (unsigned)a.c.hkv);
  // eight waves for a tile that is not split (its blocks end sooner), four
  // where there are parts enough
  const bool wide = !a.part;
#define FA_KV_A(N)                                                              \
  do {                                                                          \
    if (wide && N <= 4) kv_attn_kernel<T, TERMS, N, N <= 4 ? 8 : 4><<<grid, 512, 0, s>>>(a); \
    else kv_attn_kernel<T, TERMS, N, 4><<<grid, 256, 0, s>>>(a);                \
  } while (0)
  if (a.c.nc == 1) FA_KV_A(1);
  else if (a.c.nc == 2) FA_KV_A(2);
  else if (a.c.nc == 3) FA_KV_A(3);
  else if (a.c.nc == 4) FA_KV_A(4);
  else FA_KV_A(8);
#undef FA_KV_A
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

template <typename T, int TERMS>
int attn_t(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  const int rc = a.tile == kTileRows ? rows16_t<T, TERMS>(ctx, a, slots, s)
                                     : launch_kv_tiles_attn(ctx, a, TERMS == 3 ? FA_DT_F32 : FA_DT_BF16, slots, s);
  if (rc) return rc;
  if (a.part) {
    kv_merge_kernel<T><<<dim3((unsigned)a.c.rows, (unsigned)a.H), 256, 0, s>>>(a);
    FA_CHECK_LAUNCH(ctx);
  }
  return FA_OK;
}

}  // namespace

size_t kv_attention_scratch(const KvAttnArgs& a) {
  const Shape h = shape_of(a);
  return (size_t)h.parts * h.tile * (a.c.nc * 64 + 2) * sizeof(float);
}

int launch_kv_attention(fa_ctx* ctx, const KvAttnArgs& k, void* scratch, hipStream_t s) {
  AttnArgs a;
  a.c = k.c;
  a.q = k.q;
  a.q_st = k.q_st;
  a.q_sh = k.q_sh;
  a.H = k.H;
  a.G = k.H / k.c.hkv;
  a.causal = k.causal;
  a.window = k.window;
  a.scale2 = (float)((double)k.scale * 1.4426950408889634);
  a.out = k.out;
  const Shape h = shape_of(k);
  a.tile = h.tile;
  a.parts = h.parts;
  a.part = a.parts ? static_cast<float*>(scratch) : nullptr;
  a.vec = (reinterpret_cast<uintptr_t>(k.q) & 15) == 0 && (k.q_st | k.q_sh) % (k.dtype == FA_DT_F32 ? 4 : 8) == 0;
  a.out_vec = (reinterpret_cast<uintptr_t>(k.out) & 15) == 0 && k.c.D % 4 == 0;
  return k.dtype == FA_DT_F32 ? attn_t<float, 3>(ctx, a, h.slots, s)
                              : attn_t<uint16_t, 1>(ctx, a, h.slots, s);
}

}  // namespace fa
