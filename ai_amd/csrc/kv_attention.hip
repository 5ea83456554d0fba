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
// weights as two (17 bits: one would put an error of an output's own rounding
// beside it, relative to the sum of magnitudes and not to the output). Scores,
// statistics and sums are float32.
#include <algorithm>

#include "kv_attention.h"

namespace fa {
namespace {

// Joins the parts of query row r of item it (row tr of its tile) in their
// order, by 16 threads: thread ln the dims 64 c + 4 ln + 0..3. A few parts at
// a time, whose loads go out together.
template <typename T, int NC>
__device__ __forceinline__ void join_row(const AttnArgs& a, const KvSeq& s, const Item& it, int r, int tr, int ln) {
  const int n = it.chunks, nc = a.c.nc, Dp = nc * 64, rows = a.tile;
  const float* jstat = a.part + a.parts * rows * Dp + (it.first * rows + tr) * 2;
  const float* src = a.part + (it.first * rows + tr) * Dp + ln * 4;
  constexpr int kBatch = NC <= 2 ? 8 : NC <= 4 ? 4 : 2;
  float jM = -__builtin_inff(), jL = 0.f, o[NC * 4];
#pragma unroll
  for (int i = 0; i < NC * 4; i++) o[i] = 0.f;
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    float2 ml[kBatch], x[kBatch][NC * 2];
    float top = jM;
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      ml[i] = make_float2(-__builtin_inff(), 0.f);
#pragma unroll
      for (int c = 0; c < NC * 2; c++) x[i][c] = make_float2(0.f, 0.f);
      if (i0 + i < n) {
        ml[i] = get2(jstat + (int64_t)(i0 + i) * rows * 2);
#pragma unroll
        for (int c = 0; c < NC * 2; c++)
          if (c < nc * 2) x[i][c] = get2(src + (int64_t)(i0 + i) * rows * Dp + (c >> 1) * 64 + (c & 1) * 2);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) top = fmaxf(top, ml[i].x);
    const float mu = top == -__builtin_inff() ? 0.f : top, alpha = __builtin_amdgcn_exp2f(jM - mu);
    jM = top;
    jL *= alpha;
#pragma unroll
    for (int c = 0; c < NC * 4; c++) o[c] *= alpha;
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const float f = __builtin_amdgcn_exp2f(ml[i].x - mu);
      jL = fmaf(ml[i].y, f, jL);
#pragma unroll
      for (int c = 0; c < NC * 2; c++) {
        o[c * 2] = fmaf(x[i][c].x, f, o[c * 2]);
        o[c * 2 + 1] = fmaf(x[i][c].y, f, o[c * 2 + 1]);
      }
    }
  }
  const int tok = r / a.G, head = it.h * a.G + r - tok * a.G;
  int l0, h0;
  seen_range(a, s, tok, tok, &l0, &h0);
  const bool too_long = (int64_t)s.len > (int64_t)a.c.tstride * 64;
  const float fin = too_long ? __builtin_nanf("") : (1.f / kWeightScale) / jL;
  T* to = (T*)a.out + ((s.row0 + tok) * a.H + head) * (int64_t)a.c.D;
#pragma unroll
  for (int c = 0; c < NC; c++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int d = c * 64 + ln * 4 + e;
      if (d < a.c.D) st(to + d, h0 <= l0 ? 0.f : o[c * 4 + e] * fin);
    }
}

// Workgroups that a CU holds, by their registers.
constexpr int few_per_cu(int nc, int rt) { return nc * rt <= 4 ? 2 : 1; }

// One work item: 16 RT query rows of one key/value head over a run of blocks.
// Lane l: rows l % 16 of each 16, group l / 16. NC: slices of 64 dims.
// Its blocks go to the four waves in turn, their results are merged at the
// end. A wave loads a block's keys while it works on the scores of the block
// before, and its values while it works on the next scores, so that about a
// block (D = 128: 16 KB) is always under way: 64 sequences of up to 8192
// tokens (606 MB) take 127 us, 4.8 TB/s, against 219 without, and a large copy
// moves 5.1 TB/s. Where registers for that leave room for fewer workgroups, one
// set serves both (not AHEAD): a slice's values are loaded where its keys were,
// the next block's keys where its values were, so half a block is under way
// (64 sequences of 2000 tokens, 16 heads on 4 of 512 dims: 207 us without, 80;
// drafts of 2 to 5 tokens on windows of 512, 8 heads on 2 of 256 dims: 18.0 us with
// half a block and two workgroups a CU, 1.4 less than a block ahead).
template <typename T, int TERMS, int NC, int RT>
__global__ __launch_bounds__(256, few_per_cu(NC, RT)) void kv_attn_kernel(AttnArgs a) {
  constexpr int WT = TERMS == 3 ? 3 : 2;  // terms of a weight; TERMS: of a query
  constexpr int kRows = 16 * RT;
  constexpr bool AHEAD = NC * RT <= 2;  // loads a block ahead, else half of one
  constexpr int kWaves = 4, kThreads = kWaves * 64;
  constexpr int kMergeDims = 128;         // dims that the waves' results are merged at a time
  constexpr int kLane = kMergeDims / 16;  // and a thread's of them, 16 threads a row
  constexpr int nc = NC;
  constexpr int kQ = RT * TERMS * NC * 2 * 64;        // operands of 16 bytes
  constexpr int kM = kWaves * 16 * (kMergeDims + 4);  // floats
  __shared__ __align__(16) char lds[kQ * 16 > kM * 4 ? kQ * 16 : kM * 4];
  __shared__ float stat[kWaves][kRows][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, grp = lane >> 4;
  const bool planned = a.part != nullptr;
  const Item it = planned ? plan_item(a, blockIdx.x, 0, 0, 0) : direct_item(a, blockIdx.x, blockIdx.y, kRows);
  if (!it.ok) return;
  const KvSeq s = it.s;
  const int rows = s.n * a.G, r0 = it.tile * kRows;
  const int valid = min(kRows, rows - r0);
  T* out = (T*)a.out;
  const bool too_long = (int64_t)s.len > (int64_t)a.c.tstride * 64;  // tokens without a table entry: NaN, not a guess

  // what the tile sees, and this lane's rows of it
  int lo, hi;
  const int ta = r0 / a.G, tb = (r0 + valid - 1) / a.G;
  seen_range(a, s, ta, tb, &lo, &hi);
  if (too_long) hi = lo;
  int rlo[RT], rhi[RT], alo, ahi;  // its rows' ranges, and what every row of the tile sees
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int t = min(r0 + rt * 16 + row, rows - 1) / a.G;
    seen_range(a, s, t, t, &rlo[rt], &rhi[rt]);
  }
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
  // (not AHEAD: kr alone, a slice's values after its keys, the next keys after them)
  uint4 kr[NC * 4], vr[AHEAD ? NC * 4 : 1];
  auto part = [&](int id, int which) {
    return static_cast<const uint8_t*>(kv_part(a.c, id, it.h, which));
  };
  const uint32_t mine16 = (uint32_t)(row * 4 + grp) * 16;  // (a base that all lanes share and 32 bits of each)
  auto key = [&](const uint8_t* p, int i) {  // no such block: keys that are NaN
    return p ? *reinterpret_cast<const uint4*>(p + ((i >> 2) * 4096 + (i & 3) * 1024) + mine16) : make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
  };
  auto value = [&](const uint8_t* p, int i) {
    return p ? *reinterpret_cast<const uint4*>(p + i * 1024 + mine16) : make_uint4(0, 0, 0, 0);
  };
  auto load_k = [&](int id) {
    const uint8_t* p = id >= 0 ? part(id, 0) : nullptr;
#pragma unroll
    for (int i = 0; i < NC * 4; i++) kr[i] = key(p, i);
  };
  auto load_v = [&](int id) {
    if constexpr (AHEAD) {
      const uint8_t* p = id >= 0 ? part(id, 1) : nullptr;
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

  // the tile's queries as operands in LDS: [16 rows][term][slice of 32 dims][lane]
  uint4* qf = reinterpret_cast<uint4*>(lds);
  for (int i = tid; i < RT * nc * 2 * 64; i += kThreads) {
    const int rt = RT == 1 ? 0 : i / (nc * 2 * 64), ks = (i >> 6) - rt * nc * 2, l = i & 63, r = r0 + rt * 16 + (l & 15);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const int tok = r / a.G, head = it.h * a.G + (r - tok * a.G);
      const T* p = (const T*)a.q + (s.row0 + tok) * a.q_st + head * a.q_sh;
      load8(p, (ks >> 1) * 64 + (l >> 4) * 16 + (ks & 1) * 8, a.c.D, a.vec, v);
    }
    bf16x8 tm[TERMS];
    terms_of<TERMS>(v, tm);
#pragma unroll
    for (int k = 0; k < TERMS; k++) qf[((rt * TERMS + k) * NC * 2 + ks) * 64 + l] = __builtin_bit_cast(uint4, tm[k]);
  }
  __syncthreads();

  kvf4 acc[RT][NC * 4];
  float m[RT], l[RT];
  uint64_t nan_sum[RT][2];  // sums that are NaN: bit 4 (tile % 16) + i of word tile / 16
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
#pragma unroll
    for (int i = 0; i < NC * 4; i++) acc[rt][i] = kvf4{0.f, 0.f, 0.f, 0.f};
    m[rt] = -__builtin_inff();
    l[rt] = 0.f;
    nan_sum[rt][0] = nan_sum[rt][1] = 0;
  }

  for (int p = pg0 + wave; p < pg1; p += kWaves) {
    const int id1 = blocks.at(a, it.b, ++turn);
    const float ks = ksv.x, vs = ksv.y;
    const int j0 = p * 64;
    const uint8_t* kp1 = id1 >= 0 ? part(id1, 0) : nullptr;
    const uint8_t* vp = id >= 0 ? part(id, 1) : nullptr;

    // S^T: four tiles of 16 tokens
    kvf4 sc4[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int tt = 0; tt < 4; tt++) sc4[rt][tt] = kvf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; c++) {
      uint4 kc[4];
#pragma unroll
      for (int tt = 0; tt < 4; tt++) kc[tt] = kr[c * 4 + tt];
      if constexpr (TERMS == 1) {
        bf16x8 q[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int u = 0; u < 2; u++)
            q[rt][u] = __builtin_bit_cast(bf16x8, qf[(rt * NC * 2 + c * 2 + u) * 64 + lane]);
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
          const bf16x8 k0 = widen(kc[tt].x, kc[tt].y), k1 = widen(kc[tt].z, kc[tt].w);
#pragma unroll
          for (int rt = 0; rt < RT; rt++) {
            sc4[rt][tt] = mfma(k0, q[rt][0], sc4[rt][tt]);
            sc4[rt][tt] = mfma(k1, q[rt][1], sc4[rt][tt]);
          }
        }
      } else {
        bf16x8 kw[4][2];
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
          kw[tt][0] = widen(kc[tt].x, kc[tt].y);
          kw[tt][1] = widen(kc[tt].z, kc[tt].w);
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int k = 0; k < TERMS; k++) {
            const bf16x8 q0 = __builtin_bit_cast(bf16x8, qf[((rt * TERMS + k) * NC * 2 + c * 2) * 64 + lane]);
            const bf16x8 q1 = __builtin_bit_cast(bf16x8, qf[((rt * TERMS + k) * NC * 2 + c * 2 + 1) * 64 + lane]);
#pragma unroll
            for (int tt = 0; tt < 4; tt++) {
              sc4[rt][tt] = mfma(kw[tt][0], q0, sc4[rt][tt]);
              sc4[rt][tt] = mfma(kw[tt][1], q1, sc4[rt][tt]);
            }
          }
      }
      if constexpr (!AHEAD) {
#pragma unroll
        for (int tt = 0; tt < 4; tt++) kr[c * 4 + tt] = value(vp, c * 4 + tt);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const bool more = p + kWaves < pg1;
    if (more) {
      ksv = scales(id1);
      if constexpr (AHEAD) load_k(id1);
    }
    const float mul = a.scale2 * ks;
    const bool edge = j0 < alo || j0 + 64 > ahi;  // some row does not see some token
    const float f = vs * kWeightScale;
    bf16x8 pt[RT][2][WT];  // weights as operands: two steps of 32 tokens
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      float top = -__builtin_inff();
#pragma unroll
      for (int tt = 0; tt < 4; tt++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = sc4[rt][tt][i] * mul;
          if (edge) {
            const int j = j0 + tt * 16 + grp * 4 + i;
            x = j >= rlo[rt] && j < rhi[rt] ? x : -__builtin_inff();
          }
          sc4[rt][tt][i] = x;
          top = fmaxf(top, x);
        }
      const float mn = fmaxf(m[rt], row_max(top));
      const float mu = mn == -__builtin_inff() ? 0.f : mn;  // a row that has seen nothing yet: weights 0, not NaN
      const float alpha = __builtin_amdgcn_exp2f(m[rt] - mu);
      if (__ballot(mn != m[rt])) {
        l[rt] *= alpha;
#pragma unroll
        for (int i = 0; i < NC * 4; i++) {
          acc[rt][i] *= alpha;
        }
      }
      m[rt] = mn;
#pragma unroll
      for (int st2 = 0; st2 < 2; st2++) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float x = __builtin_amdgcn_exp2f(sc4[rt][st2 * 2 + (i >> 2)][i & 3] - mu);
          l[rt] += x;
          w[i] = x * f;
        }
        terms_of<WT>(w, pt[rt][st2]);
      }
    }
    // Tokens that no row of the tile sees may hold anything (a length ends
    // inside the block): their value codes become zero. Tokens that some rows
    // see and others do not may be NaN: a zero weight times NaN would reach
    // the others, so NaN codes are dropped and counted by a product of their
    // own against the rows that see them; those sums become NaN at the end.
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
    const bool mixed = edge && ta != tb;
    uint32_t nan = 0;
#pragma unroll
    for (int dt = 0; dt < NC * 4; dt++) {
      uint4 v = AHEAD ? vr[AHEAD ? dt : 0] : kr[dt];
      if (edge) v = make_uint4(v.x & keep[0], v.y & keep[1], v.z & keep[2], v.w & keep[3]);
      if (mixed) {
        auto drop = [&](uint32_t w) {
          const uint32_t n = nan_bytes(w);
          nan |= n;
          return w & ~((n >> 7) * 0xFFu);
        };
        v = make_uint4(drop(v.x), drop(v.y), drop(v.z), drop(v.w));
      }
      const bf16x8 v0 = widen(v.x, v.y), v1 = widen(v.z, v.w);
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int k = 0; k < WT; k++) {
          acc[rt][dt] = mfma(v0, pt[rt][0][k], acc[rt][dt]);
          acc[rt][dt] = mfma(v1, pt[rt][1][k], acc[rt][dt]);
        }
      if constexpr (!AHEAD) {
        if ((dt & 3) == 3) {
#pragma unroll
          for (int i = dt - 3; i <= dt; i++) kr[i] = key(kp1, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (mixed && __ballot(nan != 0)) {
#pragma unroll 1
      for (int dt = 0; dt < nc * 4; dt++) {
        const uint4 v = value(vp, dt);
        const uint32_t n0 = nan_bytes(v.x & keep[0]) >> 7, n1 = nan_bytes(v.y & keep[1]) >> 7;
        const uint32_t n2 = nan_bytes(v.z & keep[2]) >> 7, n3 = nan_bytes(v.w & keep[3]) >> 7;
        if (__ballot((n0 | n1 | n2 | n3) != 0) == 0) continue;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          kvf4 cnt = {0.f, 0.f, 0.f, 0.f};  // 0x01 of a NaN byte -> 0x38, the code of one
#pragma unroll
          for (int st2 = 0; st2 < 2; st2++) {
            bf16x8 see;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int j = j0 + (st2 * 2 + (i >> 2)) * 16 + grp * 4 + (i & 3);
              see[i] = (__bf16)(j >= rlo[rt] && j < rhi[rt] ? 1.f : 0.f);
            }
            cnt = mfma(st2 ? widen(n2 * 0x38u, n3 * 0x38u) : widen(n0 * 0x38u, n1 * 0x38u), see, cnt);
          }
          uint64_t bits = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) bits |= (uint64_t)(cnt[i] > 0.f) << i;
          nan_sum[rt][0] |= dt < 16 ? bits << (4 * dt) : 0;
          if (NC > 4) nan_sum[rt][1] |= dt < 16 ? 0 : bits << (4 * (dt & 15));
        }
      }
    }
    if (more) load_v(id1);
    id = id1;
  }

#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    if (__ballot((nan_sum[rt][0] | nan_sum[rt][1]) != 0)) {
#pragma unroll
      for (int dt = 0; dt < NC * 4; dt++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (nan_sum[rt][dt >> 4] >> (4 * (dt & 15) + i) & 1) acc[rt][dt][i] = __builtin_nanf("");
    }
    // merge the waves: maxima and sums, then the outputs kMergeDims at a time
    l[rt] = row_sum(l[rt]);
    if (grp == 0) {
      stat[wave][rt * 16 + row][0] = m[rt];
      stat[wave][rt * 16 + row][1] = l[rt];
    }
  }
  __syncthreads();
  const bool split = it.chunks > 1;
  const int Dp = nc * 64;
  float* stats = a.part + a.parts * kRows * Dp;
  float* buf = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    if (rt && rt * 16 >= valid) break;
    float M = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWaves; w++) M = fmaxf(M, stat[w][rt * 16 + row][0]);
    const float Mu = M == -__builtin_inff() ? 0.f : M;
    const float mine = __builtin_amdgcn_exp2f(m[rt] - Mu);
    // the output rows: 16 threads a row, each kLane dims of every kMergeDims
    const int orow = rt * 16 + (tid >> 4), oat = (tid & 15) * kLane;
    float oM = -__builtin_inff(), L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) oM = fmaxf(oM, stat[w][orow][0]);
    const float oMu = oM == -__builtin_inff() ? 0.f : oM;
#pragma unroll
    for (int w = 0; w < kWaves; w++) L += stat[w][orow][1] * __builtin_amdgcn_exp2f(stat[w][orow][0] - oMu);
    const int otok = (r0 + orow) / a.G, ohead = it.h * a.G + (r0 + orow) - otok * a.G;
    float fin = 1.f;
    if (!split) {
      int l0, h0;
      seen_range(a, s, min(otok, s.n - 1), min(otok, s.n - 1), &l0, &h0);
      fin = too_long ? __builtin_nanf("") : h0 <= l0 ? 0.f : (1.f / kWeightScale) / L;
    }
    const bool empty = !split && fin == 0.f;
#pragma unroll
    for (int c = 0; c < (NC * 64 + kMergeDims - 1) / kMergeDims; c++) {
      __syncthreads();
#pragma unroll
      for (int dt = 0; dt < kMergeDims / 16; dt++) {
        if (c * (kMergeDims / 16) + dt < NC * 4)
          *reinterpret_cast<kvf4*>(buf + (wave * 16 + row) * (kMergeDims + 4) + dt * 16 + grp * 4) =
              acc[rt][c * (kMergeDims / 16) + dt] * mine;
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
          for (int i = 0; i < kLane; i++) o[i] += buf[(w * 16 + (tid >> 4)) * (kMergeDims + 4) + oat + i];
        if (split) {
          float* to = a.part + ((it.first + it.chunk) * kRows + orow) * Dp + d;
#pragma unroll
          for (int i = 0; i < kLane; i += 2) put2(to + i, o[i], o[i + 1]);
        } else {
          T* to = out + ((s.row0 + otok) * a.H + ohead) * (int64_t)a.c.D;
#pragma unroll
          for (int i = 0; i < kLane; i++)
            if (d + i < a.c.D) st(to + d + i, empty ? 0.f : o[i] * fin);
        }
      }
    }
    if (split && oat == 0 && orow < valid) put2(stats + ((it.first + it.chunk) * kRows + orow) * 2, oM, L);
  }
  if (!split) return;
  // The workgroup that ends last of a tile's joins its parts, in their order
  // (the result does not depend on which one that is), and leaves the count
  // at zero for the next call.
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's are where every workgroup finds them
  __syncthreads();
  if (tid == 0) {
    last = __hip_atomic_fetch_add(a.count + it.first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (uint32_t)it.chunks - 1;
    if (last) __hip_atomic_store(a.count + it.first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int r = tid >> 4; r < valid; r += 16) join_row<T, NC>(a, s, it, r0 + r, r, tid & 15);
}

// Joins the parts of split tiles of many rows: a workgroup for each 16 rows.
template <typename T>
__global__ __launch_bounds__(256) void kv_join_kernel(AttnArgs a) {
  const Item t = direct_item(a, blockIdx.x, blockIdx.y, 16);
  if (!t.ok) return;
  const KvSeq s = t.s;
  const int r = t.tile * 16 + (threadIdx.x >> 4), tile = r / a.tile;
  const int len = __builtin_amdgcn_readfirstlane(a.count[kPlanWord]);
  const Item it = plan_item(a, -1, t.b, tile, t.h, len);
  if (it.ok && it.chunks > 1 && r < s.n * a.G) join_row<T, 4>(a, s, it, r, r - tile * a.tile, threadIdx.x & 15);
}

// The kernel for many rows is taken where the work in 16-row tiles, tiles times
// blocks, is kWideWork or more, and a sequence and head has over 64 rows in bf16, 95
// in float32, in the mean of the batch. Less work than that is over before its 128 rows
// and the launch that joins its parts pay. us by it and by the kernel for few rows, with
// the work: bf16, 128 dims, 8 heads, 8000 tokens, 128 rows 32 and 30 (8 k), 256 rows 39
// and 39 (16 k), 512 rows 49 and 51 (32 k); one head, 30000 tokens, 256 rows 54 and 29
// (7.5 k); 64 sequences of 8192, one head, 80 rows 61 and 80 (45 k). float32, 256 dims,
// 16 sequences of 500, 4 heads, 128 rows 57 and 32 (4 k), 500 rows 60 and 116 (16 k). At
// 64 rows in bf16, 94 in float32, on 64 sequences: of 8192 tokens, one head 55 and 61, of
// 2000, 4 heads 65 and 48, in float32 103 and 87.
//
// One kernel takes the whole call, so sequences of many rows beside others of one have
// the form that the mean asks for (bf16, 32 heads on 8 of 128 dims, a prompt beside single
// tokens of 200 to 4000: 2048 tokens and 200 others 269 us, apart 73 and 168; 512 and 64
// others 67, apart 17 and 38; 512 and 16 others 26, apart 17 and 11).
constexpr int kWideWork = 16384;

// Its tiles are split, in about a part for each workgroup that the card holds, where
// they are fewer than kWideItems; beyond that, in kWideTarget, where plan_item's rule
// finds that a longest tile is long and the card far from full: every row of a part is
// written, read and joined. Prompts of 8 x 1100 tokens, 139 tiles of float32 rows of
// 256 dims on up to 18 blocks: 99 us whole, 93 in parts; 2 x 3000, 142 tiles on 47
// blocks: 228 and 126. In bf16, 512 tokens on 8000, 32 heads on 8 of 128 dims, 136
// tiles on 125 blocks: 224 and 109; 1536 on 3000, 392 tiles on 47: 100 and 120. Where
// workgroups have a CU each, a prompt's later tiles leave the earlier ones' CUs idle
// (kUneven: 8 heads on 2 of 256 dims, 4000 tokens, 252 tiles: 224 and 176 us); where
// two share one, the longer has it to itself then (16 on 4 of 128, 4000 tokens,
// 502 tiles: 130 and 136). Parts of fewer than kWideMin blocks cost more (2 x 3000
// in float32: 144 us with 8, 126 with 16), and so do more of them than fit at once
// (512 tokens on 8000, 3 heads on one of 256 dims in float32, 13 tiles: 64 us in 256
// parts, 90 in 512).
constexpr int kWideItems = 128, kWideTarget = 512, kWideMin = 16;
constexpr float kUneven = 0.4f;

// Tiles of kPairRows rows load and widen a block once for twice the rows: where
// they still fill the card (64 sequences of up to 8192 tokens, 24 rows on each of 8
// heads of 128 dims: bf16 228 us in tiles of 16 and 152, float32 246 and 176), or
// are kPairItems and full and see kPairBlocks (64 sequences, 64 rows on one head:
// 63 and 43; on the other side 16 of 2000 tokens, 32 rows on each of 8: 25 and 29,
// and 32 of 4000, 20 rows: 53 and 56).
constexpr int kPairItems = 96, kPairBlocks = 64;

// How a call runs, from its sizes alone.
struct Shape {
  int tile;           // rows of a work item
  int target, least, cap;  // of a split: parts aimed at, blocks of a part at least
  int span;                // blocks that a tile sees at most, by its window
  int once;                // of a split with cap: workgroups aimed at in one round
  float places, uneven;    // of a split that plan_item decides on
  int64_t slots;      // tiles, at most
  int64_t parts;      // parts, at most; 0: not split
};

// Whether a call's tiles can have 32 rows, 128.
bool may_be_pairs(const KvAttnArgs& a) {
  return a.c.nc <= 4 && a.c.rows * (a.H / a.c.hkv) > (int64_t)kTileRows * a.c.nseq;
}
bool may_be_wide(const KvAttnArgs& a) {
  return a.c.nc <= 4 && a.c.rows * (a.H / a.c.hkv) > (int64_t)(a.dtype == FA_DT_BF16 ? 64 : 95) * a.c.nseq;
}

Shape shape_of(const KvAttnArgs& a, int tile = 0) {
  Shape r;
  const int G = a.H / a.c.hkv;
  const int64_t all = a.c.rows * G, nseq = a.c.nseq;
  // tiles, about and at most
  auto tiles = [&](int rows) { return std::max((all + nseq * rows / 2) / rows, std::min(nseq, all)); };
  auto most_tiles = [&](int rows) { return all / rows + nseq; };
  // blocks that a tile of some rows can see, by the window
  auto span = [&](int rows) {
    return a.window ? (int)(((int64_t)a.window * (a.causal ? 1 : 2) + rows / G + 63) / 64 + 1) : 0x7FFFFFFF;
  };
  auto seen = [&](int rows) { return (int64_t)std::min(a.c.tstride, span(rows)); };
  r.tile = tile;
  if (!tile) {
    r.tile = kTileRows;
    const int64_t pairs = tiles(kPairRows) * a.c.hkv;
    if (may_be_wide(a) && tiles(kTileRows) * a.c.hkv * seen(kTileRows) >= kWideWork)
      r.tile = kWideRows;
    else if (may_be_pairs(a) &&
             (pairs >= 256 * few_per_cu(a.c.nc, 2) || (a.c.nc <= 2 && pairs >= kPairItems &&
                                                    seen(kPairRows) >= kPairBlocks && all >= kPairRows * nseq)))
      r.tile = kPairRows;
  }
  r.slots = most_tiles(r.tile);
  const int64_t items = r.slots * a.c.hkv;
  const bool wide = r.tile == kWideRows;
  r.span = span(r.tile);
  const int64_t blocks = seen(r.tile);
  const int per_cu = wide ? kv_tiles_per_cu(a.c.nc, a.dtype) : few_per_cu(a.c.nc, 2);  // (of pairs)
  r.target = wide ? 256 * per_cu : kTarget;
  r.least = kMinChunk;
  r.cap = wide ? 0 : kRound;
  r.once = r.tile == kPairRows ? 256 * per_cu : 256;
  r.places = r.uneven = 0.f;
  bool split = wide ? items < kWideItems : tiles(r.tile) * a.c.hkv < kTarget && items < 2 * kTarget;
  if (wide && !split) {
    r.target = kWideTarget;
    r.least = kWideMin;
    r.places = 256.f * (float)per_cu;
    r.uneven = per_cu == 1 && a.causal ? kUneven : 0.f;
    split = (float)blocks * (r.places - (1.f - r.uneven) * (float)items) >= kWideGain * r.places;
  }
  // enough tiles without, or no sequence that could be cut
  if (!split || blocks <= r.least) {
    r.parts = 0;
  } else {
    // as plan_item: a part has at least `least` blocks, total / target of them, and
    // total / once up to kRound; the last part of each item may be short
    const int64_t total = items * blocks, most = (blocks + r.least - 1) / r.least;
    const int64_t cut = wide ? r.target : std::max((int64_t)r.once, std::min((int64_t)kTarget, total / kRound));
    r.parts = std::min(cut + items + 8, items * most);  // (8: the kernel's sums are rounded)
  }
  return r;
}

template <typename T, int TERMS>
int few_t(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  const dim3 grid = a.part ? dim3((unsigned)a.parts) : dim3((unsigned)slots, (unsigned)a.c.hkv);
#define FA_KV_A(N)                                                                    \
  if (a.tile == kPairRows) kv_attn_kernel<T, TERMS, N, 2><<<grid, 256, 0, s>>>(a);    \
  else kv_attn_kernel<T, TERMS, N, 1><<<grid, 256, 0, s>>>(a)
  if (a.c.nc == 1) { FA_KV_A(1); }
  else if (a.c.nc == 2) { FA_KV_A(2); }
  else if (a.c.nc == 3) { FA_KV_A(3); }
  else if (a.c.nc == 4) { FA_KV_A(4); }
  else if (a.c.nc == 5) kv_attn_kernel<T, TERMS, 5, 1><<<grid, 256, 0, s>>>(a);
  else if (a.c.nc == 6) kv_attn_kernel<T, TERMS, 6, 1><<<grid, 256, 0, s>>>(a);
  else if (a.c.nc == 7) kv_attn_kernel<T, TERMS, 7, 1><<<grid, 256, 0, s>>>(a);
  else kv_attn_kernel<T, TERMS, 8, 1><<<grid, 256, 0, s>>>(a);
#undef FA_KV_A
  FA_CHECK_LAUNCH(ctx);
  return FA_OK;
}

template <typename T, int TERMS>
int attn_t(fa_ctx* ctx, const AttnArgs& a, int64_t slots, hipStream_t s) {
  const int rc = a.tile != kWideRows ? few_t<T, TERMS>(ctx, a, slots, s)
                                     : launch_kv_tiles_attn(ctx, a, TERMS == 3 ? FA_DT_F32 : FA_DT_BF16, slots, s);
  if (rc) return rc;
  if (a.part && a.tile == kWideRows) {
    const dim3 grid((unsigned)(a.c.rows * a.G / 16 + a.c.nseq), (unsigned)a.c.hkv);
    kv_join_kernel<T><<<grid, 256, 0, s>>>(a);
    FA_CHECK_LAUNCH(ctx);
  }
  return FA_OK;
}

}  // namespace

namespace {
size_t scratch_of(const KvAttnArgs& a, const Shape& h) {
  return h.parts ? kKvCountBytes + (size_t)h.parts * h.tile * (a.c.nc * 64 + 2) * sizeof(float) : 0;
}
}  // namespace

size_t kv_attention_scratch(const KvAttnArgs& a) { return scratch_of(a, shape_of(a)); }

size_t kv_attention_scratch_any(KvAttnArgs a) {
  size_t most = 0;
  a.window = 0;  // the more blocks a tile sees, the more parts; a window can only take other tiles
  for (int dtype : {FA_DT_F32, FA_DT_BF16})
    for (int causal : {0, 1})
      for (int tile : {kTileRows, kPairRows, kWideRows}) {
        a.dtype = dtype;
        a.causal = causal;
        if (tile == kTileRows || (tile == kPairRows ? may_be_pairs(a) : may_be_wide(a)))
          most = std::max(most, scratch_of(a, shape_of(a, tile)));
      }
  return most;
}

int64_t kv_attention_grid(const KvAttnArgs& a) {
  const Shape h = shape_of(a);
  return h.parts ? h.parts : h.tile != kWideRows ? h.slots : h.slots * a.c.hkv;
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
  a.target = h.target;
  a.least = h.least;
  a.cap = h.cap;
  a.span = h.span;
  a.once = (float)h.once;
  a.places = h.places;
  a.uneven = h.uneven;
  a.parts = h.parts;
  a.count = static_cast<uint32_t*>(scratch);
  a.part = a.parts ? reinterpret_cast<float*>(static_cast<char*>(scratch) + kKvCountBytes) : nullptr;
  a.vec = (reinterpret_cast<uintptr_t>(k.q) & 15) == 0 && (k.q_st | k.q_sh) % (k.dtype == FA_DT_F32 ? 4 : 8) == 0;
  a.out_vec = (reinterpret_cast<uintptr_t>(k.out) & 15) == 0 && k.c.D % 4 == 0;
  return k.dtype == FA_DT_F32 ? attn_t<float, 3>(ctx, a, h.slots, s)
                              : attn_t<uint16_t, 1>(ctx, a, h.slots, s);
}

}  // namespace fa
