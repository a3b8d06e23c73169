// Backward pass of attention with shaped scores (see attn_mod.h).
//
// With t = tanh(s / cap), P the probabilities and dP = dO V^T:
//   dS = scale * P * (dP - delta) * (1 - t^2),  delta_i = sum_d dO_i O_i
//   dV = P^T dO,   dK = dS^T Q,   dQ = dS K
// P goes into dV rounded to bf16, as it went into O.  dS goes into dQ and dK
// as the sum of two bf16 numbers: rounded to one, its error is as large as
// that of rounding dQ and dK themselves, and both products have their other
// operand in registers already.
//
// Two kernels, each of which recomputes the scores: one walks the keys for
// 128 queries and keeps dQ in registers, the other walks the queries for 128
// keys and keeps dK and dV.  That is nine matrix products where one kernel
// would need seven, but nothing is added through memory: no fp32 copy of dQ,
// no atomics, and the same bits in every run.
//
// Bound by the matrix and the vector unit together, at the clock that they
// leave (2.05 GHz).  16384 tokens in three documents, 16 heads of 128 over 8,
// capped: dQ 947 us, 893 TFLOP/s, matrix unit 45 and vector unit 58 per cent
// busy; dK and dV 1353 us, 783 TFLOP/s, 38 and 44 per cent (a library
// product of 8192^3 on such a card: 1116 TFLOP/s).  On one where it reached
// 1166 they took 930 and 1300, and dS as one bf16 number 743 and 1140.
// Sequences of 512 in four documents, 16384 tokens, heads of 64: 78 and 95
// us, where moving the bytes takes 47 and 41.
//
// A query that sees nothing may hold anything, and so may the gradient of its
// row: dQ leaves such a row out of delta, notes its 32 queries in `blind`, and
// dK and dV stage the rows of noted tiles one by one, those as zeros.
#include "attn_mod.h"

namespace mxa {

// ---------------------------------------------------------------------------
// dQ (and delta): block = 128 queries of one head, wave = 32 queries along
// the lanes, as in the forward pass.
// ---------------------------------------------------------------------------
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void attn_mod_dq_kernel(AttnArgs a) {
  constexpr int KK = D / 16, DB = D / 32;
  constexpr int TILE = 128 * D, V0 = 2 * TILE, ID0 = 4 * TILE;
  __shared__ __align__(1024) char smem[ID0 + 512];
  lds_char* const sm = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(size_t)sm;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  int bh, rank;
  attn_block(blockIdx.x, a.B * a.H, bh, rank);
  const int qb = cdiv(a.Tq, 128) - 1 - rank;
  const int h = bh % a.H, b = bh / a.H;
  const int hk = h / a.G;
  const SeqMask m = attn_seq_mask(a, b);

  const int q0 = qb * 128 + wave * 32;
  const int qi = q0 + col;
  const bool qok = qi < a.Tq;
  const int pos = qi + m.off;
  int sq = 0;
  if (m.has_seg) sq = qok ? a.seg_q[(long)b * a.Tq + qi] : -1;

  RowSpan wav, blk;
  attn_spans(a, m, b, qb, wave, wav, blk);
  const int limit = m.has_seg && sq < 0 ? 0 : attn_limit(m, pos);
  ScoreFn f;
  f.set<CAP>(a.scale, a.cap, BIAS ? a.slopes[h] : 0.f);

  const bf16* kb = a.k + b * a.ksb + (long)hk * a.D;
  const bf16* vb = a.v + b * a.vsb + (long)hk * a.D;
  const int* skb = m.has_seg ? a.seg_k + (long)b * a.Tk : nullptr;
  const int2* rng = m.has_seg ? attn_ranges(a.rng_k, b, a.Tk) : nullptr;

  Stager<D, 64, 4> ks, vs;
  ks.init(a.kst, wave, lane);
  vs.init(a.vst, wave, lane);
  // keys that no query of the block sees may hold anything
  const int kend = max(attn_limit(m, blk.pmax), 0);
  auto stage = [&](int buf, const Tile& t) {
    const int* sg = t.neg ? skb : nullptr;
    const int r = t.t * 64;
    ks.copy(kb, a.kst, r, kend, a.D, sg, lds0 + buf * TILE, wave, lane);
    vs.copy(vb, a.vst, r, kend, a.D, sg, lds0 + V0 + buf * TILE, wave, lane);
    if (m.has_seg && wave == 0)
      attn_stage64(skb, t.t * 64, a.Tk, lds0 + ID0 + buf * 256, lane);
  };

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();

  const LaneAddr la = attn_lane_addr<D>(lane);
  TileWalk walk;
  walk.start(0, cdiv(kend, 64));
  Tile cur = walk.next(m, blk, wav, rng, lane);
  if (cur.t >= 0) stage(0, cur);
  // queries, their output gradients and delta
  bf16x8 qf[KK], gf[KK];
  float lse = MXA_INF, delta = 0.f;
  {
    const bool ok = qok && sq >= 0;
    const long row = ((long)b * a.H + h) * a.TqP + qi;
    const bf16* qp = a.q + b * a.qsb + (long)qi * a.qst + (long)h * a.D;
    const bf16* gp = a.dout + b * a.gsb + (long)qi * a.gst + (long)h * a.D;
    const bf16* op = a.o + b * a.osb + (long)qi * a.ost + (long)h * a.D;
    const bf16* lp = a.olo + (((long)b * a.Tq + qi) * a.H + h) * a.D;
    if (ok) lse = a.lse[row];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      qf[kk] = attn_load_q(qp, kk * 2 + half, a.D, ok, a.scale);
      gf[kk] = attn_load_row(gp, kk * 2 + half, a.D, ok);
      delta = dot8(gf[kk], attn_load_row(op, kk * 2 + half, a.D, ok), delta);
      delta = dot8(gf[kk], attn_load_row(lp, kk * 2 + half, a.D, ok), delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (lse == MXA_INF) {  // sees nothing: its gradient may hold anything
      delta = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) gf[kk] = bf16x8{};
    }
    if (half == 0 && qi < a.TqP) a.delta[row] = -delta;
    const bool blind = __ballot(qok && lse == MXA_INF) != 0;
    if (lane == 0 && q0 < a.TqP)
      a.blind[((long)b * a.H + h) * (a.TqP / 32) + q0 / 32] = blind;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      attn_settle(qf[kk]);
      attn_settle(gf[kk]);
    }
    asm volatile("" : "+v"(lse));
  }
  int buf = 0;
  while (cur.t >= 0) {
    attn_wait_copies<0>();
    __syncthreads();
    Tile nxt = walk.next(m, blk, wav, rng, lane);
    if (nxt.t >= 0) stage(buf ^ 1, nxt);
    if (cur.work) {
      const unsigned krow = la.row + buf * TILE, ktr = la.tr + buf * TILE;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        // short documents leave half of a wave's tiles half empty: 128 of
        // them 79 us, skipping 76; nothing to win where a tile is longer
        if (D == 64 && !(cur.work >> nb & 1)) continue;
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          s = mfma32(attn_row_frag(sm, krow, kk, nb * 64 * D), qf[kk], s);
          dp = mfma32(attn_row_frag(sm, krow, kk, V0 + nb * 64 * D), gf[kk],
                      dp);
        }
        const int j0 = cur.t * 64 + nb * 32 + 4 * half;
        const float d0 = BIAS ? (float)(pos + m.shift - j0) : 0.f;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = attn_z<CAP>(f, s[i]);
        if (cur.ids || cur.ends)
          attn_mask_keys(x, cur.ids, cur.ends, sm,
                         ID0 + buf * 256 + nb * 128 + 16 * half, sq,
                         limit - j0, attn_gone<CAP>());
        bf16x8 df[2], dl[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float ds[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int i = 8 * w + k, dj = 8 * (i >> 2) + (i & 3);
            const float off =
                BIAS ? fmaf(f.slope, fabsf(d0 - (float)dj), -lse) : -lse;
            ds[k] = fexp2(fmaf(x[i], f.mu, off)) * (dp[i] - delta);
            if (CAP) ds[k] *= attn_dtanh(x[i]);
          }
          split8(ds, df[w], dl[w]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const bf16x8 kt =
                attn_tr_frag<D>(sm, ktr, db, (nb * 2 + w) * 32 * D);
            dq[db] = mfma32(kt, df[w], dq[db]);
            dq[db] = mfma32(kt, dl[w], dq[db]);
          }
      }
    }
    cur = nxt;
    buf ^= 1;
  }

  __syncthreads();
  attn_store_rows<DB, false>(sm, wave * 64 * D, dq, attn_ds_scale<CAP>(a.scale),
                             a.dq + ((long)b * a.Tq * a.H + h) * a.D,
                             (long)a.H * a.D, q0, a.Tq, a.D, lane);
}

// ---------------------------------------------------------------------------
// dK, dV: block = 128 keys of one key head, 32 of them along the lanes of a
// wave; the queries of every head that shares them pass by in tiles of 64.
//
// D = 64: four waves that hold V as operands in registers and K in LDS: with
// K in registers as well, 193 of them, there is room for two blocks on a
// compute unit, not three (sequences of 512 in four documents 103 and 93 us,
// though 1 to 5 registers and some 50 scalars are spilled for it).
// D = 128: those 64 registers beside 128 of accumulators would leave room
// for one wave on a SIMD only, and nothing to overlap its phases with.  K
// and V lie in LDS instead, and eight waves share the keys: one half takes
// the first 32 queries of a tile, the other the last, and the two sums meet
// in LDS at the end.
//
// nsplit > 1: a block takes every nsplit-th tile and leaves its sums in the
// workspace for attn_dkv_join_kernel; for launches too small to fill the
// chip evenly.
// ---------------------------------------------------------------------------
template <int D, bool CAP, bool BIAS>
__global__
__launch_bounds__(D == 64 ? 256 : 512, D == 64 ? 3 : 2) void
attn_mod_dkv_kernel(AttnArgs a) {
  constexpr bool WIDE = D == 128;
  constexpr int KK = D / 16, DB = D / 32, NW = WIDE ? 8 : 4;
  // query and output-gradient tiles, two buffers of each; K, and V where it
  // lies here; log-sums, deltas and ids of the tiles
  constexpr int TILE = 128 * D, G0 = 2 * TILE, K0 = 4 * TILE;
  constexpr int V0 = K0 + 256 * D;
  constexpr int ST0 = WIDE ? V0 + 256 * D : V0;
  __shared__ __align__(1024) char smem[ST0 + 6 * 256];
  lds_char* const sm = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(size_t)sm;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int wk = wave & 3;  // this wave's 32 keys
  int bh, rank;  // the first keys are seen by the most queries
  attn_block(blockIdx.x, a.B * a.Hkv, bh, rank);
  const int kb = rank / a.nsplit, split = rank % a.nsplit;
  const int hk = bh % a.Hkv, b = bh / a.Hkv;
  const SeqMask m = attn_seq_mask(a, b);

  const int k0 = kb * 128 + wk * 32;
  const int kj = k0 + col;
  int sk = 0;
  if (m.has_seg) sk = kj < a.Tk ? a.seg_k[(long)b * a.Tk + kj] : -1;
  const bool kok = kj < m.kv_len && sk >= 0 &&
                   (!m.causal || kj < m.prefix || kj < a.Tq + m.off);
  // first position that sees this key (documents aside)
  const int NEVER = 0x7fffffff;
  const int first =
      !kok ? NEVER
           : (!m.causal || kj < m.prefix ? -0x7fffffff : kj);

  // spans of the wave and the block: the smallest `first` of a key that is
  // there, the largest (NEVER if one is not), ids
  auto first_of = [&](int j) {
    return !m.causal || j < m.prefix ? -0x7fffffff : j;
  };
  const int wlo = k0 < m.kv_len ? first_of(k0) : NEVER;
  const int whi = k0 + 31 < m.kv_len ? first_of(k0 + 31) : NEVER;
  const int blo = kb * 128 < m.kv_len ? first_of(kb * 128) : NEVER;
  int slo = 0, shi = 0, bslo = 0, bshi = 0;
  if (m.has_seg) {
    const int2* r = attn_ranges(a.rng_k, b, a.Tk) + kb * 4;
    const int2 w = r[wk];
    const int2 j = attn_join(attn_join(r[0], r[1]), attn_join(r[2], r[3]));
    slo = __builtin_amdgcn_readfirstlane(w.x);
    shi = __builtin_amdgcn_readfirstlane(w.y);
    bslo = __builtin_amdgcn_readfirstlane(j.x);
    bshi = __builtin_amdgcn_readfirstlane(j.y);
  }

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = zero16();

  const int ntq = cdiv(a.Tq, 64);
  const int2* rng = m.has_seg ? attn_ranges(a.rng_q, b, a.Tq) : nullptr;
  const int* sqb = m.has_seg ? a.seg_q + (long)b * a.Tq : nullptr;

  // Verdict on query tile t of a head: bit 0 block, bit 1 wave, bit 2 all
  // pairs of the wave visible, bit 3 queries that see nothing.
  auto judge = [&](int t, int g) {
    int2 r = make_int2(0, 0);
    if (m.has_seg) r = attn_join(rng[2 * t], rng[2 * t + 1]);
    ConstArgs* c = attn_args_here();
    const int2 bl = ((const int2*)c->blind)[
        ((long)b * c->H + hk * c->G + g) * ntq + t];
    const int p0 = t * 64 + m.off, p1 = min(t * 64 + 63, a.Tq - 1) + m.off;
    bool any = p1 >= blo && blo != NEVER, wany = p1 >= wlo && wlo != NEVER;
    bool all = p0 >= whi && whi != NEVER;
    if (m.has_seg) {
      any = any && max(max(bslo, r.x), 0) <= min(bshi, r.y);
      wany = wany && max(max(slo, r.x), 0) <= min(shi, r.y);
      all = all && slo == shi && r.x == slo && r.y == slo;
    }
    any = any && t % a.nsplit == split;
    return (any ? 1 : 0) | (wany ? 2 : 0) | (all ? 4 : 0) |
           (bl.x | bl.y ? 8 : 0);
  };

  int cg = 0, base = -64;
  u64 act = 0, wact = 0, wful = 0, blind = 0;
  struct QTile {
    int g, t;
    bool work, full, blind;
  };
  auto next = [&]() -> QTile {
    while (act == 0) {
      base += 64;
      if (base >= ntq) {
        base = 0;
        if (++cg >= a.G) return QTile{-1, 0, false, false, false};
      }
      int t = base + lane;
      int v = t < ntq ? judge(t, cg) : 0;
      act = __ballot(v & 1);
      wact = __ballot(v & 2);
      wful = __ballot(v & 4);
      blind = __ballot(v & 8);
    }
    int i = __builtin_ctzll(act);
    act &= act - 1;
    return QTile{cg, base + i, (bool)((wact >> i) & 1),
                 (bool)((wful >> i) & 1), (bool)((blind >> i) & 1)};
  };

  Stager<D, 64, NW> qs, gs;
  qs.init(a.qst, wave, lane);
  gs.init(a.gst, wave, lane);
  auto stage = [&](int buf, const QTile& t) {
    const int h = hk * a.G + t.g, r = t.t * 64;
    const long row = ((long)b * a.H + h) * a.TqP;
    // queries that see nothing, and their gradients, may hold anything
    const float* sg = nullptr;
    if (t.blind) sg = attn_args_here()->lse + row;
    qs.copy(a.q + b * a.qsb + (long)h * a.D, a.qst, r, a.Tq, a.D, sg,
            lds0 + buf * TILE, wave, lane);
    gs.copy(a.dout + b * a.gsb + (long)h * a.D, a.gst, r, a.Tq, a.D, sg,
            lds0 + G0 + buf * TILE, wave, lane);
    if (wave == 0)
      attn_stage64(a.lse + row, r, a.TqP, lds0 + ST0 + buf * 256, lane);
    if (wave == 1)
      attn_stage64(a.delta + row, r, a.TqP, lds0 + ST0 + 512 + buf * 256,
                   lane);
    if (wave == 2 && m.has_seg)
      attn_stage64(sqb, r, a.Tq, lds0 + ST0 + 1024 + buf * 256, lane);
  };

  const LaneAddr la = attn_lane_addr<D>(lane);
  ScoreFn f;
  QTile cur = next();
  if (cur.g >= 0) stage(0, cur);
  bf16x8 vf[WIDE ? 1 : KK];
  {
    const bf16* kp = a.k + b * a.ksb + (long)kj * a.kst + (long)hk * a.D;
    const bf16* vp = a.v + b * a.vsb + (long)kj * a.vst + (long)hk * a.D;
    // WIDE: a wave writes K or V of its keys, else K
    const bool isv = WIDE && wave >= 4;
    const int row = wk * 32 + col;
    bf16* img = (bf16*)(smem + (isv ? V0 : K0)) + row * D;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int ch = kk * 2 + half;
      bf16x8 x = isv ? attn_load_row(vp, ch, a.D, kok)
                     : attn_load_q(kp, ch, a.D, kok, a.scale);
      *(bf16x8*)&img[(ch ^ attn_key<D>(row)) << 3] = x;
      if constexpr (!WIDE) vf[kk] = attn_load_row(vp, ch, a.D, kok);
    }
    if constexpr (!WIDE) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) attn_settle(vf[kk]);
    }
  }
  int buf = 0;
  while (cur.g >= 0) {
    attn_wait_copies<0>();
    __syncthreads();
    QTile nxt = next();
    if (nxt.g >= 0) stage(buf ^ 1, nxt);
    if (cur.work) {
      f.set<CAP>(a.scale, a.cap, BIAS ? a.slopes[hk * a.G + cur.g] : 0.f);
#pragma unroll
      for (int it = 0; it < (WIDE ? 1 : 2); ++it) {
        const int nb = WIDE ? wave >> 2 : it;  // 32 queries of the tile
        const unsigned at = buf * TILE + nb * 64 * D;
        const unsigned qrow = la.row + at, qtr = la.tr + at;
        const unsigned krow = attn_here(la.row + wk * 64 * D);
        const unsigned st = ST0 + buf * 256 + nb * 128 + 16 * half;
        f32x16 s = zero16(), dp;
        // dp starts at -delta of its rows
#pragma unroll
        for (int ii = 0; ii < 4; ++ii) {
          const f32x4 e4 = attn_lds<f32x4>(sm, st + 32 * ii + 512);
#pragma unroll
          for (int i = 0; i < 4; ++i) dp[4 * ii + i] = e4[i];
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const bf16x8 kx = attn_row_frag(sm, krow, kk, K0);
          bf16x8 vx;
          if constexpr (WIDE)
            vx = attn_row_frag(sm, krow, kk, V0);
          else
            vx = vf[kk];
          s = mfma32(attn_row_frag(sm, qrow, kk, 0), kx, s);
          dp = mfma32(attn_row_frag(sm, qrow, kk, G0), vx, dp);
        }
        const int r0 = nb * 32 + 4 * half;  // this lane's first tile row
        const int p0 = cur.t * 64 + r0 + m.off;
        const float d0 = BIAS ? (float)(p0 + m.shift - kj) : 0.f;
        bf16x8 pf[2], df[2], dl[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float p[8], ds[8];
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            const int pr = p0 + 16 * w + 8 * ii;  // of four rows, pr..pr+3
            const unsigned sr = st + 64 * w + 32 * ii;
            const f32x4 l4 = attn_lds<f32x4>(sm, sr);
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = attn_z<CAP>(f, s[8 * w + 4 * ii + i]);
            if (!cur.full) {
              if (m.has_seg) {
                const i32x4 q4 = attn_lds<i32x4>(sm, sr + 1024);
                x[0] = q4.x == sk ? x[0] : attn_gone<CAP>();
                x[1] = q4.y == sk ? x[1] : attn_gone<CAP>();
                x[2] = q4.z == sk ? x[2] : attn_gone<CAP>();
                x[3] = q4.w == sk ? x[3] : attn_gone<CAP>();
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                x[i] = pr + i >= first ? x[i] : attn_gone<CAP>();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float off =
                  BIAS ? fmaf(f.slope,
                              fabsf(d0 + (float)(16 * w + 8 * ii + i)), -l4[i])
                       : -l4[i];
              const float pi = fexp2(fmaf(x[i], f.mu, off));
              float di = pi * dp[8 * w + 4 * ii + i];
              if (CAP) di *= attn_dtanh(x[i]);
              p[4 * ii + i] = pi;
              ds[4 * ii + i] = di;
            }
          }
          pf[w] = pack8(p);
          split8(ds, df[w], dl[w]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            dv[db] = mfma32(attn_tr_frag<D>(sm, qtr, db, G0 + w * 32 * D),
                            pf[w], dv[db]);
            const bf16x8 qt = attn_tr_frag<D>(sm, qtr, db, w * 32 * D);
            dk[db] = mfma32(qt, df[w], dk[db]);
            dk[db] = mfma32(qt, dl[w], dk[db]);
          }
      }
    }
    cur = nxt;
    buf ^= 1;
  }

  if constexpr (WIDE) {
    // the second half's sums pass through the query tiles' LDS: 64 KB, dK
    // and then dV of 128 keys
    f32x4* box = (f32x4*)smem + (wk * 64 + lane) * 16;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      f32x16* acc = which ? dv : dk;
      __syncthreads();
      if (wave >= 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          f32x4 y = {acc[i >> 2][(i & 3) * 4], acc[i >> 2][(i & 3) * 4 + 1],
                     acc[i >> 2][(i & 3) * 4 + 2],
                     acc[i >> 2][(i & 3) * 4 + 3]};
          box[(i + lane) & 15] = y;
        }
      }
      __syncthreads();
      if (wave < 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          f32x4 y = box[(i + lane) & 15];
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i >> 2][(i & 3) * 4 + j] += y[j];
        }
      }
    }
    if (wave >= 4) return;
  }

  const long off = ((long)b * a.Tk * a.Hkv + hk) * a.D;
  const long kst = (long)a.Hkv * a.D;
  if (a.nsplit == 1) {
    // the waves that are left may still read the LDS of others: WIDE waves
    // take theirs from K and V, which no one reads any more
    if constexpr (!WIDE) __syncthreads();
    const unsigned box = (WIDE ? K0 : 0) + wave * 64 * D;
    attn_store_rows<DB, false>(sm, box, dk, attn_ds_scale<CAP>(a.scale),
                               a.dk + off, kst, k0, a.Tk, a.D, lane);
    attn_store_rows<DB, false>(sm, box, dv, 1.f, a.dv + off, kst, k0, a.Tk,
                               a.D, lane);
  } else if (kj < a.Tk) {
    const long n = (long)a.B * a.Tk * a.Hkv * a.D;
    float* w = a.ws + (long)split * 2 * n + off + kj * kst;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int ii = 0; ii < 4; ++ii) {
        const int d = db * 32 + 8 * ii + 4 * half;
        if (d >= a.D) continue;
        f32x4 y, z;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = dk[db][ii * 4 + i] * attn_ds_scale<CAP>(a.scale);
          z[i] = dv[db][ii * 4 + i];
        }
        *(f32x4*)(w + d) = y;
        *(f32x4*)(w + n + d) = z;
      }
  }
}

// Adds the parts of a split launch in order: n values of dK, then of dV.
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(
    const float* __restrict__ ws, bf16* __restrict__ dk,
    bf16* __restrict__ dv, long n, int nsplit) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n / 4;
       i += (long)gridDim.x * 256) {
    const long at = i * 8;  // n is a multiple of 8: no group crosses over
    f32x4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
    for (int s = 0; s < nsplit; ++s) {
      const float* p = ws + (long)s * 2 * n + at;
      y += *(const f32x4*)p;
      z += *(const f32x4*)(p + 4);
    }
    float x[8] = {y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]};
    bf16* o = at < n ? dk + at : dv + (at - n);
    *(bf16x8*)o = pack8(x);
  }
}

// Blocks of 128 keys are the unit of work and differ a lot under a causal
// mask.  Few of them leave compute units idle at the end: their queries are
// divided, as long as a part keeps some 16 tiles, those of all heads of a
// group counted: with more than 16 heads to a key head there may be more parts
// than tiles, and those without one add zeros.  Heads of 64, three blocks
// on a compute unit, 8192 tokens of 16 heads over 8 without a cap: 579 us
// with 512 blocks, 395 with 1024, 425 with 1536, the join counted; 2 x 4096
// of 16 over 4: 322, 231, 245.  Heads of 128, one block on a compute unit,
// 2 x 4095: 475, 476 and 507.
int attn_dkv_splits(int B, int Hkv, int G, int Tq, int Tk, int D) {
  const long base = (long)B * Hkv * cdiv_h(Tk, 128);
  const long want = ((D <= 64 ? 1023 : 511) + base) / base;
  const long most = (long)cdiv_h(Tq, 64) * G / 16;
  const long n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

void attn_mod_bwd(const AttnArgs& a, bool need_kv, hipStream_t s) {
  dim3 gq((unsigned)((long)a.B * a.H * cdiv_h(a.Tq, 128)));
  dim3 gk((unsigned)((long)a.B * a.Hkv * cdiv_h(a.Tk, 128) * a.nsplit));
  const bool c = a.cap != 0.f, w = a.slopes != nullptr;
#define GO(D, C, W)                                 \
  do {                                              \
    attn_mod_dq_kernel<D, C, W><<<gq, 256, 0, s>>>(a);  \
    if (need_kv)                                         \
      attn_mod_dkv_kernel<D, C, W><<<gk, (D == 64 ? 256 : 512), 0, s>>>(a); \
  } while (0)
#define PICK(D)                       \
  do {                                \
    if (c && w)                       \
      GO(D, true, true);              \
    else if (c)                       \
      GO(D, true, false);             \
    else if (w)                       \
      GO(D, false, true);             \
    else                              \
      GO(D, false, false);            \
  } while (0)
  if (a.D <= 64)
    PICK(64);
  else
    PICK(128);
#undef PICK
#undef GO
  if (need_kv && a.nsplit > 1) {
    const long n = (long)a.B * a.Tk * a.Hkv * a.D;
    attn_dkv_join_kernel<<<ew_grid(n / 4), 256, 0, s>>>(a.ws, a.dk, a.dv, n,
                                                        a.nsplit);
  }
}

}  // namespace mxa
