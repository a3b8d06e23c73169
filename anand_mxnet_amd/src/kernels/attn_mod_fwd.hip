// Forward pass of attention with shaped scores (see attn_mod.h).
//
// One block: 128 queries of one head, four waves of 32 queries.  Keys and
// values pass through LDS in tiles of 64, double buffered by direct copies;
// tiles that no query of the block can see are never touched.  A wave
// computes S^T = K Q^T (queries along the lanes), so the softmax statistics
// of a query lie in one lane of each half of the wave, and feeds the rounded
// P^T straight into O^T += V^T P^T.
//
// The sum of a row is that of its rounded probabilities, so that rounding
// them leaves the weights of the values at one in all.  In training the part
// of the output that rounding takes is kept too: the backward subtracts
// delta = sum_d dO O from every dP, and with the rounded O alone that error,
// the same for a whole row, is twice all others together.
//
// The running maximum moves only when some row's scores pass it by more
// than 8 (a factor of 256, harmless in fp32 sums and bf16 probabilities), so
// the rescaling of the accumulators is skipped for almost every tile.
//
// Bound by the vector unit, with the matrix unit behind it: per score two
// exp2 and a reciprocal under a cap.  16384 tokens in three documents, 16
// heads of 128 over 8, capped: 623 us, 680 TFLOP/s; vector unit 58, matrix
// unit 34 per cent busy at 2.05 GHz (605 us on a card where a library product
// of 8192^3 reached 1166 TFLOP/s, not 1116; one document, uncapped, ran at 976
// there).  Two groups of four waves that took turns at products and softmax,
// 256 queries a block, were no faster (640 us there; prefixes of 4095 tokens
// 240, not 215).  Sequences of 512 in four documents, 16384 tokens, heads of
// 64: 54 us, where moving the bytes takes 34; a block has four tiles, and its
// first loads and its stores weigh
// as much.
#include <type_traits>

#include "attn_mod.h"

namespace mxa {

// Smallest and largest document id of every 32 rows, 4 ceil(T / 128) entries
// of a sequence; behind its end, an empty range.
__global__ __launch_bounds__(256) void attn_seg_ranges_kernel(
    const int* __restrict__ seg, int2* __restrict__ out, int T, int nr,
    long total) {
  const long w = (long)blockIdx.x * 8 + threadIdx.x / 32;
  if (w >= total) return;
  const long b = w / nr;
  const int t = (int)(w % nr) * 32 + (threadIdx.x & 31);
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
  if (t < T) lo = hi = seg[b * T + t];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o, 32));
    hi = max(hi, __shfl_xor(hi, o, 32));
  }
  if ((threadIdx.x & 31) == 0) out[w] = make_int2(lo, hi);
}

void attn_seg_ranges(const int* seg, int2* out, int B, int T,
                     hipStream_t s) {
  const int nr = 4 * cdiv_h(T, 128);
  const long total = (long)B * nr;
  attn_seg_ranges_kernel<<<(unsigned)((total + 7) / 8), 256, 0, s>>>(
      seg, out, T, nr, total);
}

// SHORT: a wave takes the halves of a tile one by one, skips those that it
// has no pairs in, and holds half as many scores: 116 registers, four blocks
// on a compute unit.
template <int D, bool CAP, bool BIAS, bool SHORT>
__global__ __launch_bounds__(256, SHORT ? 4 : 2) void attn_mod_fwd_kernel(
    AttnArgs a) {
  constexpr int KK = D / 16, DB = D / 32;
  // K and V tiles, two buffers of each; then the tiles' ids
  constexpr int TILE = 128 * D, V0 = 2 * TILE, ID0 = 4 * TILE;
  __shared__ __align__(1024) char smem[ID0 + 512];
  lds_char* const sm = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(size_t)sm;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  int bh, rank;
  attn_block(blockIdx.x, a.B * a.H, bh, rank);
  const int qb = cdiv(a.Tq, 128) - 1 - rank;  // last queries: longest rows
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

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  float mrow = M_INIT, lsum = 0.f;

  const LaneAddr la = attn_lane_addr<D>(lane);
  TileWalk walk;
  walk.start(0, cdiv(kend, 64));
  Tile cur = walk.next(m, blk, wav, rng, lane);
  if (cur.t >= 0) stage(0, cur);
  bf16x8 qf[KK];
  {
    const bf16* qp = a.q + b * a.qsb + (long)qi * a.qst + (long)h * a.D;
    const bool ok = qok && sq >= 0;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[kk] = attn_load_q(qp, kk * 2 + half, a.D, ok, a.scale);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) attn_settle(qf[kk]);
  }
  // NH times 32 keys of a tile, from its half nb0 on
  auto part = [&](auto nh, const Tile& cur, int buf, int nb0) {
    constexpr int NH = decltype(nh)::value, N = 16 * NH;
    const unsigned krow = la.row + buf * TILE + nb0 * 64 * D;
    const unsigned vtr = la.tr + buf * TILE + nb0 * 64 * D;
    const unsigned ids = ID0 + buf * 256 + 16 * half + nb0 * 128;
    f32x16 s[NH];
#pragma unroll
    for (int nb = 0; nb < NH; ++nb) s[nb] = zero16();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int nb = 0; nb < NH; ++nb)
        s[nb] = mfma32(attn_row_frag(sm, krow, kk, nb * 64 * D), qf[kk],
                       s[nb]);
    if (D == 128) {
      // eight reads of K ahead of the products: 16384 tokens, 16 heads
      // of 128 took 631 us with the two to four that the compiler keeps
      // in flight, 617 us like this, no less with twelve
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
    }

    const int j0 = cur.t * 64 + nb0 * 32 + 4 * half;
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = attn_z<CAP>(f, s[i >> 4][i & 15]);
    if (cur.ids || cur.ends) {
#pragma unroll
      for (int nb = 0; nb < NH; ++nb)
        attn_mask_keys(x + 16 * nb, cur.ids, cur.ends, sm, ids + 128 * nb, sq,
                       limit - j0 - 32 * nb, -MXA_INF);
    }
    // with a bias, x[i] + base + (i >> 2) * step becomes the score.  The
    // bias is linear in j where all keys of the tile lie before the wave's
    // queries: one addition for each four keys there.
    float mx = -MXA_INF, base = 0.f, step = 0.f;
    if (BIAS) {
      const float d0 = (float)(pos + m.shift - j0);
      if (cur.t * 64 + 63 <= wav.pmin) {
        base = f.slope * d0;
        step = -8.f * f.slope;
        const float e[4] = {0.f, -f.slope, -2.f * f.slope, -3.f * f.slope};
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(x[i], f.mu, e[i & 3]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          x[i] = fmaf(x[i], f.mu,
                      f.slope * fabsf(d0 - (float)(8 * (i >> 2) + (i & 3))));
      }
#pragma unroll
      for (int g = 0; g < N / 4; ++g)
        mx = fmaxf(mx, fmaf((float)g, step,
                            fmaxf(fmaxf(x[4 * g], x[4 * g + 1]),
                                  fmaxf(x[4 * g + 2], x[4 * g + 3]))));
      mx += base;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) mx = fmaxf(mx, x[i]);
      mx *= f.mu;
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__ballot(mx > mrow + 8.f)) {
      float mnew = fmaxf(mrow, mx);
      float al = fexp2(mrow - mnew);
      mrow = mnew;
      lsum *= al;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= al;
    }
    bf16x8 pf[2 * NH];
#pragma unroll
    for (int st = 0; st < 2 * NH; ++st) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int g = 2 * st + (i >> 2);
        p[i] = BIAS ? fexp2(x[8 * st + i] - (mrow - base - (float)g * step))
                    : fexp2(fmaf(x[8 * st + i], f.mu, -mrow));
      }
      pf[st] = pack8(p);
      lsum = dot8(pf[st], ones8(), lsum);
    }
#pragma unroll
    for (int st = 0; st < 2 * NH; ++st)
#pragma unroll
      for (int db = 0; db < DB; ++db)
        o[db] = mfma32(attn_tr_frag<D>(sm, vtr, db, V0 + st * 32 * D),
                       pf[st], o[db]);
  };
  int buf = 0;
  while (cur.t >= 0) {
    attn_wait_copies<0>();
    __syncthreads();  // this tile has landed, the other buffer is free
    Tile nxt = walk.next(m, blk, wav, rng, lane);
    if (nxt.t >= 0) stage(buf ^ 1, nxt);
    if constexpr (SHORT) {
#pragma unroll 1
      for (int nb = 0; nb < 2; ++nb)
        if (cur.work >> nb & 1)
          part(std::integral_constant<int, 1>(), cur, buf, nb);
    } else if (cur.work) {
      part(std::integral_constant<int, 2>(), cur, buf, 0);
    }
    cur = nxt;
    buf ^= 1;
  }

  lsum += __shfl_xor(lsum, 32, 64);
  // a sum of zero: nothing seen, the row is zero; a NaN stays one
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  __syncthreads();  // the tiles' LDS is free
  const unsigned box = wave * 64 * D;
  attn_store_rows<DB, false>(sm, box, o, inv,
                             a.o + b * a.osb + (long)h * a.D, a.ost, q0,
                             a.Tq, a.D, lane);
  if (a.olo)
    attn_store_rows<DB, true>(sm, box, o, inv,
                              a.olo + ((long)b * a.Tq * a.H + h) * a.D,
                              (long)a.H * a.D, q0, a.Tq, a.D, lane);
  if (a.lse && half == 0 && qi < a.TqP)
    a.lse[((long)b * a.H + h) * a.TqP + qi] =
        qok && lsum != 0.f ? mrow + __log2f(lsum) : MXA_INF;
}

void attn_mod_fwd(const AttnArgs& a, hipStream_t s) {
  dim3 g((unsigned)((long)a.B * a.H * cdiv_h(a.Tq, 128)));
  const bool c = a.cap != 0.f, w = a.slopes != nullptr;
#define GO(D, C, W, S) attn_mod_fwd_kernel<D, C, W, S><<<g, 256, 0, s>>>(a)
#define PICK(D, S)                    \
  do {                                \
    if (c && w)                       \
      GO(D, true, true, S);           \
    else if (c)                       \
      GO(D, true, false, S);          \
    else if (w)                       \
      GO(D, false, true, S);          \
    else                              \
      GO(D, false, false, S);         \
  } while (0)
  // 16384 tokens, 16 heads of 64, in us, whole tiles and halves: sequences
  // of 256 36.3 and 33.0, of 1024 65 and 63, of 2048 119 and 120, of 8192
  // 186 and 210; capped 41.2 and 38.2, 91 and 88, 154 and 150, 282 and 289;
  // capped, sequences of 512 in four documents 57.8 and 53.2.  Heads of 128
  // have no room for a third block either way.
  if (a.D > 64)
    PICK(128, false);
  else if (a.Tk <= 2048)
    PICK(64, true);
  else
    PICK(64, false);
#undef PICK
#undef GO
}

}  // namespace mxa
