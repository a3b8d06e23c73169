// Attention with shaped scores for a few queries over a long cache (see
// attn_mod.h): the form that answers token by token.
//
// Bound by reading K and V once: 64 sequences of up to 8192 keys, 16 heads of
// 128 over 4, 102 us for 522 MB, 5.1 TB/s; 4 of up to 131071, three queries
// each, 336 us for 1.95 GB, 5.8 TB/s (a copy moves 4.9, a sum reads 3.7).
// The queries of all heads that share a key head form the 32 columns of one
// product (row r = token r / G, head r % G), so a shared cache is read once
// for its whole group.  The keys of a sequence are divided among `nsplit` blocks and, tile by tile of 32, among
// the four waves of a block; a wave streams its tiles through LDS of its own
// with counted waits and no barriers: the next K is on its way while this
// tile's V is used, and the other way round.  Partial softmaxes are joined in
// LDS, then (nsplit > 1) by a second kernel, in a fixed order.
#include "attn_mod.h"

namespace mxa {

constexpr int DEC_ROWS = 32;

template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void attn_decode_kernel(
    AttnArgs a) {
  constexpr int KK = D / 16, DB = D / 32;
  constexpr int NCOPY = 32 * D / 512;  // copies of one tile
  // per wave: a K and a V tile; later the partial outputs
  constexpr int TILE = 64 * D;
  __shared__ __align__(1024) char smem[8 * TILE + 1024];
  lds_char* const sm = (lds_char*)smem;
  const unsigned lds0 = (unsigned)(size_t)sm;
  float(*smax)[32] = (float(*)[32])(smem + 8 * TILE);
  float(*ssum)[32] = smax + 4;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int R = a.Tq * a.G;
  const int nrt = cdiv(R, DEC_ROWS);
  const int sp = blockIdx.x % a.nsplit;
  const int rt = blockIdx.x / a.nsplit % nrt;
  const int bh = blockIdx.x / a.nsplit / nrt;
  const int hk = bh % a.Hkv, b = bh / a.Hkv;
  const SeqMask m = attn_seq_mask(a, b);

  const int r = rt * DEC_ROWS + col;
  const bool ok = r < R;
  const int tok = r / a.G, h = hk * a.G + r % a.G;
  const int pos = tok + m.off;
  const int limit = ok ? attn_limit(m, pos) : 0;
  const int pmin = rt * DEC_ROWS / a.G + m.off;
  const int pmax = (min(rt * DEC_ROWS + DEC_ROWS, R) - 1) / a.G + m.off;
  const int full_end = attn_limit(m, pmin);  // all rows see keys below

  ScoreFn f;
  f.set<CAP>(a.scale, a.cap, BIAS && ok ? a.slopes[h] : 0.f);
  // this block's tiles: an equal share of what the sequence has
  const int kend = max(attn_limit(m, pmax), 0);  // nobody sees the rest
  const int nt = cdiv(kend, 32);
  const int share = cdiv(nt, a.nsplit);
  const int t1 = min(nt, (sp + 1) * share);
  int t = sp * share + wave;

  const bf16* kb = a.k + b * a.ksb + (long)hk * a.D;
  const bf16* vb = a.v + b * a.vsb + (long)hk * a.D;
  Stager<D, 32, 1> ks, vs;
  ks.init(a.kst, 0, lane);
  vs.init(a.vst, 0, lane);
  const unsigned kat = wave * 2 * TILE, vat = kat + TILE;
  // the wave's own reads of a tile end before the next one is copied over it
  auto stage_k = [&](int tile) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    ks.copy(kb, a.kst, tile * 32, kend, a.D, (const int*)nullptr, lds0 + kat,
            0, lane);
  };
  auto stage_v = [&](int tile) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    vs.copy(vb, a.vst, tile * 32, kend, a.D, (const int*)nullptr, lds0 + vat,
            0, lane);
  };

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  float mrow = M_INIT, lsum = 0.f;

  const LaneAddr la = attn_lane_addr<D>(lane);
  const unsigned krow = la.row + kat, vtr = la.tr + vat;
  if (t < t1) {
    stage_k(t);
    stage_v(t);
  }
  // the queries come while the first tiles are on their way
  bf16x8 qf[KK];
  {
    const bf16* qp = a.q + b * a.qsb + (long)tok * a.qst + (long)h * a.D;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[kk] = attn_load_q(qp, kk * 2 + half, a.D, ok, a.scale);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) attn_settle(qf[kk]);
    asm volatile("" : "+v"(f.slope));
  }
  for (; t < t1; t += 4) {
    const bool more = t + 4 < t1;
    attn_wait_copies<NCOPY>();  // K is there, V may be on its way
    f32x16 s = zero16();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      s = mfma32(attn_row_frag(sm, krow, kk, 0), qf[kk], s);
    if (more) stage_k(t + 4);
    const int j0 = t * 32 + 4 * half;
    const float d0 = BIAS ? (float)(pos + m.shift - j0) : 0.f;
    float x[16], mx = -MXA_INF;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = attn_z<CAP>(f, s[i]);
    if (t * 32 + 32 > full_end)
      attn_mask_keys(x, false, true, sm, 0, 0, limit - j0, -MXA_INF);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int dj = 8 * (i >> 2) + (i & 3);
      x[i] *= f.mu;
      if (BIAS) x[i] = fmaf(f.slope, fabsf(d0 - (float)dj), x[i]);
      mx = fmaxf(mx, x[i]);
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
    bf16x8 pf[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = fexp2(x[8 * w + i] - mrow);
      }
      pf[w] = pack8(p);
      lsum = dot8(pf[w], ones8(), lsum);
    }
    if (more)
      attn_wait_copies<NCOPY>();
    else
      attn_wait_copies<0>();
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int db = 0; db < DB; ++db)
        o[db] = mfma32(attn_tr_frag<D>(sm, vtr, db, w * 32 * D), pf[w],
                       o[db]);
    if (more) stage_v(t + 4);
  }
  lsum += __shfl_xor(lsum, 32, 64);

  // ---- join the four waves ----
  // partial outputs [32][D] fp32 lie over the wave's own tiles, whose reads
  // are done; float4 slots are rotated by the row against conflicts
  float* po = (float*)(smem + kat);
  __syncthreads();
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      const int slot = (db * 8 + 2 * ii + half + col) & (D / 4 - 1);
      f32x4 y = {o[db][ii * 4], o[db][ii * 4 + 1], o[db][ii * 4 + 2],
                 o[db][ii * 4 + 3]};
      *(f32x4*)&po[col * D + slot * 4] = y;
    }
  if (half == 0) {
    smax[wave][col] = mrow;
    ssum[wave][col] = lsum;
  }
  __syncthreads();
  const int nrow = min(DEC_ROWS, R - rt * DEC_ROWS);
  for (int i = threadIdx.x; i < nrow * (D / 4); i += 256) {
    const int row = i / (D / 4), d4 = i % (D / 4);
    const int slot = (d4 + row) & (D / 4 - 1);
    float mm = M_INIT;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, smax[w][row]);
    float l = 0.f;
    f32x4 y = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = fexp2(smax[w][row] - mm);
      l += ssum[w][row] * e;
      y += *(const f32x4*)((const float*)(smem + w * 2 * TILE) + row * D + slot * 4) * e;
    }
    const int rr = rt * DEC_ROWS + row;
    if (d4 * 4 >= a.D) continue;
    if (a.nsplit == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bf16* op = a.o + b * a.osb + (long)(rr / a.G) * a.ost +
                 (long)(hk * a.G + rr % a.G) * a.D + d4 * 4;
      bf16x4 z;
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] = (bf16)(y[k] * inv);
      *(bf16x4*)op = z;
    } else {
      const long idx = ((long)bh * a.nsplit + sp) * R + rr;
      *(f32x4*)&a.ws[idx * a.D + d4 * 4] = y;
      if (d4 == 0) {
        float* wm = a.ws + (long)a.B * a.Hkv * a.nsplit * R * a.D;
        wm[idx * 2] = mm;
        wm[idx * 2 + 1] = l;
      }
    }
  }
}

// Joins the blocks of one row: a wave per row.  Lane s holds the weight of
// split s (64 at a time); the two halves of the wave add the even and the odd
// splits, four columns a lane.
__global__ __launch_bounds__(256) void attn_decode_join_kernel(AttnArgs a) {
  const int R = a.Tq * a.G;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long)a.B * a.Hkv * R) return;
  const int rr = (int)(row % R);
  const long bh = row / R;
  const int hk = (int)(bh % a.Hkv);
  const long b = bh / a.Hkv;
  const float* wm = a.ws + (long)a.B * a.Hkv * a.nsplit * R * a.D;
  const long i0 = bh * a.nsplit * R + rr;

  float mm = M_INIT;
  for (int s = lane; s < a.nsplit; s += 64)
    mm = fmaxf(mm, wm[(i0 + (long)s * R) * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
  float l = 0.f;
  f32x4 y = {0, 0, 0, 0};
  const int d = min((lane & 31) * 4, a.D - 4);  // D < 128: lanes repeat
  for (int s0 = 0; s0 < a.nsplit; s0 += 64) {
    const int n = min(64, a.nsplit - s0);
    float e = 0.f;
    if (lane < n) {
      const long i = (i0 + (long)(s0 + lane) * R) * 2;
      e = fexp2(wm[i] - mm);
      l += wm[i + 1] * e;
    }
    // eight loads in flight: the parts come from other XCDs' writes
    for (int s = 0; s < n; s += 16) {
      f32x4 x[8];
      float w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int k = min(s + 2 * u + half, n - 1);
        x[u] = *(const f32x4*)&a.ws[(i0 + (long)(s0 + k) * R) * a.D + d];
        w[u] = __shfl(e, k, 64);
        if (s + 2 * u + half >= n) w[u] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) y += x[u] * w[u];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] += __shfl_xor(y[k], 32, 64);
  if (half == 0) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16* op = a.o + b * a.osb + (long)(rr / a.G) * a.ost +
               (long)(hk * a.G + rr % a.G) * a.D + d;
    bf16x4 z;
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = (bf16)(y[k] * inv);
    *(bf16x4*)op = z;
  }
}

// Blocks a sequence's keys are divided among: enough to fill the chip twice
// over, but no more than one for each 256 keys that the cache has room for:
// eight tiles, two a wave, of a full one; the tiles that a shorter sequence
// has are shared out evenly, and some blocks may get fewer or none.
int attn_decode_splits(int B, int Hkv, int R, int Tk) {
  long base = (long)B * Hkv * cdiv_h(R, DEC_ROWS);
  long want = (1536 + base - 1) / base;
  long most = (Tk + 255) / 256;
  long n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

// Workspace of a split launch, in floats: outputs [B Hkv][nsplit][R][D], then
// a maximum and a sum for each row of them.
long attn_decode_ws(int B, int Hkv, int R, int D, int nsplit) {
  return nsplit == 1 ? 0 : (long)B * Hkv * nsplit * R * (D + 2);
}

void attn_decode(const AttnArgs& a, hipStream_t s) {
  const int R = a.Tq * a.G;
  dim3 g((unsigned)((long)a.B * a.Hkv * cdiv_h(R, DEC_ROWS) * a.nsplit));
  const bool c = a.cap != 0.f, w = a.slopes != nullptr;
#define GO(D, C, W) attn_decode_kernel<D, C, W><<<g, 256, 0, s>>>(a)
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
  if (a.nsplit > 1) {
    long rows = (long)a.B * a.Hkv * R;
    attn_decode_join_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(a);
  }
}

}  // namespace mxa
