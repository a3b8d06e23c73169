// Attention with shaped scores: what the forward, backward and few-token
// kernels share (attn_mod_fwd.hip, attn_mod_bwd.hip, attn_mod_decode.hip).
//
// For a query i at position P = query_offset + i and a key j of one sequence
//   s = scale * q.k
//   s = cap * tanh(s / cap)              (CAP)
//   s = s - slope_h * |P - j|            (BIAS)
// and j is visible to i when all of these hold
//   j < kv_length
//   j <= P or j < prefix_length          (causal)
//   seg_q[i] == seg_k[j] >= 0            (documents)
// A query that sees nothing gives a zero row and zero gradients.
//
// Scores are held in units of log2, x = mu * z + bias, so that the softmax
// needs exp2 alone and one multiply-add in front of it.  Without a cap z is
// the product q.k itself.  tanh(y) = 1 - 2 / (1 + exp(2 y)), and a softmax
// does not see a constant: with a cap z = -1 / (1 + exp(2 y)), mu = 2 cap
// log2 e.  That is one exp2 and one reciprocal, and saturates by itself:
// exp2 -> inf gives 0, exp2 -> 0 gives -1.  1 - tanh^2 = -4 (z^2 + z).  z errs
// by 2e-7 at most (exp2 and reciprocal by a unit in the last place each), so a
// score by mu times that and a probability by cap times 4e-7 of it: 2e-5 at a
// cap of 50, 4e-4 at the largest, a tenth of what rounding it to bf16 takes.
//
// Matrix operands (v_mfma_f32_32x32x16_bf16, wave of 64 lanes, l = lane):
//   A row  l & 31,  k = 8 (l >> 5) + 0..7
//   B col  l & 31,  k = 8 (l >> 5) + 0..7
//   C col  l & 31,  row 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0..15
// Products are arranged so that the softmaxed axis lies along the rows of C:
// then C of the first product, rounded to bf16, IS the B operand of the next
// one (eight consecutive i are the k of one step, in the order 0-3, 8-11 for
// the lower and 4-7, 12-15 for the upper half of the wave), and the A operand
// is fetched in the same order by transposing LDS reads of four rows each.
// Probabilities never leave the registers.
#pragma once
#include <hip/hip_runtime.h>

#include "common.h"

namespace mxa {

struct AttnArgs {
  const bf16 *q, *k, *v;
  bf16* o;
  bf16* olo;   // what rounding took from o, [B, Tq, H, D]; may be null
  float* lse;  // [B, H, TqP] log2 of the softmax sum; +inf: row sees nothing
  const bf16* dout;
  float* delta;  // [B, H, TqP] minus sum_d dout * out
  int* blind;    // [B, H, TqP / 32] whether some of 32 queries see nothing
  bf16 *dq, *dk, *dv;
  float* ws;     // partial results of a split launch
  long qsb, ksb, vsb, osb, gsb;  // batch strides, elements
  long qst, kst, vst, ost, gst;  // row strides, elements (g: dout)
  int B, H, Hkv, G, D, Tq, Tk, TqP;
  float scale, cap;
  int causal;
  const int *seg_q, *seg_k, *prefix, *kv_len, *q_off;
  const float* slopes;
  int off0;  // added to every query_offset
  // smallest and largest id of each 32 rows, 4 ceil(T / 128) of a sequence
  const int2 *rng_q, *rng_k;
  int nsplit;
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_INIT = -1.0e30f;  // running maximum before any score
#define MXA_INF __builtin_inff()

// Sixteen zero bytes that staging lanes read where a row or a chunk is out
// of range: V rows behind a sequence must be zero (0 * NaN is NaN).
static __device__ const uint4 attn_zero16[1] = {{0, 0, 0, 0}};

DEVINL float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }
DEVINL float frcp(float x) { return __builtin_amdgcn_rcpf(x); }

// LDS image of [rows][D] bf16, D = 64 or 128, in chunks of 16 bytes; chunk c
// of row r lies in slot c ^ attn_key(r).  The key is a bijection of 16 rows
// (row fragments: 16 lanes, one chunk) and gives four aligned rows times
// four aligned chunks 16 different slots (transposing reads), so both kinds
// of read are free of bank conflicts.
template <int D>
DEVINL int attn_key(int r) {
  return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3))
                  : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// The fragments of an image differ from lane to lane in a fixed way, and
// from step to step in address bits that a lane's own address only meets by
// exclusive or; whole rows are added.  A lane keeps these two addresses:
//   row  its chunk of row (l & 31), for step 0
//   tr   its place in the first transposing read of row 0, column 0
struct LaneAddr {
  unsigned row, tr;
};

template <int D>
DEVINL LaneAddr attn_lane_addr(int lane) {
  const int half = lane >> 5, col = lane & 31, a = (lane & 15) >> 2;
  const int c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  const int hi = D == 128 ? a : a >> 1;
  LaneAddr x;
  x.row = col * (2 * D) + ((half ^ attn_key<D>(col)) << 4);
  x.tr = (4 * half + a) * (2 * D) + (((hi << 2) | (c ^ half)) << 4) +
         (lane & 1) * 8;
  return x;
}

typedef __attribute__((address_space(3))) char lds_char;

// A or B operand: rows 0..31 of the image at `row` (bytes, with the lane's
// own part in it), columns 16 kk on.  `at`: a constant offset.
DEVINL bf16x8 attn_row_frag(lds_char* sm, unsigned row, int kk, int at) {
  typedef __attribute__((address_space(3))) const bf16x8 lds8;
  return *(lds8*)(sm + ((row ^ (kk << 5)) + at));
}

// A operand of the transposed image: its rows are columns 32 db..32 db + 31
// of the image, k runs over image rows {0-3, 8-11} (lower half of the wave)
// or {4-7, 12-15}; `at` adds whole rows.
template <int D>
DEVINL bf16x8 attn_tr_frag(lds_char* sm, unsigned tr, int db, int at) {
  typedef __attribute__((address_space(3))) bf16x4 lds4;
  bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      (lds4*)(sm + ((tr ^ (db << 6)) + at)));
  bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      (lds4*)(sm + ((tr ^ (db << 6) ^ 32) + at + 16 * D)));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename T>
DEVINL T attn_lds(lds_char* sm, unsigned at) {
  return *(__attribute__((address_space(3))) const T*)(sm + at);
}

// A direct copy into LDS: 16 bytes (or 4) a lane, from the lane's address to
// dst + 16 (4) * lane.  Written as assembly because the compiler waits for
// every copy in flight before any LDS read that follows a builtin one, which
// would undo the double buffering; it names no register that a load fills.
// M0 is read one state after it is written, and declared, so that a value that
// the compiler puts there itself is not taken as still in place.
// Whoever reads the tile waits with attn_wait_copies and a barrier.
DEVINL void copy_lds16(const void* g, unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
      :
      : "v"(g), "s"(__builtin_amdgcn_readfirstlane(dst))
      : "memory", "m0");
}
// Two or four of them, from base + off[p] to places 1024 bytes apart.  The
// compiler does not see that a load reads the pair that holds base: five
// states after a vector instruction wrote it (a move of a spilled pair may do
// so right before) are waited for here, once for all.
DEVINL void copy_lds16x2(const void* base, const unsigned* off,
                         unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 3\n\t"
      "global_load_lds_dwordx4 %2, %0\n\t"
      "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %0"
      :
      : "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off[0]),
        "v"(off[1])
      : "memory", "m0", "scc");
}
DEVINL void copy_lds16x4(const void* base, const unsigned* off,
                         unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 3\n\t"
      "global_load_lds_dwordx4 %2, %0\n\t"
      "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %0\n\t"
      "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %0\n\t"
      "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %5, %0"
      :
      : "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off[0]),
        "v"(off[1]), "v"(off[2]), "v"(off[3])
      : "memory", "m0", "scc");
}
DEVINL void copy_lds4(const void* g, unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
      :
      : "v"(g), "s"(__builtin_amdgcn_readfirstlane(dst))
      : "memory", "m0");
}
// All but the last N copies have landed.
template <int N>
DEVINL void attn_wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// Makes the compiler wait for x here, and not inside a later loop, where the
// wait would catch the copies in flight too.
DEVINL void attn_settle(bf16x8& x) { asm volatile("" : "+v"(x)); }

// Keeps what is computed from x inside a loop, where it costs one
// instruction, rather than in registers around it.
DEVINL unsigned attn_here(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The kernel's arguments, read where this stands: what is needed now and then
// takes no registers all the way from the kernel's start.  For kernels whose
// only argument they are.
typedef __attribute__((address_space(4))) const AttnArgs ConstArgs;
DEVINL ConstArgs* attn_args_here() {
  ConstArgs* a = (ConstArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

// A pointer that is the same in all lanes, where the compiler knows it.
DEVINL const bf16* uniform_ptr(const bf16* p) {
  const size_t x = (size_t)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(x >> 32));
  return (const bf16*)((size_t)hi << 32 | lo);
}

// Whether a row counts: its id is not negative, or its query sees something.
DEVINL bool attn_open(int id) { return id >= 0; }
DEVINL bool attn_open(float lse) { return lse != MXA_INF; }

// Copies NROW consecutive rows of a head into an image, by NW waves, each
// lane 16 bytes of N instructions.  off holds where its chunks lie behind
// the first row, so a copy costs no vector arithmetic; rows are less than
// 2**25 elements apart.
template <int D, int NROW, int NW>
struct Stager {
  static constexpr int RPI = 512 / D;  // rows of one instruction
  static constexpr int CPR = D / 8;    // chunks of a row
  static constexpr int N = NROW / RPI / NW;
  static_assert(N * RPI * NW == NROW, "rows divide among the waves");
  unsigned off[N];

  DEVINL void init(long stride, int wave, int lane) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const int r = (wave * N + p) * RPI + lane / CPR;
      const int ch = (lane % CPR) ^ attn_key<D>(r);
      off[p] = (unsigned)r * (unsigned)stride * 2u + ch * 16;
    }
  }
  // Rows row0 on; img is the image's LDS address.  Rows at or behind
  // row_end, rows that gate (it may be null) shuts out and chunks at or behind
  // Dact read as zero.
  template <typename G>
  DEVINL void copy(const bf16* base, long stride, int row0, int row_end,
                   int Dact, const G* gate, unsigned img, int wave,
                   int lane) const {
    const unsigned dst = img + wave * (N * 1024);
    const bf16* g0 = uniform_ptr(base + (long)row0 * stride);
    if (row0 + NROW <= row_end && Dact == D && gate == nullptr) {
      static_assert(N == 2 || N % 4 == 0, "copies of a wave");
      if constexpr (N == 2) {
        copy_lds16x2(g0, off, dst);
      } else {
#pragma unroll
        for (int p = 0; p < N; p += 4)
          copy_lds16x4(g0, off + p, dst + p * 1024);
      }
    } else {
#pragma unroll 1  // rare: small code counts for more
      for (int p = 0; p < N; ++p) {
        const int r = (wave * N + p) * RPI + lane / CPR;
        const int ch = (lane % CPR) ^ attn_key<D>(r);
        const bf16* g = g0 + (long)r * stride + ch * 8;
        bool ok = row0 + r < row_end && ch * 8 < Dact;
        if (ok && gate) ok = attn_open(gate[row0 + r]);
        if (!ok) g = (const bf16*)attn_zero16;
        copy_lds16(g, dst + p * 1024);
      }
    }
  }
};

// 64 words into LDS, one instruction of one wave; index clamped to [0, n).
DEVINL void attn_stage64(const void* base, int first, int n, unsigned dst,
                         int lane) {
  int j = min(first + lane, n - 1);
  copy_lds4((const unsigned int*)base + j, dst);
}

DEVINL bf16x8 attn_load_row(const bf16* p, int chunk, int Dact, bool ok) {
  bf16x8 z = {};
  return ok && chunk * 8 < Dact ? *(const bf16x8*)(p + chunk * 8) : z;
}

// Which (batch, head) and which block of its rows a launch id stands for,
// nb blocks to each of n heads; rank 0 is the block with the most work.
// Blocks with the most work of all heads come first, so that the launch ends
// evenly; where the heads divide among the 8 XCDs (ids go round them), an
// XCD keeps its heads, whose other side then stays in its L2.
DEVINL void attn_block(int id, int n, int& head, int& rank) {
  if (n % 8 == 0) {
    const int per = n / 8, li = id / 8;
    head = (id % 8) * per + li % per;
    rank = li / per;
  } else {
    head = id % n;
    rank = id / n;
  }
}

// Positions and document ids that a group of queries spans.
struct RowSpan {
  int pmin, pmax, smin, smax;
};

// One sequence's masks, uniform over a block.
struct SeqMask {
  int kv_len, prefix, off, causal, has_seg;
  // what positions are moved by for the distance bias: where all queries lie
  // behind all keys, or before them, the distances shrink by one number, which
  // a softmax does not see and 32 bits would lose weights to
  int shift;
};

DEVINL SeqMask attn_seq_mask(const AttnArgs& a, int b) {
  SeqMask m;
  m.kv_len = a.kv_len ? min(max(a.kv_len[b], 0), a.Tk) : a.Tk;
  m.prefix = a.prefix ? a.prefix[b] : 0;
  // positions and the ones behind them stay within 32 bits; Tq and Tk are
  // below 2**30, so an offset cut to that sees the same keys
  const long far = (1l << 30) - 1;
  const long off = (long)a.off0 + (a.q_off ? a.q_off[b] : 0);
  m.off = (int)min(max(off, -far), far);
  m.shift = max(min(m.off, max(m.kv_len - 1, 0)), 1 - a.Tq) - m.off;
  m.causal = a.causal;
  m.has_seg = a.seg_q != nullptr;
  return m;
}

// First key that a query at position p cannot see (documents aside).
DEVINL int attn_limit(const SeqMask& m, int p) {
  return m.causal ? min(m.kv_len, max(p + 1, m.prefix)) : m.kv_len;
}

// May any query of s see any key of the 64 from j0 on?
DEVINL bool attn_tile_any(const SeqMask& m, const RowSpan& s, int j0,
                          int2 r) {
  bool ok = j0 < attn_limit(m, s.pmax);
  if (m.has_seg) ok = ok && max(max(s.smin, r.x), 0) <= min(s.smax, r.y);
  return ok;
}

// Do all queries of s and all of these keys have one id?
DEVINL bool attn_tile_one(const SeqMask& m, const RowSpan& s, int2 r) {
  return !m.has_seg || (s.smin >= 0 && s.smin == s.smax && r.x == s.smin &&
                        r.y == s.smin);
}

DEVINL int2 attn_join(int2 x, int2 y) {
  return make_int2(min(x.x, y.x), max(x.y, y.y));
}

struct Tile {
  int t;      // index of 64 keys; negative: no more
  int work;   // the halves of it in which this wave has pairs, as two bits
  bool ids;   // its queries' and keys' ids are not all the same
  bool ends;  // some queries' last visible key lies in it
  bool neg;   // some ids are negative: stage with care
};

// Walks the key tiles a block has work in: 64 tiles are judged at once, a
// tile to a lane, and the verdicts are kept as bits.
struct TileWalk {
  int base, nt;
  u64 act, wact[2], wone, wend, neg;

  DEVINL void start(int first, int ntiles) {
    base = first - 64;
    nt = ntiles;
    act = wact[0] = wact[1] = wone = wend = neg = 0;
  }
  DEVINL Tile next(const SeqMask& m, const RowSpan& blk, const RowSpan& wav,
                   const int2* rng, int lane) {
    while (act == 0) {
      base += 64;
      if (base >= nt) return Tile{-1, 0, false, false, false};
      int t = base + lane;
      int2 r0 = make_int2(0, 0), r1 = r0;
      bool in = t < nt;
      if (in && m.has_seg) {
        r0 = rng[2 * t];
        r1 = rng[2 * t + 1];
      }
      const int2 r = attn_join(r0, r1);
      act = __ballot(in && attn_tile_any(m, blk, t * 64, r));
      const bool some = in && wav.pmax != -0x7fffffff;
      wact[0] = __ballot(some && attn_tile_any(m, wav, t * 64, r0));
      wact[1] = __ballot(some && attn_tile_any(m, wav, t * 64 + 32, r1));
      wone = __ballot(in && attn_tile_one(m, wav, r));
      wend = __ballot(in && t * 64 + 64 > attn_limit(m, wav.pmin));
      neg = __ballot(in && m.has_seg && r.x < 0);
    }
    int i = __builtin_ctzll(act);
    act &= act - 1;
    return Tile{base + i,
                (int)((wact[0] >> i) & 1) | (int)((wact[1] >> i) & 1) << 1,
                !((wone >> i) & 1),
                (bool)((wend >> i) & 1), (bool)((neg >> i) & 1)};
  }
};

// The ranges of ids of one side of sequence b.
DEVINL const int2* attn_ranges(const int2* rng, long b, int T) {
  return rng + b * (4 * cdiv(T, 128));
}

// The spans of a wave's 32 queries and of its block qb of 128.
DEVINL void attn_spans(const AttnArgs& a, const SeqMask& m, int b, int qb,
                       int wave, RowSpan& wav, RowSpan& blk) {
  const int q0 = qb * 128 + wave * 32;
  blk = {qb * 128 + m.off, min(qb * 128 + 127, a.Tq - 1) + m.off, 0, 0};
  wav = {q0 + m.off, min(q0 + 31, a.Tq - 1) + m.off, 0, 0};
  if (m.has_seg) {
    const int2* r = attn_ranges(a.rng_q, b, a.Tq) + qb * 4;
    const int2 w = r[wave];
    const int2 j = attn_join(attn_join(r[0], r[1]), attn_join(r[2], r[3]));
    wav.smin = __builtin_amdgcn_readfirstlane(w.x);
    wav.smax = __builtin_amdgcn_readfirstlane(w.y);
    blk.smin = __builtin_amdgcn_readfirstlane(j.x);
    blk.smax = __builtin_amdgcn_readfirstlane(j.y);
  }
  // a wave without rows sees no tile
  if (q0 >= a.Tq) wav.pmin = wav.pmax = -0x7fffffff;
}

// Masks 16 scores of one query (C order): ids at LDS address ksg, the first
// `lim` keys are seen.  A masked score becomes `gone`.
DEVINL void attn_mask_keys(float* x, bool ids, bool ends, lds_char* sm,
                           unsigned ksg, int sq, int lim, float gone) {
  if (ids) {
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      const i32x4 k4 = attn_lds<i32x4>(sm, ksg + 32 * ii);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[ii * 4 + i] = k4[i] == sq ? x[ii * 4 + i] : gone;
    }
  }
  if (ends) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      x[i] = 8 * (i >> 2) + (i & 3) < lim ? x[i] : gone;
  }
}

// Constants of the score function.  The sign of the scale goes to the
// queries (attn_load_q): c1 and mu are positive, and z of a masked pair is
// minus infinity.  A cap between 1e-3 and 1e3 keeps the error of mu z below
// 1e-3 and mu times attn_gone beyond any exponent.
struct ScoreFn {
  float c1, mu, slope;
  template <bool CAP>
  DEVINL void set(float scale, float cap, float slope_) {
    const float sc = scale == 0.f ? 1.f : fabsf(scale);
    c1 = CAP ? sc / cap * 2.f * LOG2E : 1.f;
    mu = CAP ? 2.f * cap * LOG2E : sc * LOG2E;
    slope = -slope_ * LOG2E;
  }
};

template <bool CAP>
DEVINL float attn_z(const ScoreFn& f, float s) {
  return CAP ? frcp(-1.f - fexp2(s * f.c1)) : s;
}

// (1 - tanh^2) / -4
DEVINL float attn_dtanh(float z) { return fmaf(z, z, z); }

// A masked z in the backward: its probability is zero like that of minus
// infinity, and attn_dtanh of it is finite.
template <bool CAP>
DEVINL float attn_gone() {
  return CAP ? -1.0e18f : -MXA_INF;
}

// What dS is to be multiplied with at the end: the scale, and -4 of the
// derivative of tanh.
template <bool CAP>
DEVINL float attn_ds_scale(float scale) {
  return CAP ? -4.f * scale : scale;
}

// Query fragments times the sign of the scale (exact).
DEVINL bf16x8 attn_load_q(const bf16* p, int chunk, int Dact, bool ok,
                          float scale) {
  bf16x8 x = attn_load_row(p, chunk, Dact, ok && scale != 0.f);
  if (scale < 0.f) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 y = __builtin_bit_cast(u32x4, x) ^ 0x80008000u;
    x = __builtin_bit_cast(bf16x8, y);
  }
  return x;
}

DEVINL bf16x8 pack8(const float* x) {
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (bf16)x[i];
  return y;
}

// x as a bf16 and the bf16 of what that rounding takes: 16 bits of it.
DEVINL void split8(const float* x, bf16x8& hi, bf16x8& lo) {
  hi = pack8(x);
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i] - (float)hi[i];
  lo = pack8(r);
}

// acc + sum of a[i] * b[i], in 32 bits
DEVINL float dot8(bf16x8 a, bf16x8 b, float acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[2 * i], a[2 * i + 1]},
                                          bf16x2{b[2 * i], b[2 * i + 1]}, acc,
                                          false);
  return acc;
}

DEVINL bf16x8 ones8() {
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (bf16)1.f;
  return y;
}

DEVINL f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

DEVINL f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Writes a wave's transposed accumulator (32 rows from row0 on, those below
// row_end) as rows of bf16.  They pass through 64 D bytes of LDS of the
// wave's own at `box`: a lane has four columns of a row at a time, and with
// stores of 8 bytes to 32 rows 128 short sequences took 64 us forward, not
// 60.
// REST writes what the rounding takes instead.
template <int DB, bool REST>
DEVINL void attn_store_rows(lds_char* sm, unsigned box, const f32x16* acc,
                            float mul, bf16* base, long stride, int row0,
                            int row_end, int Dact, int lane) {
  constexpr int D = 32 * DB, CPR = D / 8, RPI = 64 / CPR;
  typedef __attribute__((address_space(3))) bf16x4 lds4;
  const int half = lane >> 5, col = lane & 31;
  const unsigned at = box + col * (2 * D) + half * 8;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      bf16x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = acc[db][ii * 4 + i] * mul;
        y[i] = (bf16)x;
        if (REST) y[i] = (bf16)(x - (float)y[i]);
      }
      *(lds4*)(sm + (at + (((db * 4 + ii) ^ (col & 7)) << 4))) = y;
    }
#pragma unroll
  for (int p = 0; p < 32 / RPI; ++p) {
    const int r = p * RPI + lane / CPR, ch = lane % CPR;
    const bf16x8 y = attn_lds<bf16x8>(
        sm, box + r * (2 * D) + ((ch ^ (r & 7)) << 4));
    if (row0 + r < row_end && ch * 8 < Dact)
      *(bf16x8*)(base + (long)(row0 + r) * stride + ch * 8) = y;
  }
}

}  // namespace mxa
