// Embedding: scaled row lookup, and the gradient of the table.
// Reference parity: src/operator/tensor/indexing_op.cu (Embedding,
// AddTakeGrad).
//
//   out[n] = scale * W[idx[n]],   dW[r] = scale * sum_{n: idx[n] = r} dy[n]
//
// An index outside [0, vocab) gives a row of zeros and adds to nothing.
// Both directions are bound by memory.  The gradient is summed in 32 bits in
// the order of the tokens and rounded once:
//   1. emb_sort    tokens ordered by row (stable), and where each row starts;
//                  for many tokens or rows a sort by digits instead
//   2. emb_reduce  EMB_CHUNK sorted tokens to a wave: rows that lie inside a
//                  chunk are final, the two at its ends may be partial; rows
//                  without a token are cleared by further blocks
//   3. emb_join    rows that cross chunks, their parts added in a fixed order
// so a row that half of all tokens hit is spread over the chip like any
// other, nothing is added by atomics and every run gives the same bits.
// 16384 tokens, 32768 rows of 1024 in bf16: lookup 10 us (64 MB), order 14,
// sums 21 (97 MB, 4.6 TB/s), rows that cross chunks 6; a table of two rows of
// 768: 9, 13, 16 and 7.  The order is bound by the two passes that every block
// makes over all indices, from L2.
#include <hip/hip_fp16.h>

#include <algorithm>

#include "common.h"

namespace mxa {

constexpr int EMB_CHUNK = 32;

DEVINL float emb_f(float x) { return x; }
DEVINL float emb_f(bf16 x) { return (float)x; }
DEVINL float emb_f(_Float16 x) { return (float)x; }

// V values of T in one access (16 bytes where V > 1)
template <typename T, int V>
DEVINL void emb_load(const T* p, T* x) {
  if (V == 1) {
    x[0] = *p;
  } else {
    typedef T vt __attribute__((ext_vector_type(V)));
    vt v = *(const vt*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = v[i];
  }
}

template <typename T, int V>
DEVINL void emb_store(T* p, const float* x, float mul) {
  if (V == 1) {
    *p = (T)(x[0] * mul);
  } else {
    typedef T vt __attribute__((ext_vector_type(V)));
    vt v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)(x[i] * mul);
    *(vt*)p = v;
  }
}

// One block: 256 / lpr rows at a time, lpr lanes (a power of two) to a row.
template <typename T, int V, typename I>
__global__ __launch_bounds__(256) void emb_lookup_kernel(
    const I* __restrict__ idx, const T* __restrict__ W, T* __restrict__ out,
    long ntok, int D, long vocab, float scale, int lpr_log2) {
  const int lpr = 1 << lpr_log2;
  const int sub = threadIdx.x >> lpr_log2, l = threadIdx.x & (lpr - 1);
  const int rpb = 256 >> lpr_log2;
  const int nv = D / V;
  for (long t = (long)blockIdx.x * rpb + sub; t < ntok;
       t += (long)gridDim.x * rpb) {
    const long row = (long)idx[t];
    const bool ok = row >= 0 && row < vocab;
    for (int c = l; c < nv; c += lpr) {
      T x[V];
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = 0.f;
      if (ok) {
        emb_load<T, V>(W + row * D + c * V, x);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = emb_f(x[i]);
      }
      emb_store<T, V>(out + t * D + c * V, y, scale);
    }
  }
}

// ---------------------------------------------------------------------------
// 1. Order the tokens by row.  Block p owns rows [p R, p R + R): it reads all
// indices twice, a wave a contiguous sixteenth of the tokens, and keeps a
// list of those that are its own.  The first time it counts them, by row and
// by wave, and the tokens of lower rows, which tells it where its part of the
// order begins without a word from another block.  The second time it places
// them; equal rows within a wave are ranked by lane, so the order is stable.
// Most groups of 64 tokens hold none of a block's rows and cost a handful of
// instructions; some 256 blocks of rows (what a block does with its own
// tokens takes longer than all blocks' reading of the same indices from L2).
// ---------------------------------------------------------------------------
constexpr int EMB_WAVES = 16;
constexpr int EMB_ROWS = 512;    // rows of a block at most

// BATCH: groups of 64 tokens that a wave reads at once.
template <typename I, int BATCH>
__global__ __launch_bounds__(1024) void emb_sort_kernel(
    const I* __restrict__ idx, int ntok, int vocab, int R, int rlog2,
    int* __restrict__ start, int2* __restrict__ sorted) {
  __shared__ int cnt[EMB_ROWS * EMB_WAVES];  // [row][wave]
  __shared__ unsigned list[EMB_WAVES][64 * BATCH];
  __shared__ int below[EMB_WAVES], tot[EMB_WAVES];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 lower = (1ull << lane) - 1;
  const int r0 = blockIdx.x * R;
  const int nr = min(R, vocab - r0);
  for (int i = threadIdx.x; i < R * EMB_WAVES; i += 1024) cnt[i] = 0;
  __syncthreads();

  constexpr int STEP = 64 * BATCH;
  const int seg = (ntok + EMB_WAVES * 64 - 1) / (EMB_WAVES * 64) * 64;
  const int t0 = min(ntok, wave * seg), t1 = min(ntok, t0 + seg);

  // Tokens tb..tb + STEP - 1: a list of (row, place) of the block's own, in
  // order; returns how many.  low counts the tokens of lower rows.
  auto filter = [&](int tb, int& low) -> int {
    unsigned r[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int t = tb + u * 64 + lane;
      r[u] = 0xffffffffu;  // outside the table: behind all rows
      if (t < t1) {
        const I x = idx[t];
        // a negative index is a large one when read without its sign
        const bool in = sizeof(I) == 8
                            ? (u64)x < (u64)(unsigned)vocab
                            : (unsigned)x < (unsigned)vocab;
        if (in) r[u] = (unsigned)x;
      }
    }
    int n = 0;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      low += __popcll(__ballot(r[u] < (unsigned)r0));
      const bool mine = r[u] - (unsigned)r0 < (unsigned)nr;
      const u64 m = __ballot(mine);
      if (m == 0) continue;
      if (mine)
        list[wave][n + __popcll(m & lower)] =
            (r[u] - (unsigned)r0) * STEP + u * 64 + lane;
      n += __popcll(m);
    }
    return n;
  };
  // lanes whose entry has the same row as this lane's
  auto same_row = [&](unsigned row, bool on) -> u64 {
    u64 same = __ballot(on);
    if (__popcll(same) > 4) {
      for (int bit = 0; bit < rlog2; ++bit) {
        const bool one = (row >> bit) & 1;
        const u64 bal = __ballot(one);
        same &= one ? bal : ~bal;
      }
    } else {
      u64 rest = same;
      while (rest) {
        const int lead = __builtin_ctzll(rest);
        const u64 eq = __ballot(
            on && row == (unsigned)__builtin_amdgcn_readlane((int)row, lead));
        if (eq >> lane & 1) same = eq;
        rest &= ~eq;
      }
    }
    return on ? same : 0;
  };

  // a wave's list and counters are its own, and its LDS accesses stay in
  // order: one lane of each row writes for all
  int low = 0, n = 0;
  for (int tb = t0; tb < t1; tb += STEP) {
    n = filter(tb, low);
    for (int k = 0; k < n; k += 64) {
      const bool on = k + lane < n;
      const unsigned row = on ? list[wave][k + lane] / STEP : 0;
      const u64 same = same_row(row, on);
      if (same && (same & lower) == 0)
        cnt[row * EMB_WAVES + wave] += __popcll(same);
    }
  }
  if (lane == 0) below[wave] = low;
  __syncthreads();

  // exclusive sums over (row, wave); a thread takes a run of the counters
  int first = 0;
  for (int w = 0; w < EMB_WAVES; ++w) first += below[w];
  const int nc = R * EMB_WAVES, per = (nc + 1023) / 1024;
  const int a = min(nc, (int)threadIdx.x * per), e = min(nc, a + per);
  int sum = 0;
  for (int i = a; i < e; ++i) sum += cnt[i];
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    int x = __shfl_up(inc, o, 64);
    if (lane >= o) inc += x;
  }
  if (lane == 63) tot[wave] = inc;
  __syncthreads();
  int run = first + inc - sum;
  for (int w = 0; w < wave; ++w) run += tot[w];
  for (int i = a; i < e; ++i) {
    int c = cnt[i];
    cnt[i] = run;
    if (i % EMB_WAVES == 0 && i / EMB_WAVES < nr)
      start[r0 + i / EMB_WAVES] = run;
    run += c;
  }
  if (r0 + nr == vocab && threadIdx.x == 1023) start[vocab] = run;
  __syncthreads();

  const bool once = t1 - t0 <= STEP;  // the list still holds them all
  for (int tb = t0; tb < t1; tb += STEP) {
    if (!once) n = filter(tb, low);
    for (int k = 0; k < n; k += 64) {
      const bool on = k + lane < n;
      const unsigned x = on ? list[wave][k + lane] : 0, row = x / STEP;
      const u64 same = same_row(row, on);
      if (same) {
        const int rank = __popcll(same & lower);
        const int pos = cnt[row * EMB_WAVES + wave] + rank;
        sorted[pos] = make_int2(r0 + (int)row, tb + (int)(x % STEP));
        // the last lane of a row moves its counter on
        if (rank == __popcll(same) - 1) cnt[row * EMB_WAVES + wave] = pos + 1;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 1 for many tokens or rows: the work above is blocks times tokens.  A stable
// sort by digits of the row, lowest first, takes a few passes over the tokens
// instead.  Each pass divides them into segments of a block each:
//   emb_digits   counts every digit of a segment
//   emb_scan     sums a digit's counts over the segments before each
//   emb_scatter  counts once more by wave, which gives every wave its places,
//                and writes (row, token) there; equal digits within 64 tokens
//                are ranked by lane
// Tokens outside the table count as of one row behind it.  The last pass knows
// where each value of the highest digit begins; emb_start finds the rows from
// there by halving.  262144 tokens in 2 ** 22 rows, three passes: 52 us, the
// starts 21, bound by the passes' launches and the reads that follow one
// another in the halving; 2 ** 20 tokens in 10 ** 7 rows 70 and 33.
// ---------------------------------------------------------------------------
constexpr int EMB_BITS = 11;      // of a digit at most: 32 KB of counters
constexpr int EMB_SEG = 2048;     // tokens of a segment at least
constexpr int EMB_SEGS = 1024;    // segments at most

template <typename I>
struct EmbIndices {
  const I* idx;
  int vocab;
  DEVINL int2 at(int t) const {
    const I x = idx[t];
    const bool in = sizeof(I) == 8 ? (u64)x < (u64)(unsigned)vocab
                                   : (unsigned)x < (unsigned)vocab;
    return make_int2(in ? (int)x : vocab, t);
  }
};

struct EmbPairs {
  const int2* pair;
  DEVINL int2 at(int t) const { return pair[t]; }
};

template <typename S>
__global__ __launch_bounds__(256) void emb_digits_kernel(
    S src, int ntok, int len, int shift, int bits, int* __restrict__ cnt) {
  __shared__ int h[1 << EMB_BITS];
  const int nd = 1 << bits;
  for (int i = threadIdx.x; i < nd; i += 256) h[i] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * len;
  const int t1 = ntok - t0 < len ? ntok : t0 + len;
#pragma unroll 4
  for (int t = t0 + (int)threadIdx.x; t < t1; t += 256)
    atomicAdd(&h[(src.at(t).x >> shift) & (nd - 1)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < nd; i += 256)
    cnt[(long)blockIdx.x * nd + i] = h[i];
}

// cnt: [nseg][nd], every entry becomes the sum of those before it; total: [nd]
__global__ __launch_bounds__(256) void emb_scan_kernel(
    int* __restrict__ cnt, int* __restrict__ total, int nseg, int nd) {
  __shared__ int part[16][16];
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  int* const p = cnt + blockIdx.x * 16 + l;
  const int per = (nseg + 15) / 16;
  const int a = min(nseg, g * per), e = min(nseg, a + per);
  int sum = 0;
#pragma unroll 8
  for (int i = a; i < e; ++i) sum += p[(long)i * nd];
  part[g][l] = sum;
  __syncthreads();
  int run = 0;
  for (int i = 0; i < g; ++i) run += part[i][l];
  if (g == 15) total[blockIdx.x * 16 + l] = run + sum;
#pragma unroll 8
  for (int i = a; i < e; ++i) {
    const int c = p[(long)i * nd];
    p[(long)i * nd] = run;
    run += c;
  }
}

// first: [nd + 1], where each digit begins; null but in the last pass
template <typename S>
__global__ __launch_bounds__(256) void emb_scatter_kernel(
    S src, int ntok, int len, int shift, int bits,
    const int* __restrict__ cnt, const int* __restrict__ total,
    int* __restrict__ first, int2* __restrict__ out) {
  __shared__ int place[4][1 << EMB_BITS];
  __shared__ int tot[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 lower = (1ull << lane) - 1;
  const int nd = 1 << bits;
  for (int i = threadIdx.x; i < nd; i += 256)
    place[0][i] = place[1][i] = place[2][i] = place[3][i] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * len;
  const int t1 = ntok - t0 < len ? ntok : t0 + len;
  // a quarter to a wave, groups of 64 tokens whole
  const int quarter = (t1 - t0 + 255) / 256 * 64;
  const int w0 = min(t1, t0 + wave * quarter), w1 = min(t1, w0 + quarter);
#pragma unroll 4
  for (int t = w0 + lane; t < w1; t += 64)
    atomicAdd(&place[wave][(src.at(t).x >> shift) & (nd - 1)], 1);

  // a thread takes a run of the digits
  const int per = (nd + 255) / 256;
  const int a = min(nd, (int)threadIdx.x * per), e = min(nd, a + per);
  int sum = 0;
  for (int i = a; i < e; ++i) sum += total[i];
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(inc, o, 64);
    if (lane >= o) inc += x;
  }
  if (lane == 63) tot[wave] = inc;
  __syncthreads();
  int run = inc - sum;
  for (int w = 0; w < wave; ++w) run += tot[w];
  for (int i = a; i < e; ++i) {
    if (first && blockIdx.x == 0) first[i] = run;
    int at = run + cnt[(long)blockIdx.x * nd + i];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int c = place[w][i];
      place[w][i] = at;
      at += c;
    }
    run += total[i];
  }
  if (first && blockIdx.x == 0 && threadIdx.x == 0) first[nd] = ntok;
  __syncthreads();

  // a wave's counters are its own, and its LDS accesses stay in order
  constexpr int U = 4;
  for (int tb = w0; tb < w1; tb += 64 * U) {
    int2 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = tb + u * 64 + lane;
      x[u] = t < w1 ? src.at(t) : make_int2(0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = tb + u * 64 + lane < w1;
      const int digit = (x[u].x >> shift) & (nd - 1);
      u64 same = __ballot(on);
      for (int bit = 0; bit < bits; ++bit) {
        const bool one = (digit >> bit) & 1;
        const u64 bal = __ballot(one);
        same &= one ? bal : ~bal;
      }
      if (on) {
        const int rank = __popcll(same & lower);
        const int pos = place[wave][digit] + rank;
        out[pos] = x[u];
        // the last lane of a digit moves its counter on
        if (rank == __popcll(same) - 1) place[wave][digit] = pos + 1;
      }
    }
  }
}

// The first place in [lo, hi) whose row is r or higher; row(i) is the i-th.
template <typename F>
DEVINL int emb_first(F row, int lo, int hi, int r) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (row(mid) < r)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// start[r]: the first place whose row is r or higher.  A block takes 256 rows,
// or EMB_SPAN of a large table, whose tokens it halves in LDS if they fit: the
// halving in memory would be most of the time there (10 ** 7 rows 33 us, not
// 96; 2 ** 22 21 and 39; 32768 rows 29 and 5, on 16 blocks).
constexpr int EMB_SPAN = 2048, EMB_KEYS = 4096;

__global__ __launch_bounds__(256) void emb_start_kernel(
    const int2* __restrict__ sorted, const int* __restrict__ first, int ntok,
    int vocab, int shift, int span, int* __restrict__ start) {
  __shared__ int keys[EMB_KEYS];
  __shared__ int ends[2];
  const long r0 = (long)blockIdx.x * span;
  const long r1 = min(r0 + span, (long)vocab + 1);
  if (span < EMB_SPAN) {
    const long r = r0 + threadIdx.x;
    if (r < r1)
      start[r] = emb_first([&](int i) { return sorted[i].x; },
                           first[r >> shift], first[(r >> shift) + 1],
                           (int)r);
    return;
  }
  if (threadIdx.x < 2) {
    const long r = threadIdx.x ? r1 : r0;
    int at = ntok;
    if (r <= vocab)
      at = emb_first([&](int i) { return sorted[i].x; }, first[r >> shift],
                     first[(r >> shift) + 1], (int)r);
    ends[threadIdx.x] = at;
  }
  __syncthreads();
  const int lo = ends[0], n = ends[1] - lo;
  if (n <= EMB_KEYS) {
    for (int i = threadIdx.x; i < n; i += 256) keys[i] = sorted[lo + i].x;
    __syncthreads();
    for (long r = r0 + threadIdx.x; r < r1; r += 256)
      start[r] = lo + emb_first([&](int i) { return keys[i]; }, 0, n, (int)r);
  } else {
    for (long r = r0 + threadIdx.x; r < r1; r += 256)
      start[r] = emb_first([&](int i) { return sorted[i].x; },
                           max(lo, first[r >> shift]),
                           min(lo + n, first[(r >> shift) + 1]), (int)r);
  }
}

// ---------------------------------------------------------------------------
// 2. Sums.  Waves [0, nchunk * ns) take a chunk (from chunk0 on) and a slice
// of 64 V columns; the rest of the grid clears rows that no token hits.
// part: [nchunk][2][D], the sums of a chunk's first row where it began in an
// earlier chunk, and of its last row where it goes on in the next.
// ---------------------------------------------------------------------------
template <typename T, int V>
__global__ __launch_bounds__(256) void emb_reduce_kernel(
    const int2* __restrict__ sorted, const int* __restrict__ start,
    const T* __restrict__ dy, T* __restrict__ dW, float* __restrict__ part,
    int vocab, int D, float scale, int chunk0, int nchunk, int ns,
    int sumblocks, int zrows, int zlog2) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= sumblocks) {
    // zrows rows of a wave at a time, 1 << zlog2 lanes to each
    const int nv = D / V;
    const float z[V] = {};
    const int sub = lane >> zlog2, l = lane & ((1 << zlog2) - 1);
    const long step = (long)(gridDim.x - sumblocks) * 4 * zrows;
    for (long r0 = ((long)(blockIdx.x - sumblocks) * 4 + wave) * zrows;
         r0 < vocab; r0 += step) {
      const long r = r0 + lane;
      const u64 empty = __ballot(lane < zrows && r < vocab &&
                                 start[min(r, (long)vocab)] ==
                                     start[min(r + 1, (long)vocab)]);
      if (empty == 0) continue;
      for (int k = sub; k < zrows; k += 64 >> zlog2) {
        if (!(empty >> k & 1)) continue;
        for (int c = l; c < nv; c += 1 << zlog2)
          emb_store<T, V>(dW + (r0 + k) * D + (long)c * V, z, 1.f);
      }
    }
    return;
  }
  const int n = start[vocab];  // tokens inside the table
  const long w = (long)blockIdx.x * 4 + wave;
  if (w >= (long)nchunk * ns) return;
  const int chunk = chunk0 + (int)(w / ns), slice = (int)(w % ns);
  const int p0 = chunk * EMB_CHUNK, p1 = min(n, p0 + EMB_CHUNK);
  if (p0 >= p1) return;
  const int c = (slice * 64 + lane) * V;
  const bool on = c < D;

  int2 kt = make_int2(-1, 0);
  if (p0 + lane < p1 && lane < EMB_CHUNK) kt = sorted[p0 + lane];
  const int prev = p0 > 0 ? sorted[p0 - 1].x : -1;
  const int next = p1 < n ? sorted[p1].x : -1;

  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  int key = __builtin_amdgcn_readlane(kt.x, 0);
  bool head = key == prev;  // this row began in an earlier chunk
  constexpr int U = 16;     // rows in flight
  for (int b = 0; b < p1 - p0; b += U) {
    T x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = __builtin_amdgcn_readlane(kt.y, (b + u) & 63);
      if (b + u < p1 - p0 && on) emb_load<T, V>(dy + (long)t * D + c, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u >= p1 - p0) break;
      const int k = __builtin_amdgcn_readlane(kt.x, (b + u) & 63);
      if (k != key) {
        if (on) {
          if (head) {
            float* q = part + ((long)chunk * 2) * D + c;
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = acc[i];
          } else {
            emb_store<T, V>(dW + (long)key * D + c, acc, scale);
          }
        }
        head = false;
        key = k;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += emb_f(x[u][i]);
    }
  }
  if (!on) return;
  if (head || key == next) {
    // a row that fills the chunk and goes on both ways has its part first
    float* q = part + ((long)chunk * 2 + (head ? 0 : 1)) * D + c;
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = acc[i];
  } else {
    emb_store<T, V>(dW + (long)key * D + c, acc, scale);
  }
}

// ---------------------------------------------------------------------------
// 3. Rows that cross chunks.  A block looks at the last rows of per chunks; if
// one began there and goes on, the block adds its parts.  Few parts: the
// first of EMB_JOIN blocks of the chunks adds them for all columns, 1 << jlog2
// threads a chunk (262144 tokens, rows of 64 in bf16: 31 us with the block's
// chunks one after another, 5 side by side).  Many: each block takes a share
// of the columns, and groups of 1 << glog2 threads a share of the parts each,
// joined in order.
// ---------------------------------------------------------------------------
constexpr int EMB_JOIN = 8;

template <typename T, int PV>
__global__ __launch_bounds__(256) void emb_join_kernel(
    const int2* __restrict__ sorted, const int* __restrict__ start,
    const float* __restrict__ part, T* __restrict__ dW, int vocab, int D,
    float scale, int chunk0, int nchunk, int per, int jlog2, int glog2) {
  __shared__ float sums[256][PV];
  __shared__ u64 todo[2];
  const int n = start[vocab];
  const int first = chunk0 + (int)blockIdx.x * per;
  if (threadIdx.x < 64) {  // per is 64 at most
    const int chunk = first + (int)threadIdx.x;
    bool on = (int)threadIdx.x < per && chunk < nchunk - 1;
    const long end = ((long)chunk + 1) * EMB_CHUNK;
    on = on && end < n;  // else nothing follows this chunk
    bool few = false;
    if (on) {
      const int key = sorted[end - 1].x;
      const int s1 = start[key + 1];
      on = s1 > end && start[key] >= chunk * EMB_CHUNK;
      few = (s1 - 1) / EMB_CHUNK - chunk + 1 <= 32;
    }
    const u64 f = __ballot(on && few), m = __ballot(on && !few);
    if (threadIdx.x == 0) {
      todo[0] = f;
      todo[1] = m;
    }
  }
  __syncthreads();
  const int nv = D / PV;
  const u64 fews = blockIdx.y == 0 ? todo[0] : 0;
  for (int k = threadIdx.x >> jlog2; fews && k < per; k += 256 >> jlog2) {
    if (!(fews >> k & 1)) continue;
    const int chunk = first + k;
    const int key = sorted[(chunk + 1) * EMB_CHUNK - 1].x;
    const int parts = (start[key + 1] - 1) / EMB_CHUNK - chunk + 1;
    const float* p0 = part + ((long)chunk * 2 + 1) * D;  // first part
    const float* p1 = part + ((long)chunk * 2) * D;      // others: + 2 D i
    T* out = dW + (long)key * D;
    for (int v = threadIdx.x & ((1 << jlog2) - 1); v < nv; v += 1 << jlog2) {
      float y[PV], x[PV];
      emb_load<float, PV>(p0 + v * PV, y);
#pragma unroll 4
      for (int i = 1; i < parts; ++i) {
        emb_load<float, PV>(p1 + (long)i * 2 * D + v * PV, x);
#pragma unroll
        for (int c = 0; c < PV; ++c) y[c] += x[c];
      }
      emb_store<T, PV>(out + v * PV, y, scale);
    }
  }
  for (u64 left = todo[1]; left; left &= left - 1) {
    const int chunk = first + __builtin_ctzll(left);
    const int key = sorted[(chunk + 1) * EMB_CHUNK - 1].x;
    const int parts = (start[key + 1] - 1) / EMB_CHUNK - chunk + 1;
    const float* p0 = part + ((long)chunk * 2 + 1) * D;  // first part
    const float* p1 = part + ((long)chunk * 2) * D;      // others: + 2 D i
    T* out = dW + (long)key * D;
    const int lo = (int)((long)nv * blockIdx.y / EMB_JOIN);
    const int hi = (int)((long)nv * (blockIdx.y + 1) / EMB_JOIN);
    // as many groups as the block's share of the columns leaves threads for
    const int gl = 1 << glog2, ng = 256 >> glog2;
    const int g = threadIdx.x >> glog2, l = threadIdx.x & (gl - 1);
    const int share = (parts + ng - 1) / ng;
    const int a = min(parts, g * share), e = min(parts, a + share);
    for (int vb = lo; vb < hi; vb += gl) {
      const int v = vb + l;
      float y[PV] = {};
      if (v < hi) {
#pragma unroll 8
        for (int i = a; i < e; ++i) {
          float x[PV];
          emb_load<float, PV>(
              (i == 0 ? p0 : p1 + (long)i * 2 * D) + v * PV, x);
#pragma unroll
          for (int k = 0; k < PV; ++k) y[k] += x[k];
        }
      }
      // the upper half of the groups hands its sums to the lower, and so on
      for (int w = ng / 2; w > 0; w /= 2) {
        if (g >= w && g < 2 * w)
#pragma unroll
          for (int k = 0; k < PV; ++k) sums[threadIdx.x][k] = y[k];
        __syncthreads();
        if (g < w)
#pragma unroll
          for (int k = 0; k < PV; ++k)
            y[k] += sums[threadIdx.x + w * gl][k];
      }
      if (g == 0 && v < hi) emb_store<T, PV>(out + v * PV, y, scale);
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Blocks of a launch at most: the runtime takes less than 2**32 threads a
// dimension.
constexpr unsigned EMB_LAUNCH = 1u << 21;

// dtype: 0 bf16, 1 fp16, 2 fp32
#define EMB_TYPES(dtype, F)                 \
  switch (dtype) {                          \
    case 0: F(bf16, 8); break;              \
    case 1: F(_Float16, 8); break;          \
    default: F(float, 4); break;            \
  }

void emb_lookup(int dtype, bool vec, bool idx64, const void* idx,
                const void* W, void* out, long ntok, int D, long vocab,
                float scale, hipStream_t s) {
#define GO(T, V, I)                                                       \
  do {                                                                    \
    int nv = D / (V), lg = 0;                                             \
    while ((1 << lg) < nv && lg < 8) ++lg;                                \
    long nb = (ntok + (256 >> lg) - 1) / (256 >> lg);                     \
    unsigned g = (unsigned)(nb < 8192 ? nb : 8192);                       \
    emb_lookup_kernel<T, V, I><<<g, 256, 0, s>>>(                         \
        (const I*)idx, (const T*)W, (T*)out, ntok, D, vocab, scale, lg);  \
  } while (0)
#define F(T, V)             \
  if (vec && idx64)         \
    GO(T, V, long);         \
  else if (vec)             \
    GO(T, V, int);          \
  else if (idx64)           \
    GO(T, 1, long);         \
  else                      \
    GO(T, 1, int)
  EMB_TYPES(dtype, F)
#undef F
#undef GO
}

int emb_chunks(long ntok) {
  return (int)((ntok + EMB_CHUNK - 1) / EMB_CHUNK);
}

// How the tokens are ordered.  By blocks the time goes with tokens (and some
// 4096 more for a block's start) times blocks beyond one for each compute
// unit, by digits with the passes.  The whole gradient of rows of 64, in us by
// blocks and by digits:
//   1000 rows       16384 tokens 22 and 31,   65536 45 and 34
//   32768 rows      32768 tokens 34 and 45,   65536 49 and 48,  262144 181, 74
//   250000 rows     16384 tokens 43 and 55,   65536 73 and 58,  262144 208, 81
//   2 ** 20 rows    512 tokens   65 and 60,   65536 183 and 76
//   10 ** 7 rows    512 tokens   539 and 302, 16384 773 and 332
struct EmbOrder {
  int rlog2;        // rows of a block, as a power of two
  unsigned blocks;
  int bits, passes; // by digits: of this many bits; no passes: by blocks
  int len, nseg;    // and segments of this many tokens
  long ws;          // integers of workspace
};

static EmbOrder emb_order(long ntok, long vocab) {
  EmbOrder o = {};
  while ((1 << o.rlog2) < EMB_ROWS && (long)256 << o.rlog2 < vocab) ++o.rlog2;
  o.blocks = (unsigned)((vocab + (1l << o.rlog2) - 1) >> o.rlog2);
  int bits = 4;  // of the row behind the last one too
  while (vocab >> bits) ++bits;
  const int passes = (bits + EMB_BITS - 1) / EMB_BITS;
  if ((ntok + 4096) * std::max(256l, (long)o.blocks) <=
      16384l * 256 * (passes + 1))
    return o;
  o.passes = passes;
  o.bits = (bits + o.passes - 1) / o.passes;
  o.len = (int)std::max((long)EMB_SEG, (ntok + EMB_SEGS - 1) / EMB_SEGS);
  o.nseg = (int)((ntok + o.len - 1) / o.len);
  // the other buffer of (row, token); counts, totals and first places
  o.ws = (o.passes > 1 ? 2 * ntok : 0) + ((o.nseg + 2l) << o.bits) + 1;
  return o;
}

long emb_ws(long ntok, long vocab) { return emb_order(ntok, vocab).ws; }

template <typename S>
static void emb_pass(const EmbOrder& o, S src, int pass, int ntok, int* cnt,
                     int2* out, hipStream_t s) {
  const int nd = 1 << o.bits, shift = pass * o.bits;
  int* total = cnt + (long)o.nseg * nd;
  int* first = pass == o.passes - 1 ? total + nd : nullptr;
  emb_digits_kernel<S><<<o.nseg, 256, 0, s>>>(src, ntok, o.len, shift, o.bits,
                                              cnt);
  emb_scan_kernel<<<nd / 16, 256, 0, s>>>(cnt, total, o.nseg, nd);
  emb_scatter_kernel<S><<<o.nseg, 256, 0, s>>>(src, ntok, o.len, shift, o.bits,
                                               cnt, total, first, out);
}

// start: [vocab + 1], sorted: [ntok], part: [emb_chunks][2][D], ws: [emb_ws]
void emb_grad(int dtype, bool vec, bool idx64, const void* idx,
              const void* dy, void* dW, int* start, int2* sorted,
              float* part, int* ws, int ntok, int D, int vocab, float scale,
              hipStream_t s) {
  const EmbOrder o = emb_order(ntok, vocab);
  const int R = 1 << o.rlog2, lg = o.rlog2;
  const unsigned nb = o.blocks;
  // 16 groups at once keep the lists of 16384 tokens from the first pass to
  // the second: 14.2 us, not 17.8 (32768 rows).  They gain nothing for few
  // tokens (4096: 7.3 and 6.6) and leave room for one block on a compute unit
  // (250000 rows: 25 and 23).
  const bool wide = ntok > 8192 && nb <= 256;
#define GO(I, N)                                                       \
  emb_sort_kernel<I, N><<<nb, 1024, 0, s>>>((const I*)idx, ntok, vocab, \
                                            R, lg, start, sorted)
  if (o.passes) {
    int2* other = (int2*)ws;
    int* cnt = ws + (o.passes > 1 ? 2l * ntok : 0);
    for (int p = 0; p < o.passes; ++p) {
      // the last pass writes to sorted
      int2* dst = (o.passes - 1 - p) % 2 ? other : sorted;
      const int2* src = dst == sorted ? other : sorted;
      if (p > 0)
        emb_pass(o, EmbPairs{src}, p, ntok, cnt, dst, s);
      else if (idx64)
        emb_pass(o, EmbIndices<long>{(const long*)idx, vocab}, p, ntok, cnt,
                 dst, s);
      else
        emb_pass(o, EmbIndices<int>{(const int*)idx, vocab}, p, ntok, cnt,
                 dst, s);
    }
    const int span = vocab >= 1 << 20 ? EMB_SPAN : 256;
    emb_start_kernel<<<(unsigned)(vocab / span + 1), 256, 0, s>>>(
        sorted, cnt + ((o.nseg + 1l) << o.bits), ntok, vocab,
        (o.passes - 1) * o.bits, span, start);
  } else if (idx64 && wide)
    GO(long, 16);
  else if (idx64)
    GO(long, 8);
  else if (wide)
    GO(int, 16);
  else
    GO(int, 8);
#undef GO
  const int nchunk = emb_chunks(ntok);
#define GO(T, V)                                                             \
  do {                                                                       \
    const int ns = (D / (V) + 63) / 64;                                      \
    const int most = max(1, (int)(EMB_LAUNCH * 4l / ns));                    \
    /* cleared by 8192 waves, whose lanes take as many rows as they cover */ \
    int zlog2 = 0, zrows = 1;                                                \
    while (zlog2 < 6 && (1 << zlog2) < D / (V)) ++zlog2;                     \
    while (zrows < 64 &&                                                     \
           (zrows < 64 >> zlog2 || 16384l * zrows <= vocab))                 \
      zrows *= 2;                                                            \
    for (int c0 = 0; c0 < nchunk; c0 += most) {                              \
      const int nc = min(most, nchunk - c0);                                 \
      unsigned sb = (unsigned)(((long)nc * ns + 3) / 4);                     \
      unsigned zb = (unsigned)(vocab < 8192 ? (vocab + 3) / 4 : 2048);       \
      if (c0 > 0) zb = 0;                                                    \
      emb_reduce_kernel<T, V><<<sb + zb, 256, 0, s>>>(                       \
          sorted, start, (const T*)dy, (T*)dW, part, vocab, D, scale, c0,    \
          nc, ns, (int)sb, zrows, zlog2);                                    \
    }                                                                        \
    constexpr int PV = (V) == 1 ? 1 : 4;                                     \
    /* chunks of a block: few blocks start for nothing, and as many as its */ \
    /* threads take side by side while that leaves 256 blocks              */ \
    int jlog2 = 0;                                                           \
    while (jlog2 < 8 && (1 << jlog2) < D / PV) ++jlog2;                      \
    int glog2 = 0;                                                           \
    while (glog2 < 5 && (EMB_JOIN << glog2) < D / PV) ++glog2;               \
    const int per = max(                                                     \
        1, min(64, max(nchunk / 2048, min(256 >> jlog2, nchunk / 256))));    \
    const int jb = (nchunk - 2 + per) / per;                                 \
    for (int j = 0; j < jb; j += EMB_LAUNCH)                                 \
      emb_join_kernel<T, PV>                                                 \
          <<<dim3(min((int)EMB_LAUNCH, jb - j), EMB_JOIN), 256, 0, s>>>(     \
              sorted, start, part, (T*)dW, vocab, D, scale, j * per, nchunk, \
              per, jlog2, glog2);                                            \
  } while (0)
#define F(T, V) \
  if (vec)      \
    GO(T, V);   \
  else          \
    GO(T, 1)
  EMB_TYPES(dtype, F)
#undef F
#undef GO
}

}  // namespace mxa
