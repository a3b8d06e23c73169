// Embedding: scaled row lookup, and the gradient of the table.
// Reference parity: src/operator/tensor/indexing_op.cu (Embedding,
// AddTakeGrad).
//
//   out[n] = scale * W[idx[n]],   dW[r] = scale * sum_{n: idx[n] = r} dy[n]
//
// An index outside [0, vocab) gives a row of zeros and adds to nothing.
// Both directions are bound by memory.  The gradient is summed in 32 bits in
// the order of the tokens and rounded once, by three launches:
//   1. emb_sort    tokens ordered by row (stable), and where each row starts
//   2. emb_reduce  EMB_CHUNK sorted tokens to a wave: rows that lie inside a
//                  chunk are final, the two at its ends may be partial; rows
//                  without a token are cleared by further blocks
//   3. emb_join    rows that cross chunks, their parts added in order
// so a row that half of all tokens hit is spread over the chip like any
// other, nothing is added by atomics and every run gives the same bits.
// 16384 tokens, 32768 rows of 1024 in bf16: lookup 10 us (64 MB), order 14,
// sums 20 (97 MB, 5 TB/s), rows that cross chunks 5; a table of two rows of
// 768: 9, 14, 15 and 7.  The order is bound by the two passes that every block
// makes over all indices, from L2.
#include <hip/hip_fp16.h>

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
    const I* __restrict__ idx, int ntok, int vocab, int R, int rlog2, int p0,
    int* __restrict__ start, int2* __restrict__ sorted) {
  __shared__ int cnt[EMB_ROWS * EMB_WAVES];  // [row][wave]
  __shared__ unsigned list[EMB_WAVES][64 * BATCH];
  __shared__ int below[EMB_WAVES], tot[EMB_WAVES];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 lower = (1ull << lane) - 1;
  const int r0 = (p0 + (int)blockIdx.x) * R;
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
    int sumblocks) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= sumblocks) {
    const int nv = D / V;
    const float z[V] = {};
    for (long r = (blockIdx.x - sumblocks) * 4 + wave; r < vocab;
         r += (gridDim.x - sumblocks) * 4) {
      if (start[r] != start[r + 1]) continue;
      for (int c = lane; c < nv; c += 64)
        emb_store<T, V>(dW + r * D + (long)c * V, z, 1.f);
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
// 3. Rows that cross chunks.  A block looks at the last row of one chunk; if
// it began there and goes on, the block adds its parts.  Few parts: the
// first of EMB_JOIN blocks of the chunk adds them for all columns.  Many:
// each block takes a share of the columns, and 8 groups of 32 threads a
// share of the parts each, joined in order.
// ---------------------------------------------------------------------------
constexpr int EMB_JOIN = 8;

template <typename T, int PV>
__global__ __launch_bounds__(256) void emb_join_kernel(
    const int2* __restrict__ sorted, const int* __restrict__ start,
    const float* __restrict__ part, T* __restrict__ dW, int vocab, int D,
    float scale, int chunk0) {
  __shared__ float sums[8][32][PV];
  const int n = start[vocab];
  const int chunk = chunk0 + (int)blockIdx.x;
  const int end = (chunk + 1) * EMB_CHUNK;
  if (end >= n) return;  // nothing follows this chunk
  const int key = sorted[end - 1].x;
  const int s0 = start[key], s1 = start[key + 1];
  if (s1 <= end || s0 < chunk * EMB_CHUNK) return;
  const int parts = (s1 - 1) / EMB_CHUNK - chunk + 1;
  const int nv = D / PV;
  const float* p0 = part + ((long)chunk * 2 + 1) * D;  // first part
  const float* p1 = part + ((long)chunk * 2) * D;      // others: + 2 D i
  T* out = dW + (long)key * D;
  if (parts <= 32) {
    if (blockIdx.y != 0) return;
    for (int v = threadIdx.x; v < nv; v += 256) {
      float y[PV], x[PV];
      emb_load<float, PV>(p0 + v * PV, y);
#pragma unroll 4
      for (int i = 1; i < parts; ++i) {
        emb_load<float, PV>(p1 + (long)i * 2 * D + v * PV, x);
#pragma unroll
        for (int k = 0; k < PV; ++k) y[k] += x[k];
      }
      emb_store<T, PV>(out + v * PV, y, scale);
    }
    return;
  }
  const int lo = (int)((long)nv * blockIdx.y / EMB_JOIN);
  const int hi = (int)((long)nv * (blockIdx.y + 1) / EMB_JOIN);
  const int g = threadIdx.x >> 5, l = threadIdx.x & 31;
  const int share = (parts + 7) / 8;
  const int a = g * share, e = min(parts, a + share);
  for (int vb = lo; vb < hi; vb += 32) {
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
#pragma unroll
    for (int k = 0; k < PV; ++k) sums[g][l][k] = y[k];
    __syncthreads();
    if (g == 0 && v < hi) {
#pragma unroll
      for (int w = 1; w < 8; ++w)
#pragma unroll
        for (int k = 0; k < PV; ++k) y[k] += sums[w][l][k];
      emb_store<T, PV>(out + v * PV, y, scale);
    }
    __syncthreads();
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

// start: [vocab + 1], sorted: [ntok], part: [emb_chunks][2][D]
void emb_grad(int dtype, bool vec, bool idx64, const void* idx,
              const void* dy, void* dW, int* start, int2* sorted,
              float* part, int ntok, int D, int vocab, float scale,
              hipStream_t s) {
  int lg = 0;
  while ((1 << lg) < EMB_ROWS && (long)256 << lg < vocab) ++lg;
  const int R = 1 << lg;
  const unsigned nb = (unsigned)(((long)vocab + R - 1) / R);
  // 16 groups at once keep the lists of 16384 tokens from the first pass to
  // the second: 14.2 us, not 17.8 (32768 rows; 65536 tokens 48 and 51).  They
  // gain nothing for few tokens (4096: 7.3 and 6.6) and leave room for one
  // block on a compute unit (250000 rows: 25 and 23).
  const bool wide = ntok > 8192 && nb <= 256;
#define GO(I, N)                                                         \
  for (unsigned p = 0; p < nb; p += EMB_LAUNCH)                          \
  emb_sort_kernel<I, N><<<min(EMB_LAUNCH, nb - p), 1024, 0, s>>>(        \
      (const I*)idx, ntok, vocab, R, lg, (int)p, start, sorted)
  if (idx64 && wide)
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
    for (int c0 = 0; c0 < nchunk; c0 += most) {                              \
      const int nc = min(most, nchunk - c0);                                 \
      unsigned sb = (unsigned)(((long)nc * ns + 3) / 4);                     \
      unsigned zb = (unsigned)(vocab < 8192 ? (vocab + 3) / 4 : 2048);       \
      if (c0 > 0) zb = 0;                                                    \
      emb_reduce_kernel<T, V><<<sb + zb, 256, 0, s>>>(                       \
          sorted, start, (const T*)dy, (T*)dW, part, vocab, D, scale, c0,    \
          nc, ns, (int)sb);                                                  \
    }                                                                        \
    constexpr int PV = (V) == 1 ? 1 : 4;                                     \
    for (int c0 = 0; c0 < nchunk - 1; c0 += EMB_LAUNCH)                      \
      emb_join_kernel<T, PV>                                                 \
          <<<dim3(min((int)EMB_LAUNCH, nchunk - 1 - c0), EMB_JOIN), 256, 0,  \
             s>>>(sorted, start, part, (T*)dW, vocab, D, scale, c0);         \
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
