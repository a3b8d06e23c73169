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
// indices twice.  The first time it counts its own, by row and by wave (a
// wave has a contiguous sixteenth of the tokens), and those of lower rows,
// which tells it where its part of the order begins without a word from
// another block.  The second time it places them; lanes of a wave that hold
// the same row are ranked by their lane, so the order is stable.
// Reading N indices in every block is cheap beside the gradients themselves
// while there are a few hundred blocks; they come from L2.
// ---------------------------------------------------------------------------
constexpr int EMB_WAVES = 16;

template <typename I>
__global__ __launch_bounds__(1024) void emb_sort_kernel(
    const I* __restrict__ idx, int ntok, int vocab, int R, int rlog2,
    int* __restrict__ start, int2* __restrict__ sorted) {
  extern __shared__ int cnt[];  // [R][16]
  __shared__ int below[EMB_WAVES], tot[EMB_WAVES];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = blockIdx.x * R;
  const int r1 = min(r0 + R, vocab);
  for (int i = threadIdx.x; i < R * EMB_WAVES; i += 1024) cnt[i] = 0;
  __syncthreads();

  const int seg = ((ntok + EMB_WAVES * 64 - 1) / (EMB_WAVES * 64)) * 64;
  const int t0 = min(ntok, wave * seg), t1 = min(ntok, t0 + seg);
  // a row outside the table counts as behind all rows
  auto row_of = [&](int t) -> int {
    long r = (long)idx[t];
    return r < 0 || r >= vocab ? 0x7fffffff : (int)r;
  };
  int low = 0;
  for (int t = t0 + lane; t < t1; t += 64) {
    int r = row_of(t);
    low += r < r0;
    if (r >= r0 && r < r1) atomicAdd(&cnt[(r - r0) * EMB_WAVES + wave], 1);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) low += __shfl_xor(low, o, 64);
  if (lane == 0) below[wave] = low;
  __syncthreads();

  // exclusive sums over (row, wave); a thread takes a run of the counters
  int first = 0;
  for (int w = 0; w < EMB_WAVES; ++w) first += below[w];
  const int n = R * EMB_WAVES, per = (n + 1023) / 1024;
  const int a = min(n, (int)threadIdx.x * per), e = min(n, a + per);
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
    if (i % EMB_WAVES == 0 && r0 + i / EMB_WAVES < r1)
      start[r0 + i / EMB_WAVES] = run;
    run += c;
  }
  if (r1 == vocab && threadIdx.x == 1023) start[vocab] = run;
  __syncthreads();

  for (int tb = t0; tb < t1; tb += 64) {
    const int t = tb + lane;
    int r = t < t1 ? row_of(t) : 0x7fffffff;
    const bool mine = r >= r0 && r < r1;
    u64 left = __ballot(mine);
    if (left == 0) continue;
    const int lr = mine ? r - r0 : 0;
    u64 same = left;  // lanes with this lane's row
    if (__popcll(left) > 4) {
      for (int bit = 0; bit < rlog2; ++bit) {
        u64 bal = __ballot((lr >> bit) & 1);
        same &= ((lr >> bit) & 1) ? bal : ~bal;
      }
    } else {
      u64 rest = left;
      while (rest) {
        int lead = __builtin_ctzll(rest);
        u64 eq = __ballot(mine && lr == __builtin_amdgcn_readlane(lr, lead));
        if (mine && (eq >> lane & 1)) same = eq;
        rest &= ~eq;
      }
    }
    if (mine) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int at = lr * EMB_WAVES + wave;
      const int pos = cnt[at] + rank;
      sorted[pos] = make_int2(r, t);
      // the last lane of a row moves its counter on; the counters of a wave
      // are its own, and LDS accesses of a wave stay in order
      if (rank == __popcll(same) - 1) cnt[at] = pos + 1;
    }
  }
}

// ---------------------------------------------------------------------------
// 2. Sums.  Waves [0, nchunk * ns) take a chunk and a slice of 64 V columns;
// the rest of the grid clears rows that no token hits.
// part: [nchunk][2][D], the sums of a chunk's first row where it began in an
// earlier chunk, and of its last row where it goes on in the next.
// ---------------------------------------------------------------------------
template <typename T, int V>
__global__ __launch_bounds__(256) void emb_reduce_kernel(
    const int2* __restrict__ sorted, const int* __restrict__ start,
    const T* __restrict__ dy, T* __restrict__ dW, float* __restrict__ part,
    int vocab, int D, float scale, int nchunk, int ns, int sumblocks) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= sumblocks) {
    const int nv = D / V;
    const float z[V] = {};
    for (int r = (blockIdx.x - sumblocks) * 4 + wave; r < vocab;
         r += (gridDim.x - sumblocks) * 4) {
      if (start[r] != start[r + 1]) continue;
      for (int c = lane; c < nv; c += 64)
        emb_store<T, V>(dW + (long)r * D + c * V, z, 1.f);
    }
    return;
  }
  const int n = start[vocab];  // tokens inside the table
  const long w = (long)blockIdx.x * 4 + wave;
  const int chunk = (int)(w / ns), slice = (int)(w % ns);
  const int p0 = chunk * EMB_CHUNK, p1 = min(n, p0 + EMB_CHUNK);
  if (chunk >= nchunk || p0 >= p1) return;
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
  constexpr int U = 8;      // rows in flight
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
    float scale) {
  __shared__ float sums[8][32][PV];
  const int n = start[vocab];
  const int chunk = blockIdx.x;
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
  // about 256 blocks of rows: each reads every index, and fewer would leave
  // compute units idle; the counters of 512 rows take 32 KB of LDS
  int lg = 0;
  while (lg < 9 && (long)256 << lg < vocab) ++lg;
  const int R = 1 << lg;
  const unsigned nb = (unsigned)(((long)vocab + R - 1) / R);
  const size_t lds = (size_t)R * EMB_WAVES * sizeof(int);
  if (idx64)
    emb_sort_kernel<long><<<nb, 1024, lds, s>>>((const long*)idx, ntok,
                                                vocab, R, lg, start, sorted);
  else
    emb_sort_kernel<int><<<nb, 1024, lds, s>>>((const int*)idx, ntok, vocab,
                                               R, lg, start, sorted);
  const int nchunk = emb_chunks(ntok);
#define GO(T, V)                                                            \
  do {                                                                      \
    int ns = (D / (V) + 63) / 64;                                           \
    unsigned sb = (unsigned)(((long)nchunk * ns + 3) / 4);                  \
    unsigned zb = (unsigned)(vocab < 8192 ? (vocab + 3) / 4 : 2048);        \
    emb_reduce_kernel<T, V><<<sb + zb, 256, 0, s>>>(                        \
        sorted, start, (const T*)dy, (T*)dW, part, vocab, D, scale, nchunk, \
        ns, (int)sb);                                                       \
    constexpr int PV = (V) == 1 ? 1 : 4;                                    \
    dim3 jg(nchunk - 1, EMB_JOIN);                                          \
    if (nchunk > 1)                                                         \
      emb_join_kernel<T, PV><<<jg, 256, 0, s>>>(sorted, start, part,        \
                                                (T*)dW, vocab, D, scale);   \
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
