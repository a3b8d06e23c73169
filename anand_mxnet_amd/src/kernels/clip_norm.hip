// The norm over many tensors, and their clipping by it.
//
//   norm = sqrt(sum over all tensors of x^2)
//   y = x * min(1, max_norm / (norm + 1e-8))
//
// Bound by memory: every value is read twice and written once (159 arrays of
// a bottleneck network, 102 MB: 18 us at 5.5 TB/s and 34 at 6.0, what pass 2
// reads partly from caches; 370 MB of bf16 195 us).  Pass 1
// leaves one sum a block; in pass 2 every block adds those sums, in the same
// order, so the factor never visits the host and the result is the same in
// every run.  Pass 2 walks backwards: what pass 1 read last is still in the
// caches.  A factor that is not below one (a NaN norm too) leaves the values
// as they are.  Squares are summed in 64 bits: no gradient is too large or
// too small for them, and the rate of the vector unit is far above what
// memory delivers.
//
// The tensors' addresses travel in the kernel arguments, CLIP_MAX to a
// launch, so a captured graph holds them and no table is copied.
#include "common.h"

namespace mxa {

constexpr int CLIP_MAX = 164;       // entries: 24 bytes each, 4 KB in all
constexpr int CLIP_BLOCKS = 1024;   // partial sums of a launch
constexpr long CLIP_LONG = 1l << 31;  // elements of an entry at most

struct ClipList {
  const void* src[CLIP_MAX];
  void* dst[CLIP_MAX];
  unsigned n[CLIP_MAX];       // elements
  unsigned chunk0[CLIP_MAX];  // first chunk; the type in the top 4 bits
  unsigned nchunks;
  int ntens;
  int chunk;  // bytes a block takes at a time
};

constexpr unsigned CLIP_ID = 0x0fffffff;

DEVINL float clip_f(float x) { return x; }
DEVINL float clip_f(bf16 x) { return (float)x; }
DEVINL float clip_f(_Float16 x) { return (float)x; }

DEVINL int clip_find(const ClipList& l, unsigned c) {
  int lo = 0, hi = l.ntens - 1;
  while (lo < hi) {
    int mid = (lo + hi + 1) >> 1;
    if ((l.chunk0[mid] & CLIP_ID) <= c)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Elements of [a, e) before the first 16-byte boundary.
template <typename T>
DEVINL long clip_head(const T* p, long len) {
  long h = ((16 - ((size_t)p & 15)) & 15) / sizeof(T);
  return h < len ? h : len;
}

template <typename T>
DEVINL double clip_sumsq(const T* p, long len) {
  constexpr int V = 16 / sizeof(T);
  typedef T vt __attribute__((ext_vector_type(V)));
  double s = 0;
  auto one = [&](T x) {
    double d = (double)clip_f(x);
    s = fma(d, d, s);
  };
  const long h = clip_head(p, len), nv = (len - h) / V;
  const vt* q = (const vt*)(p + h);
#pragma unroll 4
  for (long i = threadIdx.x; i < nv; i += 256) {
    vt v = q[i];
#pragma unroll
    for (int k = 0; k < V; ++k) one(v[k]);
  }
  const long rest = len - nv * V;  // head and tail, one by one
  for (long i = threadIdx.x; i < rest; i += 256)
    one(p[i < h ? i : i + nv * V]);
  return s;
}

template <typename T>
DEVINL void clip_scale(const T* p, T* y, long len, float f) {
  constexpr int V = 16 / sizeof(T);
  typedef T vt __attribute__((ext_vector_type(V)));
  const bool keep = !(f < 1.f);
  auto one = [&](T x) { return keep ? x : (T)(clip_f(x) * f); };
  // both sides must reach a 16-byte boundary together
  const bool vec = (((size_t)p ^ (size_t)y) & 15) == 0;
  const long h = clip_head(p, len), nv = vec ? (len - h) / V : 0;
  const vt* q = (const vt*)(p + h);
  vt* z = (vt*)(y + h);
#pragma unroll 4
  for (long i = threadIdx.x; i < nv; i += 256) {
    vt v = q[i];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = one(v[k]);
    __builtin_nontemporal_store(v, &z[i]);
  }
  const long rest = len - nv * V;
  for (long i = threadIdx.x; i < rest; i += 256) {
    const long j = i < h || !vec ? i : i + nv * V;
    y[j] = one(p[j]);
  }
}

// All threads get the sum.
DEVINL double clip_block_sum(double s) {
  __shared__ double part[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
  return s;
}

__global__ __launch_bounds__(256) void clip_sumsq_kernel(
    ClipList l, double* __restrict__ sums) {
  double s = 0;
  for (unsigned c = blockIdx.x; c < l.nchunks; c += gridDim.x) {
    const int i = clip_find(l, c);
    const int dt = (int)(l.chunk0[i] >> 28);
    const long ce = l.chunk >> (dt == 2 ? 2 : 1);
    const long a = (long)(c - (l.chunk0[i] & CLIP_ID)) * ce;
    const long len = min(ce, (long)l.n[i] - a);
    if (dt == 0)
      s += clip_sumsq((const bf16*)l.src[i] + a, len);
    else if (dt == 1)
      s += clip_sumsq((const _Float16*)l.src[i] + a, len);
    else
      s += clip_sumsq((const float*)l.src[i] + a, len);
  }
  s = clip_block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void clip_scale_kernel(
    ClipList l, const double* __restrict__ sums, int nsum, double max_norm,
    float* __restrict__ norm_out) {
  double s = 0;
  for (int i = threadIdx.x; i < nsum; i += 256) s += sums[i];
  const double norm = sqrt(clip_block_sum(s));
  const float f = (float)(max_norm / (norm + 1e-8));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  for (unsigned b = blockIdx.x; b < l.nchunks; b += gridDim.x) {
    const unsigned c = l.nchunks - 1 - b;
    const int i = clip_find(l, c);
    if (!(f < 1.f) && l.src[i] == l.dst[i]) continue;
    const int dt = (int)(l.chunk0[i] >> 28);
    const long ce = l.chunk >> (dt == 2 ? 2 : 1);
    const long a = (long)(c - (l.chunk0[i] & CLIP_ID)) * ce;
    const long len = min(ce, (long)l.n[i] - a);
    if (dt == 0)
      clip_scale((const bf16*)l.src[i] + a, (bf16*)l.dst[i] + a, len, f);
    else if (dt == 1)
      clip_scale((const _Float16*)l.src[i] + a, (_Float16*)l.dst[i] + a, len,
                 f);
    else
      clip_scale((const float*)l.src[i] + a, (float*)l.dst[i] + a, len, f);
  }
}

// Entries of a tensor of n elements, doubles of workspace for n entries.
long clip_entries(long n) { return (n + CLIP_LONG - 1) / CLIP_LONG; }
long clip_ws(long n) { return (n + CLIP_MAX - 1) / CLIP_MAX * CLIP_BLOCKS; }

// dtype: 0 bf16, 1 fp16, 2 fp32; every numel is positive, at most CLIP_LONG
void clip_norm(const void* const* src, void* const* dst, const long* numel,
               const int* dtype, long ntens, double max_norm, double* ws,
               float* norm, hipStream_t s) {
  long bytes = 0;
  for (long i = 0; i < ntens; ++i) bytes += numel[i] * (dtype[i] == 2 ? 4 : 2);
  // finding a chunk's tensor takes about as long as reading 16 KB; where
  // every block has many chunks, larger ones
  const int chunk = bytes > 16384l * 4 * CLIP_BLOCKS ? 65536 : 16384;
  const long groups = (ntens + CLIP_MAX - 1) / CLIP_MAX;
  long nsum = 0;
  for (long step = 0; step < 2 * groups; ++step) {
    // the sums forwards, the scaling backwards
    const bool scale = step >= groups;
    const long grp = scale ? 2 * groups - 1 - step : step;
    const long t0 = grp * CLIP_MAX;
    ClipList l;
    l.ntens = (int)(ntens - t0 < CLIP_MAX ? ntens - t0 : CLIP_MAX);
    l.chunk = chunk;
    unsigned chunks = 0;
    for (int i = 0; i < l.ntens; ++i) {
      const int dt = dtype[t0 + i];
      const long ce = chunk / (dt == 2 ? 4 : 2);
      l.src[i] = src[t0 + i];
      l.dst[i] = dst[t0 + i];
      l.n[i] = (unsigned)numel[t0 + i];
      l.chunk0[i] = chunks | (unsigned)dt << 28;
      chunks += (unsigned)((numel[t0 + i] + ce - 1) / ce);
    }
    l.nchunks = chunks;
    const unsigned nb = chunks < CLIP_BLOCKS ? chunks : CLIP_BLOCKS;
    if (!scale) {
      clip_sumsq_kernel<<<nb, 256, 0, s>>>(l, ws + nsum);
      nsum += nb;
    } else {
      clip_scale_kernel<<<nb, 256, 0, s>>>(l, ws, (int)nsum, max_norm,
                                           grp == 0 ? norm : nullptr);
    }
  }
}

}  // namespace mxa
