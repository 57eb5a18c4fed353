// The global norm of many gradient tensors, their clipping by it, and the AdamW step of a flat
// parameter buffer under such a clip, for gfx950.
//
//   n = sqrt(sum_k sum_i g_ki^2)  (or max |g_ki|),  c = min(1, max_norm / (n + 1e-6)),  g <- c g
//
// What bounds them: memory (clip: one read, one read + write of every gradient; step: 4 + 28 bytes
// a parameter).  The tensors are cut into chunks, one block each.  The table of tensors travels in
// launch arguments, so a call needs no copy to the device and can be captured: one that fits the
// arguments is read there; a longer one is laid out in the workspace by small launches first, which
// costs less than a norm and a scaling launch for each piece of the list (900 tensors, in chunks of
// 16 K elements: 265 us against 327).  Squares are summed in 64 bits: no gradient of a finite norm overflows or vanishes, and the
// order is fixed (no atomics).  Up to 1024 chunks the launch that scales folds their partials itself,
// in every block alike, and a clip is two launches (24 tensors of 0.5 M together: 3.6 + 4.3 us);
// beyond, one block folds them once (150 M in bf16 into fp32: norm 87 us, 3.5 TB/s, table launches 27,
// scaling 152 us, 5.9 TB/s; in place: scaling 90 us; the norm alone, over and over, 54 us, as its 300 MB
// then come from the last-level cache in part).

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "../../include/ganamd.h"

namespace {

constexpr int kNT = 256;
constexpr long kChunkMin = 4096, kChunkMax = 8192;
constexpr int kFoldMax = 1024;      // partials that every scaling block folds by itself
constexpr int kTable = 160;         // tensors of a launch (the arguments stay under 4 KB)
constexpr int kStepVec = 4;         // vectors of each buffer a thread of the step takes
constexpr int kStepBlocks = 1024;   // partials of the flat buffer's norm

struct Entry {
  uint64_t in, out;     // address | type << 60
  uint32_t first, tail; // first chunk of this launch's numbering; elements of the last chunk
};
struct Table {
  Entry e[kTable];
  int n, chunk;         // tensors; elements per chunk
  uint32_t chunks;      // of this launch
  uint32_t base, index; // chunks and tensors of the launches before it
};
// The same laid out in the workspace: a chunk's tensor, and the tensors (their chunks numbered through).
struct Listed {
  const Entry* e;
  const uint32_t* owner;
  int n, chunk;
  uint32_t chunks;
};

__device__ __forceinline__ float bf(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ float hf(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }

template <int DT>
struct Elem;
template <> struct Elem<GANAMD_F32> { typedef uint32_t S; static constexpr int V = 4; };
template <> struct Elem<GANAMD_BF16> { typedef uint16_t S; static constexpr int V = 8; };
template <> struct Elem<GANAMD_F16> { typedef uint16_t S; static constexpr int V = 8; };

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int ALIGN> struct W16;
template <> struct W16<4> { typedef u32x4 type __attribute__((aligned(4))); };
template <> struct W16<2> { typedef u32x4 type __attribute__((aligned(2))); };

template <int DT>
__device__ __forceinline__ float conv(uint32_t s) {
  return DT == GANAMD_F32 ? __uint_as_float(s) : DT == GANAMD_BF16 ? bf(s) : hf(s);
}
template <int DT>
__device__ __forceinline__ float lane(const u32x4& w, int j) {
  return DT == GANAMD_F32 ? __uint_as_float(w[j & 3]) : conv<DT>((w[(j >> 1) & 3] >> (16 * (j & 1))) & 0xffffu);
}
template <int DT>
__device__ __forceinline__ uint32_t pack1(float f) {
  if (DT == GANAMD_F32) return __float_as_uint(f);
  if (DT == GANAMD_BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// running sum of squares (KIND 0) or largest magnitude (KIND 1, as bits: a NaN is the largest)
template <int KIND>
struct Acc {
  double s = 0;
  uint32_t m = 0;
  __device__ __forceinline__ void add(float f) {
    if (KIND == 0) {
      const double d = (double)f;
      s = fma(d, d, s);
    } else {
      m = max(m, __float_as_uint(f) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void join(double o) {      // o: another partial's value()
    if (KIND == 0)
      s += o;
    else
      m = max(m, __float_as_uint((float)o) & 0x7fffffffu);
  }
  __device__ __forceinline__ double value() const { return KIND == 0 ? s : (double)__uint_as_float(m); }
};

// over a block of NT threads; the result in every thread
template <int KIND, int NT>
__device__ __forceinline__ double block_join(Acc<KIND> a, double* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double x = __shfl_xor(a.value(), o, 64);
    a.join(x);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a.value();
  __syncthreads();
  Acc<KIND> t;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t.join(sh[i]);
  return t.value();
}

template <int KIND, int DT>
__device__ __forceinline__ void norm_chunk(const void* in, long lo, long n, Acc<KIND>& acc) {
  typedef typename Elem<DT>::S S;
  typedef typename W16<sizeof(S)>::type W;
  constexpr int V = Elem<DT>::V, U = 4;
  const S* p = static_cast<const S*>(in) + lo;
  const long nv = n / V;
  for (long i = threadIdx.x; i < nv; i += U * kNT) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = i + u * kNT < nv ? *reinterpret_cast<const W*>(p + (i + u * kNT) * V) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) acc.add(lane<DT>(w[u], j));
  }
  for (long i = nv * V + threadIdx.x; i < n; i += kNT) acc.add(conv<DT>(p[i]));
}

// The piece of a tensor that this block's chunk is.
struct Piece {
  uint64_t in, out;
  long lo, n;
};

__device__ __forceinline__ Piece piece(const Entry& e, uint32_t end, uint32_t chunk, int size) {
  return {e.in, e.out, (long)(chunk - e.first) * size, chunk + 1 == end ? (long)e.tail : (long)size};
}
// in the arguments: the lanes count the tensors that start at or before the chunk
__device__ __forceinline__ Piece find(const Table& t, uint32_t chunk) {
  int k = 0;
  for (int i = threadIdx.x & 63; i < kTable; i += 64) {
    const bool le = i < t.n && t.e[i].first <= chunk;
    k += __popcll(__ballot(le));
  }
  k = __builtin_amdgcn_readfirstlane(k) - 1;
  return piece(t.e[k], k + 1 < t.n ? t.e[k + 1].first : t.chunks, chunk, t.chunk);
}
__device__ __forceinline__ Piece find(const Listed& t, uint32_t chunk) {
  const int k = (int)t.owner[chunk];
  return piece(t.e[k], k + 1 < t.n ? t.e[k + 1].first : t.chunks, chunk, t.chunk);
}

// Lays a launch's table out in the workspace, a block per tensor.
__global__ __launch_bounds__(kNT) void list_kernel(Table t, Entry* e, uint32_t* owner) {
  const int k = blockIdx.x;
  const uint32_t first = t.e[k].first, end = k + 1 < t.n ? t.e[k + 1].first : t.chunks;
  if (threadIdx.x == 0) {
    Entry o = t.e[k];
    o.first += t.base;
    e[t.index + k] = o;
  }
  for (uint32_t c = first + threadIdx.x; c < end; c += kNT) owner[t.base + c] = t.index + k;
}

constexpr uint64_t kAddr = (1ull << 60) - 1;

template <int KIND, class Tab>
__global__ __launch_bounds__(kNT) void norm_kernel(Tab t, double* __restrict__ part) {
  __shared__ double sh[kNT / 64];
  const uint32_t chunk = blockIdx.x;
  const Piece q = find(t, chunk);
  const void* in = reinterpret_cast<const void*>(q.in & kAddr);
  const int dt = (int)(q.in >> 60);
  Acc<KIND> acc;
  if (dt == GANAMD_F32)
    norm_chunk<KIND, GANAMD_F32>(in, q.lo, q.n, acc);
  else if (dt == GANAMD_BF16)
    norm_chunk<KIND, GANAMD_BF16>(in, q.lo, q.n, acc);
  else
    norm_chunk<KIND, GANAMD_F16>(in, q.lo, q.n, acc);
  const double v = block_join<KIND, kNT>(acc, sh);
  if (threadIdx.x == 0) part[chunk] = v;
}

template <int KIND, int NT>
__device__ __forceinline__ double fold(const double* __restrict__ part, long n, double* sh) {
  Acc<KIND> acc;
#pragma unroll 4
  for (long i = threadIdx.x; i < n; i += NT) acc.join(part[i]);
  const double v = block_join<KIND, NT>(acc, sh);
  return KIND == 0 ? sqrt(v) : v;
}

// n partials -> the norm, in 64 bits too for the scaling launches (`keep`)
template <int KIND>
__global__ __launch_bounds__(1024) void norm_fold_kernel(double* part, long n, float* norm, double* keep) {
  __shared__ double sh[16];
  const double v = fold<KIND, 1024>(part, n, sh);
  if (threadIdx.x == 0) {
    *norm = (float)v;
    if (keep) *keep = v;
  }
}

__device__ __forceinline__ float clip_factor(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  return c >= 1.0 ? 1.f : (float)c;           // a NaN stays
}

template <int DI, int DO>
__device__ __forceinline__ void scale_chunk(const void* in, void* out, long lo, long n, float c) {
  typedef typename Elem<DI>::S SI;
  typedef typename Elem<DO>::S SO;
  typedef typename W16<sizeof(SI)>::type WI;
  typedef typename W16<sizeof(SO)>::type WO;
  constexpr int V = Elem<DI>::V, U = 4;
  const SI* p = static_cast<const SI*>(in) + lo;
  SO* q = static_cast<SO*>(out) + lo;
  const long nv = n / V;
  for (long i = threadIdx.x; i < nv; i += U * kNT) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kNT < nv) w[u] = *reinterpret_cast<const WI*>(p + (i + u * kNT) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kNT < nv) {
        SO* o = q + (i + u * kNT) * V;
        constexpr int WORDS = V * (int)sizeof(SO) / 4;
        uint32_t r[WORDS];
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
          if (DO == GANAMD_F32)
            r[j] = pack1<DO>(lane<DI>(w[u], j) * c);
          else
            r[j] = pack1<DO>(lane<DI>(w[u], 2 * j) * c) | pack1<DO>(lane<DI>(w[u], 2 * j + 1) * c) << 16;
        }
#pragma unroll
        for (int j = 0; j < WORDS; j += 4)
          *reinterpret_cast<WO*>(reinterpret_cast<uint32_t*>(o) + j) = u32x4{r[j], r[j + 1], r[j + 2], r[j + 3]};
      }
    }
  }
  for (long i = nv * V + threadIdx.x; i < n; i += kNT) q[i] = (SO)pack1<DO>(conv<DI>(p[i]) * c);
}

// n > 0: folds the partials itself; n == 0: part[0] is the norm.  The first block says it.
template <int KIND, class Tab>
__global__ __launch_bounds__(kNT) void scale_kernel(Tab t, const double* __restrict__ part, int n, float max_norm,
                                                    float* norm) {
  __shared__ double sh[kNT / 64];
  const uint32_t chunk = blockIdx.x;
  const Piece q = find(t, chunk);
  const double v = n > 0 ? fold<KIND, kNT>(part, n, sh) : part[0];
  if (norm && chunk == 0 && threadIdx.x == 0) *norm = (float)v;
  const float c = clip_factor(v, max_norm);
  if (c == 1.f && q.in == q.out) return;           // in place, times one
  const void* in = reinterpret_cast<const void*>(q.in & kAddr);
  void* out = reinterpret_cast<void*>(q.out & kAddr);
  const int di = (int)(q.in >> 60), dn = (int)(q.out >> 60);
  if (di == GANAMD_F32)
    scale_chunk<GANAMD_F32, GANAMD_F32>(in, out, q.lo, q.n, c);
  else if (di == GANAMD_BF16 && dn == GANAMD_BF16)
    scale_chunk<GANAMD_BF16, GANAMD_BF16>(in, out, q.lo, q.n, c);
  else if (di == GANAMD_BF16)
    scale_chunk<GANAMD_BF16, GANAMD_F32>(in, out, q.lo, q.n, c);
  else if (dn == GANAMD_F16)
    scale_chunk<GANAMD_F16, GANAMD_F16>(in, out, q.lo, q.n, c);
  else
    scale_chunk<GANAMD_F16, GANAMD_F32>(in, out, q.lo, q.n, c);
}

// ------------------------------------------------------------------ the flat buffer's step
// Partials of a flat fp32 buffer's sum of squares; block 0 also counts the step.  (362 M: 283 us, 5.1 TB/s.)
__global__ __launch_bounds__(kNT) void flat_norm_kernel(const float* __restrict__ g, long n, long per,
                                                        double* __restrict__ part, int32_t* step) {
  __shared__ double sh[kNT / 64];
  const long lo = blockIdx.x * per, len = min(per, n - lo);
  Acc<0> acc;
  norm_chunk<0, GANAMD_F32>(g, lo, len, acc);
  const double v = block_join<0, kNT>(acc, sh);
  if (threadIdx.x == 0) {
    part[blockIdx.x] = v;
    if (blockIdx.x == 0) *step += 1;
  }
}

struct AdamArgs {
  double lr, beta1, beta2, eps, wd;
  float max_norm;
};
struct AdamConst {
  float c, size, root, decay, w, b2, omb2, eps;
};

__device__ __forceinline__ void adamw_one(const AdamConst& k, float gi, float& p, float& m, float& v) {
  gi *= k.c;
  float pi = p * k.decay;
  const float mi = k.w < 0.5f ? m + k.w * (gi - m) : gi - (gi - m) * (1.f - k.w);
  const float vi = v * k.b2 + k.omb2 * gi * gi;
  p = pi + (-k.size) * (mi / (sqrtf(vi) / k.root + k.eps));
  m = mi;
  v = vi;
}

// A block takes kStepVec vectors a thread, one piece of each buffer: pieces go in launch order, so
// what is in flight stays close together in memory (362 M parameters: 2.16 ms, 5.4 TB/s; blocks that
// stride through the whole buffers: 2.58 ms; one vector a thread: 2.22).  Every block folds the
// partials of the norm itself: a kernel of its own for that measured the same and is a launch more.
__global__ __launch_bounds__(kNT) void adamw_clip_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                         float* __restrict__ m, float* __restrict__ v, long n,
                                                         const double* __restrict__ part, int parts,
                                                         const int32_t* __restrict__ step, AdamArgs a, float* norm) {
  __shared__ double sh[kNT / 64];
  __shared__ AdamConst ks;
  const double nv = fold<0, kNT>(part, parts, sh);
  if (threadIdx.x == 0) {
    const double t = (double)*step;
    ks.c = clip_factor(nv, a.max_norm);
    ks.size = (float)(a.lr / (1.0 - pow(a.beta1, t)));
    ks.root = (float)sqrt(1.0 - pow(a.beta2, t));
    ks.decay = (float)(1.0 - a.lr * a.wd);
    ks.w = (float)(1.0 - a.beta1);
    ks.b2 = (float)a.beta2;
    ks.omb2 = (float)(1.0 - a.beta2);    // (of the 64-bit beta2: 1 - 0.999f is 1.3e-5 off 0.001)
    ks.eps = (float)a.eps;
    if (blockIdx.x == 0) *norm = (float)nv;
  }
  __syncthreads();
  const AdamConst k = ks;
  typedef W16<4>::type W;
  const long quads = n / 4, lo = blockIdx.x * (long)(kNT * kStepVec), hi = min(quads, lo + kNT * kStepVec);
  for (long i = lo + threadIdx.x; i < hi; i += kNT) {
    const u32x4 gw = *reinterpret_cast<const W*>(g + 4 * i);
    u32x4 pw = *reinterpret_cast<const W*>(p + 4 * i), mw = *reinterpret_cast<const W*>(m + 4 * i),
          vw = *reinterpret_cast<const W*>(v + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float pj = __uint_as_float(pw[j]), mj = __uint_as_float(mw[j]), vj = __uint_as_float(vw[j]);
      adamw_one(k, __uint_as_float(gw[j]), pj, mj, vj);
      pw[j] = __float_as_uint(pj);
      mw[j] = __float_as_uint(mj);
      vw[j] = __float_as_uint(vj);
    }
    *reinterpret_cast<W*>(p + 4 * i) = pw;
    *reinterpret_cast<W*>(m + 4 * i) = mw;
    *reinterpret_cast<W*>(v + 4 * i) = vw;
  }
  if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
    const long i = quads * 4 + threadIdx.x;
    adamw_one(k, g[i], p[i], m[i], v[i]);
  }
}

// ------------------------------------------------------------------ host
inline int ok(hipError_t e) { return e == hipSuccess ? GANAMD_OK : GANAMD_ELAUNCH; }
inline long esize(int dt) { return dt == GANAMD_F32 ? 4 : 2; }
inline bool is_type(int dt) { return dt >= GANAMD_F32 && dt <= GANAMD_F16; }

// How a list is cut: elements per chunk (4 K while that makes at most 2048 of a list without its tails, 8 K
// beyond: 900 tensors of 150 M, 18,900 chunks, took 256 us with 8 K, 265 with 16 K, 307 with 64 K) and
// where things lie.
struct Plan {
  long chunk, chunks;
  int tensors;                        // with elements
  size_t entries, owner, total;       // behind the partials and the folded norm; total bytes
};

bool plan(const ganamd_tensor* l, int n, Plan& p) {
  if (n < 0 || (n && !l)) return false;
  long total = 0;
  p.tensors = 0;
  for (int i = 0; i < n; ++i) {
    if (l[i].n < 0 || l[i].n > (1L << 40) || !is_type(l[i].dtype) || (l[i].n && !l[i].p)) return false;
    total += l[i].n;
    p.tensors += l[i].n > 0;
  }
  p.chunk = kChunkMin;
  while (p.chunk < kChunkMax && total / p.chunk > 2048) p.chunk *= 2;
  p.chunks = 0;
  for (int i = 0; i < n; ++i) p.chunks += (l[i].n + p.chunk - 1) / p.chunk;
  if (p.chunks * kNT >= (1L << 32)) return false;      // threads of a launch
  p.entries = sizeof(double) * ((size_t)p.chunks + 1);
  p.owner = p.entries + (p.tensors > kTable ? sizeof(Entry) * (size_t)p.tensors : 0);
  p.total = p.owner + (p.tensors > kTable ? sizeof(uint32_t) * (size_t)p.chunks : 0);
  return true;
}

struct Range {
  uint64_t lo, hi;
  bool out;
};

// Whether any output shares memory with another output or with another tensor's input (blocks of
// one launch would race).  0: no, 1: yes, -1: no memory to tell.
int overlap(const ganamd_tensor* l, int n) {
  if (n == 0) return 0;
  Range* r = static_cast<Range*>(malloc(sizeof(Range) * 2 * (size_t)n));
  if (!r) return -1;
  size_t k = 0;
  for (int i = 0; i < n; ++i) {
    if (!l[i].n) continue;
    const uint64_t a = reinterpret_cast<uint64_t>(l[i].p), b = reinterpret_cast<uint64_t>(l[i].out);
    r[k++] = {b, b + l[i].n * esize(l[i].out_dtype), true};
    if (a != b || l[i].dtype != l[i].out_dtype) r[k++] = {a, a + l[i].n * esize(l[i].dtype), false};
  }
  const auto less = [](const Range& x, const Range& y) { return x.lo < y.lo; };
  std::sort(r, r + k, less);
  uint64_t out_hi = 0, any_hi = 0;
  int bad = 0;
  for (size_t i = 0; i < k && !bad; ++i) {
    bad = r[i].lo < (r[i].out ? any_hi : out_hi);
    any_hi = std::max(any_hi, r[i].hi);
    if (r[i].out) out_hi = std::max(out_hi, r[i].hi);
  }
  free(r);
  return bad;
}

// Calls f(table) for the pieces of a list that fit a launch; tensors without elements take no place.
template <class F>
int for_tables(const ganamd_tensor* l, int n, long chunk, F f) {
  Table t;
  t.n = 0;
  t.chunk = (int)chunk;
  t.chunks = t.base = t.index = 0;
  for (int i = 0; i <= n; ++i) {
    if (i == n || t.n == kTable) {
      if (t.n) {
        f(t);
        if (hipGetLastError() != hipSuccess) return GANAMD_ELAUNCH;
      }
      t.base += t.chunks;
      t.index += t.n;
      t.n = 0;
      t.chunks = 0;
      if (i == n) break;
    }
    if (!l[i].n) continue;
    Entry& e = t.e[t.n++];
    e.in = reinterpret_cast<uint64_t>(l[i].p) | (uint64_t)l[i].dtype << 60;
    e.out = reinterpret_cast<uint64_t>(l[i].out) | (uint64_t)l[i].out_dtype << 60;
    e.first = t.chunks;
    const long c = (l[i].n + chunk - 1) / chunk;
    e.tail = (uint32_t)(l[i].n - (c - 1) * chunk);
    t.chunks += (uint32_t)c;
  }
  return GANAMD_OK;
}

// f(table) once for the whole list: of the arguments' kind, or of the workspace's, laid out first.
template <class F>
int for_list(const ganamd_tensor* l, int n, const Plan& p, char* ws, bool lay, hipStream_t st, F f) {
  if (p.tensors <= kTable) return for_tables(l, n, p.chunk, f);
  Entry* e = reinterpret_cast<Entry*>(ws + p.entries);
  uint32_t* owner = reinterpret_cast<uint32_t*>(ws + p.owner);
  if (lay) {
    const int rc = for_tables(l, n, p.chunk, [&](const Table& t) {
      hipLaunchKernelGGL(list_kernel, dim3(t.n), dim3(kNT), 0, st, t, e, owner);
    });
    if (rc != GANAMD_OK) return rc;
  }
  f(Listed{e, owner, p.tensors, (int)p.chunk, (uint32_t)p.chunks});
  return ok(hipGetLastError());
}

template <int KIND>
int norm_launches(const ganamd_tensor* l, int n, const Plan& p, char* ws, hipStream_t st) {
  return for_list(l, n, p, ws, true, st, [&](const auto& t) {
    hipLaunchKernelGGL((norm_kernel<KIND, std::decay_t<decltype(t)>>), dim3(t.chunks), dim3(kNT), 0, st, t,
                       reinterpret_cast<double*>(ws));
  });
}

template <int KIND>
int fold_launch(const Plan& p, float* norm, char* ws, hipStream_t st) {
  double* part = reinterpret_cast<double*>(ws);
  hipLaunchKernelGGL(norm_fold_kernel<KIND>, dim3(1), dim3(1024), 0, st, part, p.chunks, norm, part + p.chunks);
  return ok(hipGetLastError());
}

template <int KIND>
int clip(const ganamd_tensor* l, int n, const Plan& p, float max_norm, float* norm, char* ws, hipStream_t st) {
  int rc = norm_launches<KIND>(l, n, p, ws, st);
  const bool alone = p.chunks == 0 || p.chunks > kFoldMax;
  if (rc == GANAMD_OK && alone) rc = fold_launch<KIND>(p, norm, ws, st);
  if (rc != GANAMD_OK) return rc;
  const double* part = reinterpret_cast<const double*>(ws);
  return for_list(l, n, p, ws, false, st, [&](const auto& t) {
    hipLaunchKernelGGL((scale_kernel<KIND, std::decay_t<decltype(t)>>), dim3(t.chunks), dim3(kNT), 0, st, t,
                       alone ? part + p.chunks : part, alone ? 0 : (int)p.chunks, max_norm, alone ? nullptr : norm);
  });
}

}  // namespace

extern "C" {

size_t ganamd_grad_norm_workspace(const ganamd_tensor* list, int n) {
  Plan p;
  return plan(list, n, p) ? p.total : 0;
}

int ganamd_grad_norm(const ganamd_tensor* list, int n, int kind, float* norm, void* workspace, size_t workspace_bytes,
                     hipStream_t st) {
  Plan p;
  if (!plan(list, n, p) || !norm || !workspace || workspace_bytes < p.total ||
      (kind != GANAMD_NORM_L2 && kind != GANAMD_NORM_MAX))
    return GANAMD_EINVAL;
  char* ws = static_cast<char*>(workspace);
  const int rc = kind == GANAMD_NORM_L2 ? norm_launches<0>(list, n, p, ws, st) : norm_launches<1>(list, n, p, ws, st);
  if (rc != GANAMD_OK) return rc;
  return kind == GANAMD_NORM_L2 ? fold_launch<0>(p, norm, ws, st) : fold_launch<1>(p, norm, ws, st);
}

int ganamd_grad_clip(const ganamd_tensor* list, int n, int kind, float max_norm, float* norm, void* workspace,
                     size_t workspace_bytes, hipStream_t st) {
  Plan p;
  if (!plan(list, n, p) || !norm || !workspace || workspace_bytes < p.total ||
      (kind != GANAMD_NORM_L2 && kind != GANAMD_NORM_MAX) || !(max_norm >= 0.f))
    return GANAMD_EINVAL;
  for (int i = 0; i < n; ++i)
    if ((list[i].n && !list[i].out) || (list[i].out_dtype != list[i].dtype && list[i].out_dtype != GANAMD_F32))
      return GANAMD_EINVAL;
  if (overlap(list, n) != 0) return GANAMD_EINVAL;
  char* ws = static_cast<char*>(workspace);
  return kind == GANAMD_NORM_L2 ? clip<0>(list, n, p, max_norm, norm, ws, st) : clip<1>(list, n, p, max_norm, norm, ws, st);
}

size_t ganamd_adamw_clip_workspace(void) { return sizeof(double) * kStepBlocks; }

int ganamd_adamw_clip(float* p, const float* g, float* m, float* v, long n, int32_t* step, double lr, double beta1,
                      double beta2, double eps, double weight_decay, float max_norm, float* norm, void* workspace,
                      size_t workspace_bytes, hipStream_t st) {
  const long blocks = std::max<long>(1, (n / 4 + kNT * kStepVec - 1) / (kNT * kStepVec));
  if (!p || !g || !m || !v || !step || !norm || n <= 0 || blocks * kNT >= (1L << 32) || !(max_norm >= 0.f) || !workspace ||
      workspace_bytes < ganamd_adamw_clip_workspace())
    return GANAMD_EINVAL;
  double* part = static_cast<double*>(workspace);
  const long unit = 16L * kNT;                        // whole trips of norm_chunk
  const long per = std::max(unit, ((n + kStepBlocks - 1) / kStepBlocks + unit - 1) / unit * unit);
  const int parts = (int)((n + per - 1) / per);
  hipLaunchKernelGGL(flat_norm_kernel, dim3(parts), dim3(kNT), 0, st, g, n, per, part, step);
  hipLaunchKernelGGL(adamw_clip_kernel, dim3((unsigned)blocks), dim3(kNT), 0, st, p, g, m, v, n, part, parts, step,
                     AdamArgs{lr, beta1, beta2, eps, weight_decay, max_norm}, norm);
  return ok(hipGetLastError());
}

}  // extern "C"
