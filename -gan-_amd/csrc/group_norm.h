// Group norm with its activation for gfx950: forward, backward and the backward's own backward
// (the gradient penalty), over channels-last maps x[b][l][c] and over channel rows x[c][b][l].
//
// For a sample b and a group of Cg channels, N = L * Cg values, with d = x - mean:
//   xh = d * r, r = (var + eps)^-1/2, z = xh * w[c] + b[c], y = a(z)
//   backward:  g = gy a'(z), u = w g:   gx = r (u - m(u) - xh m(u xh)),
//              gw = sum g xh, gb = sum g, gslope = sum gy z [z <= 0]           (m: mean over the group)
//   double backward, v the cotangent of gx, (cw, cb, cs) those of gw, gb, gslope:
//              q = r (v - m(v) - xh m(v xh)),  h = w q + cw xh + cb
//              t = gy a''(z) h + cs gy [z <= 0],  e = t w + g cw - r (v m(u xh) + u m(v xh))
//              g_gy = a'(z) h + cs z [z <= 0]
//              g_x = r (e - m(e) - xh m(e xh)) - r xh m(u q)
//              g_w = sum g q + t xh,  g_b = sum t,  g_slope = sum gy h [z <= 0]
// Every group mean above is a combination of per-channel sums over l that need no other mean, so
// each operator is ONE reduction over its inputs (5 to 10 sums a channel) and one elementwise pass
// whose result is linear in (g, v, d, t, 1) with per-channel coefficients.
//
// Statistics are summed and kept in 64 bits: the sign of z selects the branch of a kinked
// activation, and at fp32 accuracy a handful of values per 10^7 fall on the wrong side, each an
// error of the size of the gradient.  What is summed are the differences from a pivot, the group's first
// value: |pivot - mean| is at most sqrt(N) standard deviations, so what cancels between their mean
// square and their squared mean is at most N variances, in 64 bits, wherever the mean lies (sums of x
// and x^2 put the gradient of a group of one value 3e5 repeated off by 9 %).  The test itself is one
// fp32 comparison of x with the channel's threshold (the smallest float whose z is positive), exact
// for every x.
//
// What bounds them: memory.  Two forms:
//  * resident: one block holds all of a group's (rows: a tile of whole groups') values in
//    registers between the reduction and the elementwise part: each input is read once.
//  * split: the positions of a sample are cut over blocks; per-channel partials go to the
//    workspace, a small kernel folds them, a second pass over the data writes the result.
// No atomics: results are the same on every run.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ganamd.h"

namespace gn {

enum { FWD = 0, BWD = 1, DBL = 2 };
enum { SILU = 0, KINK = 1, SLOPE = 2 };   // SLOPE: a kinked activation whose slope has a gradient

// One operator call as the kernels see it.
struct Args {
  const void *x, *gy, *v;                       // data, in T
  void *o1, *o2;                                // y | gx | g_gy, g_x
  const void *w, *b, *slope, *cw, *cb, *cs;     // per-channel parameters and cotangents (pdt); may be null
  double* stats;                                // [B][G][2]: mean, r (written by FWD)
  double* coef;                                 // [B][G][8]: group coefficients of the elementwise pass
  float* part;                                  // [B][S][K][C] partial sums (FWD: doubles [B][S][2][C])
  float* par;                                   // [2 or 3][B][C]: each sample's terms of gw, gb (, gslope)
  float cslope;                                 // constant slope where slope is null
  float eps;
  long L, B;                                    // positions, samples
  int C, G, Cg, pdt, xdt;
  long pb, pc;                                  // elements from a sample / a channel to the next
  int TX, P;                                    // threads across the channels (rows) / planes per block; positions in flight
  int CT, nct;                                  // channels per tile, tiles
  int S;                                        // chunks of a sample's positions
  int per;                                      // positions (planes: vectors) per chunk
  bool once;                                    // outputs go past the caches
};

// ------------------------------------------------------------------ types
struct bf16 { uint16_t u; };
struct f16 { _Float16 h; };

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(bf16 x) { return __uint_as_float((uint32_t)x.u << 16); }
__device__ __forceinline__ float up(f16 x) { return (float)x.h; }
template <class T>
__device__ __forceinline__ T down(float x);
template <>
__device__ __forceinline__ float down<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 down<bf16>(float x) {
  const __bf16 h = (__bf16)x;   // round to nearest even
  return bf16{__builtin_bit_cast(uint16_t, h)};
}
template <>
__device__ __forceinline__ f16 down<f16>(float x) { return f16{(_Float16)x}; }

// V elements as the 32-bit words they come in, loaded and stored whole at any element alignment
// (rows of an odd channel count start anywhere; global memory takes unaligned vectors).  They are
// unpacked where they are used: a value kept for a second use stays packed.
template <int BYTES, int ALIGN>
struct Word;
#define GN_WORD(BYTES, TYPE, ALIGN) \
  template <> struct Word<BYTES, ALIGN> { typedef TYPE type __attribute__((aligned(ALIGN))); };
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
GN_WORD(16, u32x4, 4) GN_WORD(16, u32x4, 2) GN_WORD(8, u32x2, 4) GN_WORD(8, u32x2, 2)
GN_WORD(4, uint32_t, 4) GN_WORD(4, uint32_t, 2) GN_WORD(2, uint16_t, 2)
#undef GN_WORD

template <class T, int V>
struct Vec {
  static constexpr int N = (V * (int)sizeof(T) + 3) / 4, PER = 4 / (int)sizeof(T);
  typedef typename Word<sizeof(T) * V, sizeof(T)>::type W;
  uint32_t w[N];
  __device__ __forceinline__ float get(int j) const;
  __device__ __forceinline__ void put(const float (&f)[V]);
  // elements j < n become the value of these bits
  __device__ __forceinline__ void fill_front(int n, uint32_t v) {
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (PER == 1) {
        if (i < n) w[i] = v;
      } else {
        const int k = n - 2 * i;
        w[i] = k >= 2 ? v | v << 16 : k == 1 ? (w[i] & 0xffff0000u) | v : w[i];
      }
    }
  }
  __device__ __forceinline__ void zero_front(int n) { fill_front(n, 0); }
  // the compiler may not carry anything derived from these words past here
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i]));
  }
};
template <class T> __device__ __forceinline__ float up_bits(uint32_t w, int half);
template <> __device__ __forceinline__ float up_bits<float>(uint32_t w, int) { return __uint_as_float(w); }
template <> __device__ __forceinline__ float up_bits<bf16>(uint32_t w, int half) {
  return __uint_as_float(half ? w & 0xffff0000u : w << 16);
}
template <> __device__ __forceinline__ float up_bits<f16>(uint32_t w, int half) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(half ? w >> 16 : w));
}
template <class T> __device__ __forceinline__ uint32_t bits(T x);
template <> __device__ __forceinline__ uint32_t bits<float>(float x) { return __float_as_uint(x); }
template <> __device__ __forceinline__ uint32_t bits<bf16>(bf16 x) { return x.u; }
template <> __device__ __forceinline__ uint32_t bits<f16>(f16 x) { return __builtin_bit_cast(uint16_t, x.h); }

template <class T, int V>
__device__ __forceinline__ float Vec<T, V>::get(int j) const { return up_bits<T>(w[j / PER], j % PER); }
template <class T, int V>
__device__ __forceinline__ void Vec<T, V>::put(const float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = bits(down<T>(f[i * PER]));
    if (PER == 2 && i * PER + 1 < V) w[i] |= bits(down<T>(f[i * PER + 1 < V ? i * PER + 1 : 0])) << 16;
  }
}

template <class T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  typedef typename Vec<T, V>::W W;
  const W x = *reinterpret_cast<const W*>(p);
  Vec<T, V> v;
  if constexpr (sizeof(x) < 4)
    v.w[0] = x;
  else
    __builtin_memcpy(v.w, &x, sizeof(x));
  return v;
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& v, int skip, bool once) {
  typedef typename Vec<T, V>::W W;
  if (skip == 0) {
    W x;
    if constexpr (sizeof(x) < 4)
      x = (W)v.w[0];
    else
      __builtin_memcpy(&x, v.w, sizeof(x));
    if (once) {
      asm volatile("");                 // (else the two stores become one, without the hint)
      __builtin_nontemporal_store(x, reinterpret_cast<W*>(p));
      asm volatile("");
    } else {
      *reinterpret_cast<W*>(p) = x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j >= skip) {
        const uint32_t h = v.w[j / Vec<T, V>::PER] >> (16 * (j % Vec<T, V>::PER));
        if constexpr (sizeof(T) == 4)
          reinterpret_cast<uint32_t*>(p)[j] = h;
        else
          reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)h;
      }
  }
}

__device__ __forceinline__ float loadp(const void* p, int dt, long i) {
  if (dt == GANAMD_F32) return static_cast<const float*>(p)[i];
  if (dt == GANAMD_BF16) return up(static_cast<const bf16*>(p)[i]);
  return up(static_cast<const f16*>(p)[i]);
}

// The pivot of the group that starts with channel c, in sample b: its first value.
__device__ __forceinline__ float pivot(const Args& a, long b, int c) { return loadp(a.x, a.xdt, b * a.pb + c * a.pc); }
// The same as it is stored, so that nothing waits for the load before the value is put to use.
__device__ __forceinline__ uint32_t pivot_bits(const Args& a, long b, int c) {
  const long i = b * a.pb + c * a.pc;
  return a.xdt == GANAMD_F32 ? static_cast<const uint32_t*>(a.x)[i] : static_cast<const uint16_t*>(a.x)[i];
}
__device__ __forceinline__ float of_bits(const Args& a, uint32_t v) {
  return a.xdt == GANAMD_F32 ? __uint_as_float(v) : a.xdt == GANAMD_BF16 ? up(bf16{(uint16_t)v})
       : (float)__builtin_bit_cast(_Float16, (uint16_t)v);
}

// ------------------------------------------------------------------ which elements a thread owns
// rows (channels last): V consecutive channels, every P-th position.  planes (channel rows): one
// channel, every P-th vector of V positions.  The last vector of a row / plane is moved back to end
// with it; its first `skip` elements belong to its neighbour and add nothing to the sums here.
template <bool ROWS, int V>
struct Map {
  long base, step;     // element offset of position 0, of one position
  long last;           // planes: L - V
  int ch;              // first channel of this thread
  int slot;            // ch within the tile
  int p;               // first position
  int npos;            // positions (planes: vectors) of a sample
  int skip0;
  bool active;

  __device__ __forceinline__ Map(const Args& a, long b, int tile) {
    const int c0 = tile * a.CT, wid = min(a.CT, a.C - c0);
    if (ROWS) {
      const int tx = threadIdx.x % a.TX;
      p = threadIdx.x / a.TX;
      const int cv = c0 + tx * V;
      active = tx * V < wid && p < a.P;
      ch = max(min(cv, c0 + wid - V), 0);
      skip0 = cv - ch;
      slot = ch - c0;
      base = b * a.L * a.C + ch;
      step = a.C;
      last = 0;
      npos = (int)a.L;
    } else {
      p = threadIdx.x % a.P;
      slot = threadIdx.x / a.P;
      ch = min(c0 + slot, a.C - 1);
      active = slot < wid;
      skip0 = 0;
      base = ((long)ch * a.B + b) * a.L;
      step = V;
      last = a.L - V;
      npos = (int)((a.L + V - 1) / V);
    }
  }
  __device__ __forceinline__ long at(long i, int& skip) const {
    if (ROWS) {
      skip = skip0;
      return base + i * step;
    }
    const long l = i * V, s = l < last ? l : last;
    skip = (int)(l - s);
    return base + s;
  }
};

// ------------------------------------------------------------------ per-channel constants
__device__ __forceinline__ float kink(double mean, double rw, double b, float& sg) {
  const float a = (float)rw;
  sg = a < 0.f ? -1.f : 1.f;
  if (a == 0.f) return b > 0.0 ? -INFINITY : NAN;      // z = b whatever x is
  const double x0 = a < 0.f ? b / rw - mean : mean - b / rw;
  const float t = (float)x0;
  return (double)t <= x0 ? nextafterf(t, INFINITY) : t;
}

// What the activation needs of a channel: d = x - mf; z = d * a + o (o carries the part of the
// mean below fp32); the kink's threshold tf on sg * x (sg: the sign of a), and its slope k.
// A block's first threads make them, one channel each, and all read theirs from LDS (put / get:
// field-major, `n` channels a field).
template <int MODE, int ACT>
struct Chan {
  static constexpr bool Z = MODE == FWD || ACT != KINK;       // uses z
  static constexpr bool SIGN = MODE != FWD && ACT != SILU;    // uses the exact sign of z
  static constexpr int N = 6;
  float mf, a, o, tf, sg, k;
  __device__ __forceinline__ void set(const Args& g, double mean, double r, int c) {
    const float w = g.w ? loadp(g.w, g.pdt, c) : 1.f, bb = g.b ? loadp(g.b, g.pdt, c) : 0.f;
    mf = (float)mean;
    const double rw = r * (double)w;
    a = (float)rw;
    o = (float)((double)bb + ((double)mf - mean) * rw);
    k = 1.f;
    tf = 0.f;
    sg = 1.f;
    if (ACT != SILU) k = g.slope ? loadp(g.slope, g.pdt, c) : g.cslope;
    if (SIGN) tf = kink(mean, rw, (double)bb, sg);
  }
  template <class F>
  __device__ __forceinline__ void fields(F f) {
    f(0, mf);
    f(1, a);
    if (Z) f(2, o);
    if (SIGN) {
      f(3, tf);
      f(4, sg);
    }
    if (ACT != SILU) f(5, k);
  }
  __device__ __forceinline__ void put(float* t, int n, int c) {
    fields([&](int i, float& v) { t[i * n + c] = v; });
  }
  __device__ __forceinline__ void get(const float* t, int n, int c) {
    fields([&](int i, float& v) { v = t[i * n + c]; });
  }
};

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int MODE, int ACT>
__device__ __forceinline__ float act_fwd(const Chan<MODE, ACT>& c, float x) {
  const float z = (x - c.mf) * c.a + c.o;
  if (ACT == SILU) return z * sigmoid(z);
  return z > 0.f ? z : c.k * z;
}
// g = gy a'(z); t = gy a''(z) (SILU) or gy [z <= 0] (kinked); z itself
template <int MODE, int ACT>
__device__ __forceinline__ void act_bwd(const Chan<MODE, ACT>& c, float x, float d, float gy, float& g, float& t, float& z) {
  z = d * c.a + c.o;
  if (ACT == SILU) {
    const float s = sigmoid(z), n = 1.f - s;
    g = gy * (s * (1.f + z * n));
    t = gy * (s * n * (2.f + z * (n - s)));
  } else {
    const bool pos = c.sg * x >= c.tf;
    g = pos ? gy : c.k * gy;
    t = pos ? 0.f : gy;
  }
}
template <int MODE, int ACT>
__device__ __forceinline__ float act_d1(const Chan<MODE, ACT>& c, float x, float z) {
  if (ACT == SILU) {
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
  }
  return c.sg * x >= c.tf ? 1.f : c.k;
}

// ------------------------------------------------------------------ sums over positions
// FWD sums in double (x - pivot and its square; ch.mf holds the pivot); the others in fp32 over a
// thread's own positions.
//   BWD: g, g d (, gy z [z<=0]).   DBL: v, v d, g, g d, g v, then
//   SILU: k, k d, k d^2, k v, k v d with k = gy a''; SLOPE: s, s d, s v with s = gy [z <= 0]
template <int MODE, int ACT>
struct Sums {
  static constexpr int K = MODE == FWD ? 2 : MODE == BWD ? (ACT == SLOPE ? 3 : 2)
                                                         : (ACT == SILU ? 10 : ACT == SLOPE ? 8 : 5);
};
template <int MODE>
struct AccT { typedef float type; };
template <>
struct AccT<FWD> { typedef double type; };

template <int MODE, int ACT, bool ROWS, class T, int V, int NC, int K, class A>
__device__ __forceinline__ void accumulate(A (&acc)[K][NC], const Chan<MODE, ACT> (&ch)[NC], const Vec<T, V>& x,
                                           const Vec<T, V>& gy, const Vec<T, V>& v) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = ROWS ? j : 0;
    const float xf = x.get(j);
    if constexpr (MODE == FWD) {
      const double xd = (double)xf - (double)ch[c].mf;
      acc[0][c] += xd;
      acc[1][c] = fma(xd, xd, acc[1][c]);
    } else {
      const float d = xf - ch[c].mf;
      float g, t, z;
      act_bwd(ch[c], xf, d, gy.get(j), g, t, z);
      if constexpr (MODE == BWD) {
        acc[0][c] += g;
        acc[1][c] = fmaf(g, d, acc[1][c]);
        if constexpr (ACT == SLOPE) acc[2][c] = fmaf(t, z, acc[2][c]);
      } else {
        const float vf = v.get(j);
        acc[0][c] += vf;
        acc[1][c] = fmaf(vf, d, acc[1][c]);
        acc[2][c] += g;
        acc[3][c] = fmaf(g, d, acc[3][c]);
        acc[4][c] = fmaf(g, vf, acc[4][c]);
        if constexpr (ACT != KINK) {
          const float td = t * d;
          acc[5][c] += t;
          acc[6][c] += td;
          acc[7][c] = fmaf(t, vf, acc[7][c]);
          if constexpr (ACT == SILU) {
            acc[8][c] = fmaf(td, d, acc[8][c]);
            acc[9][c] = fmaf(td, vf, acc[9][c]);
          }
        }
      }
    }
  }
}

// v of the lane that differs in bit `STEP` of its number, or of one whose value is the same once the
// smaller steps are summed (a mirrored lane): DPP moves where there is one, half a dozen cycles
// instead of an LDS permute's latency.
template <int STEP>
__device__ __forceinline__ uint32_t other(uint32_t v) {
  if constexpr (STEP == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
  else if constexpr (STEP == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  else if constexpr (STEP == 4) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true);  // row_half_mirror
  else if constexpr (STEP == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true);  // row_mirror
  else return (uint32_t)__shfl_xor((int)v, STEP, 64);
}
template <int STEP>
__device__ __forceinline__ float other(float v) { return __uint_as_float(other<STEP>(__float_as_uint(v))); }
template <int STEP>
__device__ __forceinline__ double other(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t w = (uint64_t)other<STEP>((uint32_t)(u >> 32)) << 32 | other<STEP>((uint32_t)u);
  return __builtin_bit_cast(double, w);
}
// The sum over W (a power of two, at most 64) neighbouring lanes, in each of them.
template <class A>
__device__ __forceinline__ A lanes_sum(A v, int W) {
  if (W >= 2) v += other<1>(v);
  if (W >= 4) v += other<2>(v);
  if (W >= 8) v += other<4>(v);
  if (W >= 16) v += other<8>(v);
  if (W >= 32) v += other<16>(v);
  if (W >= 64) v += other<32>(v);
  return v;
}

// Sums that a round of a row tile's fold takes through LDS at once (32 KB of scratch).
constexpr int fold_round(int K, int NC, int nt, int size) {
  const int n = 32768 / (NC * nt * size);
  return n < 1 ? 1 : n < K ? n : K;
}

// Folds acc over the block's positions into chan[k * a.CT + slot] (LDS), in one order.  `sh`: scratch
// of rows: fold_round * NC * threads values (a thread's values nt apart: no bank conflicts), planes:
// K * 16.  Every thread of the block calls it.
template <bool ROWS, int V, int K, int NC, class A>
__device__ __forceinline__ void fold(const Args& a, const Map<ROWS, V>& m, A (&acc)[K][NC], A* sh, A* chan, int c0) {
  const int tid = threadIdx.x, nt = blockDim.x;
  if constexpr (ROWS) {
    const int R = fold_round(K, NC, nt, sizeof(A)), wid = min(a.CT, a.C - c0);
    for (int k0 = 0; k0 < K; k0 += R) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k >= k0 && k < k0 + R) {
#pragma unroll
          for (int j = 0; j < NC; ++j) sh[((k - k0) * NC + j) * nt + tid] = acc[k][j];
        }
      __syncthreads();
      const int I = min(R, K - k0) * NC * a.TX, Q = max(1, min(nt / I, a.P));
      for (int i0 = 0; i0 < I; i0 += nt) {                // one trip where Q > 1
        const int i = i0 + tid % (Q > 1 ? I : nt), q = Q > 1 ? tid / I : 0;
        const int tx = i % a.TX, kj = i / a.TX;
        A s = 0;
        if (i < I && q < Q) {
          const A* p0 = sh + kj * nt + tx;
#pragma unroll 4
          for (int p = q; p < a.P; p += Q) s += p0[p * a.TX];
        }
        if (Q > 1) {
          __syncthreads();
          if (q < Q && q > 0) sh[(q - 1) * I + i] = s;
          __syncthreads();
          if (q == 0)
            for (int o = 0; o < Q - 1; ++o) s += sh[o * I + i];
        }
        const int j = kj % NC, slot = max(min(tx * V, wid - V), -c0) + j;
        if (q == 0 && i < I && tx * V < wid && slot >= tx * V) chan[(k0 + kj / NC) * a.CT + slot] = s;
      }
    }
    __syncthreads();
  } else {
    const int lanes = a.P < 64 ? a.P : 64, nw = a.P / lanes;   // P: a power of two
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const A s = lanes_sum(m.active ? acc[k][0] : (A)0, lanes);
      if (nw == 1) {
        if (m.p == 0 && m.active) chan[k * a.CT + m.slot] = s;
      } else if ((tid & 63) == 0) {
        sh[k * 16 + (tid >> 6)] = s;
      }
    }
    __syncthreads();
    if (nw > 1) {
      for (int i = tid; i < K * (nt / a.P); i += nt) {
        const int k = i / (nt / a.P), s = i % (nt / a.P);
        if (s < a.CT) {
          A t = 0;
          for (int q = 0; q < nw; ++q) t += sh[k * 16 + s * nw + q];
          chan[k * a.CT + s] = t;
        }
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ group coefficients
// A channel's terms of the group sums and of the parameter gradients, from its sums over a sample.
// First sweep (all modes): sums that need no mean.  DBL has a second sweep that needs them.
struct Group { double mean, r; float mf; double xo; };

__device__ __forceinline__ Group group_of(double mean, double r) {
  Group q;
  q.mean = mean;
  q.r = r;
  q.mf = (float)mean;
  q.xo = ((double)q.mf - mean) * r;
  return q;
}
__device__ __forceinline__ double param(const void* p, int dt, int c, double none) {
  return p ? (double)loadp(p, dt, c) : none;
}

// BWD: out[2] = w sum g, w sum g xh; terms[3] = gw, gb, gslope
// DBL: out[4] = sum v, sum v xh, w sum g, w sum g xh
template <int MODE, int ACT, class S>
__device__ __forceinline__ void sweep1(const Args& a, const Group& q, int c, S s, double* out, double* terms) {
  const double w = param(a.w, a.pdt, c, 1.0);
  if (MODE == BWD) {
    const double g0 = s(0), gx = q.r * s(1) + q.xo * g0;
    out[0] += w * g0;
    out[1] += w * gx;
    terms[0] = gx;
    terms[1] = g0;
    terms[2] = ACT == SLOPE ? s(2) : 0.0;
  } else {
    const double v0 = s(0), g0 = s(2);
    out[0] += v0;
    out[1] += q.r * s(1) + q.xo * v0;
    out[2] += w * g0;
    out[3] += w * (q.r * s(3) + q.xo * g0);
  }
}
// DBL, m[4] the group's means of sweep1: out[3] = terms of N m(e), N m(e xh), N m(u q) beyond the means
template <int ACT, class S>
__device__ __forceinline__ void sweep2(const Args& a, const Group& q, int c, S s, const double* m, double* out,
                                       double* terms) {
  const double w = param(a.w, a.pdt, c, 1.0), cw = param(a.cw, a.pdt, c, 0.0), cb = param(a.cb, a.pdt, c, 0.0);
  const double r = q.r, xo = q.xo;
  const double g0 = s(2), gx = r * s(3) + xo * g0;
  const double Q = r * (s(4) - m[0] * g0 - m[1] * gx);
  const double h1 = w * r, h2 = cw - h1 * m[1], h3 = cb - h1 * m[0];   // h = h1 v + h2 xh + h3
  double T0 = 0.0, T1 = 0.0, sl = 0.0;
  if (ACT == SILU) {
    const double k0 = s(5), kx = r * s(6) + xo * k0;
    const double kxx = r * r * s(8) + 2.0 * r * xo * s(6) + xo * xo * k0;
    const double kv = s(7), kvx = r * s(9) + xo * kv;
    T0 = h1 * kv + h2 * kx + h3 * k0;
    T1 = h1 * kvx + h2 * kxx + h3 * kx;
  } else if (ACT == SLOPE) {
    const double cs = param(a.cs, a.pdt, c, 0.0);
    const double s0 = s(5), sx = r * s(6) + xo * s0;
    T0 = cs * s0;
    T1 = cs * sx;
    sl = h1 * s(7) + h2 * sx + h3 * s0;
  }
  out[0] += w * T0 + cw * g0;
  out[1] += w * T1 + cw * gx;
  out[2] += w * Q;
  terms[0] = Q + T1;
  terms[1] = T0;
  terms[2] = sl;
}

// coef[] of a group from its sums.  BWD: {m(u), m(u xh)}; DBL: {m(v), m(v xh), m(u xh), m(e), m(e xh) + m(u q)}
__device__ __forceinline__ void dbl_coef(const Group& q, const double* m, const double* t, double invN, double* co) {
  co[0] = m[0];
  co[1] = m[1];
  co[2] = m[3];
  co[3] = -q.r * (m[0] * m[3] + m[2] * m[1]) + t[0] * invN;
  co[4] = -2.0 * q.r * m[1] * m[3] + t[1] * invN + t[2] * invN;
}

// The elementwise pass's coefficients of one channel; the first moment of a slope's gradient needs
// no z there, so a backward's SLOPE is its KINK.
template <int MODE, int ACT>
struct Lin {
  typedef Chan<MODE, MODE == BWD && ACT == SLOPE ? KINK : ACT> C;
  static constexpr int N = C::N + (MODE == FWD ? 0 : MODE == BWD ? 2 : 7);
  C ch;
  float B1, C1;                     // BWD: gx = g a + d B1 + C1
  float H2, H3, G1, V1, D1, K1, cs; // DBL: h = v a + d H2 + H3; g_x = t a + g G1 + v V1 + d D1 + K1
  __device__ __forceinline__ void set(const Args& g, double mean, double r, const double* co, int c) {
    ch.set(g, mean, r, c);
    const double w = param(g.w, g.pdt, c, 1.0), xo = ((double)ch.mf - mean) * r;
    if (MODE == BWD) {
      B1 = (float)(-r * r * co[1]);
      C1 = (float)(-r * (co[0] + xo * co[1]));
    } else if (MODE == DBL) {
      const double cw = param(g.cw, g.pdt, c, 0.0), cb = param(g.cb, g.pdt, c, 0.0);
      const double h2 = cw - w * r * co[1];
      H2 = (float)(h2 * r);
      H3 = (float)(h2 * xo + cb - w * r * co[0]);
      G1 = (float)(r * (cw - r * w * co[1]));
      V1 = (float)(-r * r * co[2]);
      D1 = (float)(-r * r * co[4]);
      K1 = (float)(-r * (co[3] + xo * co[4]));
      cs = ACT == SLOPE ? (float)param(g.cs, g.pdt, c, 0.0) : 0.f;
    }
  }
  template <class F>
  __device__ __forceinline__ void fields(F f) {
    constexpr int n = C::N;
    ch.fields(f);
    if (MODE == BWD) {
      f(n, B1);
      f(n + 1, C1);
    } else if (MODE == DBL) {
      f(n, H2);
      f(n + 1, H3);
      f(n + 2, G1);
      f(n + 3, V1);
      f(n + 4, D1);
      f(n + 5, K1);
      if (ACT == SLOPE) f(n + 6, cs);
    }
  }
  __device__ __forceinline__ void put(float* t, int n, int c) {
    fields([&](int i, float& v) { t[i * n + c] = v; });
  }
  __device__ __forceinline__ void get(const float* t, int n, int c) {
    fields([&](int i, float& v) { v = t[i * n + c]; });
  }
};

template <int MODE, int ACT, bool ROWS, class T, int V, int NC>
__device__ __forceinline__ void apply(const Lin<MODE, ACT> (&ln)[NC], const Vec<T, V>& x, const Vec<T, V>& gy,
                                      const Vec<T, V>& v, Vec<T, V>& o1, Vec<T, V>& o2) {
  float f1[V], f2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const Lin<MODE, ACT>& l = ln[ROWS ? j : 0];
    const float xf = x.get(j);
    if constexpr (MODE == FWD) {
      f1[j] = act_fwd(l.ch, xf);
    } else {
      const float d = xf - l.ch.mf;
      float g, t, z;
      act_bwd(l.ch, xf, d, gy.get(j), g, t, z);
      if constexpr (MODE == BWD) {
        f1[j] = fmaf(g, l.ch.a, fmaf(d, l.B1, l.C1));
      } else {
        const float vf = v.get(j);
        const float h = fmaf(vf, l.ch.a, fmaf(d, l.H2, l.H3));
        float gg = act_d1(l.ch, xf, z) * h, tt = 0.f;
        if (ACT == SILU) tt = t * h;
        if (ACT == SLOPE) {
          tt = l.cs * t;
          if (!(l.ch.sg * xf >= l.ch.tf)) gg = fmaf(l.cs, z, gg);
        }
        f1[j] = gg;
        f2[j] = fmaf(tt, l.ch.a, fmaf(g, l.G1, fmaf(vf, l.V1, fmaf(d, l.D1, l.K1))));
      }
    }
  }
  o1.put(f1);
  if constexpr (MODE == DBL) o2.put(f2);
}

// ------------------------------------------------------------------ shared by the kernels
// The pivots of a thread's channels (FWD's only channel constants): asked for before its data, of the
// first two groups that the channels lie in and without a branch, so that nothing waits for them
// before the data is on its way; put to use after that (narrower groups: read one by one then).
template <int ACT, bool ROWS, class T, int V, int NC>
struct Pivots {
  const T* x;
  T p0, p1;
  int g, rest;                             // the first group's first channel, channels left in it
  __device__ __forceinline__ Pivots(const Args& a, const Map<ROWS, V>& m, long b) {
    x = static_cast<const T*>(a.x) + b * a.pb;
    g = m.ch / a.Cg * a.Cg;
    rest = a.Cg - (m.ch - g);
    p0 = x[g * a.pc];
    if (NC > 1) p1 = x[min(g + a.Cg, a.C - a.Cg) * a.pc];
  }
  __device__ __forceinline__ void get(const Args& a, Chan<FWD, ACT> (&ch)[NC]) const {
#pragma unroll
    for (int j = 0; j < NC; ++j) ch[j].mf = NC == 1 || j < rest ? up(p0) : up(p1);
    if (NC > 1 && a.Cg + 1 < NC)
#pragma unroll
      for (int j = 1; j < NC; ++j) ch[j].mf = up(x[(g + (a.Cg - rest + j) / a.Cg * a.Cg) * a.pc]);
  }
};

// A tile's channel constants for the sums (BWD, DBL): made in `tab`, read by every thread.
template <int MODE, int ACT, bool ROWS, int V, int NC>
__device__ __forceinline__ void load_chan(const Args& a, const Map<ROWS, V>& m, long b, int c0, float* tab,
                                          Chan<MODE, ACT> (&ch)[NC]) {
  if constexpr (MODE != FWD) {
    const int wid = min(a.CT, a.C - c0);
    for (int c = threadIdx.x; c < wid; c += blockDim.x) {
      const double* s = a.stats + 2 * (b * a.G + (c0 + c) / a.Cg);
      Chan<MODE, ACT> q;
      q.set(a, s[0], s[1], c0 + c);
      q.put(tab, a.CT, c);
    }
    __syncthreads();
    if (m.active) {
#pragma unroll
      for (int j = 0; j < NC; ++j) ch[j].get(tab, a.CT, max(m.slot + j, 0));   // (a moved-back front is not counted)
    }
    __syncthreads();                       // tab's memory becomes the sums'
  }
}

// The same for the elementwise pass; co: the tile's first group's coefficients, 8 a group.
template <int MODE, int ACT, bool ROWS, int V, int NC>
__device__ __forceinline__ void load_lin(const Args& a, const Map<ROWS, V>& m, long b, int c0, const double* st,
                                         int st_step, const double* co, float* tab, Lin<MODE, ACT> (&ln)[NC]) {
  const int wid = min(a.CT, a.C - c0), g0 = c0 / a.Cg;
  for (int c = threadIdx.x; c < wid; c += blockDim.x) {
    const int g = (c0 + c) / a.Cg - g0;
    Lin<MODE, ACT> q;
    q.set(a, st[(long)g * st_step], st[(long)g * st_step + 1], co + 8L * g, c0 + c);
    q.put(tab, a.CT, c);
  }
  __syncthreads();
  if (m.active) {
#pragma unroll
    for (int j = 0; j < NC; ++j) ln[j].get(tab, a.CT, max(m.slot + j, 0));      // (nor stored)
  }
}

// Groups c0 / Cg .. of sample b from their channels' sums chan[k * stride + c], W lanes each (the
// channels of a group, at most a wave): statistics or coefficients to gco[8 a group] (FWD: which holds the
// pivots in field 7), a sample's terms of the parameter gradients to par.
template <int MODE, int ACT, class A>
__device__ __forceinline__ void finish_groups(const Args& a, long b, int c0, int ng, const A* chan, long stride,
                                              double* gco, bool tell) {
  int W = 1;
  while (W < a.Cg && W < 64) W *= 2;
  const int lane = threadIdx.x & (W - 1), g0 = c0 / a.Cg;
  const double invN = 1.0 / ((double)a.L * a.Cg);
  for (int gi = threadIdx.x / W; gi < ng; gi += blockDim.x / W) {
    const int cg = gi * a.Cg;
    double* st = a.stats + 2 * (b * a.G + g0 + gi);
    double* co = gco + 8L * gi;
    if constexpr (MODE == FWD) {
      double s = 0, q = 0;
      for (int c = lane; c < a.Cg; c += W) {
        s += chan[cg + c];
        q += chan[stride + cg + c];
      }
      s = lanes_sum(s, W);
      q = lanes_sum(q, W);
      const double md = s * invN, mean = co[7] + md, var = fmax(q * invN - md * md, 0.0);
      const double nan = s - s + (q - q);            // fmax drops a NaN: put it back
      const double r = 1.0 / sqrt(var + nan + (double)a.eps);
      if (lane == 0) {
        co[0] = mean;
        co[1] = r;
        if (tell) {
          st[0] = mean;
          st[1] = r;
        }
      }
    } else {
      const Group q = group_of(st[0], st[1]);
      const int cc = c0 + cg;
      double m1[4] = {0, 0, 0, 0};
      for (int c = lane; c < a.Cg; c += W) {
        double terms[3];
        sweep1<MODE, ACT>(a, q, cc + c, [&](int k) { return (double)chan[k * stride + cg + c]; }, m1, terms);
        if (MODE == BWD && tell && a.par)
#pragma unroll
          for (int k = 0; k < Sums<BWD, ACT>::K; ++k) a.par[(k * a.B + b) * a.C + cc + c] = (float)terms[k];
      }
#pragma unroll
      for (int k = 0; k < (MODE == BWD ? 2 : 4); ++k) m1[k] = lanes_sum(m1[k], W) * invN;
      if (MODE == BWD) {
        if (lane == 0) {
          co[0] = m1[0];
          co[1] = m1[1];
        }
      } else {
        double m2[3] = {0, 0, 0};
        for (int c = lane; c < a.Cg; c += W) {
          double terms[3];
          sweep2<ACT>(a, q, cc + c, [&](int k) { return (double)chan[k * stride + cg + c]; }, m1, m2, terms);
          if (tell && a.par)
#pragma unroll
            for (int k = 0; k < (ACT == SLOPE ? 3 : 2); ++k) a.par[(k * a.B + b) * a.C + cc + c] = (float)terms[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) m2[k] = lanes_sum(m2[k], W);
        if (lane == 0) dbl_coef(q, m1, m2, invN, co);
      }
    }
  }
}

template <int MODE, int ACT, bool ROWS, class T, int V, int NC>
__device__ __forceinline__ void write(const Args& a, const Lin<MODE, ACT> (&ln)[NC], long at, int skip,
                                      const Vec<T, V>& x, const Vec<T, V>& gy, const Vec<T, V>& v) {
  Vec<T, V> o1, o2;
  apply<MODE, ACT, ROWS, T, V, NC>(ln, x, gy, v, o1, o2);
  if (MODE != BWD || a.o1) store(static_cast<T*>(a.o1) + at, o1, skip, a.once);
  if constexpr (MODE == DBL) store(static_cast<T*>(a.o2) + at, o2, skip, a.once);
}

// ------------------------------------------------------------------ the resident form
// Block (tile of whole groups, sample): RMAX vectors a thread, held between sums and result, so each
// input is read once.  What is left above a copy's time is that a block's phases follow each other
// (load, fold, coefficients, store): 64 samples of 48 channel rows of 64x64 in fp32, forward 20 us
// (5.0 TB/s), backward 35 (4.3); of 128 rows of 32x32 forward 16, backward 20, double backward 36 (4.7);
// in bf16 16, 22 and 12, 14, 22 (half the bytes: the phases weigh more).
template <int MODE, int ACT, bool ROWS, class T, int V, int RMAX, int NTMAX>
__global__ __launch_bounds__(NTMAX) void resident_kernel(Args a) {
  typedef typename AccT<MODE>::type A;
  constexpr int NC = ROWS ? V : 1, K = Sums<MODE, ACT>::K;
  extern __shared__ __align__(16) char lds[];
  const int tile = blockIdx.x % a.nct;
  const long b = blockIdx.x / a.nct;
  const Map<ROWS, V> m(a, b, tile);
  const int gt = a.CT / a.Cg;                       // groups of a tile (the last may hold fewer)
  double* gco = reinterpret_cast<double*>(lds);     // [gt][8] (FWD: mean, r)
  float* tab = reinterpret_cast<float*>(gco + gt * 8);
  A* chan = reinterpret_cast<A*>(tab);              // [K][CT]
  A* sh = chan + K * a.CT;
  const T* px = static_cast<const T*>(a.x);
  const T* pg = static_cast<const T*>(a.gy);
  const T* pv = static_cast<const T*>(a.v);

  const int c0 = tile * a.CT, g0 = c0 / a.Cg, ng = min(gt, a.G - g0);
  Chan<MODE, ACT> ch[NC];
  const Pivots<ACT, ROWS, T, V, NC> piv(a, m, b);
  const T mine = static_cast<const T*>(a.x)[b * a.pb + (c0 + min((int)threadIdx.x, ng - 1) * a.Cg) * a.pc];
  Vec<T, V> x[RMAX], gy[MODE >= BWD ? RMAX : 1], v[MODE == DBL ? RMAX : 1];
#pragma unroll
  for (int k = 0; k < RMAX; ++k) {
    const int i = m.p + k * a.P;
    int skip = V;
    if (m.active && i < m.npos) {
      const long at = m.at(i, skip);
      x[k] = load<T, V>(px + at);
      if constexpr (MODE >= BWD) gy[k] = load<T, V>(pg + at);
      if constexpr (MODE == DBL) v[k] = load<T, V>(pv + at);
    }
    if (MODE != FWD && skip == V) x[k].zero_front(skip);
    if constexpr (MODE >= BWD) gy[k].zero_front(skip);
    if constexpr (MODE == DBL) v[k].zero_front(skip);
  }
  if constexpr (MODE == FWD) {
    if ((int)threadIdx.x < ng) gco[8 * threadIdx.x + 7] = (double)up(mine);
    for (int g = threadIdx.x + blockDim.x; g < ng; g += blockDim.x) gco[8 * g + 7] = (double)pivot(a, b, c0 + g * a.Cg);
    piv.get(a, ch);
  }
  load_chan<MODE, ACT, ROWS, V, NC>(a, m, b, c0, tab, ch);
  A acc[K][NC];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[k][j] = 0;
#pragma unroll
  for (int k = 0; k < RMAX; ++k) {
    if constexpr (MODE == FWD) {
      const int i = m.p + k * a.P;
      if (!m.active || i >= m.npos) continue;
      if (!ROWS && a.L % V) {              // (rows: the fold leaves a moved-back front out)
        int skip;
        m.at(i, skip);
        x[k].fill_front(skip, bits(down<T>(ch[0].mf)));
      }
    } else if (!m.active || (k > 0 && k * a.P >= m.npos)) {
      continue;
    }
    accumulate<MODE, ACT, ROWS, T, V, NC>(acc, ch, x[k], gy[MODE >= BWD ? k : 0], v[MODE == DBL ? k : 0]);
  }
#pragma unroll
  for (int k = 0; k < RMAX; ++k) {
    x[k].pin();
    if constexpr (MODE >= BWD) gy[k].pin();
    if constexpr (MODE == DBL) v[k].pin();
  }
  fold<ROWS, V, K, NC>(a, m, acc, sh, chan, c0);
  finish_groups<MODE, ACT>(a, b, c0, ng, chan, (long)a.CT, gco, true);
  __syncthreads();
  Lin<MODE, ACT> ln[NC];
  if (MODE == FWD)
    load_lin<MODE, ACT, ROWS, V, NC>(a, m, b, c0, gco, 8, gco, tab, ln);
  else
    load_lin<MODE, ACT, ROWS, V, NC>(a, m, b, c0, a.stats + 2 * (b * a.G + g0), 2, gco, tab, ln);
  if (!m.active) return;
#pragma unroll
  for (int k = 0; k < RMAX; ++k) {
    const int i = m.p + k * a.P;
    if (i < m.npos) {
      int skip;
      const long at = m.at(i, skip);
      write<MODE, ACT, ROWS, T, V, NC>(a, ln, at, skip, x[k], gy[MODE >= BWD ? k : 0], v[MODE == DBL ? k : 0]);
    }
  }
}

// ------------------------------------------------------------------ the split form
// For groups that no block can hold (channels last, a group's values lie a few channels wide over all
// positions: reading one alone would fetch every line for each group).  The second pass reads the
// inputs again: 64 maps of 64x64x96 in bf16, forward 15 us of sums and 20 of the elementwise pass; 256
// of them 43 and 62 (4.7 and 6.5 TB/s), backward 68 and 108 (5.9 and 5.6).  Neither waits on the
// vector units (a leaky slope takes the same time as SiLU).
constexpr int kNT = 512;

// The loop of both passes over a chunk: U positions a trip, the next ones loaded before the present
// ones are used; `first` runs between the first loads and their use.  use(at, skip, x, gy, v) gets
// skip == 0 where nothing is moved back (rows: a thread's own skip0); only the last trip looks at
// the chunk's end, and at the end of a plane.
template <int MODE, bool ROWS, class T, int V, int U, class First, class Use>
__device__ __forceinline__ void stream(const Args& a, const Map<ROWS, V>& m, int lo, int hi, First first, Use use) {
  const T* px = static_cast<const T*>(a.x);
  const T* pg = static_cast<const T*>(a.gy);
  const T* pv = static_cast<const T*>(a.v);
  Vec<T, V> x[U], gy[MODE >= BWD ? U : 1], v[MODE == DBL ? U : 1];
  const int whole = ROWS ? hi : min(hi, (int)(a.L / V));       // positions before it are whole vectors
  const long hop = (long)a.P * m.step;
  int i0 = lo + m.p;
  auto fetch = [&](int i, bool full) {
    const long at = m.base + i * m.step;
    if (full) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = load<T, V>(px + at + u * hop);
        if constexpr (MODE >= BWD) gy[u] = load<T, V>(pg + at + u * hop);
        if constexpr (MODE == DBL) v[u] = load<T, V>(pv + at + u * hop);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * a.P < hi) {
          int skip;
          const long q = m.at(i + u * a.P, skip);
          x[u] = load<T, V>(px + q);
          if constexpr (MODE >= BWD) gy[u] = load<T, V>(pg + q);
          if constexpr (MODE == DBL) v[u] = load<T, V>(pv + q);
        }
    }
  };
  bool full = i0 + (U - 1) * a.P < whole;
  if (m.active) fetch(i0, full);
  first();
  if (!m.active) return;
  while (full) {
    Vec<T, V> cx[U], cg[MODE >= BWD ? U : 1], cv[MODE == DBL ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      cx[u] = x[u];
      if constexpr (MODE >= BWD) cg[u] = gy[u];
      if constexpr (MODE == DBL) cv[u] = v[u];
    }
    const long at = m.base + i0 * m.step;
    i0 += U * a.P;
    full = i0 + (U - 1) * a.P < whole;
    fetch(i0, full);
#pragma unroll
    for (int u = 0; u < U; ++u)
      use(at + u * hop, ROWS ? m.skip0 : 0, cx[u], cg[MODE >= BWD ? u : 0], cv[MODE == DBL ? u : 0]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i0 + u * a.P < hi) {
      int skip;
      const long at = m.at(i0 + u * a.P, skip);
      use(at, skip, x[u], gy[MODE >= BWD ? u : 0], v[MODE == DBL ? u : 0]);
    }
}

// blockIdx.x = (sample, tile, chunk), chunk fastest
template <int MODE, int ACT, bool ROWS, class T, int V>
__global__ __launch_bounds__(kNT) void sums_kernel(Args a) {
  typedef typename AccT<MODE>::type A;
  constexpr int NC = ROWS ? V : 1, K = Sums<MODE, ACT>::K, U = 2;
  extern __shared__ __align__(16) char lds[];
  const int s = blockIdx.x % a.S, tile = blockIdx.x / a.S % a.nct;
  const int bi = blockIdx.x / a.S / a.nct;
  const long b = bi;
  const Map<ROWS, V> m(a, b, tile);
  float* tab = reinterpret_cast<float*>(lds);
  A* chan = reinterpret_cast<A*>(lds);
  A* sh = chan + K * a.CT;
  const int c0 = tile * a.CT, wid = min(a.CT, a.C - c0);
  const int hi = (int)min((long)m.npos, (long)(s + 1) * a.per);
  Chan<MODE, ACT> ch[NC];
  const Pivots<ACT, ROWS, T, V, NC> piv(a, m, b);
  A acc[K][NC];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[k][j] = 0;
  stream<MODE, ROWS, T, V, U>(
      a, m, s * a.per, hi, [&] {
        if constexpr (MODE == FWD) piv.get(a, ch);
        load_chan<MODE, ACT, ROWS, V, NC>(a, m, b, c0, tab, ch);
      },
      [&](long, int skip, Vec<T, V>& x, Vec<T, V>& gy, Vec<T, V>& v) {
        if constexpr (!ROWS) {                 // (rows: the fold leaves a moved-back front out)
          if (MODE == FWD) x.fill_front(skip, bits(down<T>(ch[0].mf)));
          if constexpr (MODE >= BWD) gy.zero_front(skip);
          if constexpr (MODE == DBL) v.zero_front(skip);
        }
        accumulate<MODE, ACT, ROWS, T, V, NC>(acc, ch, x, gy, v);
      });
  fold<ROWS, V, K, NC>(a, m, acc, sh, chan, c0);
  A* part = reinterpret_cast<A*>(a.part) + ((long)bi * a.S + s) * K * a.C;
  for (int i = threadIdx.x; i < K * wid; i += blockDim.x)
    part[(long)(i / wid) * a.C + c0 + i % wid] = chan[i / wid * a.CT + i % wid];
}

// Many chunks: every 32 of a channel's into the first of them, so that the group blocks' loop is short.
constexpr int kFold = 32;

template <class A>
__global__ __launch_bounds__(256) void chunk_kernel(A* part, int S, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x, s0 = blockIdx.y * kFold;
  if (i >= n) return;
  A* p = part + ((long)blockIdx.z * S + s0) * n + i;
  double t = 0;
#pragma unroll 8
  for (int s = 0; s < min(kFold, S - s0); ++s) t += (double)p[(long)s * n];
  *p = (A)t;
}

// Block (sample, gpb groups): the chunks' sums folded in double and in one order into the first
// chunk's place, then the groups' statistics or coefficients.
template <int MODE, int ACT>
__global__ __launch_bounds__(256) void group_kernel(Args a, int gpb, int sstep) {
  typedef typename AccT<MODE>::type A;
  constexpr int K = Sums<MODE, ACT>::K;
  const int nb = (a.G + gpb - 1) / gpb, g0 = blockIdx.x % nb * gpb, bi = blockIdx.x / nb;
  const long b = bi;
  extern __shared__ __align__(16) double gco[];      // (FWD)
  const int ng = min(gpb, a.G - g0), nc = ng * a.Cg, pairs = K * nc, ns = (a.S + sstep - 1) / sstep;
  A* part = reinterpret_cast<A*>(a.part) + (long)bi * a.S * K * a.C + g0 * a.Cg;
  const uint32_t mine = MODE == FWD ? pivot_bits(a, b, (g0 + min((int)threadIdx.x, ng - 1)) * a.Cg) : 0;
  if (ns > 1) {
    int sw = 1;                                       // lanes that share a channel's chunks
    while (sw * 2 * pairs <= 256 && sw * 2 <= ns && sw < 64) sw *= 2;
    const int q = threadIdx.x & (sw - 1);
    const long hop = (long)sstep * K * a.C;
    for (int i0 = 0; i0 < pairs; i0 += 256 / sw) {
      const int i = i0 + threadIdx.x / sw;
      A* p = part + (long)(i / nc) * a.C + i % nc;
      double t = 0;
      if (i < pairs) {
#pragma unroll 8
        for (int s = q; s < ns; s += sw) t += (double)p[s * hop];
      }
      t = lanes_sum(t, sw);
      if (q == 0 && i < pairs) *p = (A)t;
    }
  }
  if (MODE == FWD && (int)threadIdx.x < ng) gco[8 * threadIdx.x + 7] = (double)of_bits(a, mine);   // (gpb <= 128)
  if (MODE == FWD || ns > 1) __syncthreads();
  // (FWD writes the statistics; the coefficients have their own place)
  finish_groups<MODE, ACT>(a, b, g0 * a.Cg, ng, part, (long)a.C, MODE == FWD ? gco : a.coef + 8 * (b * a.G + g0),
                           true);
}

// FOLD: each block folds its sample's chunks and finishes the groups itself (rows, one tile of all
// channels; a.part holds fold_S chunks), one launch less; else a group_kernel went before.
template <int MODE, int ACT, bool ROWS, class T, int V, bool FOLD>
__global__ __launch_bounds__(kNT) void apply_kernel(Args a, int fold_S) {
  typedef typename AccT<MODE>::type A;
  constexpr int NC = ROWS ? V : 1, K = Sums<MODE, ACT>::K, U = 2;
  extern __shared__ __align__(16) char lds[];
  const int s = blockIdx.x % a.S, tile = blockIdx.x / a.S % a.nct;
  const long b = blockIdx.x / a.S / a.nct;
  const Map<ROWS, V> m(a, b, tile);
  const int c0 = tile * a.CT;
  const int hi = (int)min((long)m.npos, (long)(s + 1) * a.per);
  const long g0 = b * a.G + c0 / a.Cg;
  Lin<MODE, ACT> ln[NC];
  stream<MODE, ROWS, T, V, U>(
      a, m, s * a.per, hi,
      [&] {
        if constexpr (FOLD) {
          double* gco = reinterpret_cast<double*>(lds);
          A* chan = reinterpret_cast<A*>(gco + 8L * a.G);            // [K][C]; then the coefficients
          const A* part = reinterpret_cast<const A*>(a.part) + b * fold_S * K * a.C;
          const T mine = static_cast<const T*>(a.x)[b * a.pb + min((int)threadIdx.x, a.G - 1) * a.Cg * a.pc];
          for (int i = threadIdx.x; i < K * a.C; i += blockDim.x) {
            double t = 0;
#pragma unroll 4
            for (int k = 0; k < fold_S; ++k) t += (double)part[(long)k * K * a.C + i];
            chan[i] = (A)t;
          }
          if (MODE == FWD) {
            if ((int)threadIdx.x < a.G) gco[8 * threadIdx.x + 7] = (double)up(mine);
            for (int g = threadIdx.x + blockDim.x; g < a.G; g += blockDim.x) gco[8 * g + 7] = (double)pivot(a, b, g * a.Cg);
          }
          __syncthreads();
          finish_groups<MODE, ACT>(a, b, 0, a.G, chan, (long)a.C, gco, s == 0);
          __syncthreads();
          load_lin<MODE, ACT, ROWS, V, NC>(a, m, b, 0, MODE == FWD ? gco : a.stats + 2 * g0, MODE == FWD ? 8 : 2, gco,
                                           reinterpret_cast<float*>(chan), ln);
        } else {
          load_lin<MODE, ACT, ROWS, V, NC>(a, m, b, c0, a.stats + 2 * g0, 2, a.coef + 8 * g0,
                                           reinterpret_cast<float*>(lds), ln);
        }
      },
      [&](long at, int skip, Vec<T, V>& x, Vec<T, V>& gy, Vec<T, V>& v) {
        write<MODE, ACT, ROWS, T, V, NC>(a, ln, at, skip, x, gy, v);
      });
}

// ------------------------------------------------------------------ launches
// Threads of a resident block and the vectors of each input that a thread can hold: what fits 128
// registers a thread (1024 threads) or 256 (512).
constexpr int resident_threads(int mode, bool rows) { return rows || mode == DBL ? 512 : 1024; }
constexpr int resident_vectors(int mode, bool rows) { return mode == DBL || (mode == BWD && !rows) ? 8 : 16; }

// How one call runs (group_norm.hip makes it from sizes and type alone).
struct Plan {
  int mode, act;
  bool rows, resident;
  int V, rmax, nt;
  size_t lds, apply_lds;
  int apply_S, apply_per; // the elementwise pass's own chunks
  bool fold_apply;        // its blocks fold the sums' chunks themselves
  int gpb, sstep;         // groups a folding block takes; chunks are folded by 32 before (or 1)
};

template <int MODE, int ACT, bool ROWS, class T, int V, int RMAX>
int launch_resident(const Plan& p, const Args& a, hipStream_t st) {
  constexpr int NTMAX = resident_threads(MODE, ROWS);
  hipLaunchKernelGGL((resident_kernel<MODE, ACT, ROWS, T, V, RMAX, NTMAX>), dim3((unsigned)(a.B * a.nct)), dim3(p.nt),
                     p.lds, st, a);
  return hipGetLastError() == hipSuccess ? GANAMD_OK : GANAMD_ELAUNCH;
}

template <int MODE, int ACT, bool ROWS, class T, int V>
int launch_v(const Plan& p, const Args& a, hipStream_t st) {
  if (p.resident) {
    constexpr int MOST = resident_vectors(MODE, ROWS);
    if (p.rmax <= 2) return launch_resident<MODE, ACT, ROWS, T, V, 2>(p, a, st);
    if (p.rmax <= 4) return launch_resident<MODE, ACT, ROWS, T, V, 4>(p, a, st);
    if (p.rmax <= 8) return launch_resident<MODE, ACT, ROWS, T, V, 8>(p, a, st);
    if constexpr (MOST > 8) return launch_resident<MODE, ACT, ROWS, T, V, MOST>(p, a, st);
    return GANAMD_EINVAL;
  }
  const dim3 grid((unsigned)(a.B * a.nct * a.S));
  hipLaunchKernelGGL((sums_kernel<MODE, ACT, ROWS, T, V>), grid, dim3(p.nt), p.lds, st, a);
  Args b = a;
  b.S = p.apply_S;
  b.per = p.apply_per;
  const dim3 apply_grid((unsigned)(a.B * a.nct * b.S));
  if constexpr (ROWS) {
    if (p.fold_apply && (MODE != BWD || a.o1)) {
      hipLaunchKernelGGL((apply_kernel<MODE, ACT, ROWS, T, V, true>), apply_grid, dim3(p.nt), p.apply_lds, st, b, a.S);
      return hipGetLastError() == hipSuccess ? GANAMD_OK : GANAMD_ELAUNCH;
    }
  }
  if (p.sstep > 1) {
    typedef typename AccT<MODE>::type A;
    const int n = Sums<MODE, ACT>::K * a.C;
    hipLaunchKernelGGL(chunk_kernel<A>, dim3((n + 255) / 256, (a.S + kFold - 1) / kFold, (unsigned)a.B), dim3(256), 0,
                       st, reinterpret_cast<A*>(a.part), a.S, n);
  }
  hipLaunchKernelGGL((group_kernel<MODE, ACT>), dim3((unsigned)(a.B * ((a.G + p.gpb - 1) / p.gpb))), dim3(256),
                     MODE == FWD ? 64 * (size_t)p.gpb : 0, st, a, p.gpb, p.sstep);
  if (MODE != BWD || a.o1)
    hipLaunchKernelGGL((apply_kernel<MODE, ACT, ROWS, T, V, false>), apply_grid, dim3(p.nt), p.apply_lds, st, b, a.S);
  return hipGetLastError() == hipSuccess ? GANAMD_OK : GANAMD_ELAUNCH;
}

// Vector width of an element type: 16 bytes; in the double backward of rows, where a thread carries
// ten sums and a dozen coefficients of each of its channels, 4 elements; 1 where rows or planes are
// shorter than that.
constexpr int vec_width(int mode, bool rows, int size) { return rows && mode == DBL ? 4 : 16 / size; }

template <int MODE, int ACT, class T>
int launch_t(const Plan& p, const Args& a, hipStream_t st) {
  constexpr int VR = vec_width(MODE, true, sizeof(T)), VP = vec_width(MODE, false, sizeof(T));
  if (p.rows) return p.V == 1 ? launch_v<MODE, ACT, true, T, 1>(p, a, st) : launch_v<MODE, ACT, true, T, VR>(p, a, st);
  return p.V == 1 ? launch_v<MODE, ACT, false, T, 1>(p, a, st) : launch_v<MODE, ACT, false, T, VP>(p, a, st);
}

template <class T>
int launch(const Plan& p, const Args& a, hipStream_t st) {
  if (p.mode == FWD)
    return p.act == SILU ? launch_t<FWD, SILU, T>(p, a, st) : launch_t<FWD, KINK, T>(p, a, st);
  if (p.mode == BWD)
    return p.act == SILU ? launch_t<BWD, SILU, T>(p, a, st)
         : p.act == KINK ? launch_t<BWD, KINK, T>(p, a, st) : launch_t<BWD, SLOPE, T>(p, a, st);
  return p.act == SILU ? launch_t<DBL, SILU, T>(p, a, st)
       : p.act == KINK ? launch_t<DBL, KINK, T>(p, a, st) : launch_t<DBL, SLOPE, T>(p, a, st);
}

// one translation unit per element type (compiled in parallel)
int launch_f32(const Plan& p, const Args& a, hipStream_t st);
int launch_bf16(const Plan& p, const Args& a, hipStream_t st);
int launch_f16(const Plan& p, const Args& a, hipStream_t st);

}  // namespace gn
