// Group norm with its activation: plans, workspaces and the C entry points (kernels: group_norm.h).
#include "group_norm.h"

#include <algorithm>

namespace {

using gn::Args;
using gn::Plan;

inline long up_to(long a, long b) { return (a + b - 1) / b; }
inline long pow2_at_least(long n) {
  long p = 1;
  while (p < n) p *= 2;
  return p;
}

bool valid(const ganamd_norm_desc* d) {
  return d && d->B > 0 && d->C > 0 && d->L > 0 && d->L <= (1L << 30) && d->G > 0 && d->C % d->G == 0 &&
         d->C <= (1 << 24) && (d->layout == GANAMD_NORM_ROWS || d->layout == GANAMD_NORM_PLANES) &&
         d->dtype >= GANAMD_F32 && d->dtype <= GANAMD_F16 && d->param_dtype >= GANAMD_F32 &&
         d->param_dtype <= GANAMD_F16 && d->act >= GANAMD_NORM_NONE && d->act <= GANAMD_NORM_PRELU && d->eps > 0.f;
}

int esize(int dt) { return dt == GANAMD_F32 ? 4 : 2; }

struct Full {
  Plan p;
  Args a;                          // the sizes; no pointers
  size_t part, coef, par, fold, total;   // workspace offsets and size
};

constexpr int kFoldB = 512;        // samples a parameter-gradient block folds

// Which kernels a call takes and how its work is cut, from the sizes and the type alone.
bool make_plan(const ganamd_norm_desc* d, int mode, Full& f) {
  if (!valid(d)) return false;
  Plan& p = f.p;
  Args& a = f.a;
  a = Args{};
  const int esz = esize(d->dtype);
  const int C = d->C, G = d->G, Cg = C / G;
  const long L = d->L, B = d->B;
  p.mode = mode;
  p.rows = d->layout == GANAMD_NORM_ROWS;
  p.act = d->act == GANAMD_NORM_SILU ? gn::SILU
        : d->act == GANAMD_NORM_PRELU && mode != gn::FWD ? gn::SLOPE : gn::KINK;
  p.V = gn::vec_width(mode, p.rows, esz);
  if ((p.rows ? (long)C : L) < p.V) p.V = 1;
  const int K = mode == gn::FWD ? 2 : mode == gn::BWD ? (p.act == gn::SLOPE ? 3 : 2)
              : (p.act == gn::SILU ? 10 : p.act == gn::SLOPE ? 8 : 5);
  const size_t asz = mode == gn::FWD ? 8 : 4;
  const int tabs = mode == gn::FWD ? 6 : mode == gn::BWD ? 8 : 13;      // fields of a channel's coefficients
  const int rcap = gn::resident_vectors(mode, p.rows), most = gn::resident_threads(mode, p.rows);
  // Resident blocks are made smaller, down to 256 threads, as long as a thread then holds no more than
  // this many vectors of an input: several blocks a CU overlap their phases (64 samples of 128 rows
  // of 32x32, calls back to back: forward 13.4 us against 16.7 with the widest blocks, backward 23.9 against
  // 25.9).
  const long few = mode == gn::DBL ? 4 : 8;
  // A block of the resident form that holds so few values beats the split form's launches however few the
  // blocks are (one fp32 sample, resident against split: forward of 64 channels of 16x16, 8 K values a block,
  // 6.3 us against 9.6, of 32x32, 32 K, 9.5 against 10.1; backward 11.1 against 14.0, of 16x32, 16 K, 12.0 against
  // 13.6).  A larger one takes longer than they do (forward of 4 bf16 samples of 32x32x128, 64 K, 16.2 against
  // 13.4; backward of one sample of 64 channels of 32x32 17.2 against 13.5) until there are many blocks
  // (that one, 96 blocks: forward 11.7 against 14.9, backward 23.1 against 21.1; 192: 13.8 against 19.4, 25.1
  // against 32.3).
  const long small = mode == gn::FWD ? 32 << 10 : 16 << 10, many = 96;
  a.L = L; a.B = B; a.C = C; a.G = G; a.Cg = Cg; a.eps = d->eps; a.pdt = d->param_dtype;
  a.xdt = d->dtype; a.pb = p.rows ? L * C : L; a.pc = p.rows ? 1 : B * L;
  a.cslope = d->act == GANAMD_NORM_LEAKY ? d->slope : 1.f;
  // A call whose tensors are well beyond the 256 MB of the last-level cache: its outputs are stored past
  // the caches (forward and a copy of its output, 256 maps of 64x64x96 in bf16: 190 us against 212;
  // for smaller ones the call itself gains too, but the kernel that reads its output loses as much:
  // 64 maps of 64x64x64 in fp32 with the copy 69 against 67).
  const long data = (mode == gn::FWD ? 2 : mode == gn::BWD ? 3 : 5) * B * L * C * esz;
  const bool large = data >= (384L << 20);
  a.once = large;
  p.resident = false;
  const long nv = up_to(L, p.V);
  if (p.rows) {
    // a tile of whole groups, at least a cache line wide
    long gt = 1;
    while (gt < G && (gt * Cg * esz < 128 || gt * Cg < p.V)) ++gt;
    for (long t = gt; t <= G && t < gt + p.V; ++t)
      if (t * Cg % p.V == 0) { gt = t; break; }
    if (gt * Cg < p.V) gt = G;
    const long CT = gt * Cg, TX = up_to(CT, p.V);
    if (TX <= most) {
      const long P = std::min(most / TX, std::max(up_to(L, few), std::min(L, 256 / TX)));
      const long R = up_to(L, P), nct = up_to(G, gt);
      if (R <= rcap && (CT * L <= small || B * nct >= many)) {
        p.resident = true;
        a.TX = (int)TX; a.P = (int)P; a.CT = (int)CT; a.nct = (int)nct; p.rmax = (int)R;
        p.nt = (int)up_to(TX * P, 64) * 64;
      }
    }
  } else if (Cg <= most) {
    long P = std::min(pow2_at_least(nv), pow2_at_least(most / Cg + 1) / 2), gt = 1;
    // Small planes: several groups a block, up to 512 threads while two blocks a CU are left (forward of 1024
    // samples of 64 planes of 4x4, groups of 2: 6.1 us, one group a block 24; 256 samples of 128 planes of 8x8,
    // groups of 4: 6.9 us, up to 256 threads 7.9; 512 bf16 samples of 32 planes of 8x8: 5.2 us, with four
    // blocks a CU left 5.9, with one 5.3).
    while (gt < G && (gt + 1) * Cg * P <= 512 && B * up_to(G, gt + 1) >= 512) ++gt;
    gt = up_to(G, up_to(G, gt));           // (as many blocks, evenly filled)
    while (P > 1 && up_to(nv, P / 2) <= few && gt * Cg * P > 256) P /= 2;
    const long R = up_to(nv, P), nct = up_to(G, gt);
    if (R <= rcap && (gt * Cg * L <= small || B * nct >= many)) {
      p.resident = true;
      a.TX = (int)(gt * Cg); a.P = (int)P; a.CT = (int)(gt * Cg); a.nct = (int)nct; p.rmax = (int)R;
      p.nt = (int)up_to(a.TX * P, 64) * 64;
    }
  }
  if (p.resident) {
    p.fold_apply = false;
    a.S = p.apply_S = 1;
    a.per = p.apply_per = 0;
    const size_t sh = p.rows ? (size_t)gn::fold_round(K, p.V, p.nt, asz) * p.V * p.nt : (size_t)K * 16;
    p.lds = (size_t)(a.CT / Cg) * 64 + std::max(asz * ((size_t)K * a.CT + sh), 4 * (size_t)tabs * a.CT);
    if (p.lds > 64 * 1024) p.resident = false;
  }
  if (!p.resident) {
    long npos;
    if (p.rows) {
      const long all = up_to(C, p.V);
      // (a tile's channels: their sums or coefficients, and the fold's scratch, share 64 KB)
      a.nct = (int)std::max(up_to(all, gn::kNT), up_to(all * p.V * std::max<long>(K * asz, 4 * tabs), 24 * 1024));
      a.TX = (int)up_to(all, a.nct);
      a.CT = a.TX * p.V;
      a.nct = (int)up_to(C, a.CT);
      a.P = (int)std::min<long>(gn::kNT / a.TX, L);
      p.nt = (int)up_to((long)a.TX * a.P, 64) * 64;
      npos = L;
    } else {
      a.P = (int)std::min<long>(gn::kNT, pow2_at_least(nv));
      a.CT = a.TX = (int)std::min<long>(gn::kNT / a.P, C);
      a.nct = (int)up_to(C, a.CT);
      p.nt = (int)up_to((long)a.TX * a.P, 64) * 64;
      npos = nv;
    }
    // The sums: two blocks of eight waves a CU, but four vectors a thread at least (more blocks are
    // more folds: 64 maps of 64x64x96 in bf16 took 37 us with 512 blocks, 42 with 1024, 48 with
    // 2048), and at most 128 values of a channel in one thread's fp32 sums.
    long S = std::max<long>(1, std::min(up_to(512, B * a.nct), up_to(npos, 4L * a.P)));
    S = std::max(S, up_to(npos, (p.rows ? 128L : 128L / p.V) * a.P));
    a.per = (int)(up_to(up_to(npos, S), a.P) * a.P);
    a.S = (int)up_to(npos, a.per);
    // The elementwise pass: as many; for large calls pieces in launch order, which keep what is in flight
    // together in memory (the same maps: forward 128 us with 8192 blocks, 133 with 512, backward 203
    // and 229; but the 335 MB double backward of 64 maps of 64x64x64 in fp32 121 and 116).
    const long SA = std::max<long>(1, std::min(up_to(large ? 8192 : 512, B * a.nct), up_to(npos, 4L * a.P)));
    p.apply_per = (int)(up_to(up_to(npos, SA), a.P) * a.P);
    p.apply_S = (int)up_to(npos, p.apply_per);
    const size_t sh = p.rows ? (size_t)gn::fold_round(K, p.V, p.nt, asz) * p.V * p.nt : (size_t)K * 16;
    p.lds = std::max(asz * ((size_t)K * a.CT + sh), 4 * (size_t)tabs * a.CT);
    p.apply_lds = 4 * (size_t)tabs * a.CT;
    // Few blocks, few chunks, all of a sample's groups in a block's reach: the elementwise blocks fold
    // and a launch goes (64 maps of 64x64x96 in bf16 forward: 35.5 us, with a group kernel 37.5; the
    // backward of 64 maps of 64x64x64 in fp32 69.8 against 72.8, of 7 maps of 33x31x100 15.1 against 18.5).
    const size_t fold_lds = 64 * (size_t)G + std::max(asz * (size_t)K * C, p.apply_lds);
    p.fold_apply = p.rows && a.nct == 1 && a.S <= 16 && B * p.apply_S <= 1024 && fold_lds <= 32 * 1024;
    if (p.fold_apply) p.apply_lds = fold_lds;
  }
  p.gpb = (int)std::max<long>(1, std::min<long>(G, 256 / ((long)K * Cg)));
  p.sstep = a.S > 2 * gn::kFold ? gn::kFold : 1;
  // A launch holds fewer than 2^32 threads across x and 2^16 blocks across y or z; the kernels' block numbers
  // are 32 bits.  (In doubles: the products of absurd sizes pass 64 bits.)
  const double blocks = (double)B * a.nct * std::max(a.S, p.apply_S), most_threads = 4294967295.0;
  if (blocks >= 2147483648.0 || blocks * p.nt > most_threads || (double)B * G >= 2147483648.0 || p.lds > 64 * 1024 ||
      up_to(B, kFoldB) > 65535 || (p.sstep > 1 && B > 65535) ||
      (!p.resident && (double)B * up_to(G, p.gpb) * 256 > most_threads))
    return false;
  // workspace
  const size_t pars = p.act == gn::SLOPE ? 3 : 2;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
  f.part = p.resident ? 0 : take(asz * (size_t)K * C * a.S * B);
  f.coef = p.resident || mode == gn::FWD ? 0 : take(64 * (size_t)B * G);
  f.par = mode == gn::FWD ? 0 : take(4 * pars * (size_t)B * C);
  f.fold = mode == gn::FWD || B <= kFoldB ? 0 : take(4 * pars * (size_t)up_to(B, kFoldB) * C);
  f.total = at;
  return true;
}

__device__ __forceinline__ void put(void* out, int dt, long i, double v, int accumulate) {
  if (dt == GANAMD_F32) {
    float* o = static_cast<float*>(out) + i;
    *o = accumulate ? *o + (float)v : (float)v;
  } else if (dt == GANAMD_BF16) {
    gn::bf16* o = static_cast<gn::bf16*>(out) + i;
    *o = gn::down<gn::bf16>((accumulate ? gn::up(*o) : 0.f) + (float)v);
  } else {
    gn::f16* o = static_cast<gn::f16*>(out) + i;
    *o = gn::down<gn::f16>((accumulate ? gn::up(*o) : 0.f) + (float)v);
  }
}

// Sums in[k][b][c] over chunks of `n` samples, in double and one order; the last stage writes the
// gradients, an earlier one in's successor mid[k][chunk][c].  Block: 64 channels x 16 samples.
__global__ __launch_bounds__(1024) void param_kernel(const float* __restrict__ in, long B, int C, int n, float* mid,
                                                     void* g0, void* g1, void* g2, int dt, int accumulate) {
  __shared__ double sh[16][64];
  const int k = blockIdx.y, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const long chunk = blockIdx.z, c = blockIdx.x * 64L + x;
  void* out = k == 0 ? g0 : k == 1 ? g1 : g2;
  if (!mid && !out) return;
  const long hi = min(B, (chunk + 1) * n);
  double t = 0;
  if (c < C) {
#pragma unroll 4
    for (long b = chunk * n + y; b < hi; b += 16) t += (double)in[(k * B + b) * C + c];
  }
  sh[y][x] = t;
  __syncthreads();
  if (y != 0 || c >= C) return;
  for (int i = 1; i < 16; ++i) t += sh[i][x];
  if (mid)
    mid[((long)k * gridDim.z + chunk) * C + c] = (float)t;
  else
    put(out, dt, c, t, accumulate);
}

int fold_params(const Full& f, char* ws, int K, void* gw, void* gb, void* gs, int dt, int accumulate, hipStream_t st) {
  if (!gw && !gb && !gs) return GANAMD_OK;
  const float* in = reinterpret_cast<const float*>(ws + f.par);
  long B = f.a.B;
  const int C = f.a.C;
  const unsigned gx = (unsigned)up_to(C, 64);
  if (B > kFoldB) {
    float* mid = reinterpret_cast<float*>(ws + f.fold);
    const long nc = up_to(B, kFoldB);
    hipLaunchKernelGGL(param_kernel, dim3(gx, K, (unsigned)nc), dim3(1024), 0, st, in, B, C, kFoldB, mid, gw, gb, gs, dt, 0);
    in = mid;
    B = nc;
  }
  hipLaunchKernelGGL(param_kernel, dim3(gx, K, 1), dim3(1024), 0, st, in, B, C, (int)B, (float*)nullptr, gw, gb, gs,
                     dt, accumulate);
  return hipGetLastError() == hipSuccess ? GANAMD_OK : GANAMD_ELAUNCH;
}

int run(const ganamd_norm_desc* d, const Full& f, Args a, char* ws, hipStream_t st) {
  a.part = reinterpret_cast<float*>(ws + f.part);
  a.coef = reinterpret_cast<double*>(ws + f.coef);
  return d->dtype == GANAMD_F32 ? gn::launch_f32(f.p, a, st)
       : d->dtype == GANAMD_BF16 ? gn::launch_bf16(f.p, a, st) : gn::launch_f16(f.p, a, st);
}

}  // namespace

extern "C" {

int ganamd_group_norm_workspace(const ganamd_norm_desc* d, int op, size_t* bytes) {
  Full f;
  if (!bytes || op < gn::FWD || op > gn::DBL || !make_plan(d, op, f)) return GANAMD_EINVAL;
  *bytes = f.total;
  return GANAMD_OK;
}

int ganamd_group_norm_plan_info(const ganamd_norm_desc* d, int op, int* info) {
  Full f;
  if (!info || op < gn::FWD || op > gn::DBL || !make_plan(d, op, f)) return GANAMD_EINVAL;
  const int v[11] = {f.p.resident, f.p.V,  f.p.nt, f.a.TX,      f.a.P,        f.a.CT,
                     f.a.nct,      f.a.S, f.a.per, f.p.apply_S, f.p.apply_per};
  for (int i = 0; i < 11; ++i) info[i] = v[i];
  return GANAMD_OK;
}

int ganamd_group_norm_fwd(const ganamd_norm_desc* d, const void* x, const void* w, const void* b, const void* slope,
                          void* y, double* stats, void* workspace, size_t workspace_bytes, hipStream_t st) {
  Full f;
  if (!make_plan(d, gn::FWD, f) || !x || !y || !stats || (d->act == GANAMD_NORM_PRELU && !slope) ||
      workspace_bytes < f.total || (f.total && !workspace))
    return GANAMD_EINVAL;
  // in place, no elementwise block may read a pivot that another one has overwritten: a group kernel goes before
  if (x == y) f.p.fold_apply = false;
  Args a = f.a;
  a.x = x; a.w = w; a.b = b; a.slope = d->act == GANAMD_NORM_PRELU ? slope : nullptr;
  a.o1 = y; a.stats = stats;
  return run(d, f, a, static_cast<char*>(workspace), st);
}

int ganamd_group_norm_bwd(const ganamd_norm_desc* d, const void* gy, const void* x, const void* w, const void* b,
                          const void* slope, const double* stats, void* gx, void* gw, void* gb, void* gslope,
                          int accumulate, void* workspace, size_t workspace_bytes, hipStream_t st) {
  Full f;
  if (!make_plan(d, gn::BWD, f) || !gy || !x || !stats || (d->act == GANAMD_NORM_PRELU && !slope) ||
      (gslope && d->act != GANAMD_NORM_PRELU) || workspace_bytes < f.total || (f.total && !workspace))
    return GANAMD_EINVAL;
  if (!gx && !gw && !gb && !gslope) return GANAMD_OK;
  char* ws = static_cast<char*>(workspace);
  Args a = f.a;
  a.x = x; a.gy = gy; a.w = w; a.b = b; a.slope = d->act == GANAMD_NORM_PRELU ? slope : nullptr;
  a.o1 = gx; a.stats = const_cast<double*>(stats);
  a.par = gw || gb || gslope ? reinterpret_cast<float*>(ws + f.par) : nullptr;
  const int rc = run(d, f, a, ws, st);
  return rc != GANAMD_OK ? rc : fold_params(f, ws, gslope ? 3 : 2, gw, gb, gslope, d->param_dtype, accumulate, st);
}

int ganamd_group_norm_bwd_bwd(const ganamd_norm_desc* d, const void* ggx, const void* ggw, const void* ggb,
                              const void* ggslope, const void* gy, const void* x, const void* w, const void* b,
                              const void* slope, const double* stats, void* g_gy, void* g_x, void* g_w, void* g_b,
                              void* g_slope, int accumulate, void* workspace, size_t workspace_bytes, hipStream_t st) {
  Full f;
  if (!make_plan(d, gn::DBL, f) || !ggx || !gy || !x || !stats || !g_gy || !g_x ||
      (d->act == GANAMD_NORM_PRELU && !slope) || ((g_slope || ggslope) && d->act != GANAMD_NORM_PRELU) ||
      workspace_bytes < f.total || (f.total && !workspace))
    return GANAMD_EINVAL;
  char* ws = static_cast<char*>(workspace);
  Args a = f.a;
  a.x = x; a.gy = gy; a.v = ggx; a.w = w; a.b = b; a.slope = d->act == GANAMD_NORM_PRELU ? slope : nullptr;
  a.cw = ggw; a.cb = ggb; a.cs = ggslope;
  a.o1 = g_gy; a.o2 = g_x; a.stats = const_cast<double*>(stats);
  a.par = g_w || g_b || g_slope ? reinterpret_cast<float*>(ws + f.par) : nullptr;
  const int rc = run(d, f, a, ws, st);
  return rc != GANAMD_OK ? rc : fold_params(f, ws, g_slope ? 3 : 2, g_w, g_b, g_slope, d->param_dtype, accumulate, st);
}

}  // extern "C"
