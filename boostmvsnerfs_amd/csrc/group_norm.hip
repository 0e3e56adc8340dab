// Group normalisation with an activation, forward and backward, on channel-last and planar maps: what stands in for
// csrc/bn.hip where a step sees one image (batch statistics of one image are that image's own, differ between training and
// inference and have to be exchanged between ranks; a group's statistics are per sample and none of that).
//
//   mean, var over the M = C / G * S values of a (sample, group);  z = (x - mean) rstd w_c + b_c;  y = act(z)
//   g = dy act'(z);  db_c = sum g;  dw_c = sum g xhat;  dx = rstd (g w - (sum_g g w + xhat sum_g g w xhat) / M)
//   act(v) = v > 0 ? v : slope v (1 none, 0 ReLU, 0.01 leaky ReLU), or v / (1 + exp(-v)) (SiLU)
//
// Numbers.  Sums are 64-bit; the backward adds four terms at a time in 32 bits first.  Mean and variance are sum d and sum d^2 of
// d = x - pivot, the pivot the group's first value: (mean - pivot)^2 <= M var whatever the values are, so the difference that
// gives the variance loses at most M 2^-52 of it.  (Of x itself it would lose (mean / std)^2 2^-52: half a percent at an offset of 5e6
// standard deviations, which fp32 maps can hold.)  64 bits are not only for long sums: act' of the ReLUs jumps at z = 0, so
// the backward has to decide the sign of z as the exact value has it.  It computes z in 32 bits and, where |z| is within 2^-18 of
// its terms (a few values in a million), again in 64 with the saved 64-bit statistics.  x - mean is taken as (x - mh) - ml with
// mean = mh + ml, so a large common offset costs no accuracy.
//
// What bounds it: bytes, and for small maps the launches.  Two launches each way: sums of a chunk per workgroup -> partials; then
// every workgroup joins the partials of the groups it touches (always in the same order: bit-reproducible, no atomics) and writes
// its chunk.  The forward's two launches have the same chunk -> workgroup map, so it finds the chunk in its XCD's L2; the
// backward's second has the workgroups of dw and db in front (ceil(C / 8): another XCD where that is no multiple of 8) and finds it
// in the last-level cache.  Where a workgroup holds all of a group in registers the forward is one launch.  Averages of 20 runs:
//   3 x 8 x 512 x 640 fp32 (31.5 MB), ReLU: forward 10.9 + 11.8 us (the second 5.3 TB/s), backward 17.1 + 17.5 (5.4 TB/s)
//   4 x 320 x 64 x 64 bf16 (10.5 MB), SiLU: forward 19.3 us, the pair among others;  1 x 64 x 8 x 8 x 10 fp32: 6.4 us, one launch
//   1 x 8 x 64 x 64 x 80 planar (10.5 MB), leaky: forward 6.1 + 7.4 us, backward 7.7 + 8.2
#include <algorithm>

#include "bmv_common.hpp"

namespace bmv {

constexpr int kGnThreads = 256, kGnWaves = kGnThreads / 64;

template <int DT> struct GnType;
template <> struct GnType<0> { using T = float; };
template <> struct GnType<1> { using T = __bf16; };
template <> struct GnType<2> { using T = _Float16; };

// V values of T, loaded and stored as one access of V * sizeof(T) <= 16 bytes
template <typename T, int V>
struct alignas(sizeof(T) * V) GnVec {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ GnVec<T, V> gn_load(const T* p) {
  return *reinterpret_cast<const GnVec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void gn_store(T* p, const float* f) {
  GnVec<T, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = (T)f[j];      // to nearest even: the one rounding of a result
  *reinterpret_cast<GnVec<T, V>*>(p) = o;
}

// affine parameters: 32 bits (wdt 0) or the map's type
template <typename T>
__device__ __forceinline__ float gn_param(const void* p, int c, int wdt, float dflt) {
  if (!p) return dflt;
  return wdt == 0 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}

struct GnArgs {
  const void *x, *dy, *w, *b;
  void *out, *dw, *db;           // y / dx; dw, db (backward)
  double *mean, *rstd;           // (N, G): written by the forward, read by the backward
  double2* part;                 // [N * G][pieces]: (sum, sum of squares) / (sum g w, sum g w xhat)
  double2* partc;                // backward: per channel and piece (sum g, sum g xhat), element n * pcn + k * pck + c * pcc
  long S, M;
  long pcn, pck, pcc;
  int N, C, G, cg, wdt;
  int chunks, slabs, width;      // channel-last: row chunks, channel slabs of `width` channels.  planar: chunks of a plane
  long per;                      // rows (values of a plane) of a chunk
  int pieces, npc;               // pieces a (sample, group) is joined from; pieces per channel of partc
  int slab_pieces;               // channel-last: slabs that share a group (1 where slabs hold whole groups)
  int dwb;                       // backward: workgroups in front of the map's that finish dw and db
  float slope;
  double eps;
};

__device__ __forceinline__ double gn_wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// sum of the pieces of one (sample, group), by one wave, every lane gets it
__device__ __forceinline__ double2 gn_join(const double2* __restrict__ p, int pieces) {
  double a = 0., b = 0.;
  for (int k = threadIdx.x & 63; k < pieces; k += 64) a += p[k].x, b += p[k].y;
  return {gn_wave_sum(a), gn_wave_sum(b)};
}

struct GnStat {
  double mean, rstd;
};
// (s: of the differences from the pivot)
__device__ __forceinline__ GnStat gn_stat(double2 s, double pivot, double M, double eps) {
  const double d = s.x / M, var = s.y / M - d * d;
  return {pivot + d, 1. / sqrt((var > 0. || var != var ? var : 0.) + eps)};
}
// the pivot of group g of sample n
template <typename T>
__device__ __forceinline__ double gn_pivot_cl(const GnArgs& a, int n, int g) {
  return (double)(float)static_cast<const T*>(a.x)[(long)n * a.S * a.C + g * a.cg];
}
template <typename T>
__device__ __forceinline__ double gn_pivot_pl(const GnArgs& a, int n, int g) {
  return (double)(float)static_cast<const T*>(a.x)[((long)n * a.C + g * a.cg) * a.S];
}

// z > 0 as the exact z has it (see above)
__device__ __forceinline__ bool gn_positive(float z, float dsc, float b, float x, double mean, double rstd, float w) {
  if (fabsf(z) > 0x1p-18f * (fabsf(dsc) + fabsf(b))) return z > 0.f;
  return ((double)x - mean) * (rstd * (double)w) + (double)b > 0.;
}

template <bool SILU>
__device__ __forceinline__ float gn_act(float z, float slope) {
  if (SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));      // (1 ulp; a division is ten instructions)
  return z > 0.f ? z : (slope == 0.f ? (z != z ? z : 0.f) : slope * z);   // (0 * -inf would be NaN)
}

// g = dy act'(z)
template <bool SILU>
__device__ __forceinline__ float gn_grad(float dy, float x, float d, float sc, float b, float w, float slope, double mean,
                                         double rstd) {
  const float dsc = d * sc, z = dsc + b;
  if (SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return dy * s * (1.f + z * (1.f - s));
  }
  if (slope == 1.f) return dy;
  return gn_positive(z, dsc, b, x, mean, rstd, w) ? dy : (slope == 0.f ? 0.f : slope * dy);
}

// ---- channel-last ----------------------------------------------------------------------------------------------------
// Workgroup = (sample, channel slab, row chunk); thread = V consecutive channels (one 16-byte access where C allows) of
// every `rpi`-th row, so a thread's channels never change.  Lanes run over the slab's channels first: accesses are coalesced
// whatever C is.  ONE: V channels always lie in one group (C / G a multiple of V): one pair of sums instead of V.
struct GnCl {
  int n, slab, k, c0, nch, wv, cv, r0, rpi, c;
  long begin, end;
  bool on;
};
template <int V>
__device__ __forceinline__ GnCl gn_cl(const GnArgs& a, int bid) {
  GnCl t;
  t.k = bid % a.chunks;
  bid /= a.chunks;
  t.slab = bid % a.slabs, t.n = bid / a.slabs;
  t.c0 = t.slab * a.width, t.nch = min(a.width, a.C - t.c0);
  t.wv = t.nch / V, t.rpi = kGnThreads / t.wv;
  t.r0 = threadIdx.x / t.wv, t.cv = threadIdx.x - t.r0 * t.wv;
  t.on = t.r0 < t.rpi, t.c = t.c0 + t.cv * V;
  t.begin = min(t.k * a.per, a.S), t.end = min(t.begin + a.per, a.S);
  return t;
}

// A thread's V channels as E sums: 1 where they always lie in one group (C / G a multiple of V), 2 where groups have V channels
// or more (what is in front of a group border, what is behind it), else V.
// (cut: channels of the first up to its group's border)
template <int V, int E>
__device__ __forceinline__ int gn_entry(int cut, int j) {
  return E == V ? j : E == 1 ? 0 : j >= cut;
}
// the groups of channels c ... c + V - 1, one division
template <int V>
__device__ __forceinline__ void gn_group_of(int c, int cg, int* g) {
  int k = c / cg, left = (k + 1) * cg - c;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j && left == 0) ++k, left = cg;
    g[j] = k, --left;
  }
}

// sh: [row of the workgroup][vector of the slab][E] -> row 0: the sum over the workgroup's rows
template <int TH>
__device__ __forceinline__ void gn_cl_rows(const GnCl& t, int ne, double2* sh) {
  __syncthreads();
  int half = 1;
  while (half < t.rpi) half <<= 1;
  for (half >>= 1; half >= 1; half >>= 1) {          // rows r0 + half onto r0
    for (int i = threadIdx.x; i < half * ne; i += TH)
      if (i + half * ne < t.rpi * ne) sh[i].x += sh[i + half * ne].x, sh[i].y += sh[i + half * ne].y;
    __syncthreads();
  }
}
// ... and of it, group by group of the slab: lane 0 of a wave hands the group's two sums to `to`
template <int V, int E, int TH, typename F>
__device__ __forceinline__ void gn_cl_groups(const GnArgs& a, const GnCl& t, const double2* sh, F to) {
  const int lane = threadIdx.x & 63, g0 = t.c0 / a.cg, g1 = (t.c0 + t.nch - 1) / a.cg;
  for (int g = g0 + (int)(threadIdx.x >> 6); g <= g1; g += TH / 64) {
    const int lo = max(g * a.cg, t.c0) - t.c0, hi = min((g + 1) * a.cg, t.c0 + t.nch) - t.c0;   // channels of the slab
    double x = 0., y = 0.;
    if (E == V)
      for (int i = lo + lane; i < hi; i += 64) x += sh[i].x, y += sh[i].y;
    else
      for (int i = lo / V + lane; i <= (hi - 1) / V; i += 64) {
        const double2 v = sh[i * E + (E == 2 && (t.c0 + i * V) / a.cg != g)];
        x += v.x, y += v.y;
      }
    x = gn_wave_sum(x), y = gn_wave_sum(y);
    if (lane == 0) to(g, x, y);
  }
}
// the workgroup's piece of every group of its slab
template <int V, int E>
__device__ __forceinline__ void gn_cl_pieces(const GnArgs& a, const GnCl& t, const double2* sh) {
  gn_cl_groups<V, E, kGnThreads>(a, t, sh, [&](int g, double x, double y) {
    const int first = g * a.cg / a.width, last = ((g + 1) * a.cg - 1) / a.width;      // the slabs that share the group
    double2* to = a.part + ((long)t.n * a.G + g) * a.pieces + t.k;
    to[(t.slab - first) * a.chunks] = {x, y};
    if (t.slab == last)                              // (fewer than others share: the missing pieces are zero)
      for (int k = last - first + 1; k < a.slab_pieces; ++k) to[k * a.chunks] = {0., 0.};
  });
}

template <int V, int E>
__device__ __forceinline__ void gn_fold(const GnArgs& a, const GnCl& t, const double* s, const double* q, double2* sh) {
  double2 v[E];
  const int cut = (t.c / a.cg + 1) * a.cg - t.c;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = {0., 0.};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = gn_entry<V, E>(cut, j);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e == at) v[e].x += s[j], v[e].y += q[j];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sh[threadIdx.x * E + e] = v[e];
}

template <int DT, int V, int E>
__global__ void __launch_bounds__(kGnThreads) gn_cl_stats_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  __shared__ double2 sh[kGnThreads * E];
  const GnCl t = gn_cl<V>(a, blockIdx.x);
  if (t.on) {
    constexpr int A = E == 1 ? 1 : V;                // accumulators
    double s[V] = {}, q[V] = {}, pv[V];
    int gs[V];
    gn_group_of<V>(t.c, a.cg, gs);
#pragma unroll
    for (int j = 0; j < A; ++j) pv[j] = gn_pivot_cl<T>(a, t.n, gs[j]);
    const T* p = static_cast<const T*>(a.x) + (long)t.n * a.S * a.C + t.c;
    constexpr int U = 4;
    for (long r = t.begin + t.r0; r < t.end; r += U * t.rpi) {
      GnVec<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = gn_load<T, V>(p + min(r + u * t.rpi, t.end - 1) * a.C);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * t.rpi >= t.end) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double f = (double)(float)v[u].v[j] - pv[A == 1 ? 0 : j];
          s[A == 1 ? 0 : j] += f, q[A == 1 ? 0 : j] += f * f;
        }
      }
    }
    if (E == 1) sh[threadIdx.x] = {s[0], q[0]};
    else gn_fold<V, E>(a, t, s, q, sh);
  }
  gn_cl_rows<kGnThreads>(t, t.wv * E, sh);
  gn_cl_pieces<V, E>(a, t, sh);
}

// one piece per (sample, group) out of many: in front of the apply launch where its workgroups would join too many
__global__ void __launch_bounds__(kGnThreads) gn_finish_kernel(const double2* __restrict__ part, int pieces, long n,
                                                               double2* __restrict__ out) {
  const long i = (long)blockIdx.x * kGnWaves + (threadIdx.x >> 6);
  if (i >= n) return;
  const double2 s = gn_join(part + i * pieces, pieces);
  if ((threadIdx.x & 63) == 0) out[i] = s;
}

template <int DT, int V, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_cl_apply_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  extern __shared__ GnStat st[];                     // the slab's groups
  constexpr int U = 4;
  const GnCl t = gn_cl<V>(a, blockIdx.x);
  const long off = (long)t.n * a.S * a.C + t.c;
  const T* p = static_cast<const T*>(a.x) + off;
  T* o = static_cast<T*>(a.out) + off;
  // the first rows and the parameters are on their way while the partials are joined
  GnVec<T, V> v[U];
  float sc[V], b[V];
  if (t.on && t.begin < t.end) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = gn_load<T, V>(p + min(t.begin + t.r0 + u * t.rpi, t.end - 1) * a.C);
#pragma unroll
    for (int j = 0; j < V; ++j) sc[j] = gn_param<T>(a.w, t.c + j, a.wdt, 1.f), b[j] = gn_param<T>(a.b, t.c + j, a.wdt, 0.f);
  }
  const int g0 = t.c0 / a.cg, g1 = (t.c0 + t.nch - 1) / a.cg;
  for (int g = g0 + (threadIdx.x >> 6); g <= g1; g += kGnWaves) {
    const long i = (long)t.n * a.G + g;
    const GnStat s = gn_stat(gn_join(a.part + i * a.pieces, a.pieces), gn_pivot_cl<T>(a, t.n, g), (double)a.M, a.eps);
    if ((threadIdx.x & 63) == 0) {
      st[g - g0] = s;
      if (t.k == 0) a.mean[i] = s.mean, a.rstd[i] = s.rstd;     // (slabs that share a group write the same value)
    }
  }
  __syncthreads();
  if (!t.on) return;
  float mh[V], ml[V];
  int g[V];
  gn_group_of<V>(t.c, a.cg, g);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const GnStat s = st[g[j] - g0];
    mh[j] = (float)s.mean, ml[j] = (float)(s.mean - (double)mh[j]), sc[j] = (float)(s.rstd * (double)sc[j]);
  }
  for (long r = t.begin + t.r0; r < t.end; r += U * t.rpi) {
    GnVec<T, V> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = v[u];
    if (r + U * t.rpi < t.end) {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = gn_load<T, V>(p + min(r + (U + u) * t.rpi, t.end - 1) * a.C);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * t.rpi >= t.end) break;
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = gn_act<SILU>((((float)w[u].v[j] - mh[j]) - ml[j]) * sc[j] + b[j], a.slope);
      gn_store<T, V>(o + (r + u * t.rpi) * a.C, f);
    }
  }
}

// A whole (sample, slab of groups) in the registers of one workgroup, R accesses a thread: one launch instead of two
constexpr int kGnHold = 8;
template <int DT, int V, int E, int TH, bool SILU>
__global__ void __launch_bounds__(TH) gn_cl_whole_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  constexpr int R = kGnHold;
  __shared__ double2 sh[TH * E];
  extern __shared__ GnStat st[];                     // the slab's groups
  GnCl t = gn_cl<V>(a, blockIdx.x);
  t.rpi = TH / t.wv, t.on = t.r0 < t.rpi;            // (gn_cl counts 256 threads)
  const long off = (long)t.n * a.S * a.C + t.c;
  const T* p = static_cast<const T*>(a.x) + off;
  GnVec<T, V> v[R];
  double s[V] = {}, q[V] = {}, pv[V];
  int gs[V];
  if (t.on) {
    gn_group_of<V>(t.c, a.cg, gs);
#pragma unroll
    for (int u = 0; u < R; ++u) v[u] = gn_load<T, V>(p + min((long)t.r0 + u * t.rpi, a.S - 1) * a.C);
#pragma unroll
    for (int j = 0; j < (E == 1 ? 1 : V); ++j) pv[j] = gn_pivot_cl<T>(a, t.n, gs[j]);
#pragma unroll
    for (int u = 0; u < R; ++u) {
      if (t.r0 + u * t.rpi >= a.S) break;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double f = (double)(float)v[u].v[j] - pv[E == 1 ? 0 : j];
        s[E == 1 ? 0 : j] += f, q[E == 1 ? 0 : j] += f * f;
      }
    }
  }
  const int g0 = t.c0 / a.cg;
  if (E == 1 && a.width == a.cg) {                   // one group: a sum over all threads
    const double x = gn_wave_sum(s[0]), y = gn_wave_sum(q[0]);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = {x, y};
    __syncthreads();
    double2 sum = {0., 0.};
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) sum.x += sh[i].x, sum.y += sh[i].y;
    const GnStat m = gn_stat(sum, gn_pivot_cl<T>(a, t.n, g0), (double)a.M, a.eps);
    if (threadIdx.x == 0) st[0] = m, a.mean[(long)t.n * a.G + g0] = m.mean, a.rstd[(long)t.n * a.G + g0] = m.rstd;
  } else {
    if (t.on) {
      if (E == 1) sh[threadIdx.x] = {s[0], q[0]};
      else gn_fold<V, E>(a, t, s, q, sh);
    }
    gn_cl_rows<TH>(t, t.wv * E, sh);
    gn_cl_groups<V, E, TH>(a, t, sh, [&](int g, double x, double y) {
      const GnStat m = gn_stat({x, y}, gn_pivot_cl<T>(a, t.n, g), (double)a.M, a.eps);
      st[g - g0] = m;
      a.mean[(long)t.n * a.G + g] = m.mean, a.rstd[(long)t.n * a.G + g] = m.rstd;
    });
  }
  __syncthreads();
  if (!t.on) return;
  float mh[V], ml[V], sc[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const GnStat m = st[gs[j] - g0];
    mh[j] = (float)m.mean, ml[j] = (float)(m.mean - (double)mh[j]);
    sc[j] = (float)(m.rstd * (double)gn_param<T>(a.w, t.c + j, a.wdt, 1.f)), b[j] = gn_param<T>(a.b, t.c + j, a.wdt, 0.f);
  }
  T* o = static_cast<T*>(a.out) + off;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    if (t.r0 + u * t.rpi >= a.S) break;
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = gn_act<SILU>((((float)v[u].v[j] - mh[j]) - ml[j]) * sc[j] + b[j], a.slope);
    gn_store<T, V>(o + ((long)t.r0 + u * t.rpi) * a.C, f);
  }
}

template <int DT, int V, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_cl_bwd_reduce_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  __shared__ double2 sh[kGnThreads * V];
  const GnCl t = gn_cl<V>(a, blockIdx.x);
  if (t.on) {
    float mh[V], ml[V], sc[V], b[V], w[V];
    double mean[V], rstd[V], s[V], q[V];
    int gs[V];
    gn_group_of<V>(t.c, a.cg, gs);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const long i = (long)t.n * a.G + gs[j];
      mean[j] = a.mean[i], rstd[j] = a.rstd[i], s[j] = q[j] = 0.;
      mh[j] = (float)mean[j], ml[j] = (float)(mean[j] - (double)mh[j]);
      w[j] = gn_param<T>(a.w, t.c + j, a.wdt, 1.f), b[j] = gn_param<T>(a.b, t.c + j, a.wdt, 0.f);
      sc[j] = (float)(rstd[j] * (double)w[j]);
    }
    const long off = (long)t.n * a.S * a.C + t.c;
    const T *p = static_cast<const T*>(a.x) + off, *pd = static_cast<const T*>(a.dy) + off;
    constexpr int U = 4;
    for (long r = t.begin + t.r0; r < t.end; r += U * t.rpi) {
      GnVec<T, V> v[U], e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long ru = min(r + u * t.rpi, t.end - 1);      // (rows behind the chunk: read again, counted below as zero)
        v[u] = gn_load<T, V>(p + ru * a.C), e[u] = gn_load<T, V>(pd + ru * a.C);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // four terms in 32 bits, their sum in 64: a sum of four adds one 32-bit rounding to the terms' own
        float fs = 0.f, fq = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float x = (float)v[u].v[j], d = (x - mh[j]) - ml[j];
          const float g = gn_grad<SILU>((float)e[u].v[j], x, d, sc[j], b[j], w[j], a.slope, mean[j], rstd[j]);
          if (r + u * t.rpi < t.end) fs += g, fq += g * d;
        }
        s[j] += (double)fs, q[j] += (double)fq;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sh[threadIdx.x * V + j] = {s[j], q[j] * rstd[j]};
  }
  gn_cl_rows<kGnThreads>(t, t.nch, sh);
  for (int i = threadIdx.x; i < t.nch; i += kGnThreads) {
    const double2 v = sh[i];
    const int c = t.c0 + i;
    if (a.partc) a.partc[t.n * a.pcn + t.k * a.pck + c * a.pcc] = v;
    const double w = (double)gn_param<T>(a.w, c, a.wdt, 1.f);
    sh[i] = {v.x * w, v.y * w};
  }
  __syncthreads();
  gn_cl_pieces<V, V>(a, t, sh);
}

// dw and db out of the pieces: 8 channels a workgroup, 32 threads each, the samples and pieces of a channel in a fixed order
template <int DT>
__device__ __forceinline__ void gn_param_grads(const GnArgs& a, int wg) {
  using T = typename GnType<DT>::T;
  __shared__ double2 sw[kGnThreads];
  const int cl = threadIdx.x & 7, q = threadIdx.x >> 3, c = wg * 8 + cl;
  double x = 0., y = 0.;
  if (c < a.C)
    for (int i = q; i < a.N * a.npc; i += 32) {
      const int n = i / a.npc, k = i - n * a.npc;
      const double2 v = a.partc[n * a.pcn + k * a.pck + c * a.pcc];
      x += v.x, y += v.y;
    }
  sw[threadIdx.x] = {x, y};
  __syncthreads();
  if (q || c >= a.C) return;
  for (int i = 1; i < 32; ++i) x += sw[i * 8 + cl].x, y += sw[i * 8 + cl].y;
  if (a.wdt == 0) {
    if (a.db) static_cast<float*>(a.db)[c] = (float)x;
    if (a.dw) static_cast<float*>(a.dw)[c] = (float)y;
  } else {
    if (a.db) static_cast<T*>(a.db)[c] = (T)(float)x;
    if (a.dw) static_cast<T*>(a.dw)[c] = (T)(float)y;
  }
}

template <int DT, int V, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_cl_bwd_apply_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  extern __shared__ double2 sg[];                    // the slab's groups: the two sums over M
  if ((int)blockIdx.x < a.dwb) return gn_param_grads<DT>(a, blockIdx.x);
  constexpr int U = 4;
  const GnCl t = gn_cl<V>(a, blockIdx.x - a.dwb);
  const long off = (long)t.n * a.S * a.C + t.c;
  const T *p = static_cast<const T*>(a.x) + off, *pd = static_cast<const T*>(a.dy) + off;
  T* o = static_cast<T*>(a.out) + off;
  // the first rows, the statistics and the parameters are on their way while the partials are joined
  GnVec<T, V> v[U], e[U];
  float w[V], b[V];
  double mean[V], rstd[V];
  int gs[V];
  if (t.on && t.begin < t.end) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long at = min(t.begin + t.r0 + u * t.rpi, t.end - 1) * a.C;
      v[u] = gn_load<T, V>(p + at), e[u] = gn_load<T, V>(pd + at);
    }
    gn_group_of<V>(t.c, a.cg, gs);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const long i = (long)t.n * a.G + gs[j];
      mean[j] = a.mean[i], rstd[j] = a.rstd[i];
      w[j] = gn_param<T>(a.w, t.c + j, a.wdt, 1.f), b[j] = gn_param<T>(a.b, t.c + j, a.wdt, 0.f);
    }
  }
  const int g0 = t.c0 / a.cg, g1 = (t.c0 + t.nch - 1) / a.cg;
  for (int g = g0 + (threadIdx.x >> 6); g <= g1; g += kGnWaves) {
    const double2 s = gn_join(a.part + ((long)t.n * a.G + g) * a.pieces, a.pieces);
    if ((threadIdx.x & 63) == 0) sg[g - g0] = {s.x / (double)a.M, s.y / (double)a.M};
  }
  __syncthreads();
  if (!t.on || t.begin >= t.end) return;
  // dx = rstd w g - rstd m1 - (x - mean) rstd^2 m2
  float mh[V], ml[V], sc[V], c1[V], c2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const double2 m = sg[gs[j] - g0];
    mh[j] = (float)mean[j], ml[j] = (float)(mean[j] - (double)mh[j]);
    sc[j] = (float)(rstd[j] * (double)w[j]);
    c1[j] = (float)(rstd[j] * m.x), c2[j] = (float)(rstd[j] * rstd[j] * m.y);
  }
  for (long r = t.begin + t.r0; r < t.end; r += U * t.rpi) {
    GnVec<T, V> vn[U], en[U];
    if (r + U * t.rpi < t.end) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long at = min(r + (U + u) * t.rpi, t.end - 1) * a.C;
        vn[u] = gn_load<T, V>(p + at), en[u] = gn_load<T, V>(pd + at);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * t.rpi >= t.end) break;
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = (float)v[u].v[j], d = (x - mh[j]) - ml[j];
        const float g = gn_grad<SILU>((float)e[u].v[j], x, d, sc[j], b[j], w[j], a.slope, mean[j], rstd[j]);
        f[j] = (sc[j] * g - c1[j]) - d * c2[j];
      }
      gn_store<T, V>(o + (r + u * t.rpi) * a.C, f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = vn[u], e[u] = en[u];
  }
}

// ---- planar ----------------------------------------------------------------------------------------------------------
// Unit = (sample, channel, chunk of the plane), by a workgroup (TPU 256) or, where planes are short, by a wave (TPU 64);
// V values of the plane per access.
struct GnPl {
  long plane, begin, end;
  int n, c, k, t;
  bool on;
};
template <int TPU>
__device__ __forceinline__ GnPl gn_pl(const GnArgs& a, long bid) {
  GnPl p;
  const unsigned unit = (unsigned)bid * (kGnThreads / TPU) + (TPU == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  p.on = unit < (unsigned)a.N * a.C * a.chunks;           // (at most max(N C, 8192) units: gn_plan, gn_bad)
  p.t = threadIdx.x & (TPU - 1);
  const unsigned plane = unit / a.chunks;
  p.k = (int)(unit - plane * a.chunks), p.plane = plane;
  p.n = (int)(plane / a.C), p.c = (int)(plane - (unsigned)p.n * a.C);
  p.begin = min(p.k * a.per, a.S), p.end = min(p.begin + a.per, a.S);      // (chunks begin at 16-byte borders of the plane)
  return p;
}
// sum over the unit; every thread of a wave-unit, thread 0 of a workgroup-unit has it
template <int TPU>
__device__ __forceinline__ double2 gn_unit_sum(double x, double y) {
  x = gn_wave_sum(x), y = gn_wave_sum(y);
  if (TPU == 64) return {x, y};
  __shared__ double2 sh[kGnWaves];
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = {x, y};
  __syncthreads();
  x = y = 0.;
#pragma unroll
  for (int i = 0; i < kGnWaves; ++i) x += sh[i].x, y += sh[i].y;
  return {x, y};
}

template <int DT, int V, int TPU>
__global__ void __launch_bounds__(kGnThreads) gn_pl_stats_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  const GnPl t = gn_pl<TPU>(a, blockIdx.x);
  double s = 0., q = 0.;
  if (t.on) {
    const T* p = static_cast<const T*>(a.x) + t.plane * a.S;
    const double pivot = gn_pivot_pl<T>(a, t.n, t.c / a.cg);
    constexpr int U = 4;
    long i = t.begin + t.t * V;
    for (; i + (U - 1) * TPU * V < t.end; i += U * TPU * V) {
      GnVec<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = gn_load<T, V>(p + i + u * TPU * V);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double f = (double)(float)v[u].v[j] - pivot;
          s += f, q += f * f;
        }
    }
    for (; i < t.end; i += TPU * V) {
      const GnVec<T, V> v = gn_load<T, V>(p + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double f = (double)(float)v.v[j] - pivot;
        s += f, q += f * f;
      }
    }
  }
  const double2 v = gn_unit_sum<TPU>(s, q);
  if (t.on && t.t == 0) {
    const int g = t.c / a.cg;
    a.part[((long)t.n * a.G + g) * a.pieces + (t.c - g * a.cg) * a.chunks + t.k] = v;
  }
}

template <int DT, int V, int TPU, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_pl_apply_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  const GnPl t = gn_pl<TPU>(a, blockIdx.x);
  if (!t.on) return;                                 // (workgroup-units: the whole workgroup)
  const int g = t.c / a.cg;
  const long ig = (long)t.n * a.G + g;
  const GnStat s = gn_stat(gn_join(a.part + ig * a.pieces, a.pieces), gn_pivot_pl<T>(a, t.n, g), (double)a.M, a.eps);
  if (t.t == 0 && t.k == 0 && t.c == g * a.cg) a.mean[ig] = s.mean, a.rstd[ig] = s.rstd;
  const float mh = (float)s.mean, ml = (float)(s.mean - (double)mh);
  const float sc = (float)(s.rstd * (double)gn_param<T>(a.w, t.c, a.wdt, 1.f)), b = gn_param<T>(a.b, t.c, a.wdt, 0.f);
  const T* p = static_cast<const T*>(a.x) + t.plane * a.S;
  T* o = static_cast<T*>(a.out) + t.plane * a.S;
  for (long i = t.begin + t.t * V; i < t.end; i += TPU * V) {
    const GnVec<T, V> v = gn_load<T, V>(p + i);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = gn_act<SILU>((((float)v.v[j] - mh) - ml) * sc + b, a.slope);
    gn_store<T, V>(o + i, f);
  }
}

// A whole (sample, group) -- one run of C / G planes -- in the registers of one workgroup
template <int DT, int V, int TH, bool SILU>
__global__ void __launch_bounds__(TH) gn_pl_whole_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  constexpr int R = kGnHold;
  __shared__ double2 sh[TH / 64];
  const int n = blockIdx.x / a.G, g = blockIdx.x - n * a.G, sv = (int)(a.S / V), nv = a.cg * sv;      // accesses of a plane, of the group
  const long off = ((long)n * a.C + (long)g * a.cg) * a.S;
  const T* p = static_cast<const T*>(a.x) + off;
  GnVec<T, V> v[R];
  double s = 0., q = 0.;
  const double pivot = (double)(float)p[0];
#pragma unroll
  for (int u = 0; u < R; ++u) v[u] = gn_load<T, V>(p + (long)min((int)threadIdx.x + u * TH, nv - 1) * V);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    if ((int)threadIdx.x + u * TH >= nv) break;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double f = (double)(float)v[u].v[j] - pivot;
      s += f, q += f * f;
    }
  }
  s = gn_wave_sum(s), q = gn_wave_sum(q);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = {s, q};
  __syncthreads();
  s = q = 0.;
#pragma unroll
  for (int i = 0; i < TH / 64; ++i) s += sh[i].x, q += sh[i].y;
  const GnStat m = gn_stat({s, q}, pivot, (double)a.M, a.eps);
  if (threadIdx.x == 0) a.mean[blockIdx.x] = m.mean, a.rstd[blockIdx.x] = m.rstd;
  const float mh = (float)m.mean, ml = (float)(m.mean - (double)mh);
  T* o = static_cast<T*>(a.out) + off;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int i = threadIdx.x + u * TH;
    if (i >= nv) break;
    const int c = g * a.cg + i / sv;
    const float sc = (float)(m.rstd * (double)gn_param<T>(a.w, c, a.wdt, 1.f)), b = gn_param<T>(a.b, c, a.wdt, 0.f);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = gn_act<SILU>((((float)v[u].v[j] - mh) - ml) * sc + b, a.slope);
    gn_store<T, V>(o + (long)i * V, f);
  }
}

template <int DT, int V, int TPU, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_pl_bwd_reduce_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  const GnPl t = gn_pl<TPU>(a, blockIdx.x);
  double s = 0., q = 0., rstd = 0.;
  float w = 0.f;
  if (t.on) {
    const long ig = (long)t.n * a.G + t.c / a.cg;
    const double mean = a.mean[ig];
    rstd = a.rstd[ig];
    const float mh = (float)mean, ml = (float)(mean - (double)mh), b = gn_param<T>(a.b, t.c, a.wdt, 0.f);
    w = gn_param<T>(a.w, t.c, a.wdt, 1.f);
    const float sc = (float)(rstd * (double)w);
    const T *p = static_cast<const T*>(a.x) + t.plane * a.S, *pd = static_cast<const T*>(a.dy) + t.plane * a.S;
    constexpr int U = 4;
    for (long i = t.begin + t.t * V; i < t.end; i += U * TPU * V) {
      GnVec<T, V> v[U], e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long iu = i + u * TPU * V < t.end ? i + u * TPU * V : i;
        v[u] = gn_load<T, V>(p + iu), e[u] = gn_load<T, V>(pd + iu);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float fs = 0.f, fq = 0.f;                         // (four terms in 32 bits, their sum in 64, as in gn_cl_bwd_reduce_kernel)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float x = (float)v[u].v[j], d = (x - mh) - ml;
          const float gr = gn_grad<SILU>((float)e[u].v[j], x, d, sc, b, w, a.slope, mean, rstd);
          if (i + u * TPU * V < t.end) fs += gr, fq += gr * d;
        }
        s += (double)fs, q += (double)fq;
      }
    }
  }
  double2 v = gn_unit_sum<TPU>(s, q);
  if (t.on && t.t == 0) {
    v.y *= rstd;
    if (a.partc) a.partc[t.n * a.pcn + t.k * a.pck + t.c * a.pcc] = v;
    const int g = t.c / a.cg;
    a.part[((long)t.n * a.G + g) * a.pieces + (t.c - g * a.cg) * a.chunks + t.k] = {v.x * (double)w, v.y * (double)w};
  }
}

template <int DT, int V, int TPU, bool SILU>
__global__ void __launch_bounds__(kGnThreads) gn_pl_bwd_apply_kernel(GnArgs a) {
  using T = typename GnType<DT>::T;
  if ((int)blockIdx.x < a.dwb) return gn_param_grads<DT>(a, blockIdx.x);
  const GnPl t = gn_pl<TPU>(a, (long)blockIdx.x - a.dwb);
  if (!t.on) return;
  const long ig = (long)t.n * a.G + t.c / a.cg;
  const double2 sum = gn_join(a.part + ig * a.pieces, a.pieces);
  const double mean = a.mean[ig], rstd = a.rstd[ig];
  const float mh = (float)mean, ml = (float)(mean - (double)mh), b = gn_param<T>(a.b, t.c, a.wdt, 0.f);
  const float w = gn_param<T>(a.w, t.c, a.wdt, 1.f), sc = (float)(rstd * (double)w);
  const float c1 = (float)(rstd * sum.x / (double)a.M), c2 = (float)(rstd * rstd * sum.y / (double)a.M);
  const T *p = static_cast<const T*>(a.x) + t.plane * a.S, *pd = static_cast<const T*>(a.dy) + t.plane * a.S;
  T* o = static_cast<T*>(a.out) + t.plane * a.S;
  for (long i = t.begin + t.t * V; i < t.end; i += TPU * V) {
    const GnVec<T, V> v = gn_load<T, V>(p + i), e = gn_load<T, V>(pd + i);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = (float)v.v[j], d = (x - mh) - ml;
      f[j] = (sc * gn_grad<SILU>((float)e.v[j], x, d, sc, b, w, a.slope, mean, rstd) - c1) - d * c2;
    }
    gn_store<T, V>(o + i, f);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr long kGnThreadsMost = (1l << 32) - 1;      // of a launch
constexpr int kGnMaxJoin = 1024;      // double2 that a workgroup of the apply launch joins; above, one more launch does
constexpr int kGnFew = 384;           // workgroups, fewer of which cost more than that launch (200416 x 19 fp16, 19 groups: 80 us with 53, 33)

struct GnPlan {
  GnArgs a;
  int V, tpu;
  int whole, held;                     // forward in one launch: its workgroups' threads, or 0; channels that one holds
  bool last, finish;
  long wgs, part, partc, fin;          // workgroups of the map; double2 of the workspace's three parts
};

static int gn_vec(long n, int size) {  // values per access: 16 bytes where the contiguous extent allows it
  for (int v = 16 / size; v > 1; v >>= 1)
    if (n % v == 0) return v;
  return 1;
}
// threads of a workgroup that holds `accesses` of them, kGnHold a thread; 0: too many
static int gn_whole(long accesses) { return accesses <= 256 * kGnHold ? 256 : accesses <= 1024 * kGnHold ? 1024 : 0; }

static GnPlan gn_plan(int N, int C, long S, int G, int dtype, int last, bool backward) {
  GnPlan p{};
  GnArgs& a = p.a;
  a.N = N, a.C = C, a.S = S, a.G = G, a.cg = C / G, a.M = (long)a.cg * S;
  const int size = dtype == 0 ? 4 : 2;
  p.last = last != 0;
  if (p.last) {
    p.V = gn_vec(C, size);
    const int cv = C / p.V;
    // A slab is whole groups where 256 accesses hold one: the fewest that are 128 bytes of a row (a cache line), or the number
    // among the next three that leaves the fewest of the 256 threads without a column.  Wide groups are cut in equal slabs.
    int unit = a.cg / p.V;             // accesses from one group border that is an access border to the next
    if (a.cg % p.V) {
      int lcm = a.cg;
      while (lcm % p.V) lcm += a.cg;
      unit = lcm / p.V;
    }
    int wv;
    if (unit > kGnThreads) {
      const int k = (cv + kGnThreads - 1) / kGnThreads;
      wv = (cv + k - 1) / k;
    } else {
      const int line = (128 / (p.V * size) + unit - 1) / unit;
      int best = -1;
      wv = unit;
      for (int k = line; k < line + 4; ++k) {
        const int w = std::min(unit * k, cv), used = w <= kGnThreads ? kGnThreads / w * w : 0;
        if (used > best + 8) best = used, wv = w;
      }
      if (best <= 0) wv = unit;
    }
    a.width = wv * p.V, a.slabs = (C + a.width - 1) / a.width;
    a.slab_pieces = 1;
    if (a.width % a.cg)
      for (int g = 0; g < G; ++g) {
        const int shared = ((g + 1) * a.cg - 1) / a.width - g * a.cg / a.width + 1;
        if (shared > a.slab_pieces) a.slab_pieces = shared;
      }
    // Rows of a chunk: 512 workgroups (two on a compute unit), of at least 2 accesses a thread.  What a workgroup does besides its
    // rows -- joining the pieces, adding its rows' sums -- costs about as much as 8 accesses a thread, and more workgroups are more
    // pieces to join: 3 x 32 x 128 x 160 backward 29.4 us with 1024, 17.6 with 512; 4 x 320 x 64 x 64 bf16 41.7, 30.6.  The forward's
    // is less: 1024 where they have 7 accesses or more (3 x 8 x 512 x 640 23.4 -> 22.0 us, 3 x 32 x 512 x 640 72.8 -> 67.5).  And
    // so few that their pieces need no launch of their own (1 x 256 x 128 x 128 bf16 forward 21 -> 16.4 us).
    const long rpi = kGnThreads / wv, touched = std::min<long>((a.width + a.cg - 1) / a.cg + 1, G);
    const long target = !backward && (long)N * a.slabs * S >= 7 * rpi * 1024 ? 1024 : 512;
    const long few = kGnMaxJoin / (touched * a.slab_pieces), most = target / ((long)N * a.slabs);
    const long wgs = std::max(1l, few * N * a.slabs >= kGnFew ? std::min(most, few) : most);
    a.per = std::max(2 * rpi, ((S + wgs - 1) / wgs + rpi - 1) / rpi * rpi);
    const long chunks = (S + a.per - 1) / a.per;
    a.chunks = (int)chunks, a.pieces = a.chunks * a.slab_pieces, a.npc = a.chunks;
    a.pcn = (long)a.chunks * C, a.pck = C, a.pcc = 1;
    p.wgs = (long)N * a.slabs * a.chunks;
    p.finish = touched * a.pieces > kGnMaxJoin;
    // (one launch: the fewest channels that are whole groups and whole accesses; kGnHold passes of threads / accesses rows)
    if (unit <= kGnThreads) {
      p.held = unit * p.V;
      p.whole = S <= 256 / unit * kGnHold ? 256 : S <= 1024 / unit * kGnHold && (a.cg % p.V == 0 || a.cg >= p.V) ? 1024 : 0;
    }
  } else {
    p.V = gn_vec(S, size);
    p.tpu = S >= 4096 ? 256 : 64;
    long chunks = (S + p.tpu * p.V * 4 - 1) / (p.tpu * p.V * 4);
    long cap = 2048 / ((long)N * C) * (256 / p.tpu);
    if (cap < 1) cap = 1;
    if (chunks > cap) chunks = cap;
    a.per = ((S + chunks - 1) / chunks + 15) & ~15l;
    a.chunks = (int)chunks, a.pieces = a.cg * a.chunks, a.npc = a.chunks;
    a.pcn = (long)C * a.chunks, a.pck = 1, a.pcc = a.chunks;
    p.wgs = ((long)N * C * a.chunks * p.tpu + 255) / 256;
    p.finish = a.pieces > (p.tpu == 64 ? kGnMaxJoin / 4 : kGnMaxJoin);
    p.whole = gn_whole(a.M / p.V);
  }
  if ((long)N * (p.last ? C / std::max(p.held, 1) : G) * p.whole > kGnThreadsMost) p.whole = 0;
  a.dwb = (C + 7) / 8;
  p.part = (long)N * G * a.pieces, p.fin = p.finish ? (long)N * G : 0, p.partc = (long)N * C * a.npc;
  return p;
}

template <int DT, int V, bool SILU>
static void gn_whole_launch(const GnPlan& p, const GnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((long)a.N * (p.last ? a.C / p.held : a.G)));
  if (!p.last) {
    if (p.whole == 256) hipLaunchKernelGGL((gn_pl_whole_kernel<DT, V, 256, SILU>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((gn_pl_whole_kernel<DT, V, 1024, SILU>), grid, dim3(1024), 0, st, a);
    return;
  }
  GnArgs b = a;
  b.chunks = 1, b.width = p.held, b.slabs = a.C / p.held;
  const unsigned lds = (unsigned)(p.held / a.cg) * sizeof(GnStat);
#define BMV_GN_WHOLE(E, TH) hipLaunchKernelGGL((gn_cl_whole_kernel<DT, V, E, TH, SILU>), grid, dim3(TH), lds, st, b)
  if (a.cg % V == 0) {
    if (p.whole == 256) BMV_GN_WHOLE(1, 256);
    else BMV_GN_WHOLE(1, 1024);
  } else if (a.cg >= V) {
    if (p.whole == 256) BMV_GN_WHOLE((V < 2 ? 1 : 2), 256);
    else BMV_GN_WHOLE((V < 2 ? 1 : 2), 1024);
  } else BMV_GN_WHOLE(V, 256);
#undef BMV_GN_WHOLE
}

template <int DT, int V>
static void gn_fwd_launch(const GnPlan& p, GnArgs a, bool silu, hipStream_t st) {
  if (p.whole) {
    if (silu) gn_whole_launch<DT, V, true>(p, a, st);
    else gn_whole_launch<DT, V, false>(p, a, st);
    return;
  }
  const dim3 grid((unsigned)p.wgs), block(kGnThreads);
  if (p.last) {
    if (a.cg % V == 0) hipLaunchKernelGGL((gn_cl_stats_kernel<DT, V, 1>), grid, block, 0, st, a);
    else if (a.cg >= V) hipLaunchKernelGGL((gn_cl_stats_kernel<DT, V, (V < 2 ? 1 : 2)>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gn_cl_stats_kernel<DT, V, V>), grid, block, 0, st, a);
  } else if (p.tpu == 256) hipLaunchKernelGGL((gn_pl_stats_kernel<DT, V, 256>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((gn_pl_stats_kernel<DT, V, 64>), grid, block, 0, st, a);
  if (p.finish) {
    hipLaunchKernelGGL(gn_finish_kernel, dim3(cdiv((long)a.N * a.G, kGnWaves)), block, 0, st, a.part, a.pieces, (long)a.N * a.G, a.part + p.part);
    a.part += p.part, a.pieces = 1;
  }
  const unsigned lds = (unsigned)((a.width + a.cg - 1) / a.cg + 1) * sizeof(GnStat);
#define BMV_GN_APPLY(SILU)                                                                                      \
  if (p.last) hipLaunchKernelGGL((gn_cl_apply_kernel<DT, V, SILU>), grid, block, lds, st, a);                   \
  else if (p.tpu == 256) hipLaunchKernelGGL((gn_pl_apply_kernel<DT, V, 256, SILU>), grid, block, 0, st, a);     \
  else hipLaunchKernelGGL((gn_pl_apply_kernel<DT, V, 64, SILU>), grid, block, 0, st, a)
  if (silu) { BMV_GN_APPLY(true); } else { BMV_GN_APPLY(false); }
#undef BMV_GN_APPLY
}

template <int DT, int V, bool SILU>
static void gn_bwd_launch(const GnPlan& p, GnArgs a, hipStream_t st) {
  const dim3 grid((unsigned)p.wgs), block(kGnThreads);
  if (!a.partc) a.dwb = 0;
  if (p.last) hipLaunchKernelGGL((gn_cl_bwd_reduce_kernel<DT, V, SILU>), grid, block, 0, st, a);
  else if (p.tpu == 256) hipLaunchKernelGGL((gn_pl_bwd_reduce_kernel<DT, V, 256, SILU>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((gn_pl_bwd_reduce_kernel<DT, V, 64, SILU>), grid, block, 0, st, a);
  if (p.finish) {
    hipLaunchKernelGGL(gn_finish_kernel, dim3(cdiv((long)a.N * a.G, kGnWaves)), block, 0, st, a.part, a.pieces, (long)a.N * a.G, a.part + p.part);
    a.part += p.part, a.pieces = 1;
  }
  const dim3 grid2((unsigned)(p.wgs + a.dwb));
  const unsigned lds = (unsigned)((a.width + a.cg - 1) / a.cg + 1) * sizeof(double2);
  if (p.last) hipLaunchKernelGGL((gn_cl_bwd_apply_kernel<DT, V, SILU>), grid2, block, lds, st, a);
  else if (p.tpu == 256) hipLaunchKernelGGL((gn_pl_bwd_apply_kernel<DT, V, 256, SILU>), grid2, block, 0, st, a);
  else hipLaunchKernelGGL((gn_pl_bwd_apply_kernel<DT, V, 64, SILU>), grid2, block, 0, st, a);
}

template <int DT, int V>
static void gn_launch(const GnPlan& p, const GnArgs& a, bool bwd, bool silu, hipStream_t st) {
  if (!bwd) gn_fwd_launch<DT, V>(p, a, silu, st);
  else if (silu) gn_bwd_launch<DT, V, true>(p, a, st);
  else gn_bwd_launch<DT, V, false>(p, a, st);
}

static void gn_dispatch(const GnPlan& p, const GnArgs& a, int dtype, bool bwd, bool silu, hipStream_t st) {
#define BMV_GN_V(DT, VEC) if (p.V == VEC) return gn_launch<DT, VEC>(p, a, bwd, silu, st)
  if (dtype == 0) {
    BMV_GN_V(0, 4);
    BMV_GN_V(0, 2);
    BMV_GN_V(0, 1);
  } else if (dtype == 1) {
    BMV_GN_V(1, 8);
    BMV_GN_V(1, 4);
    BMV_GN_V(1, 2);
    BMV_GN_V(1, 1);
  } else {
    BMV_GN_V(2, 8);
    BMV_GN_V(2, 4);
    BMV_GN_V(2, 2);
    BMV_GN_V(2, 1);
  }
#undef BMV_GN_V
}

static bool gn_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static const char* gn_bad(const bmv_group_norm_spec* s) {
  if (!s) return "no spec";
  if (s->N <= 0 || s->C <= 0 || s->S <= 0) return "bad shape";
  if (s->G <= 0 || s->C % s->G) return "the channels are no multiple of the groups";
  if (s->dtype < 0 || s->dtype > 2) return "unknown type";
  if (s->param_dtype != 0 && s->param_dtype != s->dtype) return "weight and bias are 32-bit or of the map's type";
  if (s->act != 0 && s->act != 1) return "unknown activation";
  if (!(s->eps >= 0.)) return "eps must not be negative";
  if ((long)s->N * s->C > (1l << 24) || s->S > (1l << 40) / ((long)s->N * s->C)) return "the map is too large (N C up to 2^24, N C S up to 2^40)";
  return nullptr;
}
// the plan of a call, or why there is none
static const char* gn_plan_of(const bmv_group_norm_spec* s, bool backward, GnPlan& p) {
  if (const char* bad = gn_bad(s)) return bad;
  p = gn_plan(s->N, s->C, s->S, s->G, s->dtype, s->channels_last, backward);
  return (p.wgs + p.a.dwb) * kGnThreads > kGnThreadsMost ? "the map has too many workgroups for a launch" : nullptr;
}

}  // namespace bmv

using namespace bmv;

extern "C" {

long bmv_group_norm_workspace(const bmv_group_norm_spec* spec, int backward) {
  GnPlan p;
  const char* bad = gn_plan_of(spec, backward != 0, p);
  BMV_REQUIRE(!bad, "bmv_group_norm_workspace: %s", bad);
  return 2 * (p.part + p.fin + (backward ? p.partc : 0));
}

int bmv_group_norm_fwd(const bmv_group_norm_spec* spec, const void* x, const void* weight, const void* bias, double* stats,
                       double* workspace, void* y, bmv_stream_t stream) {
  GnPlan p;
  const char* bad = gn_plan_of(spec, false, p);
  BMV_REQUIRE(!bad, "bmv_group_norm_fwd: %s", bad);
  BMV_REQUIRE(x && stats && workspace && y, "bmv_group_norm_fwd: null pointer");
  BMV_REQUIRE(gn_aligned(x) && gn_aligned(y) && gn_aligned(workspace), "bmv_group_norm_fwd: x, y and workspace begin at 16-byte addresses");
  GnArgs a = p.a;
  a.x = x, a.w = weight, a.b = bias, a.out = y, a.wdt = spec->param_dtype, a.eps = spec->eps, a.slope = spec->slope;
  a.mean = stats, a.rstd = stats + (long)a.N * a.G;
  a.part = reinterpret_cast<double2*>(workspace);
  gn_dispatch(p, a, spec->dtype, false, spec->act == 1, as_stream(stream));
  BMV_LAUNCH_END("bmv_group_norm_fwd");
}

int bmv_group_norm_bwd(const bmv_group_norm_spec* spec, const void* x, const void* dy, const void* weight, const void* bias,
                       const double* stats, double* workspace, void* dx, void* dweight, void* dbias, bmv_stream_t stream) {
  GnPlan p;
  const char* bad = gn_plan_of(spec, true, p);
  BMV_REQUIRE(!bad, "bmv_group_norm_bwd: %s", bad);
  BMV_REQUIRE(x && dy && stats && workspace && dx, "bmv_group_norm_bwd: null pointer");
  BMV_REQUIRE(gn_aligned(x) && gn_aligned(dy) && gn_aligned(dx) && gn_aligned(workspace),
              "bmv_group_norm_bwd: x, dy, dx and workspace begin at 16-byte addresses");
  GnArgs a = p.a;
  a.x = x, a.dy = dy, a.w = weight, a.b = bias, a.out = dx, a.dw = dweight, a.db = dbias, a.wdt = spec->param_dtype, a.slope = spec->slope;
  a.mean = const_cast<double*>(stats), a.rstd = a.mean + (long)a.N * a.G;
  a.part = reinterpret_cast<double2*>(workspace);
  a.partc = dweight || dbias ? a.part + p.part + p.fin : nullptr;
  gn_dispatch(p, a, spec->dtype, true, spec->act == 1, as_stream(stream));
  BMV_LAUNCH_END("bmv_group_norm_bwd");
}

}  // extern "C"
