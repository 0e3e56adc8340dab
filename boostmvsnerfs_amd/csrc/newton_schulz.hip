// Newton-Schulz orthogonalisation of a list of matrices, and the optimiser's step around it (momentum before, the decayed
// update of the weights behind it): what train.py's Adam step is to element-wise updates, for whole matrices.
//
//   X_0 = U / max(|U|_F, eps) with the short side as rows (m <= n); steps times:
//   A = X X^T,  Q = a I + b A + c A A,  X <- Q X.       The polynomial moves every singular value towards 1.
//   Step: buf <- mu buf + (1 - mu) g,  U = (1 - mu) g + mu buf (Nesterov) or buf,  w <- w (1 - lr decay) - lr scale X.
//
// Numbers.  A near-zero singular value grows by a = 3.4 a step, and with it whatever error X carried in its direction: the
// products need fp32 accuracy, whatever type the matrices have.  They run on the bf16 matrix cores with every fp32 operand as
// three bf16 pieces (hi + mid + lo: its 24 significand bits exactly) and the six products that are not below 2^-25, sums in
// fp32: 2.5 PFLOP/s / 6 against the 0.157 of the fp32 matrix instructions.  |U|_F is a 64-bit sum.
//
// Every operand is kept as its three pieces from the moment it is computed (one split per value, not one per use), in the
// orientation in which its k axis is contiguous, so all three products are L R^T of row-major operands and LDS tiles are
// filled by 16-byte DMA with no registers in between: A from X (k = n), A A from the symmetric A (k = m), Q X from Q and X^T
// (k = m); X is therefore written in both orientations.  A and Q are symmetric: only tiles on and below the diagonal are
// computed, the others are written as their transposes.
// One launch per stage for the whole list: a workgroup finds its matrix and tile in a table of the kernel arguments.
#include <algorithm>
#include <vector>

#include "bmv_common.hpp"

namespace bmv {

using nsb8 = __attribute__((ext_vector_type(8))) __bf16;
using nsf16 = __attribute__((ext_vector_type(16))) float;
using nsi4 = __attribute__((ext_vector_type(4))) int;

constexpr int kNsList = 40;      // matrices per launch (the table travels in the kernel arguments)
constexpr int kNsTile = 128;     // output tile of a workgroup; matrices are padded to it with zeros
constexpr int kNsStrip = 512;    // columns of a preparing workgroup's strip of 64 rows

struct NsItem {
  const void* src;      // U, or the gradient
  void* dst;            // the result, or the weights that the step updates
  float* buf;           // momentum (step), or null
  long ws;              // byte offset of this matrix' pieces in the workspace
  int rows, cols;       // of src / dst
  float scale;          // step: lr * scale of this matrix
  int wg0;              // first workgroup of this matrix in the launch
};
struct NsArgs {
  NsItem it[kNsList];
  char* ws;
  double* sq;           // partial sums of squares: [item][strip], kNsList * sqn of them
  int count, sqn, dtype, muon, nesterov, first, last, flip;
  float a, b, c, eps, mu, nu, keep;      // nu: 1 - mu, rounded once
};

// short side m, long side n, padded
struct NsShape {
  int m, n, mp, np;
  bool tall;            // the source is n x m: X is its transpose
  __host__ __device__ NsShape(int rows, int cols) {
    tall = rows > cols;
    m = tall ? cols : rows, n = tall ? rows : cols;
    mp = (m + kNsTile - 1) & ~(kNsTile - 1), np = (n + kNsTile - 1) & ~(kNsTile - 1);
  }
  __host__ __device__ long big() const { return (long)mp * np; }
  __host__ __device__ long sym() const { return (long)mp * mp; }
};
// the pieces of a matrix: plane p of an operand begins p * (elements of a plane) behind its first
struct NsPlanes {
  __bf16 *x, *xt, *xt1, *a, *q;      // xt, xt1: X^T before and after a step, in turn
  __device__ NsPlanes(char* ws, const NsShape& s) {
    x = reinterpret_cast<__bf16*>(ws);
    xt = x + 3 * s.big(), xt1 = xt + 3 * s.big(), a = xt1 + 3 * s.big(), q = a + 3 * s.sym();
  }
};
static long ns_bytes(const NsShape& s) { return (9 * s.big() + 6 * s.sym()) * 2; }

__device__ __forceinline__ int ns_find(const NsArgs& g, int wg) {
  int i = 0;
  while (i + 1 < g.count && g.it[i + 1].wg0 <= wg) ++i;
  return __builtin_amdgcn_readfirstlane(i);
}

__device__ __forceinline__ float ns_read(const void* p, long i, int dtype) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  if (dtype == 1) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void ns_write(void* p, long i, int dtype, float v) {
  if (dtype == 0) static_cast<float*>(p)[i] = v;
  else if (dtype == 1) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}
// what the iteration starts from, before its norm is divided out; `fresh`: the momentum is moved first
__device__ __forceinline__ float ns_start(const NsArgs& g, const NsItem& it, long i, bool fresh) {
  const float v = ns_read(it.src, i, g.dtype);
  if (!g.muon) return v;
  float m = it.buf[i];
  if (fresh) m = g.mu * m + g.nu * v, it.buf[i] = m;
  return g.nesterov ? g.nu * v + g.mu * m : m;
}
__device__ __forceinline__ void ns_result(const NsArgs& g, const NsItem& it, long i, float x) {
  ns_write(it.dst, i, g.dtype, g.muon ? ns_read(it.dst, i, g.dtype) * g.keep - it.scale * x : x);
}

// x = p[0] + p[1] + p[2], exactly: every piece is the nearest bf16 to what the pieces before it leave (to nearest, not
// truncated: what the dropped products of the pieces amount to is then below 2^-25 and of either sign, not 2^-21 of one)
__device__ __forceinline__ void ns_split(float x, __bf16 p[3]) {
  p[0] = (__bf16)x;
  const float r = x - (float)p[0];
  p[1] = (__bf16)r;
  p[2] = (__bf16)(r - (float)p[1]);
}
// eight consecutive values as three 16-byte stores
__device__ __forceinline__ void ns_store8(__bf16* p, long plane, const float* v) {
  nsb8 o[3];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    __bf16 q[3];
    ns_split(v[j], q);
#pragma unroll
    for (int k = 0; k < 3; ++k) o[k][j] = q[k];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<nsb8*>(p + k * plane) = o[k];
}

// ---- the start: momentum and sum of squares; then scaled, split, both orientations --------------------------------------
__global__ void __launch_bounds__(256) ns_norm_kernel(NsArgs g) {
  const int i = ns_find(g, blockIdx.x);
  const NsItem it = g.it[i];
  const int wg = blockIdx.x - it.wg0, nc = (it.cols + kNsStrip - 1) / kNsStrip;
  const int r0 = wg / nc * 64, c0 = wg % nc * kNsStrip;
  const int r1 = min(r0 + 64, it.rows), c1 = min(c0 + kNsStrip, it.cols);
  double s = 0.;
  for (int r = r0 + (threadIdx.x >> 6); r < r1; r += 4)
    for (int c = c0 + (threadIdx.x & 63); c < c1; c += 64) {
      const double v = (double)ns_start(g, it, (long)r * it.cols + c, true);
      s += v * v;
    }
  __shared__ double sh[4];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) g.sq[(long)i * g.sqn + wg] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__global__ void __launch_bounds__(256) ns_split_kernel(NsArgs g) {
  const int i = ns_find(g, blockIdx.x);
  const NsItem it = g.it[i];
  const NsShape s(it.rows, it.cols);
  const NsPlanes p(g.ws + it.ws, s);
  const int wg = blockIdx.x - it.wg0, nt = s.np / 64;
  const int k0 = wg / nt * 64, j0 = wg % nt * 64;       // rows and columns of X
  __shared__ float tile[64][65];                         // [row of X][column of X]
  __shared__ double sh[4];
  double sq = 0.;
  const int strips = ((it.rows + 63) / 64) * ((it.cols + kNsStrip - 1) / kNsStrip);
  for (int k = threadIdx.x; k < strips; k += 256) sq += g.sq[(long)i * g.sqn + k];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sq += __shfl_xor(sq, m, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sq;
  __syncthreads();
  const double norm = sqrt((sh[0] + sh[1]) + (sh[2] + sh[3]));
  const float scale = (float)(1. / (norm > (double)g.eps || norm != norm ? norm : (double)g.eps));
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    const int hi = e >> 6, lo = e & 63;                  // the source's row and column inside the tile
    const int r = (s.tall ? j0 : k0) + hi, c = (s.tall ? k0 : j0) + lo;
    const float v = r < it.rows && c < it.cols ? ns_start(g, it, (long)r * it.cols + c, false) * scale : 0.f;
    if (s.tall) tile[lo][hi] = v;
    else tile[hi][lo] = v;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e) {                          // 64 lines of 8 pieces of 8 values, each way
    const int line = (threadIdx.x >> 3) + 32 * e, at = (threadIdx.x & 7) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[line][at + j];
    ns_store8(p.x + (long)(k0 + line) * s.np + j0 + at, s.big(), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[at + j][line];
    ns_store8(p.xt + (long)(j0 + line) * s.mp + k0 + at, s.big(), v);
  }
}

// ---- the products --------------------------------------------------------------------------------------------------------
enum { kNsGram = 0, kNsPoly = 1, kNsApply = 2 };

// tile t of the lower triangle, row by row
__device__ __forceinline__ void ns_triangle(int t, int& i, int& j) {
  i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((long)(i + 1) * (i + 2) / 2 <= t) ++i;
  while ((long)i * (i + 1) / 2 > t) --i;
  j = t - (int)((long)i * (i + 1) / 2);
}

// A workgroup = 128 x 128 of L R^T, four waves of 64 x 64 (2 x 2 accumulators of v_mfma_f32_32x32x16_bf16); 32 k-values a
// stage, two stages in LDS.  LDS tile of one operand piece: 128 rows of 64 bytes = 4 x 16-byte cells; the cell of k-octet o
// of row r is o ^ (r >> 2 & 3), so that the 16 lanes of a phase of ds_read_b128 (16 rows, one octet) touch all 64 banks once.
// The DMA writes lane l's 16 bytes at cell l: the swizzle is applied to the address that the lane reads from.
constexpr int kNsPiece = kNsTile * 64;                    // bytes of one piece's tile
constexpr int kNsStage = 6 * kNsPiece;                    // L and R, three pieces each
constexpr int kNsPitch = kNsTile + 4;                     // floats: the finished tile in LDS
constexpr int kNsLds = 2 * kNsStage > kNsTile * kNsPitch * 4 ? 2 * kNsStage : kNsTile * kNsPitch * 4;

template <int STAGE>
__global__ void __launch_bounds__(256, 1) ns_product_kernel(NsArgs g) {
  extern __shared__ __align__(16) char lds[];
  const int i = ns_find(g, blockIdx.x);
  const NsItem it = g.it[i];
  const NsShape s(it.rows, it.cols);
  const NsPlanes p(g.ws + it.ws, s);
  const int t = blockIdx.x - it.wg0;
  int ti, tj;
  if (STAGE == kNsApply) ti = t / (s.np / kNsTile), tj = t % (s.np / kNsTile);
  else ns_triangle(t, ti, tj);
  const int K = STAGE == kNsGram ? s.np : s.mp;
  const __bf16* L = STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : p.q;
  const __bf16* R = STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : (g.flip ? p.xt1 : p.xt);
  const long lplane = STAGE == kNsGram ? s.big() : s.sym(), rplane = STAGE == kNsApply ? s.big() : lplane;
  L += (long)ti * kNsTile * K, R += (long)tj * kNsTile * K;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // DMA: wave w fills rows 16 (w + 4 h) .. + 15 (h = 0, 1) of each of the six tiles: lane -> row lane >> 2, cell lane & 3
  const int drow = wave * 16 + (lane >> 2), dcell = (lane & 3) ^ (drow >> 2 & 3);
  const long doff = (long)drow * K + dcell * 8;           // (row + 64: r >> 2 & 3 is the same)
  auto fill = [&](int buf, int k) {
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        char* to = lds + buf * kNsStage + q * kNsPiece + (wave * 16 + h * 64) * 64;
        const long off = doff + (long)h * 64 * K + k;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(L + q * lplane + off),
                                         (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(R + q * rplane + off),
                                         (__attribute__((address_space(3))) void*)(to + 3 * kNsPiece), 16, 0, 0);
      }
  };
  const int lr = (wave >> 1) * 64 + (lane & 31), rr = (wave & 1) * 64 + (lane & 31), oct = lane >> 5;
  auto read = [&](int buf, int operand, int q, int row, int o) {
    return *reinterpret_cast<const nsb8*>(lds + buf * kNsStage + (operand * 3 + q) * kNsPiece + row * 64 + ((o ^ (row >> 2 & 3)) * 16));
  };
  // hi hi goes to accumulators of its own: the other five products are 2^-8 of it, and adding them into the large sums would
  // round those six times instead of once per 16 k-values
  nsf16 acc[2][2] = {}, low[2][2] = {};
  fill(0, 0);
  const int stages = K / 32;
  for (int k = 0; k < stages; ++k) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's part of stage k is in LDS
    __syncthreads();                                      // everybody's, and nobody reads the other buffer any more
    if (k + 1 < stages) fill((k + 1) & 1, (k + 1) * 32);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      nsb8 lf[2][3], rf[2][3];
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          lf[e][q] = read(k & 1, 0, q, lr + 32 * e, half * 2 + oct);
          rf[e][q] = read(k & 1, 1, q, rr + 32 * e, half * 2 + oct);
        }
      // the six products, small ones first
#pragma unroll
      for (int sum = 2; sum >= 0; --sum)
#pragma unroll
        for (int q = 0; q <= sum; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f)
              if (sum) low[e][f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lf[e][q], rf[f][sum - q], low[e][f], 0, 0, 0);
              else acc[e][f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lf[e][q], rf[f][sum - q], acc[e][f], 0, 0, 0);
    }
  }
  __syncthreads();
  // the tile into LDS (accumulator register r of lane l: row 8 (r >> 2) + 4 (l >> 5) + (r & 3), column l & 31)
  float* tile = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = (wave >> 1) * 64 + e * 32 + 8 * (r >> 2) + 4 * oct + (r & 3);
        tile[row * kNsPitch + (wave & 1) * 64 + f * 32 + (lane & 31)] = acc[e][f][r] + low[e][f][r];
      }
  __syncthreads();
  const int row0 = ti * kNsTile, col0 = tj * kNsTile;
  if (STAGE == kNsPoly) {                                 // a I + b A + c A A, in place
    for (int e = threadIdx.x; e < kNsTile * kNsTile / 8; e += 256) {
      const int r = e >> 4, c = (e & 15) * 8;
      const __bf16* ap = p.a + (long)(row0 + r) * s.mp + col0 + c;
      const nsb8 h = *reinterpret_cast<const nsb8*>(ap), m = *reinterpret_cast<const nsb8*>(ap + s.sym()),
                 l = *reinterpret_cast<const nsb8*>(ap + 2 * s.sym());
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float av = ((float)h[j] + (float)m[j]) + (float)l[j];
        float v = g.b * av + g.c * tile[r * kNsPitch + c + j];
        if (row0 + r == col0 + c + j && row0 + r < s.m) v += g.a;
        tile[r * kNsPitch + c + j] = v;
      }
    }
    __syncthreads();
  }
  if (STAGE == kNsApply && g.last) {
    for (int e = threadIdx.x; e < kNsTile * kNsTile; e += 256) {
      const int hi = e >> 7, lo = e & 127;                // row and column of the source inside the tile
      const int r = (s.tall ? col0 : row0) + hi, c = (s.tall ? row0 : col0) + lo;
      if (r < it.rows && c < it.cols) ns_result(g, it, (long)r * it.cols + c, s.tall ? tile[lo * kNsPitch + hi] : tile[hi * kNsPitch + lo]);
    }
    return;
  }
  // both orientations, as pieces
  __bf16* out = STAGE == kNsGram ? p.a : STAGE == kNsPoly ? p.q : p.x;
  __bf16* outt = STAGE == kNsApply ? (g.flip ? p.xt : p.xt1) : out;
  const int pitch = STAGE == kNsApply ? s.np : s.mp;
  const long plane = STAGE == kNsApply ? s.big() : s.sym();
  for (int e = threadIdx.x; e < kNsTile * kNsTile / 8; e += 256) {
    const int r = e >> 4, c = (e & 15) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[r * kNsPitch + c + j];
    ns_store8(out + (long)(row0 + r) * pitch + col0 + c, plane, v);
  }
  if (STAGE != kNsApply && ti == tj) return;
  for (int e = threadIdx.x; e < kNsTile * kNsTile / 8; e += 256) {
    const int c = e >> 4, r = (e & 15) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[(r + j) * kNsPitch + c];
    ns_store8(outt + (long)(col0 + c) * s.mp + row0 + r, plane, v);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
static const char* ns_bad(int count, const int* rows, const int* cols) {
  if (count < 0 || (count > 0 && (!rows || !cols))) return "bad list";
  for (int i = 0; i < count; ++i)
    if (rows[i] <= 0 || cols[i] <= 0 || rows[i] > (1 << 16) || cols[i] > (1 << 16)) return "a side is not in 1 ... 65536";
  return nullptr;
}
// what a call writes overlaps nothing else that it reads or writes
static bool ns_apart(int count, const int* rows, const int* cols, int size, const void* const* in, const void* const* out,
                     const void* const* out32) {
  struct Span {
    uintptr_t lo, hi;
    bool writes;
  };
  std::vector<Span> v;
  v.reserve(3 * count);
  for (int i = 0; i < count; ++i) {
    const uintptr_t n = (uintptr_t)rows[i] * cols[i];
    v.push_back({(uintptr_t)in[i], (uintptr_t)in[i] + n * size, false});
    v.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + n * size, true});
    if (out32) v.push_back({(uintptr_t)out32[i], (uintptr_t)out32[i] + n * 4, true});
  }
  std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t read = 0, written = 0;      // the furthest ends so far
  for (const Span& s : v) {
    if (s.lo < written || (s.writes && s.lo < read)) return false;
    (s.writes ? written : read) = std::max(s.writes ? written : read, s.hi);
  }
  return true;
}
static int ns_strips(int rows, int cols) { return ((rows + 63) / 64) * ((cols + kNsStrip - 1) / kNsStrip); }

// the list in runs of kNsList; a run's pieces share the workspace with the next run's
static long ns_workspace(int count, const int* rows, const int* cols) {
  long most = 0;
  for (int b = 0; b < count; b += kNsList) {
    long bytes = 0;
    int sqn = 1;
    for (int i = b; i < count && i < b + kNsList; ++i) {
      bytes += ns_bytes(NsShape(rows[i], cols[i]));
      if (ns_strips(rows[i], cols[i]) > sqn) sqn = ns_strips(rows[i], cols[i]);
    }
    bytes += (long)kNsList * sqn * sizeof(double);
    if (bytes > most) most = bytes;
  }
  return most;
}

static int ns_run(NsArgs g, int count, const void* const* src, void* const* dst, float* const* buf, const int* rows,
                  const int* cols, const float* scales, int steps, char* ws, hipStream_t st) {
  static const bool ready = [] {      // (96 KB of LDS: above what a kernel gets without asking)
    const void* k[3] = {(const void*)ns_product_kernel<kNsGram>, (const void*)ns_product_kernel<kNsPoly>, (const void*)ns_product_kernel<kNsApply>};
    for (const void* f : k)
      if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kNsLds) != hipSuccess) return false;
    return true;
  }();
  if (!ready) return -1;
  for (int b = 0; b < count; b += kNsList) {
    g.count = count - b < kNsList ? count - b : kNsList;
    long off = 0;
    g.sqn = 1;
    for (int i = 0; i < g.count; ++i) {
      NsItem& it = g.it[i];
      it.src = src[b + i], it.dst = dst[b + i], it.buf = buf ? buf[b + i] : nullptr, it.rows = rows[b + i], it.cols = cols[b + i];
      it.scale = scales ? scales[b + i] : 1.f, it.ws = off;
      off += ns_bytes(NsShape(it.rows, it.cols));
      if (ns_strips(it.rows, it.cols) > g.sqn) g.sqn = ns_strips(it.rows, it.cols);
    }
    g.ws = ws, g.sq = reinterpret_cast<double*>(ws + off);
    // workgroups of the launch: fills wg0
    auto table = [&](auto&& wgs) {
      long n = 0;
      for (int i = 0; i < g.count; ++i) g.it[i].wg0 = (int)n, n += wgs(g.it[i], NsShape(g.it[i].rows, g.it[i].cols));
      return dim3((unsigned)n);
    };
    const dim3 block(256);
    hipLaunchKernelGGL(ns_norm_kernel, table([](const NsItem& it, const NsShape&) { return (long)ns_strips(it.rows, it.cols); }), block, 0, st, g);
    hipLaunchKernelGGL(ns_split_kernel, table([](const NsItem&, const NsShape& s) { return s.big() / (64 * 64); }), block, 0, st, g);
    auto triangle = [](const NsItem&, const NsShape& s) { return (long)(s.mp / kNsTile) * (s.mp / kNsTile + 1) / 2; };
    for (int k = 0; k < steps; ++k) {
      g.last = k + 1 == steps, g.flip = k & 1;
      dim3 grid = table(triangle);
      hipLaunchKernelGGL(ns_product_kernel<kNsGram>, grid, block, kNsLds, st, g);
      hipLaunchKernelGGL(ns_product_kernel<kNsPoly>, grid, block, kNsLds, st, g);
      grid = table([](const NsItem&, const NsShape& s) { return s.big() / (kNsTile * kNsTile); });
      hipLaunchKernelGGL(ns_product_kernel<kNsApply>, grid, block, kNsLds, st, g);
    }
  }
  return 0;
}

}  // namespace bmv

using namespace bmv;

extern "C" {

long bmv_newton_schulz_workspace(int count, const int* rows, const int* cols) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_newton_schulz_workspace: %s", bad);
  return ns_workspace(count, rows, cols);
}

int bmv_newton_schulz(int count, const void* const* src, void* const* dst, const int* rows, const int* cols, int dtype, int steps,
                      float a, float b, float c, float eps, void* workspace, bmv_stream_t stream) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_newton_schulz: %s", bad);
  BMV_REQUIRE(dtype >= 0 && dtype <= 2, "bmv_newton_schulz: unknown type %d", dtype);
  BMV_REQUIRE(steps > 0 && eps >= 1e-12f, "bmv_newton_schulz: at least one step and eps >= 1e-12 (got %d, %g)", steps, (double)eps);
  if (count == 0) return BMV_OK;
  BMV_REQUIRE(src && dst && workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "bmv_newton_schulz: null pointer, or a workspace off its 256-byte border");
  for (int i = 0; i < count; ++i) BMV_REQUIRE(src[i] && dst[i], "bmv_newton_schulz: null pointer (matrix %d)", i);
  BMV_REQUIRE(ns_apart(count, rows, cols, dtype == 0 ? 4 : 2, src, dst, nullptr), "bmv_newton_schulz: a result overlaps another matrix");
  NsArgs g{};
  g.dtype = dtype, g.a = a, g.b = b, g.c = c, g.eps = eps;
  BMV_REQUIRE(ns_run(g, count, src, dst, nullptr, rows, cols, nullptr, steps, static_cast<char*>(workspace), as_stream(stream)) == 0,
              "bmv_newton_schulz: %d bytes of LDS refused", kNsLds);
  BMV_LAUNCH_END("bmv_newton_schulz");
}

int bmv_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta, const int* rows, const int* cols,
                  const float* scales, int dtype, double momentum, int nesterov, double keep, int steps, float a, float b, float c,
                  float eps, void* workspace, bmv_stream_t stream) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_muon_step: %s", bad);
  BMV_REQUIRE(dtype >= 0 && dtype <= 2, "bmv_muon_step: unknown type %d", dtype);
  BMV_REQUIRE(steps > 0 && eps >= 1e-12f, "bmv_muon_step: at least one step and eps >= 1e-12 (got %d, %g)", steps, (double)eps);
  if (count == 0) return BMV_OK;
  BMV_REQUIRE(params && grads && momenta && scales && workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
              "bmv_muon_step: null pointer, or a workspace off its 256-byte border");
  for (int i = 0; i < count; ++i) BMV_REQUIRE(params[i] && grads[i] && momenta[i], "bmv_muon_step: null pointer (matrix %d)", i);
  BMV_REQUIRE(ns_apart(count, rows, cols, dtype == 0 ? 4 : 2, grads, params, reinterpret_cast<const void* const*>(momenta)),
              "bmv_muon_step: a weight or a momentum overlaps another tensor (is one listed twice?)");
  NsArgs g{};
  g.dtype = dtype, g.a = a, g.b = b, g.c = c, g.eps = eps, g.muon = 1, g.nesterov = nesterov, g.mu = (float)momentum, g.nu = (float)(1. - momentum), g.keep = (float)keep;
  BMV_REQUIRE(ns_run(g, count, grads, params, momenta, rows, cols, scales, steps, static_cast<char*>(workspace), as_stream(stream)) == 0,
              "bmv_muon_step: %d bytes of LDS refused", kNsLds);
  BMV_LAUNCH_END("bmv_muon_step");
}

}  // extern "C"
