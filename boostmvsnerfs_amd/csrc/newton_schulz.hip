// Newton-Schulz orthogonalisation of a list of matrices, and the optimiser's step around it (momentum before, the decayed
// update of the weights behind it): what train.py's Adam step is to element-wise updates, for whole matrices.
//
//   X_0 = U / max(|U|_F, eps) with the short side as rows (m <= n); steps times:
//   A = X X^T,  Q = a I + b A + c A A,  X <- Q X.       The polynomial moves every singular value towards 1.
//   Step: buf <- mu buf + (1 - mu) g,  U = (1 - mu) g + mu buf (Nesterov) or buf,  w <- w (1 - lr decay) - lr scale X.
//
// Numbers.  A near-zero singular value grows by a = 3.4 a step, and with it whatever error X carried in its direction: the
// products need more accuracy than the result's type has.  They run on the bf16 matrix cores with every fp32 operand as
// three bf16 pieces (hi + mid + lo: its 24 significand bits exactly) and the six products that are not below 2^-25, sums in
// fp32: 2.5 PFLOP/s / 6 against the 0.157 of the fp32 matrix instructions.  |U|_F is a 64-bit sum; for short sides of up to 128
// it is the root of the fp32 trace of U U^T, so a norm of more than 1.8e19 makes the result NaN there.
//
// All types: a bf16 or fp16 matrix' result is the fp32 result of the same values, rounded once.
//
// Layout.  Every operand is kept as its pieces from the moment it is computed (one split per value, not one per use), in the
// orientation in which its k axis is contiguous, so all three products are L R^T: A from X (k = n), A A from the symmetric A
// (k = m), Q X from Q and X^T (k = m); X is therefore written in both orientations.  And it is kept in the order in which the
// products stage it: panels of 128 rows, in them blocks of 16 k-values, in a block piece after piece, 128 rows of 32 bytes.
// What a stage of a product loads is one run of memory per operand, moved to LDS by 16-byte DMA with no registers and next to
// no address arithmetic.  A and Q are symmetric: only tiles on and below the diagonal are computed.
//
// Work.  Matrices of up to 1000 or so: a product is one launch of 64 x 64 blocks (ns_block_kernel).  Above, its tiles of 128 x 128
// are as many workgroups while they fill the card; the rest is cut along k into equal runs of stages over all compute units, whose
// partial tiles the joining launch adds in a fixed order.  That launch also applies the polynomial, splits the values and writes
// both orientations.  A product of the whole list is one launch: a workgroup finds its matrix in a table of the kernel arguments.
//
// What bounds it.  4096 x 4096 fp32: Q X takes 612 ... 647 us by the card, 1275 ... 1347 TFLOP/s of bf16 products -- a large product
// of the library reaches 1247 --, with the matrix pipe 66 % busy at the 1.9 GHz that its power leaves.  Joins are 7 ... 20 % on
// top (4096 x 4096: 100 of 1365 ... 1410 us a step) and move their bytes at 4 ... 5 TB/s.  Below 1000 or so it is the chain: 15
// launches, of which 7.5 us each are start, first operands and end.
//
// Matrices with a short side of up to 128 (every layer of the networks here) go another way, one launch a step: see below.
#include <algorithm>
#include <atomic>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "bmv_common.hpp"

namespace bmv {

using nsb8 = __attribute__((ext_vector_type(8))) __bf16;
using nsf4 = __attribute__((ext_vector_type(4))) float;
using nsf16 = __attribute__((ext_vector_type(16))) float;

constexpr int kNsList = 40;      // matrices per launch (the table travels in the kernel arguments)
constexpr int kNsTile = 128;     // output tile of a workgroup; matrices are padded to it with zeros
constexpr int kNsP = 3;          // bf16 pieces of an operand
constexpr int kNsK = 16;         // k-values of a stage
constexpr int kNsCell = 2048;    // elements of a piece of a block: 128 rows of 16 k-values
constexpr int kNsChunk = 8192;   // elements of a workgroup of the norm
constexpr int kNsUnits = 256, kNsLdsBytes = 160 * 1024;    // compute units, LDS of one
constexpr int kNsSlots = 512;    // workgroups that run at once: two on each of 256 compute units

struct NsItem {
  const void* src;      // U, or the gradient
  void* dst;            // the result, or the weights that the step updates
  float* buf;           // momentum (step), or null
  long ws;              // byte offset of this matrix' pieces in the workspace
  int rows, cols;       // of src / dst
  float scale;          // step: lr * scale of this matrix
  int at;               // first workgroup / tile of this matrix in the launch
};
struct NsArgs {
  NsItem it[kNsList];
  char* ws;
  double* sq;           // partial sums of squares: [item][chunk], kNsList * sqn of them
  float* part;          // partial tiles
  int count, sqn, dtype, muon, nesterov, first, last, flip;
  int least, spread;    // short sides: columns of a workgroup at least; slots of matrices that all XCDs share
  int full, run;        // a product's tiles that are a workgroup each; stages of a run of the others
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
  __host__ __device__ int mt() const { return mp / kNsTile; }
  __host__ __device__ int nt() const { return np / kNsTile; }
  __host__ __device__ long triangle() const { return (long)mt() * (mt() + 1) / 2; }
};
// the operands of a matrix, kNsP pieces each
struct NsPlanes {
  __bf16 *x, *xt, *xt1, *a, *q;      // xt, xt1: X^T before and after a step, in turn
  __device__ NsPlanes(char* ws, const NsShape& s) {
    x = reinterpret_cast<__bf16*>(ws);
    xt = x + kNsP * s.big(), xt1 = xt + kNsP * s.big(), a = xt1 + kNsP * s.big(), q = a + kNsP * s.sym();
  }
};
static long ns_bytes(const NsShape& s) { return (3 * s.big() + 2 * s.sym()) * 2 * kNsP; }

// the 8 k-values k ... k + 7 (k % 8 == 0) of row r, piece 0, of an operand with K k-values; piece q is kNsCell * q behind.
// The two 16-byte cells of a row in a block are in turn swapped every 8 rows: the 16 lanes of a phase of ds_read_b128 (rows at
// one k) then touch all 64 banks once.
__device__ __forceinline__ long ns_cell(int r, int k, int K) {
  return ((long)(r >> 7) * (K / kNsK) + k / kNsK) * (kNsP * kNsCell) + (r & 127) * kNsK + (((k >> 3) ^ (r >> 3)) & 1) * 8;
}

// the matrix that holds `at`: the last whose first is not behind it (one load a lane instead of a chain of them)
__device__ __forceinline__ int ns_find(const NsArgs& g, int at) {
  static_assert(kNsList <= 64, "a lane each");
  const int lane = threadIdx.x & 63;
  if (g.count == 1) return 0;                             // (0.2 us of a launch)
  return __popcll(__ballot(lane < g.count && g.it[min(lane, kNsList - 1)].at <= at)) - 1;
}

// N values of what the iteration starts from, before its norm is divided out; `fresh`: the momentum is moved first.  at(j): the
// index of value j, or -1 for a zero.  (All loads before the first use: a branch or a conversion between them waits for each.
// Fused products are written out: the same roundings for all types.)
template <int DT, bool MUON, int N, typename F>
__device__ __forceinline__ void ns_start(const NsArgs& g, const NsItem& it, bool fresh, F at, float* v) {
  using T = std::conditional_t<DT == 0, float, std::conditional_t<DT == 1, __bf16, _Float16>>;
  long i[N];
  T raw[N];
  float m[N];
#pragma unroll
  for (int j = 0; j < N; ++j) i[j] = at(j);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    raw[j] = static_cast<const T*>(it.src)[max(i[j], 0l)];
    if (MUON) m[j] = it.buf[max(i[j], 0l)];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float x = (float)raw[j];
    if (MUON) {
      if (fresh) m[j] = fmaf(g.mu, m[j], g.nu * x);
      if (fresh && i[j] >= 0) it.buf[i[j]] = m[j];
      x = g.nesterov ? fmaf(g.mu, m[j], g.nu * x) : m[j];
    }
    v[j] = i[j] >= 0 ? x : 0.f;
  }
}
// N results, value j of index at(j) (-1: none): the iterate itself, or the weight that it steps, rounded once (the fused product is
// written out: one order of the roundings for all types)
template <int N, typename F>
__device__ __forceinline__ void ns_results(const NsArgs& g, const NsItem& it, F at, const float* x) {
  long i[N];
#pragma unroll
  for (int j = 0; j < N; ++j) i[j] = at(j);
  auto run = [&](auto* dst) {
    std::remove_pointer_t<decltype(dst)> w[N];
    if (g.muon) {
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = dst[max(i[j], 0l)];
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i[j] >= 0) dst[i[j]] = (std::remove_pointer_t<decltype(dst)>)(g.muon ? fmaf(-it.scale, x[j], (float)w[j] * g.keep) : x[j]);
  };
  if (g.dtype == 0) run(static_cast<float*>(it.dst));
  else if (g.dtype == 1) run(static_cast<__bf16*>(it.dst));
  else run(static_cast<_Float16*>(it.dst));
}

// x = p[0] + p[1] + p[2], exactly: every piece is the nearest bf16 to what the pieces before it leave (to nearest, not
// truncated: what the dropped products of the pieces amount to is then below 2^-25 and of either sign, not 2^-21 of one).
// Eight consecutive values as kNsP 16-byte stores.
__device__ __forceinline__ void ns_store8(__bf16* p, const float* v) {
  nsb8 o[kNsP];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float r = v[j];
#pragma unroll
    for (int q = 0; q < kNsP; ++q) o[q][j] = (__bf16)r, r -= (float)o[q][j];
  }
#pragma unroll
  for (int q = 0; q < kNsP; ++q) *reinterpret_cast<nsb8*>(p + q * kNsCell) = o[q];
}

// A 64 x 64 block of values in LDS, rows r0 ..., columns c0 ... of a matrix, as cells of the operand whose k axis is the
// columns (out, K = its columns) and of its transpose (outt, Kt); either may be null.
constexpr int kNsPitch = 65;
__device__ __forceinline__ void ns_store_block(const float* t, int r0, int c0, __bf16* out, int K, __bf16* outt, int Kt) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = threadIdx.x + 256 * e, line = i >> 1 & 63, k = (i >> 7) * 16 + (i & 1) * 8;     // lanes along a block's run
    float v[8];
    if (out) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = t[line * kNsPitch + k + j];
      ns_store8(out + ns_cell(r0 + line, c0 + k, K), v);
    }
    if (outt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = t[(k + j) * kNsPitch + line];
      ns_store8(outt + ns_cell(c0 + line, r0 + k, Kt), v);
    }
  }
}

// ---- the start: momentum and sum of squares; then scaled, split, both orientations --------------------------------------
template <int DT, bool MUON>
__global__ void __launch_bounds__(256) ns_norm_kernel(NsArgs g) {
  const int i = ns_find(g, blockIdx.x);
  const NsItem it = g.it[i];
  const int wg = blockIdx.x - it.at;
  const long numel = (long)it.rows * it.cols, base = (long)wg * kNsChunk;
  double s = 0.;
  for (int k = 0; k < kNsChunk / 256; k += 8) {
    float v[8];
    ns_start<DT, MUON, 8>(g, it, true, [&](int j) {
      const long at = base + (k + j) * 256 + threadIdx.x;
      return at < numel ? at : -1l;
    }, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)v[j] * (double)v[j];
  }
  __shared__ double sh[4];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) g.sq[(long)i * g.sqn + wg] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

template <int DT, bool MUON>
__global__ void __launch_bounds__(256) ns_split_kernel(NsArgs g) {
  const int i = ns_find(g, blockIdx.x);
  const NsItem it = g.it[i];
  const NsShape s(it.rows, it.cols);
  const NsPlanes p(g.ws + it.ws, s);
  const int wg = blockIdx.x - it.at, nt = s.np / 64;
  const int k0 = wg / nt * 64, j0 = wg % nt * 64;       // rows and columns of X
  __shared__ float tile[64 * kNsPitch];                  // [row of X][column of X]
  __shared__ double sh[4];
  double sq = 0.;
  const int chunks = (int)(((long)it.rows * it.cols + kNsChunk - 1) / kNsChunk);
  for (int k = threadIdx.x; k < chunks; k += 256) sq += g.sq[(long)i * g.sqn + k];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sq += __shfl_xor(sq, m, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sq;
  __syncthreads();
  const double norm = sqrt((sh[0] + sh[1]) + (sh[2] + sh[3]));
  const float scale = (float)(1. / (norm > (double)g.eps || norm != norm ? norm : (double)g.eps));
#pragma unroll
  for (int k = 0; k < 16; k += 8) {
    float v[8];
    ns_start<DT, MUON, 8>(g, it, false, [&](int j) {
      const int e = threadIdx.x + 256 * (k + j), r = (s.tall ? j0 : k0) + (e >> 6), c = (s.tall ? k0 : j0) + (e & 63);
      return r < it.rows && c < it.cols ? (long)r * it.cols + c : -1l;
    }, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = threadIdx.x + 256 * (k + j), hi = e >> 6, lo = e & 63;      // the source's row and column inside the tile
      tile[s.tall ? lo * kNsPitch + hi : hi * kNsPitch + lo] = v[j] * scale;
    }
  }
  __syncthreads();
  ns_store_block(tile, k0, j0, p.x, s.np, p.xt, s.mp);
}

// ---- the products --------------------------------------------------------------------------------------------------------
enum { kNsGram = 0, kNsPoly = 1, kNsApply = 2 };

// Tile t of a product: super-rows of 8 tile rows, in them column by column, so that neighbouring workgroups (the 64 of an XCD
// at a time) share 8 + 8 panels of operands in its L2.  Symmetric products: only columns up to the row.
__device__ __forceinline__ void ns_tile(int t, int mt, int nt, bool symmetric, int& i, int& j) {
  if (!symmetric) {
    const int per = 8 * nt, sr = t / per, h = min(8, mt - 8 * sr);
    t -= sr * per;
    i = 8 * sr + t % h, j = t / h;
    return;
  }
  int sr = 0;
  while (32 * (sr + 1) * (sr + 1) + 4 * (sr + 1) <= t) ++sr;      // (tiles above super-row sr: 32 sr^2 + 4 sr)
  t -= 32 * sr * sr + 4 * sr;
  const int h = min(8, mt - 8 * sr);
  if (t < 8 * sr * h) {
    i = 8 * sr + t % h, j = t / h;
    return;
  }
  t -= 8 * sr * h;
  int col = 0;
  while (t >= h - col) t -= h - col, ++col;
  i = 8 * sr + col + t, j = 8 * sr + col;
}
__device__ __forceinline__ int ns_tiles(const NsShape& s, int stage) { return stage == kNsApply ? s.mt() * s.nt() : (int)s.triangle(); }
__host__ __device__ __forceinline__ int ns_stages(const NsShape& s, int stage) { return (stage == kNsGram ? s.np : s.mp) / kNsK; }

// A finished 64 x 64 block of a product in LDS, by its workgroup: the polynomial (kNsPoly), then both orientations as pieces, or
// the result
template <int STAGE>
__device__ __forceinline__ void ns_finish(const NsArgs& g, const NsItem& it, const NsShape& s, const NsPlanes& p, int row0, int col0,
                                          bool diagonal, float* tile) {
  if (STAGE == kNsPoly) {                                 // a I + b A + c A A, in place
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = threadIdx.x + 256 * e, r = k >> 1 & 63, c = (k >> 7) * 16 + (k & 1) * 8;
      const __bf16* ap = p.a + ns_cell(row0 + r, col0 + c, s.mp);
      float av[8] = {};
#pragma unroll
      for (int q = kNsP - 1; q >= 0; --q) {
        const nsb8 piece = *reinterpret_cast<const nsb8*>(ap + q * kNsCell);
#pragma unroll
        for (int j = 0; j < 8; ++j) av[j] += (float)piece[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float* to = tile + r * kNsPitch + c + j;
        *to = g.b * av[j] + g.c * *to + (row0 + r == col0 + c + j && row0 + r < s.m ? g.a : 0.f);
      }
    }
    __syncthreads();
  }
  if (STAGE == kNsApply && g.last) {
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = threadIdx.x + 256 * (k + j), hi = e >> 6, lo = e & 63;      // row and column of the source inside the block
        v[j] = tile[s.tall ? lo * kNsPitch + hi : hi * kNsPitch + lo];
      }
      ns_results<8>(g, it, [&](int j) {
        const int e = threadIdx.x + 256 * (k + j), r = (s.tall ? col0 : row0) + (e >> 6), c = (s.tall ? row0 : col0) + (e & 63);
        return r < it.rows && c < it.cols ? (long)r * it.cols + c : -1l;
      }, v);
    }
    return;
  }
  __bf16* out = STAGE == kNsGram ? p.a : STAGE == kNsPoly ? p.q : p.x;
  if (STAGE == kNsApply) ns_store_block(tile, row0, col0, out, s.np, g.flip ? p.xt : p.xt1, s.mp);
  else ns_store_block(tile, row0, col0, out, s.mp, diagonal ? nullptr : out, s.mp);
}

// A workgroup = 128 x 128 of L R^T, four waves of 64 x 64 (2 x 2 accumulators of v_mfma_f32_32x32x16_bf16, twice: hi hi goes to
// accumulators of its own, because the other products are 2^-8 of it and adding them into the large sums would round those
// once more for each).  Three stages of 16 k-values in LDS: one being multiplied, two on their way.  The finished tile leaves
// in the order of the accumulators, 16 bytes a lane; the joining launch knows that order.
template <int STAGE>
__global__ void __launch_bounds__(256, 2) ns_product_kernel(NsArgs g) {
  constexpr int kBufs = 3;
  constexpr int kHalf = kNsP * kNsCell;                   // elements of an operand's stage
  constexpr int kStage = 2 * kHalf;                       // L's, then R's
  constexpr int kLoads = kStage * 2 / 1024 / 4;           // 1 KB DMAs of a wave for a stage
  __shared__ __align__(16) __bf16 lds[kBufs * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool whole = (int)blockIdx.x < g.full;
  // the unit range of this workgroup: unit = stage of a tile behind the whole ones
  int t = whole ? xcd_contiguous(blockIdx.x, g.full) : g.full;
  long skip = whole ? 0 : (long)(blockIdx.x - g.full) * g.run, left = whole ? 1l << 40 : g.run;
  int i = ns_find(g, t);
  while (left > 0) {
    const NsItem it = g.it[i];
    const NsShape s(it.rows, it.cols);
    const int stages = ns_stages(s, STAGE), tiles = ns_tiles(s, STAGE);
    if (!whole) {                                         // go to the tile that holds the next unit
      const long jump = min(skip / stages, (long)(it.at + tiles - t));
      t += (int)jump, skip -= jump * stages;
      if (t >= it.at + tiles) {
        if (++i >= g.count) return;
        continue;
      }
    }
    const int first = (int)skip, count = (int)min(left, (long)stages - first);
    skip = 0, left -= whole ? left : count;
    int ti, tj;
    ns_tile(t - it.at, s.mt(), s.nt(), STAGE != kNsApply, ti, tj);
    const NsPlanes p(g.ws + it.ws, s);
    const __bf16* L = STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : p.q;
    const __bf16* R = STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : (g.flip ? p.xt1 : p.xt);
    L += ((long)ti * stages + first) * kHalf, R += ((long)tj * stages + first) * kHalf;
    auto fill = [&](int k) {                              // stage k into buffer k % kBufs
      __bf16* to = lds + k % kBufs * kStage;
#pragma unroll
      for (int h = 0; h < kLoads; ++h) {
        const int c = wave + 4 * h, off = c % (kLoads * 2) * 512;      // (1 KB = 512 elements; L's first, then R's)
        const __bf16* from = (c < kLoads * 2 ? L : R) + (long)k * kHalf + off;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + lane * 8),
                                         (__attribute__((address_space(3))) void*)(to + c * 512), 16, 0, 0);
      }
    };
    const int lr = (wave >> 1) * 64 + (lane & 31), rr = (wave & 1) * 64 + (lane & 31), oct = lane >> 5;
    auto read = [&](int k, int operand, int q, int row) {
      return *reinterpret_cast<const nsb8*>(lds + k % kBufs * kStage + operand * kHalf + q * kNsCell + row * kNsK + ((oct ^ row >> 3) & 1) * 8);
    };
    nsf16 acc[2][2] = {}, low[2][2] = {};
    fill(0);
    if (count > 1) fill(1);
    for (int k = 0; k < count; ++k) {
      // this wave's part of stage k is in LDS (of the newer loads only those of stage k + 1 may be on their way), then
      // everybody's, and nobody reads stage k - 1 any more
      if (k + 1 < count) asm volatile("s_waitcnt vmcnt(%0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::"n"(kLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (k + kBufs - 1 < count) fill(k + kBufs - 1);
      nsb8 lf[2][kNsP], rf[2][kNsP];
#pragma unroll
      for (int q = kNsP - 1; q >= 0; --q)
#pragma unroll
        for (int e = 0; e < 2; ++e) lf[e][q] = read(k, 0, q, lr + 32 * e), rf[e][kNsP - 1 - q] = read(k, 1, kNsP - 1 - q, rr + 32 * e);
      // the products of pieces whose numbers add up to at most kNsP - 1, small ones first
#pragma unroll
      for (int sum = kNsP - 1; sum >= 0; --sum)
#pragma unroll
        for (int q = sum; q >= 0; --q)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f)
              if (sum) low[e][f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lf[e][q], rf[f][sum - q], low[e][f], 0, 0, 0);
              else acc[e][f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lf[e][q], rf[f][sum - q], acc[e][f], 0, 0, 0);
    }
    // slot: a whole tile's number; behind those, run + tile, which grows by one from each run's piece of a tile to the next
    const long slot = whole ? t : t + (long)(blockIdx.x - g.full);
    nsf4* out = reinterpret_cast<nsf4*>(g.part) + slot * (kNsTile * kNsTile / 4) + threadIdx.x;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          nsf4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[e][f][4 * r + j] + low[e][f][4 * r + j];
          out[((e * 2 + f) * 4 + r) * 256] = v;
        }
    if (whole) return;
    // (the next tile's first stages go over this one's, and its waits count loads alone)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (++t >= it.at + tiles) {
      if (++i >= g.count) return;
    }
  }
}

// A workgroup = a wave's 64 x 64 quarter of a tile: its partial sums in the order of the runs, then the polynomial
// (kNsPoly), then both orientations as pieces, or the result.
template <int STAGE>
__global__ void __launch_bounds__(256) ns_join_kernel(NsArgs g) {
  __shared__ float tile[64 * kNsPitch];
  const int t = blockIdx.x >> 2, quarter = blockIdx.x & 3, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = ns_find(g, t);
  const NsItem it = g.it[i];
  const NsShape s(it.rows, it.cols);
  const NsPlanes p(g.ws + it.ws, s);
  int ti, tj;
  ns_tile(t - it.at, s.mt(), s.nt(), STAGE != kNsApply, ti, tj);
  // the slots that hold this tile: its own number, or one for each run that has stages of it
  long lo = t, hi = t;
  if (t >= g.full) {
    long unit = 0;                                        // the tile's first unit
    for (int k = 0; k < i; ++k) {
      const NsShape o(g.it[k].rows, g.it[k].cols);
      const int begin = max(g.it[k].at, g.full), end = g.it[k].at + ns_tiles(o, STAGE);
      if (end > begin) unit += (long)(end - begin) * ns_stages(o, STAGE);
    }
    const int stages = ns_stages(s, STAGE);
    unit += (long)(t - max(it.at, g.full)) * stages;
    lo = t + unit / g.run, hi = t + (unit + stages - 1) / g.run;
  }
  const nsf4* part = reinterpret_cast<const nsf4*>(g.part) + quarter * 64 + lane;
  nsf4 v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = part[lo * (kNsTile * kNsTile / 4) + (wave * 4 + r) * 256];
  for (long k = lo + 1; k <= hi; ++k)
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += part[k * (kNsTile * kNsTile / 4) + (wave * 4 + r) * 256];
  // accumulator register 4 r + j of lane l: row 8 r + 4 (l >> 5) + j, column l & 31 of the 32 x 32 block (wave >> 1, wave & 1)
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      tile[((wave >> 1) * 32 + 8 * r + 4 * (lane >> 5) + j) * kNsPitch + (wave & 1) * 32 + (lane & 31)] = v[r][j];
  __syncthreads();
  ns_finish<STAGE>(g, it, s, p, ti * kNsTile + (quarter >> 1) * 64, tj * kNsTile + (quarter & 1) * 64, ti == tj, tile);
}

// The same products whole and in one launch, 64 x 64 a workgroup: more bytes an operation, but no partial tiles and no joining
// launch.  A compute unit has one workgroup, so nothing else hides its waits: each of the four waves takes every fourth block of 16
// k-values for all of the 64 x 64, through a ring of stages of its own that it fills and reads without any barrier -- half the LDS
// reads of waves that share stages, and none waits for another.  Their four sums meet at the end.
constexpr int kNsBlockBufs = 3;
constexpr int kNsBlockLds = 4 * kNsBlockBufs * kNsP * 4 * 1024;      // waves, stages, pieces of 64 + 64 rows of 16 k-values
__host__ __device__ __forceinline__ int ns_block_count(const NsShape& s, int stage) {
  return stage == kNsApply ? 4 * s.mt() * s.nt() : s.mt() * (2 * s.mt() + 1);
}
template <int STAGE>
__global__ void __launch_bounds__(256, 1) ns_block_kernel(NsArgs g) {
  constexpr int kBufs = kNsBlockBufs;
  constexpr int kLeft = kNsP * 1024, kStage = 2 * kLeft, kLoads = 4 * kNsP;      // elements of an operand's part, of a stage; 1 KB DMAs
  constexpr int kSum = 64 * kNsPitch;                     // floats of the finished tile, beside which the shares have room
  static_assert(4 * kBufs * kStage * 2 == kNsBlockLds && (kSum + 3 * 1024) * 4 <= kBufs * kStage * 2 && kSum % 4 == 0, "LDS");
  extern __shared__ __align__(16) __bf16 stages_[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // an XCD has an eighth of every matrix' blocks, one run of them
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, i = ns_find(g, slot);
  const NsItem it = g.it[i];
  const NsShape s(it.rows, it.cols);
  const int blocks = ns_block_count(s, STAGE), t = xcd * ((blocks + 7) / 8) + slot - it.at;
  if (t >= blocks || slot - it.at >= (blocks + 7) / 8) return;
  const NsPlanes p(g.ws + it.ws, s);
  int ti, tj;
  ns_tile(t, 2 * s.mt(), 2 * s.nt(), STAGE != kNsApply, ti, tj);
  const int K = STAGE == kNsGram ? s.np : s.mp, count = K / (kNsK * 4);
  // (a half panel: rows 64 (t & 1) ... of every block's pieces)
  const long panel = (long)(K / kNsK) * (kNsP * kNsCell), mine = (long)wave * (kNsP * kNsCell) + lane * 8;
  const __bf16* L = (STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : p.q) + (ti >> 1) * panel + (ti & 1) * 1024 + mine;
  const __bf16* R = (STAGE == kNsGram ? p.x : STAGE == kNsPoly ? p.a : (g.flip ? p.xt1 : p.xt)) + (tj >> 1) * panel + (tj & 1) * 1024 + mine;
  __bf16* ring = stages_ + wave * (kBufs * kStage);
  auto fill = [&](int k) {
    __bf16* to = ring + k % kBufs * kStage;
    const long at = (long)k * (4 * kNsP * kNsCell);
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {                    // (1 KB = 32 rows of a piece of a block; L's first, then R's)
      const int h = c % (2 * kNsP), d = h / 2 * kNsCell + h % 2 * 512;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((c < 2 * kNsP ? L : R) + at + d),
                                       (__attribute__((address_space(3))) void*)(to + c * 512), 16, 0, 0);
    }
  };
  const int row = lane & 31, oct = lane >> 5, cell = row * kNsK + ((oct ^ row >> 3) & 1) * 8;      // (32 rows on: the same cell)
  nsf16 acc[2][2] = {}, low[2][2] = {};                   // (low: sums of their own for the small products)
  nsb8 lf[2][2][kNsP], rf[2][2][kNsP];                    // operands of the stage that is multiplied, and of the next
  auto fetch = [&](int k, int into) {
    const __bf16* b = ring + k % kBufs * kStage + cell;
#pragma unroll
    for (int q = 0; q < kNsP; ++q) {
#pragma unroll
      for (int e = 0; e < 2; ++e) lf[into][e][q] = *reinterpret_cast<const nsb8*>(b + (q * 2 + e) * 512);
#pragma unroll
      for (int f = 0; f < 2; ++f) rf[into][f][q] = *reinterpret_cast<const nsb8*>(b + kLeft + (q * 2 + f) * 512);
    }
  };
  // stage k is in LDS (behind it up to kBufs - 2 may be on their way), and the operands of stage k - 1 in registers
  auto arrive = [&](int k) {
    if (k + kBufs - 2 < count) asm volatile("s_waitcnt vmcnt(%0)\n\ts_waitcnt lgkmcnt(0)" ::"n"((kBufs - 2) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)" ::: "memory");
  };
  for (int k = 0; k < kBufs - 1 && k < count; ++k) fill(k);
  arrive(0);
  if (kBufs - 1 < count) fill(kBufs - 1);
  fetch(0, 0);
  for (int k = 0; k < count; k += 2)                      // (an even number of stages: K is a multiple of 128)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // the next stage's operands are read under this one's products (behind the last stage: that one again, unused)
      arrive(k + u + 1);
      if (k + u + kBufs < count) fill(k + u + kBufs);
      fetch(min(k + u + 1, count - 1), u ^ 1);
#pragma unroll
      for (int sum = kNsP - 1; sum >= 0; --sum)
#pragma unroll
        for (int q = sum; q >= 0; --q)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              nsf16& to = sum ? low[e][f] : acc[e][f];
              to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lf[u][e][q], rf[u][f][sum - q], to, 0, 0, 0);
            }
    }
  // Wave w finishes 32 x 32 block w of the sums: the others' shares of it come through their rings
  arrive(count);
  constexpr int kRing = kBufs * kStage / 2;               // floats
  float* tile = reinterpret_cast<float*>(stages_);
  nsf4 own[4];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      nsf4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = acc[b >> 1][b & 1][4 * r + j] + low[b >> 1][b & 1][4 * r + j];
      if (b == wave) own[r] = v;
      else *reinterpret_cast<nsf4*>(tile + wave * kRing + kSum + ((b - wave - 1 & 3) * 4 + r) * 256 + lane * 4) = v;
    }
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int from = wave + d & 3;                        // (its shares: blocks from + 1, from + 2, from + 3)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      own[r] += *reinterpret_cast<const nsf4*>(tile + from * kRing + kSum + ((wave - from - 1 & 3) * 4 + r) * 256 + lane * 4);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[((wave >> 1) * 32 + 8 * r + 4 * oct + j) * kNsPitch + (wave & 1) * 32 + row] = own[r][j];
  __syncthreads();
  ns_finish<STAGE>(g, it, s, p, ti * 64, tj * 64, ti == tj, tile);
}

// ---- short sides of up to 128 ------------------------------------------------------------------------------------------------
// A step of such a matrix is launches, not work: the three products and their joins are six launches of 3 to 6 us each that
// leave the card nearly empty.  Here a workgroup owns T columns of X for all steps (X^T and A in LDS, fp32) and a step is ONE
// launch: it adds up the other workgroups' shares of A = X X^T, takes Y = A X and X <- a X + b Y + c A Y of its columns
// (2 m^2 T operations twice instead of m^3 and 2 m^2 T: A A would be computed by every workgroup again), and leaves its
// share of the next A.  |U|_F^2 is the trace of the first A: no launch of its own.  fp32 matrix instructions (16x16x4): the
// products are too small for the split of the operands to pay.
// LDS rows are m + 4 floats (m a multiple of 16): rows 4 apart are 16 banks apart, which keeps both the 16-byte reads along k
// (16 rows, one k) and the 4-byte reads across rows (16 values of rows 4 apart) free of conflicts.
// T.  More columns cost a workgroup more, and every workgroup fewer shares of A to add up.  Five steps of 128 x 256 take 70 us
// with 16 columns and 75 with 32, 128 x 512 103 and 89; 64 x 864 takes 51 us with 32 and 56 with 64, 64 x 1728 71 and 68.  A list
// that has more workgroups than fit the card at once gets more columns each: cheaper than a second round.  (64 columns of more
// than 64 rows would be four blocks a wave: 10 % slower at 128 x 2048 than 32.)
// Long sides: the shares that everybody adds up grow with n^2.  Above 64 rows up to 2048 (128 x 2048 181 us, through the large
// matrices' way 187; 128 x 3000 229 and 174); below them 64 x 8192 takes 134 us (226), 64 x 16384 218 (320).
// A step's time: 128 x 128 10 us, 64 x 1728 12.5 us; the network of MVSNeRF, 29 matrices, 13.5 us.  4 us of it is one launch
// behind another; the rest is a chain of shares, two products and the next share, of which the products are a quarter.
constexpr int kNsShort = 128;                            // short side, and long side (below), up to which this way is taken
__host__ __device__ __forceinline__ int ns_short_long(int m) { return m <= 64 ? 16384 : 2048; }
__host__ __device__ __forceinline__ int ns_columns(int m, int n, int least) {
  const int t = n <= 288 ? 16 : n <= 1152 ? 32 : 64, u = t > least ? t : least;
  return m > 64 && u > 32 ? 32 : u;
}
struct NsShort {
  int m, n, mp, mb, T, parts, blocks, pitch;            // m in 16s: mp = 16 mb; columns of a workgroup; workgroups; 16 x 16 blocks of A's lower triangle
  __host__ __device__ NsShort(const NsShape& s, int least) {
    m = s.m, n = s.n, mp = (m + 15) & ~15, mb = mp / 16, T = ns_columns(m, n, least);
    parts = (n + T - 1) / T, blocks = mb * (mb + 1) / 2, pitch = mp + 4;
  }
  __host__ __device__ long x() const { return (long)n * mp; }                     // floats of X^T
  __host__ __device__ long share() const { return (long)parts * blocks * 256; }   // floats of A's shares
  __host__ __device__ long bytes() const { return (x() + 2 * share()) * 4; }
  __host__ __device__ int lds() const { return (2 * T + mp) * pitch * 4; }
};

// block b of the lower triangle of at most 8 x 8, row by row
__device__ __forceinline__ void ns_triangle(int b, int& i, int& j) {
  i = (b >= 1) + (b >= 3) + (b >= 6) + (b >= 10) + (b >= 15) + (b >= 21) + (b >= 28);
  j = b - i * (i + 1) / 2;
}

// it.at of the matrices that have an XCD of their own: XCD << kNsXcd | slot
constexpr int kNsXcd = 24;

// (DT, MUON: the start's alone; the steps' kernel is one for all)
template <bool START, int DT, bool MUON>
__global__ void __launch_bounds__(512) ns_short_kernel(NsArgs g) {
  extern __shared__ __align__(16) float sm[];
  // (ns_place) workgroups go to the XCDs in turn: slot s of XCD x
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, key = slot < g.spread ? slot : xcd << kNsXcd | slot, i = ns_find(g, key);
  const NsItem it = g.it[i];
  const NsShape shape(it.rows, it.cols);
  const NsShort s(shape, g.least);
  const int wg = slot < g.spread ? (slot - it.at) * 8 + xcd : key - it.at;
  if (wg >= s.parts) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, c16 = lane & 15;
  const int j0 = wg * s.T, nj = min(s.T, s.n - j0);
  float *xs = sm, *ys = xs + s.T * s.pitch, *as = ys + s.T * s.pitch;      // [column][row], [column][row], [row][row]
  float* x = reinterpret_cast<float*>(g.ws + it.ws);
  nsf4* in = reinterpret_cast<nsf4*>(x + s.x() + (g.flip ? s.share() : 0));
  nsf4* out = reinterpret_cast<nsf4*>(x + s.x() + (g.flip ? 0 : s.share()));
  // columns of the tile as rows of m values, 16 bytes a lane, two columns a wave
  const int k4 = lane & 31, jw = wave * 2 + (lane >> 5);
  if (START) {
    // 8 values a thread at a time: of a column (tall: one wave a column) or of a row
    const int sh = 31 - __clz(s.T), all = shape.tall ? s.T * 128 : s.mp << sh;
    for (int e0 = threadIdx.x; e0 < all; e0 += 8 * 512) {
      float v[8];
      int to[8];
      ns_start<DT, MUON, 8>(g, it, true, [&](int u) {
        const int e = e0 + 512 * u, j = shape.tall ? e >> 7 : e & (s.T - 1), k = shape.tall ? e & 127 : e >> sh;
        to[u] = e < all && k < s.mp ? j * s.pitch + k : -1;
        return e < all && j < nj && k < s.m ? (shape.tall ? (long)(j0 + j) * it.cols + k : (long)k * it.cols + j0 + j) : -1l;
      }, v);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (to[u] >= 0) xs[to[u]] = v[u];
    }
    __syncthreads();
  } else {
    // all of the wave's loads in flight at once: its columns of X, then its (at most five) blocks of the shares
    nsf4 xv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = jw + 16 * e;
      xv[e] = j < nj && k4 < s.mp / 4 ? *reinterpret_cast<const nsf4*>(x + (long)(j0 + j) * s.mp + 4 * k4) : nsf4{};
    }
    auto gather = [&](auto nb) {                          // blocks wave, wave + 8, ...: nb of them (the last one again where there are fewer)
      constexpr int NB = decltype(nb)::value;
      nsf4 v[NB] = {};
      const nsf4* from[NB];
#pragma unroll
      for (int e = 0; e < NB; ++e) from[e] = in + min(wave + 8 * e, s.blocks - 1) * 64 + lane;
      const int step = s.blocks * 64;
      int p = 0;
      for (; p + 4 <= s.parts; p += 4) {
        nsf4 w[NB][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < NB; ++e) w[e][u] = from[e][(p + u) * step];
#pragma unroll
        for (int e = 0; e < NB; ++e) v[e] += (w[e][0] + w[e][1]) + (w[e][2] + w[e][3]);
      }
      for (; p < s.parts; ++p)
#pragma unroll
        for (int e = 0; e < NB; ++e) v[e] += from[e][p * step];
#pragma unroll
      for (int e = 0; e < NB; ++e) {
        int bi, bj;
        ns_triangle(min(wave + 8 * e, s.blocks - 1), bi, bj);
#pragma unroll
        for (int r = 0; r < 4; ++r) as[(16 * bi + 4 * q + r) * s.pitch + 16 * bj + c16] = v[e][r];
        *reinterpret_cast<nsf4*>(as + (16 * bj + c16) * s.pitch + 16 * bi + 4 * q) = v[e];
      }
    };
    if (s.blocks <= 8) gather(std::integral_constant<int, 1>{});
    else if (s.blocks <= 16) gather(std::integral_constant<int, 2>{});
    else gather(std::integral_constant<int, 5>{});
    if (k4 < s.mp / 4) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (jw + 16 * e < s.T) *reinterpret_cast<nsf4*>(xs + (jw + 16 * e) * s.pitch + 4 * k4) = xv[e];
      for (int j = jw + 32; j < s.T; j += 16)             // (64 columns)
        *reinterpret_cast<nsf4*>(xs + j * s.pitch + 4 * k4) = j < nj ? *reinterpret_cast<const nsf4*>(x + (long)(j0 + j) * s.mp + 4 * k4) : nsf4{};
    }
    __syncthreads();
    if (g.first) {                                        // X = U / max(|U|, eps), A = (X X^T) / the same squared
      float tr = 0.f;
      for (int k = lane; k < s.mp; k += 64) tr += as[k * s.pitch + k];
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) tr += __shfl_xor(tr, m, 64);
      const float norm = sqrtf(tr), f = 1.f / (norm > g.eps || norm != norm ? norm : g.eps);
      __syncthreads();
      for (int e = threadIdx.x; e < s.mp * s.pitch; e += 512) as[e] = as[e] * f * f;
      for (int e = threadIdx.x; e < s.T * s.pitch; e += 512) xs[e] *= f;
      __syncthreads();
    }
    // block b of the tile: rows 16 (b % mb) ..., columns 16 (b / mb) ...; NE of them a wave: wave, wave + 8, ...  (a wave without
    // a block of its own computes the last one again and writes the same values)
    auto step = [&](auto ne) {
      constexpr int NE = decltype(ne)::value;
      const int tiles = s.mb * (s.T / 16);
      int at[NE], ar[NE], vc[NE];
      nsf4 acc[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int b = min(wave + 8 * e, tiles - 1), rb = b % s.mb, cb = b / s.mb;
        ar[e] = (16 * rb + c16) * s.pitch + 4 * q, vc[e] = (16 * cb + c16) * s.pitch + 4 * q;
        at[e] = (16 * cb + c16) * s.pitch + 16 * rb + 4 * q;      // the lane's four rows of its column
      }
      // A v: the lane's four k-values are 4 q ... 4 q + 3 of every 16, each summed on its own (a chain of m / 4 roundings, not m)
      auto product = [&](const float* v) {
        nsf4 sum[NE][4] = {};
        for (int k = 0; k < s.mp; k += 16)
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            const nsf4 av = *reinterpret_cast<const nsf4*>(as + ar[e] + k), bv = *reinterpret_cast<const nsf4*>(v + vc[e] + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[e][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j], bv[j], sum[e][j], 0, 0, 0);
          }
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[e] = (sum[e][0] + sum[e][1]) + (sum[e][2] + sum[e][3]);
      };
      product(xs);
#pragma unroll
      for (int e = 0; e < NE; ++e) *reinterpret_cast<nsf4*>(ys + at[e]) = acc[e];
      __syncthreads();
      product(ys);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const nsf4 xv = *reinterpret_cast<const nsf4*>(xs + at[e]), yv = *reinterpret_cast<const nsf4*>(ys + at[e]);
        acc[e] = g.a * xv + (g.b * yv + g.c * acc[e]);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < NE; ++e) *reinterpret_cast<nsf4*>(xs + at[e]) = acc[e];
      __syncthreads();
    };
    const int tiles = s.mb * (s.T / 16);
    if (tiles <= 8) step(std::integral_constant<int, 1>{});
    else step(std::integral_constant<int, 2>{});
    if (g.last) {
      const int sh = 31 - __clz(s.T), all = shape.tall ? nj * 128 : s.m << sh;
      for (int e0 = threadIdx.x; e0 < all; e0 += 8 * 512) {
        float v[8];
        long at[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int e = min(e0 + 512 * u, all - 1), j = shape.tall ? e >> 7 : e & (s.T - 1), k = shape.tall ? e & 127 : e >> sh;
          const bool on = e0 + 512 * u < all && j < nj && k < s.m;
          at[u] = on ? (shape.tall ? (long)(j0 + j) * it.cols + k : (long)k * it.cols + j0 + j) : -1l;
          v[u] = on ? xs[j * s.pitch + k] : 0.f;
        }
        ns_results<8>(g, it, [&](int u) { return at[u]; }, v);
      }
      return;
    }
  }
  if (k4 < s.mp / 4)
    for (int j = jw; j < nj; j += 16)
      *reinterpret_cast<nsf4*>(x + (long)(j0 + j) * s.mp + 4 * k4) = *reinterpret_cast<const nsf4*>(xs + j * s.pitch + 4 * k4);
  // this tile's share of X X^T, blocks of the lower triangle in the order of the accumulators
  for (int b = wave; b < s.blocks; b += 8) {
    int bi, bj;
    ns_triangle(b, bi, bj);
    nsf4 sum[4] = {};
    for (int j = 0; j < s.T; j += 16)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* col = xs + (j + e + 4 * q) * s.pitch + c16;
        sum[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(col[16 * bi], col[16 * bj], sum[e], 0, 0, 0);
      }
    out[((long)wg * s.blocks + b) * 64 + lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
static const char* ns_bad(int count, const int* rows, const int* cols) {
  if (count < 0 || (count > 0 && (!rows || !cols))) return "bad list";
  for (int i = 0; i < count; ++i)
    if (rows[i] <= 0 || cols[i] <= 0 || rows[i] > (1 << 16) || cols[i] > (1 << 16)) return "a side is not in 1 ... 65536";
  return nullptr;
}
// the host's lists are the only thing of a call that can throw
template <typename F>
static auto ns_no_throw(F f) -> decltype(f()) {
  try {
    return f();
  } catch (const std::exception&) {
    set_error("Newton-Schulz: out of host memory");
    return BMV_ERR_INVALID;
  }
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
static int ns_chunks(int rows, int cols) { return (int)(((long)rows * cols + kNsChunk - 1) / kNsChunk); }

// limit: of the short side, what BMV_NS_SHORT is at the call (read once: the workspace's layout goes by it)
static int ns_limit() { return std::min(kNsShort, tuning("BMV_NS_SHORT", kNsShort)); }
static bool ns_is_short(int rows, int cols, int limit) {
  const int m = std::min(rows, cols);
  return m <= limit && std::max(rows, cols) <= ns_short_long(m);
}
// Workspace of a part of the list (indices): the short ones' X and shares, or the others' pieces, then the norm's partial
// sums, then partial tiles
// a workgroup's columns at least: the fewest with which the list runs at once (or nearly)
static int ns_short_least(const int* rows, const int* cols, const int* idx, int n) {
  for (int least = 16; least < 64; least *= 2) {
    long wgs = 0;
    int lds = 1;
    for (int k = 0; k < n; ++k) {
      const NsShort s(NsShape(rows[idx[k]], cols[idx[k]]), least);
      wgs += s.parts, lds = std::max(lds, s.lds());
    }
    if (wgs <= kNsUnits * std::min(4, kNsLdsBytes / lds)) return least;
  }
  return 64;
}
static long ns_short_room(const int* rows, const int* cols, const int* idx, int n) {
  const int least = ns_short_least(rows, cols, idx, n);
  long bytes = 0;
  for (int k = 0; k < n; ++k) bytes += NsShort(NsShape(rows[idx[k]], cols[idx[k]]), least).bytes();
  return bytes;
}
struct NsRoom {
  long pieces = 0, tiles = 0;
  int sqn = 1;
  NsRoom(const int* rows, const int* cols, const int* idx, int n) {
    for (int k = 0; k < n; ++k) {
      const int i = idx[k];
      const NsShape s(rows[i], cols[i]);
      pieces += ns_bytes(s), tiles += (long)s.mt() * s.nt();      // (no fewer than the symmetric products')
      sqn = std::max(sqn, ns_chunks(rows[i], cols[i]));
    }
  }
  long bytes() const { return pieces + (long)kNsList * sqn * sizeof(double) + (tiles + kNsSlots) * (kNsTile * kNsTile * 4l); }
};
// the list's indices: the short ones, then the others
static std::vector<int> ns_order(int count, const int* rows, const int* cols, int limit, int& shorts) {
  std::vector<int> v;
  v.reserve(count);
  for (int i = 0; i < count; ++i)
    if (ns_is_short(rows[i], cols[i], limit)) v.push_back(i);
  shorts = (int)v.size();
  for (int i = 0; i < count; ++i)
    if (!ns_is_short(rows[i], cols[i], limit)) v.push_back(i);
  return v;
}
// a list is done in parts of kNsList, which share the workspace
static long ns_workspace(int count, const int* rows, const int* cols, const std::vector<int>& v, int shorts) {
  long most = 0;
  for (int b = 0; b < shorts; b += kNsList) most = std::max(most, ns_short_room(rows, cols, &v[b], std::min(shorts - b, kNsList)));
  for (int b = shorts; b < count; b += kNsList) most = std::max(most, NsRoom(rows, cols, &v[b], std::min(count - b, kNsList)).bytes());
  return most;
}

// 64 x 64 blocks, where rounds of them on all compute units are cheaper than tiles, a cut along k and a join: that goes by the k
// a compute unit walks.  A launch of them is 7.5 us and 0.2 us for 32 k-values -- k = 384 9.9 us, 1024 13.7 ... 19.3
// by how many blocks share the caches --, cut tiles and the launch that joins them 14 ... 25.  Five steps with blocks up to 2048
// and up to 1024: 1024 x 2048 402 us and 428, 768 x 2048 334 and 350, 512 x 2048 251 and 246.
constexpr int kNsBlockK = 2048;
template <int STAGE>
static void ns_block_launch(NsArgs& g, hipStream_t st) {
  // (the longest first: an item's blocks begin in the order of the list)
  std::stable_sort(g.it, g.it + g.count, [](const NsItem& a, const NsItem& b) {
    auto k = [](const NsItem& i) { const NsShape s(i.rows, i.cols); return STAGE == kNsGram ? s.np : s.mp; };
    return k(a) > k(b);
  });
  int slots = 0;
  for (int i = 0; i < g.count; ++i) g.it[i].at = slots, slots += (ns_block_count(NsShape(g.it[i].rows, g.it[i].cols), STAGE) + 7) / 8;
  hipLaunchKernelGGL((ns_block_kernel<STAGE>), dim3(8u * slots), dim3(256), kNsBlockLds, st, g);
}
template <int STAGE>
static bool ns_blocks(NsArgs& g, hipStream_t st) {
  long blocks = 0, most = 0;
  for (int i = 0; i < g.count; ++i) {
    const NsShape s(g.it[i].rows, g.it[i].cols);
    blocks += ns_block_count(s, STAGE), most = std::max<long>(most, STAGE == kNsGram ? s.np : s.mp);
  }
  if ((blocks + kNsUnits - 1) / kNsUnits * most > tuning("BMV_NS_BLOCK_K", kNsBlockK)) return false;
  ns_block_launch<STAGE>(g, st);
  return true;
}

template <int STAGE>
static void ns_product(NsArgs& g, hipStream_t st) {
  if (ns_blocks<STAGE>(g, st)) return;
  long tiles = 0, units = 0;
  for (int i = 0; i < g.count; ++i) {
    const NsShape s(g.it[i].rows, g.it[i].cols);
    g.it[i].at = (int)tiles;
    tiles += STAGE == kNsApply ? (long)s.mt() * s.nt() : s.triangle();
  }
  g.full = (int)(tiles / kNsSlots * kNsSlots);
  for (int i = 0; i < g.count; ++i) {
    const NsShape s(g.it[i].rows, g.it[i].cols);
    const long end = i + 1 < g.count ? g.it[i + 1].at : tiles, begin = std::max<long>(g.it[i].at, g.full);
    if (end > begin) units += (end - begin) * ns_stages(s, STAGE);
  }
  // A run for every compute unit (two for each hide more latency, but a partial tile is 64 KB through memory: 512 x 4096 331 us, one
  // 319), but of at least 256 k-values for the same reason: 160 x 8192 283 us, with 128 322 and with 384 295.  Panels are multiples
  // of 128 long.
  g.run = (int)std::max<long>((units + kNsUnits - 1) / kNsUnits, 256 / kNsK);
  hipLaunchKernelGGL((ns_product_kernel<STAGE>), dim3((unsigned)(g.full + (units + g.run - 1) / g.run)), dim3(256), 0, st, g);
  hipLaunchKernelGGL((ns_join_kernel<STAGE>), dim3((unsigned)(4 * tiles)), dim3(256), 0, st, g);
}

struct NsLists {
  const void* const* src;
  void* const* dst;
  float* const* buf;
  const int *rows, *cols;
  const float* scales;
};
static void ns_fill(NsArgs& g, const NsLists& l, const int* idx, int n) {
  g.count = n;
  for (int k = 0; k < n; ++k) {
    NsItem& it = g.it[k];
    const int i = idx[k];
    it.src = l.src[i], it.dst = l.dst[i], it.buf = l.buf ? l.buf[i] : nullptr, it.rows = l.rows[i], it.cols = l.cols[i];
    it.scale = l.scales ? l.scales[i] : 1.f;
  }
}

// f with the call's type and kind as constants
template <typename F>
static void ns_typed(const NsArgs& g, F f) {
  auto kind = [&](auto dt) {
    if (g.muon) f(dt, std::true_type{});
    else f(dt, std::false_type{});
  };
  if (g.dtype == 0) kind(std::integral_constant<int, 0>{});
  else if (g.dtype == 1) kind(std::integral_constant<int, 1>{});
  else kind(std::integral_constant<int, 2>{});
}

// Which XCD computes which matrix; returns the workgroups of a launch.  Every workgroup of a matrix reads the shares of all others
// of the launch before: on one XCD they are in its L2 (128 x 128 61.7 -> 55.2 us).  The matrices go to the XCDs by their work, the
// largest first, each to the one that has least; one of more workgroups than an XCD has compute units is spread over all.
static unsigned ns_place(NsArgs& g, int least) {
  int parts[kNsList], order[kNsList], alone = 0, slots[8], most = 0;
  long work[kNsList], load[8] = {};
  g.spread = 0;
  for (int i = 0; i < g.count; ++i) {
    const NsShort s(NsShape(g.it[i].rows, g.it[i].cols), least);
    parts[i] = s.parts;
    if (s.parts > kNsUnits / 8) g.it[i].at = g.spread, g.spread += (s.parts + 7) / 8;
    else {
      // (0.01 us: a workgroup 2 us, and 0.0053 us for each block and column, 0.0094 for each block and share)
      work[i] = (long)s.parts * (200 + s.blocks * (s.T / 2 + s.parts));
      int k = alone++;
      for (; k > 0 && work[order[k - 1]] < work[i]; --k) order[k] = order[k - 1];
      order[k] = i;
    }
  }
  for (int x = 0; x < 8; ++x) slots[x] = g.spread;
  for (int k = 0; k < alone; ++k) {
    const int i = order[k], x = (int)(std::min_element(load, load + 8) - load);
    g.it[i].at = x << kNsXcd | slots[x];
    load[x] += work[i], slots[x] += parts[i];
  }
  for (int x = 0; x < 8; ++x) most = std::max(most, slots[x]);
  std::sort(g.it, g.it + g.count, [](const NsItem& a, const NsItem& b) { return a.at < b.at; });
  return 8u * most;
}

static void ns_run_short(NsArgs& g, int least, int steps, char* ws, hipStream_t st) {
  long off = 0;
  int lds = 0;
  g.ws = ws, g.least = least;
  const dim3 grid(ns_place(g, least));
  for (int i = 0; i < g.count; ++i) {
    const NsShort s(NsShape(g.it[i].rows, g.it[i].cols), least);
    g.it[i].ws = off, off += s.bytes(), lds = std::max(lds, s.lds());
  }
  g.flip = 1;                                             // (the first shares go to where step 0 reads)
  ns_typed(g, [&](auto dt, auto muon) { hipLaunchKernelGGL((ns_short_kernel<true, decltype(dt)::value, decltype(muon)::value>), grid, dim3(512), lds, st, g); });
  for (int k = 0; k < steps; ++k) {
    g.first = k == 0, g.last = k + 1 == steps, g.flip = k & 1;
    hipLaunchKernelGGL((ns_short_kernel<false, 0, false>), grid, dim3(512), lds, st, g);
  }
}

static void ns_run_long(NsArgs& g, const NsRoom& room, int steps, char* ws, hipStream_t st) {
  g.ws = ws, g.sqn = room.sqn, g.sq = reinterpret_cast<double*>(ws + room.pieces);
  g.part = reinterpret_cast<float*>(g.sq + (long)kNsList * g.sqn);
  long off = 0, chunks = 0, blocks = 0;
  for (int i = 0; i < g.count; ++i) {
    NsItem& it = g.it[i];
    it.ws = off, it.at = (int)chunks;
    off += ns_bytes(NsShape(it.rows, it.cols)), chunks += ns_chunks(it.rows, it.cols);
  }
  ns_typed(g, [&](auto dt, auto muon) { hipLaunchKernelGGL((ns_norm_kernel<decltype(dt)::value, decltype(muon)::value>), dim3((unsigned)chunks), dim3(256), 0, st, g); });
  for (int i = 0; i < g.count; ++i) g.it[i].at = (int)blocks, blocks += NsShape(g.it[i].rows, g.it[i].cols).big() / (64 * 64);
  ns_typed(g, [&](auto dt, auto muon) { hipLaunchKernelGGL((ns_split_kernel<decltype(dt)::value, decltype(muon)::value>), dim3((unsigned)blocks), dim3(256), 0, st, g); });
  for (int k = 0; k < steps; ++k) {
    g.last = k + 1 == steps, g.flip = k & 1;
    ns_product<kNsGram>(g, st);
    ns_product<kNsPoly>(g, st);
    ns_product<kNsApply>(g, st);
  }
}

// More than 64 KB of LDS, which a kernel gets only where it was asked for, on each device
static bool ns_lds() {
  static constexpr int kLds = (2 * 32 + 128) * (128 + 4) * 4;    // the largest NsShort::lds()
  static std::atomic<unsigned long> ready{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const unsigned long bit = dev < 64 ? 1ul << dev : 0;
  if (ready.load(std::memory_order_acquire) & bit) return true;
  const std::pair<const void*, int> f[] = {{(const void*)ns_short_kernel<true, 0, false>, kLds},
                                           {(const void*)ns_short_kernel<true, 1, false>, kLds},
                                           {(const void*)ns_short_kernel<true, 2, false>, kLds},
                                           {(const void*)ns_short_kernel<true, 0, true>, kLds},
                                           {(const void*)ns_short_kernel<true, 1, true>, kLds},
                                           {(const void*)ns_short_kernel<true, 2, true>, kLds},
                                           {(const void*)ns_short_kernel<false, 0, false>, kLds},
                                           {(const void*)ns_block_kernel<kNsGram>, kNsBlockLds},
                                           {(const void*)ns_block_kernel<kNsPoly>, kNsBlockLds},
                                           {(const void*)ns_block_kernel<kNsApply>, kNsBlockLds}};
  for (const auto& k : f)
    if (hipFuncSetAttribute(k.first, hipFuncAttributeMaxDynamicSharedMemorySize, k.second) != hipSuccess) return false;
  ready.fetch_or(bit, std::memory_order_release);
  return true;
}

static const char* ns_run(NsArgs g, int count, const NsLists& l, int steps, void* workspace, long bytes, hipStream_t st) {
  int shorts;
  const std::vector<int> v = ns_order(count, l.rows, l.cols, ns_limit(), shorts);
  if (ns_workspace(count, l.rows, l.cols, v, shorts) > bytes) return "the workspace is too small";
  if (!ns_lds()) return "LDS refused";
  char* ws = static_cast<char*>(workspace);
  for (int b = 0; b < shorts; b += kNsList) {
    const int n = std::min(shorts - b, kNsList);
    ns_fill(g, l, &v[b], n);
    ns_run_short(g, ns_short_least(l.rows, l.cols, &v[b], n), steps, ws, st);
  }
  for (int b = shorts; b < count; b += kNsList) {
    const int n = std::min(count - b, kNsList);
    ns_fill(g, l, &v[b], n);
    ns_run_long(g, NsRoom(l.rows, l.cols, &v[b], n), steps, ws, st);
  }
  return nullptr;
}

}  // namespace bmv

using namespace bmv;

extern "C" {

long bmv_newton_schulz_workspace(int count, const int* rows, const int* cols, int dtype) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_newton_schulz_workspace: %s", bad);
  BMV_REQUIRE(dtype >= 0 && dtype <= 2, "bmv_newton_schulz_workspace: unknown type %d", dtype);
  return ns_no_throw([&]() -> long {
    int shorts;
    const std::vector<int> v = ns_order(count, rows, cols, ns_limit(), shorts);
    return ns_workspace(count, rows, cols, v, shorts);
  });
}

int bmv_newton_schulz(int count, const void* const* src, void* const* dst, const int* rows, const int* cols, int dtype, int steps,
                      float a, float b, float c, float eps, void* workspace, long workspace_bytes, bmv_stream_t stream) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_newton_schulz: %s", bad);
  BMV_REQUIRE(dtype >= 0 && dtype <= 2, "bmv_newton_schulz: unknown type %d", dtype);
  BMV_REQUIRE(steps > 0 && eps >= 1e-12f, "bmv_newton_schulz: at least one step and eps >= 1e-12 (got %d, %g)", steps, (double)eps);
  if (count == 0) return BMV_OK;
  BMV_REQUIRE(src && dst && workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "bmv_newton_schulz: null pointer, or a workspace off its 256-byte border");
  for (int i = 0; i < count; ++i) BMV_REQUIRE(src[i] && dst[i], "bmv_newton_schulz: null pointer (matrix %d)", i);
  return ns_no_throw([&]() -> int {
    BMV_REQUIRE(ns_apart(count, rows, cols, dtype == 0 ? 4 : 2, src, dst, nullptr), "bmv_newton_schulz: a result overlaps another matrix");
    NsArgs g{};
    g.dtype = dtype, g.a = a, g.b = b, g.c = c, g.eps = eps;
    const NsLists l{src, dst, nullptr, rows, cols, nullptr};
    bad = ns_run(g, count, l, steps, workspace, workspace_bytes, as_stream(stream));
    BMV_REQUIRE(!bad, "bmv_newton_schulz: %s", bad);
    BMV_LAUNCH_END("bmv_newton_schulz");
  });
}

int bmv_muon_step(int count, void* const* params, const void* const* grads, float* const* momenta, const int* rows, const int* cols,
                  const float* scales, int dtype, double momentum, int nesterov, double keep, int steps, float a, float b, float c,
                  float eps, void* workspace, long workspace_bytes, bmv_stream_t stream) {
  const char* bad = ns_bad(count, rows, cols);
  BMV_REQUIRE(!bad, "bmv_muon_step: %s", bad);
  BMV_REQUIRE(dtype >= 0 && dtype <= 2, "bmv_muon_step: unknown type %d", dtype);
  BMV_REQUIRE(steps > 0 && eps >= 1e-12f, "bmv_muon_step: at least one step and eps >= 1e-12 (got %d, %g)", steps, (double)eps);
  if (count == 0) return BMV_OK;
  BMV_REQUIRE(params && grads && momenta && scales && workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
              "bmv_muon_step: null pointer, or a workspace off its 256-byte border");
  for (int i = 0; i < count; ++i) BMV_REQUIRE(params[i] && grads[i] && momenta[i], "bmv_muon_step: null pointer (matrix %d)", i);
  return ns_no_throw([&]() -> int {
    BMV_REQUIRE(ns_apart(count, rows, cols, dtype == 0 ? 4 : 2, grads, params, reinterpret_cast<const void* const*>(momenta)),
                "bmv_muon_step: a weight or a momentum overlaps another tensor (is one listed twice?)");
    NsArgs g{};
    g.dtype = dtype, g.a = a, g.b = b, g.c = c, g.eps = eps, g.muon = 1, g.nesterov = nesterov, g.mu = (float)momentum, g.nu = (float)(1. - momentum), g.keep = (float)keep;
    const NsLists l{grads, params, momenta, rows, cols, scales};
    bad = ns_run(g, count, l, steps, workspace, workspace_bytes, as_stream(stream));
    BMV_REQUIRE(!bad, "bmv_muon_step: %s", bad);
    BMV_LAUNCH_END("bmv_muon_step");
  });
}

}  // extern "C"
