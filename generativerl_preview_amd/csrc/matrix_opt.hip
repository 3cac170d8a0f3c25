// Newton-Schulz orthogonalisation of a group of matrices, and the optimiser step around it (contract: include/grlhip.h,
// grlhip_orthogonalize / grlhip_muon_step).
//
// With m <= n (a matrix with more rows is taken transposed, by its strides), X = G / max(|G|, eps) and, `steps` times,
//     A = X X^T;   B = b A + c A A;   X <- a X + B X,
// an odd polynomial of the singular values that moves them towards 1.  3 m m n + m^3 multiply-adds a step (A and B are
// symmetric: only tiles on and below the diagonal are computed, and written twice).
//
// Every value lives in memory as two fp16 pieces scaled by 2^14 (gemm_core.hip.inc): |X|, |A|, |B| <= 3.9 (checked for the
// coefficients on the host) stay below fp16's largest value, and the second piece of a value of 2^-14 is still no subnormal.  That
// is fp32's rounding level: small singular values grow by a factor of a in every step, and so does what single fp16 pieces
// round away (measured: relative error 2e-3 to 2e-2, with two pieces 1e-6 to 1e-5, fp32 products the same).
//
// One launch per product for all matrices of a call, whatever their number: 3 steps + 2 launches.  A call whose matrices all fit into the
// LDS of one workgroup each (64 x 192 padded) is ONE launch, a workgroup per matrix (k_orth_small).
#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/grlhip.h"
#include "errors.hpp"
#include "gemm_core.hip.inc"

namespace grlhip {
int device_cus();
namespace {
using namespace mx;

constexpr float S = 16384.f;        // scale of X, A, B
constexpr int GROUP = 32;           // matrices described by the kernel arguments of one launch (graphs keep them)
constexpr int64_t MAX_SIDE = 1 << 16;

enum Stage { GRAM, POLY, UPDATE, LAST };

// One matrix, oriented to m <= n.  Strides in elements: [0] along m, [1] along n.
struct Mat {
  const void* g;      // matrix / gradient
  void* out;          // result / parameter
  float* buf;         // momentum (muon) or null
  char* ws;           // its part of the workspace, see Parts
  int64_t gs[2], os[2], bs[2];
  int m, n;
  float rate;         // muon: learning rate of this matrix
  int first[4];       // its first block of the norm and split launches, and its first tile of the GRAM, POLY and UPDATE launches
};
struct Numbers {
  float ca, cb, cc, eps;
  float momentum, fresh, keep;   // muon: momentum; 1 - momentum, from 64 bits; 1 - lr * weight decay
  int nesterov;
};
// What the launches after the first know of the matrices lies in the workspace: `first` of all matrices, [4][count], and the
// descriptions themselves.
// To the products a lone matrix comes with the kernel arguments instead: two trips to memory less in each of these launches.
struct Table { const int* first; const Mat* mat; int count; double* part; Mat one; };
struct Group {
  Mat mat[GROUP];
  int count, from;    // matrices here; matrices before them in the table
  int blocks0;        // blocks before this launch
  int* first; Mat* table; int all; double* part;
  Numbers num;
};
static_assert(sizeof(Group) <= 4000, "kernel arguments");

__host__ __device__ inline int64_t up32(int64_t v) { return (v + 31) / 32 * 32; }
__host__ __device__ inline int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }
// Pieces of a matrix in the workspace: two X, two X^T (a step reads one and writes the other), A, B.
struct Parts {
  int64_t mp, np, x, a;   // padded sides; bytes of an X, of an A
  __host__ __device__ Parts(int m, int n) : mp(up32(m)), np(up32(n)) { x = mp * np * 4; a = mp * mp * 4; }
  __host__ __device__ int64_t bytes() const { return (4 * x + 2 * a + 255) / 256 * 256; }
  __host__ __device__ int blocks() const { return (int)((mp + 63) / 64 * ((np + 63) / 64)); }
  __device__ _Float16* X(char* ws, int k) const { return (_Float16*)(ws + k * x); }
  __device__ _Float16* XT(char* ws, int k) const { return (_Float16*)(ws + (2 + k) * x); }
  __device__ _Float16* A(char* ws) const { return (_Float16*)(ws + 4 * x); }
  __device__ _Float16* B(char* ws) const { return (_Float16*)(ws + 4 * x + a); }
};
// entry (row, col) of a piece array with `cols` columns: the high piece, the low one 32 further
__device__ __forceinline__ int64_t at(int64_t row, int col, int64_t cols) { return row * 2 * cols + (col >> 5) * 64 + (col & 31); }

// The matrix that block / tile `id` of a launch belongs to: the last one that starts at or before it.  One load a lane, one
// ballot: a search would wait for memory at every step.
__device__ __forceinline__ int find(const int* first, int count, int id) {
  int below = 0;
  for (int at = 0; at < count; at += 64) {
    const int k = at + (int)(threadIdx.x & 63);
    below += __popcll(__ballot(k < count && first[k] <= id));
  }
  return __builtin_amdgcn_readfirstlane(below - 1);
}

template <class T> __device__ __forceinline__ float load(const T* p) { return (float)*p; }

// Thread t's elements of a 64 x 64 block: i0 + k di, j; along the axis that is contiguous in memory, for whole lines.
struct Walk { int i, j, di, dj; };
__device__ __forceinline__ Walk walk(bool along_n) {
  const int t = threadIdx.x;
  return along_n ? Walk{t >> 6, t & 63, 4, 0} : Walk{t & 63, t >> 6, 0, 4};
}

// buf = momentum buf + (1 - momentum) g and the direction u, or u = g, of N entries of a thread (entry e at (r[e], c[e]); outside the matrix:
// 0).  FIRST: the pass that updates buf; later ones find it updated.  All loads come before the first store, which may
// alias them as far as the compiler knows: one trip to memory, not N.
template <class T, bool MUON, bool FIRST, int N, class F>
__device__ __forceinline__ void directions(const Numbers& g, const Mat& a, F&& place, float (&u)[N]) {
  float v[MUON ? N : 1];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    int r, c;
    const bool in = place(e, r, c);
    u[e] = in ? load((const T*)a.g + r * a.gs[0] + c * a.gs[1]) : 0.f;
    if (MUON) v[MUON ? e : 0] = in ? a.buf[r * a.bs[0] + c * a.bs[1]] : 0.f;
  }
  if (!MUON) return;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    int r, c;
    const bool in = place(e, r, c);
    float& b = v[MUON ? e : 0];
    if (FIRST) {
      b = g.momentum * b + g.fresh * u[e];
      if (in) a.buf[r * a.bs[0] + c * a.bs[1]] = b;
    }
    u[e] = g.nesterov ? g.fresh * u[e] + g.momentum * b : b;
  }
}

// Sum over the block, in one order; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* sh) {
  sh[threadIdx.x] = v;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    __syncthreads();
  }
  return sh[0];
}
// What u is multiplied by: in 64 bits, as the quotient can pass fp32's range where the elements are tiny.
__device__ __forceinline__ double factor_of(double squares, float eps) {
  const double norm = sqrt(squares);
  return (double)S / (norm > eps || norm != norm ? norm : (double)eps);
}

// Pass 1: momentum, and the sum of squares of each 64 x 64 block in 64 bits (a sum that every later product depends on).  The
// first block also leaves the descriptions for the launches to come.
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_norm(Group g) {
  if (blockIdx.x == 0)
    for (int k = threadIdx.x; k < g.count; k += 256) {
      g.table[g.from + k] = g.mat[k];
#pragma unroll
      for (int f = 0; f < 4; ++f) g.first[f * g.all + g.from + k] = g.mat[k].first[f];
    }
  const int id = blockIdx.x + g.blocks0;
  // the last matrix that starts at or before this block: a lane looks at each
  const int lane = threadIdx.x & 63;
  const int e = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < g.count && g.mat[lane < GROUP ? lane : 0].first[0] <= id)) - 1);
  const Mat& a = g.mat[e];
  const int nb = (int)(up64(a.n) / 64), b = id - a.first[0];
  const int i0 = b / nb * 64, j0 = b % nb * 64;
  const Walk w = walk(a.gs[1] <= a.gs[0]);
  float u[16];
  directions<T, MUON, true>(g.num, a, [&](int k, int& i, int& j) { i = i0 + w.i + k * w.di; j = j0 + w.j + k * w.dj; return i < a.m && j < a.n; }, u);
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += (double)u[k] * u[k];
  __shared__ double sh[256];
  s = block_sum(s, sh);
  if (threadIdx.x == 0) g.part[id] = s;
}

// Pass 2: X = S u / max(|u|, eps) as pieces, and X^T.  Every block adds its matrix' partial sums, in the same order.
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_split(Table t, Numbers g) {
  const Mat& a = t.mat[find(t.first, t.count, blockIdx.x)];
  const Parts p(a.m, a.n);
  const int nb = (int)((p.np + 63) / 64), b = blockIdx.x - a.first[0], all = p.blocks();
  __shared__ double sh[256];
  __shared__ float tile[64][65];
  const int i0 = b / nb * 64, j0 = b % nb * 64;
  const Walk w = walk(a.gs[1] <= a.gs[0]);
  float u[16];
  directions<T, MUON, false>(g, a, [&](int k, int& i, int& j) { i = i0 + w.i + k * w.di; j = j0 + w.j + k * w.dj; return i < a.m && j < a.n; }, u);
  double s = 0.0;
  for (int k = threadIdx.x; k < all; k += 256) s += t.part[a.first[0] + k];
  const double inv = factor_of(block_sum(s, sh), g.eps);
#pragma unroll
  for (int k = 0; k < 16; ++k) tile[w.i + k * w.di][w.j + k * w.dj] = (float)(u[k] * inv);
  __syncthreads();
  // 8 threads write the 128 bytes of 32 entries of a row: 4 their high pieces, 4 the low ones; X, then X^T
  const int chunk = threadIdx.x & 7, low = chunk >> 2, c8 = (chunk & 3) * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int q = (threadIdx.x >> 3) + 32 * k, row = q >> 1, col = (q & 1) * 32;
    f16x8 x, xt;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 hi, lo;
      split2(tile[row][col + c8 + e], hi, lo);
      x[e] = low ? lo : hi;
      split2(tile[col + c8 + e][row], hi, lo);
      xt[e] = low ? lo : hi;
    }
    // the sides are padded to 32 only
    if (i0 + row < p.mp && j0 + col < p.np) *(f16x8*)(p.X(a.ws, 0) + at(i0 + row, j0 + col, p.np) + low * 32 + c8) = x;
    if (j0 + row < p.np && i0 + col < p.mp) *(f16x8*)(p.XT(a.ws, 0) + at(j0 + row, i0 + col, p.mp) + low * 32 + c8) = xt;
  }
}

// One product of every matrix.  k: which X is read.
template <class C, int STAGE, class T, bool MUON>
__global__ __launch_bounds__(C::THREADS, C::LDS > 81920 || C::THREADS < 256 ? (C::THREADS + 255) / 256 : C::THREADS / 128) void k_orth_product(Table t, Numbers g, int k) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  constexpr bool SYM = STAGE == GRAM || STAGE == POLY;
  constexpr int FIRST = STAGE == LAST ? 3 : STAGE + 1;
  Mat a;
  if (t.count == 1) a = t.one;
  else a = t.mat[find(t.first + FIRST * t.count, t.count, blockIdx.x)];
  const Parts p(a.m, a.n);
  const int tm = (int)((p.mp + C::BM - 1) / C::BM), tn = SYM ? tm : (int)((p.np + C::BN - 1) / C::BN);
  // the XCDs' ranges are taken inside each matrix: matrices differ in the length of their tiles
  const int u = xcd_order(blockIdx.x - a.first[FIRST], SYM ? tm * (tm + 1) / 2 : tm * tn);
  int im, in;
  if (SYM) {   // tile u of the lower triangle, row by row
    im = (int)((sqrtf(8.f * u + 1.f) - 1.f) * 0.5f);
    while (im * (im + 1) / 2 > u) --im;
    while ((im + 1) * (im + 2) / 2 <= u) ++im;
    in = u - im * (im + 1) / 2;
  } else {
    tile_at(u, tm, tn, im, in);
  }
  const int64_t m0 = (int64_t)im * C::BM, n0 = (int64_t)in * C::BN;
  f32x16 acc[C::TM][C::TN];
  const int64_t xp = p.np * 4, ap = p.mp * 4;   // row pitches in bytes
  const Lane L = lane_of();
  const int wm = L.wave / C::WN % C::WM, wn = L.wave % C::WN;
  // The operand that the epilogue adds (A of the polynomial, X of the update; read transposed: 4 consecutive entries).  Small
  // tiles ask for it before their last block: its latency, 1 us from another XCD's stores, is a good part of such a launch.  (Asked for
  // before the product it stood in front of the tiles' own loads: a product of 256 x 256 took 4.0 us instead of 2.7.)
  constexpr bool OWN = STAGE != GRAM, EARLY = OWN && C::TM * C::TN == 1;
  f16x4 own[EARLY ? 8 : 1];
  auto load_own = [&](int64_t mb, int64_t n, f16x4* hi, f16x4* lo) {
    const _Float16* o = STAGE == POLY ? p.A(a.ws) + at(n, (int)mb, p.mp) : p.XT(a.ws, k) + at(n, (int)mb, p.mp);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      hi[c] = *(const f16x4*)(o + 8 * c + 4 * L.h);
      lo[c] = *(const f16x4*)(o + 32 + 8 * c + 4 * L.h);
    }
  };
  auto late = [&] {
    const int64_t mb = m0 + wm * 32, nb = n0 + wn * 32;
    if (EARLY && mb < p.mp && nb < (SYM ? p.mp : p.np)) load_own(mb, nb + L.j, own, own + (EARLY ? 4 : 0));
  };
  if (STAGE == GRAM) {
    const char* x = (const char*)p.X(a.ws, k);
    if (!product<_Float16, 2, C>(x + m0 * xp, xp, p.mp - m0, x + n0 * xp, xp, p.mp - n0, (int)(p.np / 32), lds, acc)) return;
  } else if (STAGE == POLY) {
    const char* x = (const char*)p.A(a.ws);
    if (!product<_Float16, 2, C>(x + m0 * ap, ap, p.mp - m0, x + n0 * ap, ap, p.mp - n0, (int)(p.mp / 32), lds, acc, late)) return;
  } else {
    if (!product<_Float16, 2, C>((const char*)p.B(a.ws) + m0 * ap, ap, p.mp - m0, (const char*)p.XT(a.ws, k) + n0 * ap, ap, p.np - n0,
                                 (int)(p.mp / 32), lds, acc, late)) return;
  }
  unsigned* patch = (unsigned*)(lds + L.wave * PATCH);
#pragma unroll
  for (int y = 0; y < C::TM; ++y) {
#pragma unroll
    for (int x = 0; x < C::TN; ++x) {
      const int64_t mb = m0 + (wm * C::TM + y) * 32, nb = n0 + (wn * C::TN + x) * 32;
      if (mb >= p.mp || nb >= (SYM ? p.mp : p.np)) continue;   // sides are padded to 32: whole blocks only
      const int64_t n = nb + L.j;
      float v[16];
      if (STAGE == GRAM) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = acc[y][x][r] * (1.f / S);
      } else {
        const float f = STAGE == POLY ? g.cb : g.ca, q = (STAGE == POLY ? g.cc : 1.f) * (1.f / S);
        f16x4 late[EARLY ? 1 : 8];
        if constexpr (!EARLY) load_own(mb, n, late, late + 4);
        const f16x4 *hi = EARLY ? own : late, *lo = EARLY ? own + 4 : late + 4;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * c + i] = f * ((float)hi[c][i] + (float)lo[c][i]) + q * acc[y][x][4 * c + i];
      }
      if (SYM) {
        _Float16* D = STAGE == GRAM ? p.A(a.ws) : p.B(a.ws);
        store_t_f16x2(D + at(nb, (int)mb, p.mp), 2 * p.mp, patch, L, 32, v);
        if (im != in) store_n_f16x2(D + at(mb, (int)nb, p.mp), 2 * p.mp, patch, L, 32, v);
      } else if (STAGE == UPDATE) {
        store_t_f16x2(p.XT(a.ws, k ^ 1) + at(nb, (int)mb, p.mp), 2 * p.mp, patch, L, 32, v);
        store_n_f16x2(p.X(a.ws, k ^ 1) + at(mb, (int)nb, p.np), 2 * p.np, patch, L, 32, v);
      } else {   // the result, in the matrix' own type and place: the one rounding to that type
        const bool turned = a.os[0] < a.os[1];   // dense along m: turned round in LDS, so that lanes follow memory
        if (turned) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *(f32x4v*)((float*)patch + L.j * 36 + 8 * c + 4 * L.h) = f32x4v{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = ((float*)patch)[(2 * i + L.h) * 36 + L.j];
        }
        T* const o = (T*)a.out + (turned ? (mb + L.j) * a.os[0] + (nb + L.h) * a.os[1] : (mb + 4 * L.h) * a.os[0] + n * a.os[1]);
        auto offset = [&](int r) { return turned ? 2 * r * a.os[1] : (8 * (r >> 2) + (r & 3)) * a.os[0]; };
        auto inside = [&](int r) { return turned ? mb + L.j < a.m && nb + 2 * r + L.h < a.n : mb + 8 * (r >> 2) + 4 * L.h + (r & 3) < a.m && n < a.n; };
        float old[16];   // all loads before the first store: they may alias as far as the compiler knows
#pragma unroll
        for (int r = 0; r < 16; ++r) old[r] = MUON && inside(r) ? (float)o[offset(r)] : 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float d = v[r] * (1.f / S);
          if (inside(r)) o[offset(r)] = MUON ? (T)(g.keep * old[r] - a.rate * d) : (T)d;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------- small matrices
// A matrix whose sides are at most 64 and 192 stays in one workgroup's LDS from the first load to the last store: X, X^T, A and B as
// pieces, a barrier between products.  One launch for the group where the chain has 17, each of which lasts 4 us however little
// it does: 128 x 64 in 28 us (chain: 75), 16 x 16 in 12.  What bounds it is latency -- 9 500 cycles a step of 128 x 64 --, hence 16 waves with a 16 x 16 block each (16x16x32 instructions, a third of the 32 x 32 block's
// dependent time), one accumulator for each of the three products of pieces.
constexpr int SMALL_M = 64, SMALL_N = 192, SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64;
constexpr int SMALL_X = SMALL_M * (SMALL_N * 4 + 16), SMALL_XT = SMALL_N * (SMALL_M * 4 + 16), SMALL_A = SMALL_M * (SMALL_M * 4 + 16);
constexpr int SMALL_LDS = SMALL_X + SMALL_XT + 2 * SMALL_A;

// Rows of K blocks (32 high pieces, 32 low ones), 16 bytes apart from a multiple of 128: 16 rows of one chunk then lie in different banks
struct Plane {
  unsigned char* p; int pitch;   // bytes
  __device__ Plane(unsigned char* at_, int cols) : p(at_), pitch(cols * 4 + 16) {}
  __device__ unsigned char* at(int row, int col) const { return p + row * pitch + (col >> 5) * 128 + (col & 31) * 2; }   // the high piece; the low one is 64 further
  __device__ void put(int row, int col, _Float16 hi, _Float16 lo) const {
    unsigned char* q = at(row, col);
    *(_Float16*)q = hi;
    *(_Float16*)(q + 64) = lo;
  }
};
typedef float f32x4a __attribute__((ext_vector_type(4)));
// Sum over kb of rows ra.. of a and rows rb.. of b: a lane's entries are rows 4 (lane / 16) + i of a, row lane % 16 of b.
__device__ __forceinline__ f32x4a small_product(Plane a, int ra, Plane b, int rb, int nkb, int lane) {
  f32x4a hh = {0.f, 0.f, 0.f, 0.f}, hl = hh, lh = hh;
  const unsigned char *pa = a.p + (ra + (lane & 15)) * a.pitch + (lane >> 4) * 16, *pb = b.p + (rb + (lane & 15)) * b.pitch + (lane >> 4) * 16;
#pragma unroll 2
  for (int kb = 0; kb < nkb; ++kb) {
    const f16x8 ah = *(const f16x8*)(pa + kb * 128), al = *(const f16x8*)(pa + kb * 128 + 64);
    const f16x8 bh = *(const f16x8*)(pb + kb * 128), bl = *(const f16x8*)(pb + kb * 128 + 64);
    hl = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, hl, 0, 0, 0);
    lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, lh, 0, 0, 0);
    hh = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, hh, 0, 0, 0);
  }
  return hh + (hl + lh);
}
// Values of a block -> row n, 4 entries from m of `t`, and (both) rows m.., entry n of `d`.
__device__ __forceinline__ void small_store(Plane t, Plane d, bool both, int m, int n, f32x4a v) {
  f16x4 hi, lo;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    _Float16 x, y;
    split2(v[i], x, y);
    hi[i] = x;
    lo[i] = y;
    if (both) d.put(m + i, n, x, y);
  }
  unsigned char* q = t.at(n, m);
  *(f16x4*)q = hi;
  *(f16x4*)(q + 64) = lo;
}
__device__ __forceinline__ f32x4a small_load(Plane t, int m, int n) {
  const unsigned char* q = t.at(n, m);
  const f16x4 hi = *(const f16x4*)q, lo = *(const f16x4*)(q + 64);
  f32x4a v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)hi[i] + (float)lo[i];
  return v;
}

// entry k of a matrix, counted along the axis that is dense in memory.  The quotient of k < 2^14 by a side < 2^8 in fp32: off by less
// than the 1 / 2^9 that (k + 1/2) / side keeps from the next integer.
struct Spread {
  bool along; int inner; float inverse;
  __device__ Spread(bool along_n, const Mat& a) : along(along_n), inner(along_n ? a.n : a.m) { inverse = 1.f / inner; }
  __device__ void at(int k, int& r, int& c) const {
    const int o = (int)((k + 0.5f) * inverse), i = k - o * inner;
    r = along ? o : i;
    c = along ? i : o;
  }
};

template <class T, bool MUON>
__global__ __launch_bounds__(SMALL_THREADS, 4) void k_orth_small(Group g, int steps) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  __shared__ double sh[SMALL_WAVES];
  const Mat& a = g.mat[blockIdx.x];
  const int mp = (int)up32(a.m), np = (int)up32(a.n);
  const Lane L = lane_of();
  const Plane X(lds, np), XT(lds + SMALL_X, mp), A(lds + SMALL_X + SMALL_XT, mp), B(lds + SMALL_X + SMALL_XT + SMALL_A, mp);
  // momentum and norm; threads along the axis that is dense in memory, all of a thread's loads in flight at once
  constexpr int PER = SMALL_M * SMALL_N / SMALL_THREADS;
  const int all = a.m * a.n;
  const Spread in{a.gs[1] <= a.gs[0], a}, to{a.os[1] <= a.os[0], a};
  float u[PER];
  directions<T, MUON, true>(g.num, a, [&](int e, int& r, int& c) { const int k = threadIdx.x + e * SMALL_THREADS; in.at(k, r, c); return k < all; }, u);
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < PER; ++e) s += (double)u[e] * u[e];
  for (int k = threadIdx.x; k < (SMALL_X + SMALL_XT) / 16; k += SMALL_THREADS) ((u32x4*)lds)[k] = u32x4{0, 0, 0, 0};   // the padding stays zero
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  if (L.lane == 0) sh[L.wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int k = 0; k < SMALL_WAVES; ++k) s += sh[k];
  const double inv = factor_of(s, g.num.eps);
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int k = threadIdx.x + e * SMALL_THREADS;
    if (k >= all) continue;
    int r, c;
    in.at(k, r, c);
    _Float16 hi, lo;
    split2((float)(u[e] * inv), hi, lo);
    X.put(r, c, hi, lo);
    XT.put(c, r, hi, lo);
  }
  __syncthreads();

  constexpr int EACH = SMALL_M / 16 * (SMALL_N / 16) / SMALL_WAVES;
  const int lane = L.lane, m4 = 4 * (lane >> 4), n1 = lane & 15, tm = mp / 16, tn = np / 16;
  // the symmetric products: block w of the lower triangle by wave w
  int bm = 0;
  while ((bm + 1) * (bm + 2) / 2 <= L.wave) ++bm;
  const int bn = L.wave - bm * (bm + 1) / 2;
  const bool sym = bm < tm;
  for (int step = 0; step < steps; ++step) {
    if (sym) small_store(A, A, bm != bn, bm * 16 + m4, bn * 16 + n1, small_product(X, bm * 16, X, bn * 16, np / 32, lane) * (1.f / S));
    __syncthreads();
    if (sym) {
      const f32x4a own = small_load(A, bm * 16 + m4, bn * 16 + n1);
      small_store(B, B, bm != bn, bm * 16 + m4, bn * 16 + n1,
                  g.num.cb * own + (g.num.cc * (1.f / S)) * small_product(A, bm * 16, A, bn * 16, mp / 32, lane));
    }
    __syncthreads();
    f32x4a v[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int b = L.wave + e * SMALL_WAVES, im = b % tm * 16, in = b / tm * 16;
      if (b < tm * tn) v[e] = g.num.ca * small_load(XT, im + m4, in + n1) + (1.f / S) * small_product(B, im, XT, in, mp / 32, lane);
    }
    __syncthreads();   // everybody has read X before it is written
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int b = L.wave + e * SMALL_WAVES, im = b % tm * 16, in = b / tm * 16;
      if (b < tm * tn) small_store(XT, X, true, im + m4, in + n1, v[e]);
    }
    __syncthreads();
  }
  // the result, threads along memory again: the one rounding to the matrix' type (pieces hold 22 bits)
  float old[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int k = threadIdx.x + e * SMALL_THREADS;
    int r, c;
    to.at(k, r, c);
    old[e] = MUON && k < all ? (float)((T*)a.out)[r * a.os[0] + c * a.os[1]] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int k = threadIdx.x + e * SMALL_THREADS;
    if (k >= all) continue;
    int r, c;
    to.at(k, r, c);
    const float d = ((float)*(_Float16*)X.at(r, c) + (float)*(_Float16*)(X.at(r, c) + 64)) * (1.f / S);
    ((T*)a.out)[r * a.os[0] + c * a.os[1]] = MUON ? (T)(g.num.keep * old[e] - a.rate * d) : (T)d;
  }
}

// steps == 0: the normalised matrix itself
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_join(Table t, Numbers g) {
  const Mat& a = t.mat[find(t.first, t.count, blockIdx.x)];
  const Parts p(a.m, a.n);
  const int nb = (int)((p.np + 63) / 64), b = blockIdx.x - a.first[0];
  const int i0 = b / nb * 64, j0 = b % nb * 64;
  const Walk w = walk(a.os[1] <= a.os[0]);
  for (int k = 0; k < 16; ++k) {
    const int i = i0 + w.i + k * w.di, j = j0 + w.j + k * w.dj;
    if (i < a.m && j < a.n) {
      const _Float16* x = p.X(a.ws, 0) + at(i, j, p.np);
      const float d = ((float)x[0] + (float)x[32]) * (1.f / S);
      T* o = (T*)a.out + i * a.os[0] + j * a.os[1];
      *o = MUON ? (T)(g.keep * (float)*o - a.rate * d) : (T)d;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- host
struct Call {
  const void* const* src; void* const* dst; float* const* buf;
  const int64_t* shapes;    // [count][2] rows, cols
  const int64_t* strides;   // [count][6] row and column strides of src, dst, buf in elements, or null: contiguous
  int count, steps;
  float ca, cb, cc, eps;
  const float* rate;        // [count] or null
  double momentum;
  float keep;
  int nesterov;
};

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
Parts parts_of(const int64_t* shape) {
  const int64_t r = shape[0], c = shape[1];
  return Parts((int)(r < c ? r : c), (int)(r < c ? c : r));
}
int64_t workspace_bytes(const int64_t* shapes, int count) {
  int64_t bytes = 0, blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (shapes[2 * i] <= 0 || shapes[2 * i + 1] <= 0) continue;
    const Parts p = parts_of(shapes + 2 * i);
    bytes += p.bytes();
    blocks += p.blocks();
  }
  return bytes + up256(blocks * 8) + up256((int64_t)count * sizeof(Mat)) + up256((int64_t)count * 16) + 256;
}

int check_shapes(const char* who, const int64_t* shapes, int count) {
  if (count < 0 || (count > 0 && !shapes)) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": null shapes or negative count");
  for (int i = 0; i < count; ++i)
    for (int k = 0; k < 2; ++k)
      if (shapes[2 * i + k] < 0 || shapes[2 * i + k] > MAX_SIDE)
        return set_error(GRLHIP_ERR_UNSUPPORTED, std::string(who) + ": a side of matrix " + std::to_string(i) + " is negative or over 65536");
  return 0;
}

// The pieces hold values up to 3.9 in magnitude: follow the largest singular value (1 after the division by the Frobenius norm)
// through the steps, on a grid, and the largest eigenvalue of B.
int check_coefficients(const char* who, float a, float b, float c, int steps) {
  if (steps < 0 || steps > 32) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": steps must be between 0 and 32");
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": coefficients must be finite");
  double top = 1.0;
  for (int s = 0; s < steps; ++s) {
    double x_most = 0.0, b_most = 0.0;
    for (int k = 0; k <= 512; ++k) {
      const double x = top * k / 512, q = x * x, p = b * q + c * q * q;
      x_most = std::fmax(x_most, std::fabs((a + p) * x));
      b_most = std::fmax(b_most, std::fabs(p));
    }
    if (x_most > 1.9 || b_most > 3.8)
      return set_error(GRLHIP_ERR_UNSUPPORTED, std::string(who) + ": with these coefficients a singular value passes 1.9 or b s^2 + c s^4 passes 3.8 "
                                                                  "in magnitude, beyond the range of the fp16 pieces");
    top = x_most;
  }
  return 0;
}

// The shapes of tiles.  Products of plain square operands by kind in the order below, us:
//   512 x 512 x 512: 4.2, 4.6, 5.7, 6.2, 7.5, 9.4, 11.4, 12.5, 30;  1024 x 1024 x 1024: 18, 15, 12.5, 10.7, 13.3, 16.6, 20.5, 23.6, 57;
//   2048 x 2048 x 1024: -, -, -, 38, -, 35, 25.4, 28.3, 61;  8192 x 8192 x 2048: 774 (128), 698 (256: 1180 TFLOP/s of MFMAs).
typedef Tile<32, 32, 1, 1, 3, 4> Orth32K;      // 96 KiB, one a CU: three stages cover the latency of few tiles
typedef Tile<32, 32, 1, 1, 2, 4> Orth32;       // 64 KiB, two a CU
typedef Tile<32, 32, 1, 1, 2, 2> Orth32S;      // 32 KiB, five a CU: many short tiles
typedef Tile<64, 64, 2, 2, 3, 2> Orth64K;      // 96 KiB
typedef Tile<64, 64, 2, 2, 2, 2> Orth64;       // 64 KiB
typedef Tile<96, 96, 1, 3, 2, 3> Orth96K;      // 144 KiB: the triangle of 2048 is 253 of these, and 136 of 128
typedef Tile<128, 128, 2, 2, 2, 2> Orth128K;   // 128 KiB
typedef Tile<128, 128, 2, 2, 2> Orth128;       // 64 KiB
typedef Tile<256, 256, 2, 4, 2> Orth256;       // 128 KiB
constexpr int KINDS = 9, SIDE[KINDS] = {32, 32, 32, 64, 64, 96, 128, 128, 256}, BESIDE[KINDS] = {1, 2, 5, 1, 2, 1, 1, 2, 1};   // workgroups a CU
// A launch, in us: ALONE is a K block of 32 (two pieces, 3 MFMAs) of a tile with its CU to itself, FULL the CU's time for one of a full chip,
// FIXED what a tile costs whatever its length, shared by the workgroups beside each other, EPILOGUE an entry's stores and loads.
// Fitted to the times of 28 groups of matrices (one of 128 x 128 to 24 of 1024 x 4096) with each kind in each of the three products in turn:
// in all of them but one the kind that the rule takes is within 1.5 % of the best call, and in that one within 3 %; 18 other groups: 2 %, and 5 % in one.
// Near its ties it errs by more: of 135 random groups whose choice changes when FULL of the two-a-CU 64-wide tile is 5 % higher, the other
// choice was 1.5 % slower on average, but 12 % faster in the best one (3 x 1000 x 777: 345 us by the fit, 329 by the other).
constexpr double ALONE[KINDS] = {0.096, 0.131, 0.26, 0.224, 0.333, 0.48, 0.584, 0.646, 1.58};
constexpr double FULL[KINDS] = {0.104, 0.09, 0.093, 0.222, 0.212, 0.474, 0.641, 0.563, 2.24};
constexpr double FIXED[KINDS] = {1.74, 1.46, 1.19, 1.79, 1.16, 0.88, 2.72, 3.17, 2.64}, EPILOGUE = 1.2e-3;

int64_t tiles_of(const Parts& p, int stage, int side) {
  const int64_t tm = (p.mp + side - 1) / side, tn = (p.np + side - 1) / side;
  return stage == UPDATE ? tm * tn : tm * (tm + 1) / 2;
}
struct Plan { int kind[3]; int64_t tiles[3]; int64_t blocks; };   // by stage
// A launch lasts as long as its longest tile, or as its tiles together on all CUs, in whole tiles a CU.
Plan plan_of(const int64_t* shapes, int count) {
  Plan plan = {};
  double longest[3][KINDS] = {}, sum[3][KINDS] = {}, best[3] = {};
  int64_t tiles[3][KINDS] = {};
  for (int i = 0; i < count; ++i) {
    if (shapes[2 * i] <= 0 || shapes[2 * i + 1] <= 0) continue;
    const Parts p = parts_of(shapes + 2 * i);
    plan.blocks += p.blocks();
    for (int s = 0; s < 3; ++s)
      for (int k = 0; k < KINDS; ++k) {
        const double kb = (double)(s == GRAM ? p.np : p.mp) / 32;
        const int64_t t = tiles_of(p, s, SIDE[k]);
        tiles[s][k] += t;
        sum[s][k] += t * (kb * FULL[k] + FIXED[k] / BESIDE[k]);
        longest[s][k] = std::fmax(longest[s][k], kb * ALONE[k]);
      }
  }
  const double cus = device_cus();
  for (int s = 0; s < 3; ++s) {
    for (int k = 0; k < KINDS; ++k) {
      const double rounds = tiles[s][k] / cus, all = rounds > 1 ? sum[s][k] / cus * std::ceil(rounds) / rounds : 0.0;
      const double us = std::fmax(longest[s][k] + FIXED[k], all) + rounds * SIDE[k] * SIDE[k] * EPILOGUE;
      if (k == 0 || us < best[s]) {
        best[s] = us;
        plan.kind[s] = k;
      }
    }
    plan.tiles[s] = tiles[s][plan.kind[s]];
  }
  return plan;
}

bool all_small(const int64_t* shapes, int count) {
  for (int i = 0; i < count; ++i) {
    const Parts p = parts_of(shapes + 2 * i);
    if (p.mp > 0 && p.np > 0 && (p.mp > SMALL_M || p.np > SMALL_N)) return false;
  }
  return true;
}

template <class C, int STAGE, class T, bool MUON>
int launch(const Table& t, const Numbers& num, int k, int64_t tiles, hipStream_t stream) {
  const auto kernel = k_orth_product<C, STAGE, T, MUON>;
  if (C::LDS > 65536) LAUNCH_TRY(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS));
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(C::THREADS), C::LDS, stream, t, num, k);
  return 0;
}
template <int STAGE, class T, bool MUON>
int product_launch(int kind, const Table& t, const Numbers& num, int k, int64_t tiles, hipStream_t stream) {
  switch (kind) {
    case 0: return launch<Orth32K, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 1: return launch<Orth32, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 2: return launch<Orth32S, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 3: return launch<Orth64K, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 4: return launch<Orth64, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 5: return launch<Orth96K, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 6: return launch<Orth128K, STAGE, T, MUON>(t, num, k, tiles, stream);
    case 7: return launch<Orth128, STAGE, T, MUON>(t, num, k, tiles, stream);
    default: return launch<Orth256, STAGE, T, MUON>(t, num, k, tiles, stream);
  }
}

template <bool MUON>
Mat describe(const Call& c, int i) {
  Mat a = {};
  const int64_t r = c.shapes[2 * i], q = c.shapes[2 * i + 1];
  const int flip = r > q;   // more rows than columns: the transposed matrix
  a.g = c.src[i];
  a.out = c.dst[i];
  a.buf = MUON ? c.buf[i] : nullptr;
  for (int k = 0; k < 2; ++k) {
    const int64_t dense = k == 0 ? q : 1;
    a.gs[k ^ flip] = c.strides ? c.strides[6 * i + k] : dense;
    a.os[k ^ flip] = c.strides ? c.strides[6 * i + 2 + k] : dense;
    a.bs[k ^ flip] = c.strides ? c.strides[6 * i + 4 + k] : dense;
  }
  a.m = (int)(flip ? q : r);
  a.n = (int)(flip ? r : q);
  a.rate = c.rate ? c.rate[i] : 0.f;
  return a;
}

// Whether a dense matrix that is written (parameter, momentum) lies over another one.
bool dense_overlap(const Call& c) {
  struct Span { const char *at, *end; bool written; };
  std::vector<Span> spans;
  for (int i = 0; i < c.count; ++i) {
    const int64_t bytes = c.shapes[2 * i] * c.shapes[2 * i + 1] * 4;
    if (bytes == 0) continue;
    const void* const all[3] = {c.src[i], c.dst[i], c.buf[i]};
    for (int k = 0; k < 3; ++k) spans.push_back({(const char*)all[k], (const char*)all[k] + bytes, k > 0});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.at < y.at; });
  const char *written = nullptr, *read = nullptr;   // where those so far end
  for (const Span& s : spans) {
    if (s.at < written || (s.written && s.at < read)) return true;
    (s.written ? written : read) = std::max(s.written ? written : read, s.end);
  }
  return false;
}

template <class T, bool MUON>
int run(const char* who, const Call& c, char* ws, size_t ws_bytes, hipStream_t stream) {
  const int64_t need = workspace_bytes(c.shapes, c.count);
  if (need > (int64_t)ws_bytes || (!ws && c.count > 0)) return set_error(GRLHIP_ERR_WORKSPACE, std::string(who) + ": workspace too small: need " + std::to_string(need));
  if ((size_t)ws & 255) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": the workspace must be aligned to 256 bytes");
  if (MUON && !c.strides && dense_overlap(c)) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": parameters, gradients and momentum buffers must not share memory");
  // the matrices with the longest sums first, so that a launch does not end with them
  std::vector<int> order;
  for (int i = 0; i < c.count; ++i)
    if (c.shapes[2 * i] > 0 && c.shapes[2 * i + 1] > 0) order.push_back(i);
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) {
    const Parts p = parts_of(c.shapes + 2 * x), q = parts_of(c.shapes + 2 * y);
    return p.np != q.np ? p.np > q.np : p.mp > q.mp;
  });
  const int present = (int)order.size();
  if (present == 0) return 0;
  const Numbers num{c.ca, c.cb, c.cc, c.eps, (float)c.momentum, (float)(1.0 - c.momentum), c.keep, c.nesterov};
  if (all_small(c.shapes, c.count)) {
    const auto kernel = k_orth_small<T, MUON>;
    LAUNCH_TRY(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SMALL_LDS));
    for (int done = 0; done < present;) {
      Group g = {};
      for (; done < present && g.count < GROUP; ++done) g.mat[g.count++] = describe<MUON>(c, order[done]);
      g.num = num;
      hipLaunchKernelGGL(kernel, dim3((unsigned)g.count), dim3(SMALL_THREADS), SMALL_LDS, stream, g, c.steps);
    }
    LAUNCH_TRY(hipGetLastError());
    return 0;
  }
  const Plan plan = plan_of(c.shapes, c.count);
  if (plan.blocks > 1 << 30 || plan.tiles[0] > 1 << 22 || plan.tiles[1] > 1 << 22 || plan.tiles[2] > 1 << 22)
    return set_error(GRLHIP_ERR_UNSUPPORTED, std::string(who) + ": too many matrices for one call");
  // workspace: descriptions, firsts, partial sums, then the matrices
  char* at = ws;
  auto take = [&](int64_t bytes) { char* p = at; at += up256(bytes); return p; };
  Mat* table = (Mat*)take((int64_t)c.count * sizeof(Mat));
  int* first = (int*)take((int64_t)c.count * 16);
  double* part = (double*)take(plan.blocks * 8);
  Mat lone = {};
  int64_t seen[4] = {0, 0, 0, 0};
  for (int done = 0; done < present;) {
    Group g = {};
    g.from = done;
    g.blocks0 = (int)seen[0];
    for (; done < present && g.count < GROUP; ++done) {
      const int i = order[done];
      const Parts p = parts_of(c.shapes + 2 * i);
      Mat& a = g.mat[g.count++];
      a = describe<MUON>(c, i);
      a.ws = at;
      at += p.bytes();
      a.first[0] = (int)seen[0];
      seen[0] += p.blocks();
      for (int s = 0; s < 3; ++s) {
        a.first[s + 1] = (int)seen[s + 1];
        seen[s + 1] += tiles_of(p, s, SIDE[plan.kind[s]]);
      }
    }
    g.first = first;
    g.table = table;
    g.all = present;
    g.part = part;
    g.num = num;
    lone = g.mat[0];   // used where there is one only
    hipLaunchKernelGGL((k_orth_norm<T, MUON>), dim3((unsigned)(seen[0] - g.blocks0)), dim3(256), 0, stream, g);
  }
  const Table t{first, table, present, part, lone};
  hipLaunchKernelGGL((k_orth_split<T, MUON>), dim3((unsigned)plan.blocks), dim3(256), 0, stream, t, num);
  if (c.steps == 0) hipLaunchKernelGGL((k_orth_join<T, MUON>), dim3((unsigned)plan.blocks), dim3(256), 0, stream, t, num);
  for (int s = 0; s < c.steps; ++s) {   // the stages before the last know nothing of the matrices' type
    if (const int rc = product_launch<GRAM, float, false>(plan.kind[GRAM], t, num, s & 1, plan.tiles[GRAM], stream)) return rc;
    if (const int rc = product_launch<POLY, float, false>(plan.kind[POLY], t, num, s & 1, plan.tiles[POLY], stream)) return rc;
    const int rc = s + 1 < c.steps ? product_launch<UPDATE, float, false>(plan.kind[UPDATE], t, num, s & 1, plan.tiles[UPDATE], stream)
                                   : product_launch<LAST, T, MUON>(plan.kind[UPDATE], t, num, s & 1, plan.tiles[UPDATE], stream);
    if (rc) return rc;
  }
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

int check_pointers(const char* who, const Call& c, bool muon) {
  for (int i = 0; i < c.count; ++i) {
    if (c.shapes[2 * i] == 0 || c.shapes[2 * i + 1] == 0) continue;
    if (!c.src || !c.dst || !c.src[i] || !c.dst[i] || (muon && (!c.buf || !c.buf[i])))
      return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": null pointer for matrix " + std::to_string(i));
  }
  return 0;
}

}  // namespace
}  // namespace grlhip

using namespace grlhip;

extern "C" {

size_t grlhip_orthogonalize_workspace_bytes(const int64_t* shapes, int32_t count) {
  return guarded_size([&]() -> size_t { return check_shapes("orthogonalize", shapes, count) ? 0 : (size_t)workspace_bytes(shapes, count); });
}

int grlhip_orthogonalize_tiles(const int64_t* shapes, int32_t count, int32_t* kinds) {
  return guarded([&]() -> int {
    if (const int rc = check_shapes("orthogonalize", shapes, count)) return rc;
    if (!kinds) return set_error(GRLHIP_ERR_INVALID, "orthogonalize_tiles: null kinds");
    const bool small = all_small(shapes, count);
    const Plan plan = plan_of(shapes, count);
    for (int s = 0; s < 3; ++s) kinds[s] = small ? -1 : plan.kind[s];
    return 0;
  });
}

int grlhip_orthogonalize(const void* const* src, void* const* dst, const int64_t* shapes, const int64_t* strides, int32_t count, int elem,
                         int32_t steps, float a, float b, float c, float eps, void* workspace, size_t workspace_bytes_, void* stream) {
  return guarded([&]() -> int {
    const char* who = "orthogonalize";
    int rc = check_shapes(who, shapes, count);
    if (rc || (rc = check_coefficients(who, a, b, c, steps))) return rc;
    if (!(eps > 0.f)) return set_error(GRLHIP_ERR_INVALID, "orthogonalize: eps must be positive");
    Call call{src, dst, nullptr, shapes, strides, count, steps, a, b, c, eps, nullptr, 0.0, 1.f, 0};
    if ((rc = check_pointers(who, call, false))) return rc;
    if (elem == GRLHIP_ELEM_F32) return run<float, false>(who, call, (char*)workspace, workspace_bytes_, (hipStream_t)stream);
    if (elem == GRLHIP_ELEM_BF16) return run<__bf16, false>(who, call, (char*)workspace, workspace_bytes_, (hipStream_t)stream);
    if (elem == GRLHIP_ELEM_F16) return run<_Float16, false>(who, call, (char*)workspace, workspace_bytes_, (hipStream_t)stream);
    return set_error(GRLHIP_ERR_INVALID, "orthogonalize: unknown element type");
  });
}

int grlhip_muon_step(float* const* params, const float* const* grads, float* const* momentum_buffers, const int64_t* shapes,
                     const int64_t* strides, const float* rates, int32_t count, double momentum, int nesterov, float keep, int32_t steps,
                     float a, float b, float c, float eps, void* workspace, size_t workspace_bytes_, void* stream) {
  return guarded([&]() -> int {
    const char* who = "muon_step";
    int rc = check_shapes(who, shapes, count);
    if (rc || (rc = check_coefficients(who, a, b, c, steps))) return rc;
    if (!(eps > 0.f) || !(momentum >= 0.0 && momentum < 1.0)) return set_error(GRLHIP_ERR_INVALID, "muon_step: eps must be positive, momentum in [0, 1)");
    if (count > 0 && !rates) return set_error(GRLHIP_ERR_INVALID, "muon_step: null rates");
    Call call{(const void* const*)grads, (void* const*)params, momentum_buffers, shapes, strides, count, steps, a, b, c, eps, rates, momentum, keep, nesterov != 0};
    if ((rc = check_pointers(who, call, true))) return rc;
    return run<float, true>(who, call, (char*)workspace, workspace_bytes_, (hipStream_t)stream);
  });
}

}  // extern "C"
