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
// One launch per product for the whole group (a network's matrices), so a step of the optimiser is 3 steps + 2 launches.
#include <cmath>
#include <cstdio>
#include <string>

#include "../../include/grlhip.h"
#include "errors.hpp"
#include "gemm_core.hip.inc"

namespace grlhip {
int device_cus();
namespace {
using namespace mx;

constexpr float S = 16384.f;        // scale of X, A, B
constexpr int GROUP = 24;           // matrices of one launch: their descriptions are kernel arguments (graphs keep them)
constexpr int64_t MAX_SIDE = 1 << 16;

// One matrix, oriented to m <= n.  Strides in elements: [0] along m, [1] along n.
struct Mat {
  const void* g;      // matrix / gradient
  void* out;          // result / parameter
  float* buf;         // momentum (muon) or null
  char* ws;           // its part of the workspace, see Parts
  int64_t gs[2], os[2], bs[2];
  int m, n;
  int blk0;           // first 64 x 64 block of the norm and split launches
  int tsym, tupd;     // first tile of the symmetric / update launches
  float rate;         // muon: learning rate of this matrix
};
struct Group {
  Mat mat[GROUP];
  int count, blocks, nsym, nupd;
  double* part;       // blocks partial sums of squares
  float ca, cb, cc, eps;
  float momentum, fresh, keep;   // muon: momentum; 1 - momentum, from 64 bits; 1 - lr * weight decay
  int nesterov;
};
static_assert(sizeof(Group) <= 4000, "kernel arguments");

__host__ __device__ inline int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }
// Pieces of a matrix in the workspace: two X, two X^T (a step reads one and writes the other), A, B.
struct Parts {
  int64_t mp, np, x, a;   // padded sides; bytes of an X, of an A
  __host__ __device__ Parts(int m, int n) : mp(up64(m)), np(up64(n)) { x = mp * np * 4; a = mp * mp * 4; }
  __host__ __device__ int64_t bytes() const { return 4 * x + 2 * a; }
  __device__ _Float16* X(char* ws, int k) const { return (_Float16*)(ws + k * x); }
  __device__ _Float16* XT(char* ws, int k) const { return (_Float16*)(ws + (2 + k) * x); }
  __device__ _Float16* A(char* ws) const { return (_Float16*)(ws + 4 * x); }
  __device__ _Float16* B(char* ws) const { return (_Float16*)(ws + 4 * x + a); }
};
// entry (row, col) of a piece array with `cols` columns: the high piece, the low one 32 further
__device__ __forceinline__ int64_t at(int64_t row, int col, int64_t cols) { return row * 2 * cols + (col >> 5) * 64 + (col & 31); }

template <int FIELD>   // the matrix that block / tile `id` belongs to: the last one that starts at or before it
__device__ __forceinline__ int find(const Group& g, int id) {
  int lo = 0, hi = g.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const int first = FIELD == 0 ? g.mat[mid].blk0 : FIELD == 1 ? g.mat[mid].tsym : g.mat[mid].tupd;
    if (first <= id) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <class T> __device__ __forceinline__ float load(const T* p) { return (float)*p; }

// Thread t's elements of a 64 x 64 block: i0 + k di, j; along the axis that is contiguous in memory, for whole lines.
struct Walk { int i, j, di, dj; };
__device__ __forceinline__ Walk walk(bool along_n) {
  const int t = threadIdx.x;
  return along_n ? Walk{t >> 6, t & 63, 4, 0} : Walk{t & 63, t >> 6, 0, 4};
}

// buf = momentum buf + (1 - momentum) g and the direction u; or u = g.  WRITE: store buf.
template <class T, bool MUON, bool WRITE>
__device__ __forceinline__ float direction(const Group& g, const Mat& a, int64_t i, int64_t j) {
  const float x = load((const T*)a.g + i * a.gs[0] + j * a.gs[1]);
  if (!MUON) return x;
  float* b = a.buf + i * a.bs[0] + j * a.bs[1];
  float v = *b;
  if (WRITE) { v = g.momentum * v + g.fresh * x; *b = v; }
  return g.nesterov ? g.fresh * x + g.momentum * v : v;
}

// Pass 1: momentum, and the sum of squares of each 64 x 64 block in 64 bits (a sum that every later product depends on).
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_norm(Group g) {
  const int e = find<0>(g, blockIdx.x);
  const Mat& a = g.mat[e];
  const int nb = (int)(up64(a.n) / 64), b = blockIdx.x - a.blk0;
  const int i0 = b / nb * 64, j0 = b % nb * 64;
  const Walk w = walk(a.gs[1] <= a.gs[0]);
  double s = 0.0;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int i = i0 + w.i + k * w.di, j = j0 + w.j + k * w.dj;
    if (i < a.m && j < a.n) {
      const double u = direction<T, MUON, true>(g, a, i, j);
      s += u * u;
    }
  }
  __shared__ double sh[256];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) g.part[blockIdx.x] = sh[0];
}

// Pass 2: X = S u / max(|u|, eps) as pieces, and X^T.  Every block adds its matrix' partial sums, in the same order.
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_split(Group g) {
  const int e = find<0>(g, blockIdx.x);
  const Mat& a = g.mat[e];
  const Parts p(a.m, a.n);
  const int nb = (int)(p.np / 64), b = blockIdx.x - a.blk0, all = (int)(p.mp / 64) * nb;
  __shared__ double sh[256];
  __shared__ float tile[64][65];
  double s = 0.0;
  for (int k = threadIdx.x; k < all; k += 256) s += g.part[a.blk0 + k];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    __syncthreads();
  }
  const double norm = sqrt(sh[0]);
  // in 64 bits: the quotient can pass fp32's range where the elements are tiny
  const double inv = (double)S / (norm > g.eps || norm != norm ? norm : (double)g.eps);
  const int i0 = b / nb * 64, j0 = b % nb * 64;
  const Walk w = walk(a.gs[1] <= a.gs[0]);
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int i = w.i + k * w.di, j = w.j + k * w.dj;
    tile[i][j] = i0 + i < a.m && j0 + j < a.n ? (float)(direction<T, MUON, false>(g, a, i0 + i, j0 + j) * inv) : 0.f;
  }
  __syncthreads();
  // a thread writes 16 consecutive entries of one row of X, then of X^T
  const int row = threadIdx.x >> 2, col = (threadIdx.x & 3) * 16;
  _Float16* X = p.X(a.ws, 0) + at(i0 + row, j0 + col, p.np);
  _Float16* XT = p.XT(a.ws, 0) + at(j0 + row, i0 + col, p.mp);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    f16x8 h, l, ht, lt;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      _Float16 x, y;
      split2(tile[row][col + c * 8 + k], x, y);
      h[k] = x;
      l[k] = y;
      split2(tile[col + c * 8 + k][row], x, y);
      ht[k] = x;
      lt[k] = y;
    }
    *(f16x8*)(X + c * 8) = h;
    *(f16x8*)(X + 32 + c * 8) = l;
    *(f16x8*)(XT + c * 8) = ht;
    *(f16x8*)(XT + 32 + c * 8) = lt;
  }
}

enum Stage { GRAM, POLY, UPDATE, LAST };

// One product of every matrix of the group.  k: which X is read.
template <class C, int STAGE, class T, bool MUON>
__global__ __launch_bounds__(C::THREADS, 2) void k_orth_product(Group g, int k) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  constexpr bool SYM = STAGE == GRAM || STAGE == POLY;
  const int id = xcd_order(blockIdx.x, SYM ? g.nsym : g.nupd);
  const Mat& a = g.mat[find<SYM ? 1 : 2>(g, id)];
  const Parts p(a.m, a.n);
  const int tm = (int)((p.mp + C::BM - 1) / C::BM);
  int im, in;
  if (SYM) {   // tile t of the lower triangle, row by row
    const int t = id - a.tsym;
    im = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (im * (im + 1) / 2 > t) --im;
    while ((im + 1) * (im + 2) / 2 <= t) ++im;
    in = t - im * (im + 1) / 2;
  } else {
    tile_at(id - a.tupd, tm, (int)((p.np + C::BN - 1) / C::BN), im, in);
  }
  const int64_t m0 = (int64_t)im * C::BM, n0 = (int64_t)in * C::BN;
  f32x16 acc[C::TM][C::TN];
  const int64_t xp = p.np * 4, ap = p.mp * 4;   // row pitches in bytes
  if (STAGE == GRAM) {
    const char* x = (const char*)p.X(a.ws, k);
    product<_Float16, 2, C>(x + m0 * xp, xp, p.mp - m0, x + n0 * xp, xp, p.mp - n0, (int)(p.np / 32), lds, acc);
  } else if (STAGE == POLY) {
    const char* x = (const char*)p.A(a.ws);
    product<_Float16, 2, C>(x + m0 * ap, ap, p.mp - m0, x + n0 * ap, ap, p.mp - n0, (int)(p.mp / 32), lds, acc);
  } else {
    product<_Float16, 2, C>((const char*)p.B(a.ws) + m0 * ap, ap, p.mp - m0, (const char*)p.XT(a.ws, k) + n0 * ap, ap, p.np - n0,
                            (int)(p.mp / 32), lds, acc);
  }
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  unsigned* patch = (unsigned*)(lds + L.wave * PATCH);
#pragma unroll
  for (int y = 0; y < C::TM; ++y) {
#pragma unroll
    for (int x = 0; x < C::TN; ++x) {
      const int64_t mb = m0 + (wm * C::TM + y) * 32, nb = n0 + (wn * C::TN + x) * 32;
      if (mb >= p.mp || nb >= (SYM ? p.mp : p.np)) continue;   // sides are padded to 64: whole blocks only
      const int64_t n = nb + L.j;
      float v[16];
      if (STAGE == GRAM) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = acc[y][x][r] * (1.f / S);
      } else {   // add the operand itself: A of the polynomial, X (read transposed: 4 consecutive entries) of the update
        const _Float16* own = STAGE == POLY ? p.A(a.ws) + at(n, (int)mb, p.mp) : p.XT(a.ws, k) + at(n, (int)mb, p.mp);
        const float f = STAGE == POLY ? g.cb : g.ca, q = (STAGE == POLY ? g.cc : 1.f) * (1.f / S);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f16x4 hi = *(const f16x4*)(own + 8 * c + 4 * L.h), lo = *(const f16x4*)(own + 32 + 8 * c + 4 * L.h);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * c + i] = f * ((float)hi[i] + (float)lo[i]) + q * acc[y][x][4 * c + i];
        }
      }
      if (SYM) {
        _Float16* D = STAGE == GRAM ? p.A(a.ws) : p.B(a.ws);
        store_t_f16x2(D + at(n, (int)mb, p.mp), L.h, v);
        if (im != in) store_n_f16x2(D + at(mb, (int)nb, p.mp), 2 * p.mp, patch, L, 32, v);
      } else if (STAGE == UPDATE) {
        store_t_f16x2(p.XT(a.ws, k ^ 1) + at(n, (int)mb, p.mp), L.h, v);
        store_n_f16x2(p.X(a.ws, k ^ 1) + at(mb, (int)nb, p.np), 2 * p.np, patch, L, 32, v);
      } else if (n < a.n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t m = mb + 8 * (r >> 2) + 4 * L.h + (r & 3);
          if (m >= a.m) continue;
          T* o = (T*)a.out + m * a.os[0] + n * a.os[1];
          const float d = v[r] * (1.f / S);
          *o = MUON ? (T)(g.keep * (float)*o - a.rate * d) : (T)d;   // the one rounding to the matrix' type
        }
      }
    }
  }
}

// steps == 0: the normalised matrix itself
template <class T, bool MUON>
__global__ __launch_bounds__(256) void k_orth_join(Group g) {
  const Mat& a = g.mat[find<0>(g, blockIdx.x)];
  const Parts p(a.m, a.n);
  const int nb = (int)(p.np / 64), b = blockIdx.x - a.blk0;
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

// Workspace of the matrices [from, to): their pieces, and the partial sums.
int64_t span_bytes(const int64_t* shapes, int from, int to) {
  int64_t bytes = 0, blocks = 0;
  for (int i = from; i < to; ++i) {
    const int64_t r = shapes[2 * i], c = shapes[2 * i + 1];
    if (r <= 0 || c <= 0) continue;
    const Parts p((int)(r < c ? r : c), (int)(r < c ? c : r));
    bytes += p.bytes();
    blocks += p.mp / 64 * (p.np / 64);
  }
  return bytes + blocks * 8 + 256;
}
int64_t workspace_bytes(const int64_t* shapes, int count) {
  int64_t most = 256;
  for (int i = 0; i < count; i += GROUP) {
    const int64_t b = span_bytes(shapes, i, i + GROUP < count ? i + GROUP : count);
    if (b > most) most = b;
  }
  return most;
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

template <class C>
void set_tiles(Group& g) {
  int sym = 0, upd = 0;
  for (int i = 0; i < g.count; ++i) {
    Mat& a = g.mat[i];
    const Parts p(a.m, a.n);
    const int tm = (int)((p.mp + C::BM - 1) / C::BM), tn = (int)((p.np + C::BN - 1) / C::BN);
    a.tsym = sym;
    a.tupd = upd;
    sym += tm * (tm + 1) / 2;
    upd += tm * tn;
  }
  g.nsym = sym;
  g.nupd = upd;
}

template <class C, class T, bool MUON>
int iterate(Group& g, int steps, hipStream_t stream) {
  set_tiles<C>(g);
  // the stages before the last know nothing of the matrices' type
  const auto gram = k_orth_product<C, GRAM, float, false>, poly = k_orth_product<C, POLY, float, false>, update = k_orth_product<C, UPDATE, float, false>,
             last = k_orth_product<C, LAST, T, MUON>;
  if (C::LDS > 65536)
    for (const auto f : {gram, poly, update, last})
      LAUNCH_TRY(hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS));
  for (int s = 0; s < steps; ++s) {
    hipLaunchKernelGGL(gram, dim3(g.nsym), dim3(C::THREADS), C::LDS, stream, g, s & 1);
    hipLaunchKernelGGL(poly, dim3(g.nsym), dim3(C::THREADS), C::LDS, stream, g, s & 1);
    hipLaunchKernelGGL(s + 1 < steps ? update : last, dim3(g.nupd), dim3(C::THREADS), C::LDS, stream, g, s & 1);
  }
  return 0;
}

template <class T, bool MUON>
int run_group(Group& g, int steps, hipStream_t stream) {
  hipLaunchKernelGGL((k_orth_norm<T, MUON>), dim3(g.blocks), dim3(256), 0, stream, g);
  hipLaunchKernelGGL((k_orth_split<T, MUON>), dim3(g.blocks), dim3(256), 0, stream, g);
  if (steps == 0) {
    hipLaunchKernelGGL((k_orth_join<T, MUON>), dim3(g.blocks), dim3(256), 0, stream, g);
    LAUNCH_TRY(hipGetLastError());
    return 0;
  }
  const int rc = iterate<Tile64, T, MUON>(g, steps, stream);
  if (rc) return rc;
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

template <class T, bool MUON>
int run(const char* who, const Call& c, char* ws, size_t ws_bytes, hipStream_t stream) {
  if (workspace_bytes(c.shapes, c.count) > (int64_t)ws_bytes || (!ws && c.count > 0))
    return set_error(GRLHIP_ERR_WORKSPACE, std::string(who) + ": workspace too small: need " + std::to_string(workspace_bytes(c.shapes, c.count)));
  if ((size_t)ws & 255) return set_error(GRLHIP_ERR_INVALID, std::string(who) + ": the workspace must be aligned to 256 bytes");
  for (int from = 0; from < c.count; from += GROUP) {
    Group g = {};
    char* at = ws;
    for (int i = from; i < c.count && i < from + GROUP; ++i) {
      const int64_t r = c.shapes[2 * i], q = c.shapes[2 * i + 1];
      if (r == 0 || q == 0) continue;
      Mat& a = g.mat[g.count++];
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
      const Parts p(a.m, a.n);
      a.ws = at;
      at += p.bytes();
      a.blk0 = g.blocks;
      g.blocks += (int)(p.mp / 64 * (p.np / 64));
    }
    if (g.count == 0) continue;
    g.part = (double*)at;
    g.ca = c.ca;
    g.cb = c.cb;
    g.cc = c.cc;
    g.eps = c.eps;
    g.momentum = (float)c.momentum;
    g.fresh = (float)(1.0 - c.momentum);
    g.keep = c.keep;
    g.nesterov = c.nesterov;
    const int rc = run_group<T, MUON>(g, c.steps, stream);
    if (rc) return rc;
  }
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
