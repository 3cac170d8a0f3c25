// Softmax cross entropy of z = hidden W^T + bias over a large vocabulary, and its gradients, without the logits (contract:
// include/grlhip.h, grlhip_linear_ce_forward / grlhip_linear_ce_backward).
//
// Forward: a tile of z lives in accumulators only; its epilogue leaves each row's maximum and sum of exponentials, and the
// target's logit; one pass over these partials gives logsumexp and the loss.  2 N V H flops.
// Backward, one piece of the vocabulary at a time: z again (the same products in the same order), D = softmax - onehot written
// in 16 bits both ways round, D as [row][v] for dH += D W and D scaled by the row's gradient as [v][row] for dW = D^T H.  6 N V H
// flops; the workspace holds D of one piece.  Recomputing z costs a third more products than keeping it would, and N V
// floats less memory.
//
// fp32 operands are two fp16 pieces a value (gemm_core.hip.inc), scaled by a power of two per tensor that brings its largest
// entry to 2^13..2^14: what is lost of a value is at most 2^-23 of it or 2^-39 of the largest.  16-bit operands are used as they
// are.  D is rounded once, to the operands' type (bf16 2^-8, fp16 2^-11 relative; the sums over it stay in fp32): the gradients are
// rounded to that type anyway.  All sums are taken in a fixed order: results repeat bit for bit.
#include <cmath>
#include <string>

#include "../../include/grlhip.h"
#include "errors.hpp"
#include "gemm_core.hip.inc"

namespace grlhip {
int device_cus();
namespace {
using namespace mx;

constexpr int64_t MAX_ROWS = 1 << 20, MAX_VOCAB = 1 << 21, MAX_HIDDEN = 1 << 16;
constexpr int64_t PIECE = 1ll << 27;      // entries of D in one piece of the vocabulary
__host__ __device__ inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// What the kernels share through the workspace.
struct Scalars { unsigned hmax, wmax, gmax; unsigned pad; };   // largest finite magnitudes, as bits (their order is the floats')

// the power of two that brings the largest magnitude to 2^13..2^14; 1 for nothing but zeros
__device__ __forceinline__ float scale_of(unsigned bits) {
  if (bits == 0) return 1.f;
  int e = (int)(bits >> 23) - 127;
  e = e < -100 ? -100 : e;
  return __builtin_ldexpf(1.f, 13 - e);
}
// the smallest power of two that no gradient factor passes
__device__ __forceinline__ float ceil_of(unsigned bits) {
  if (bits == 0) return 1.f;
  const int e = (int)(bits >> 23) - 126;
  return __builtin_ldexpf(1.f, e > 127 ? 127 : e);
}

__global__ void k_ce_clear(Scalars* s) {
  if (threadIdx.x < 4) ((unsigned*)s)[threadIdx.x] = 0u;
}

struct View { const void* p; int64_t s0, s1; int rows, cols; };   // element strides

__device__ __forceinline__ void keep_max(unsigned* to, float v) {
  unsigned m = __builtin_isfinite(v) ? __builtin_bit_cast(unsigned, v) & 0x7fffffffu : 0u;
  for (int d = 32; d > 0; d >>= 1) {
    const unsigned o = __shfl_xor(m, d);
    m = o > m ? o : m;
  }
  if ((threadIdx.x & 63) == 0 && m) atomicMax(to, m);
}
// the largest finite magnitudes of hidden (blocks [0, hb)) and weight (the others): a maximum, whatever the order
__global__ __launch_bounds__(256) void k_ce_absmax(View h, View w, int hb, Scalars* s) {
  const bool is_h = (int)blockIdx.x < hb;
  const View& v = is_h ? h : w;
  const int64_t first = (is_h ? (int64_t)blockIdx.x : (int64_t)blockIdx.x - hb) * 256 + threadIdx.x;
  const int64_t step = (int64_t)(is_h ? hb : (int)gridDim.x - hb) * 256, all = (int64_t)v.rows * v.cols;
  float m = 0.f;
  for (int64_t k = first; k < all; k += step) {
    const int64_t r = k / v.cols, c = k - r * v.cols;
    const float x = fabsf(((const float*)v.p)[r * v.s0 + c * v.s1]);
    if (__builtin_isfinite(x) && x > m) m = x;
  }
  keep_max(is_h ? &s->hmax : &s->wmax, m);
}

// A 64 x 64 block of a view -> the operand layout, as it stands (n: rows of the view) and transposed (t: its columns), either
// may be null; columns beyond the view and up to the pitch become zeros.  P == 2: scaled fp16 pieces.  A row that does not
// count becomes zeros: whatever it holds must not reach a sum over rows.
template <class T> struct Piece { typedef T type; };
template <> struct Piece<float> { typedef _Float16 type; };
template <class T>
__global__ __launch_bounds__(256) void k_ce_pack(View v, void* n, int64_t n_cols, void* t, int64_t t_cols, const unsigned* most,
                                                 const int64_t* target, int64_t ignore, const float* row_weight) {
  typedef typename Piece<T>::type E;
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  typedef E e8 __attribute__((ext_vector_type(8)));
  __shared__ float tile[64][65];
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, tid = threadIdx.x;
  const float s = P == 2 ? scale_of(*most) : 1.f;
  const bool along = v.s1 <= v.s0;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int i = along ? (tid >> 6) + 4 * k : tid & 63, j = along ? tid & 63 : (tid >> 6) + 4 * k;
    float x = 0.f;
    if (i0 + i < v.rows && j0 + j < v.cols) {
      const bool counts = !target || (target[i0 + i] != ignore && !(row_weight && row_weight[i0 + i] == 0.f));
      if (counts) x = (float)((const T*)v.p)[(int64_t)(i0 + i) * v.s0 + (int64_t)(j0 + j) * v.s1] * s;
    }
    tile[i][j] = x;
  }
  __syncthreads();
  const int row = tid >> 2, col = (tid & 3) * 16;
#pragma unroll
  for (int way = 0; way < 2; ++way) {
    E* out = (E*)(way ? t : n);
    if (!out) continue;
    const int r = (way ? j0 : i0) + row, c = (way ? i0 : j0) + col;
    const int64_t cols = way ? t_cols : n_cols;
    if (r >= (way ? v.cols : v.rows) || c >= cols) continue;
    E* dst = out + (int64_t)r * P * cols + (P == 2 ? (c >> 5) * 64 + (c & 31) : c);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      e8 hi, lo;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = way ? tile[col + q * 8 + k][row] : tile[row][col + q * 8 + k];
        if constexpr (P == 2) {
          _Float16 a, b;
          split2(x, a, b);
          hi[k] = a;
          lo[k] = b;
        } else {
          hi[k] = (E)x;
        }
      }
      *(e8*)(dst + q * 8) = hi;
      if (P == 2) *(e8*)(dst + 32 + q * 8) = lo;
    }
  }
}

struct Operand { const char* p; int64_t pitch; };   // K-contiguous rows; pitch in bytes

struct Logits {
  Operand w, h;             // rows of the weight piece, rows of hidden
  const float* bias;        // of the piece, or null
  const int64_t* target;
  const float* row_weight;
  const float* lse;         // backward
  const float* scale;       // backward: gradient of each row's loss (0: the row does not count)
  const Scalars* s;
  int64_t ignore;
  int rows, v0, cols;       // rows; first vocabulary entry and entries of the piece
  int nkb;                  // K blocks
  // forward
  float2* part;             // [vocabulary tiles][rows] maximum, sum
  float* picked;            // [rows] the target's logit
  // backward
  char* d; int64_t d_cols;  // [rows][d_cols] D
  char* dt; int64_t dt_cols;  // [cols][dt_cols] D times the row's gradient
  float* bpart;             // [row tiles][cols] partial sums of the bias' gradient, or null
};

// z of one 32 x 32 block
template <int P>
__device__ __forceinline__ void logits_of(const Logits& a, const f32x16& acc, int mb, int h, float fh, float fw, float (&z)[16]) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = mb + 8 * (r >> 2) + 4 * h + (r & 3);
    float v = acc[r];
    if (P == 2) v = v * fh * fw;
    if (a.bias && m < a.cols) v += a.bias[m];
    z[r] = v;
  }
}

template <class T, int P, class C>
__global__ __launch_bounds__(C::THREADS, 2) void k_ce_forward(Logits a, int tm, int tn) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  int im, in;
  tile_at(xcd_order(blockIdx.x, gridDim.x), tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  f32x16 acc[C::TM][C::TN];
  product<T, P, C>(a.w.p + m0 * a.w.pitch, a.w.pitch, a.cols - m0, a.h.p + n0 * a.h.pitch, a.h.pitch, a.rows - n0, a.nkb, lds, acc);   // KG == 1: every wave goes on
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  const float fh = P == 2 ? 1.f / scale_of(a.s->hmax) : 1.f, fw = P == 2 ? 1.f / scale_of(a.s->wmax) : 1.f;
  float* tops = (float*)lds;                  // [WM][BN] maxima, then sums
  float* sums = tops + C::WM * C::BN;
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int nl = (wn * C::TN + x) * 32 + L.j, n = n0 + nl;
    const int64_t t = n < a.rows ? a.target[n] - a.v0 : -1;
    float top = -INFINITY, z[C::TM][16];
#pragma unroll
    for (int y = 0; y < C::TM; ++y) {
      const int mb = m0 + (wm * C::TM + y) * 32;
      logits_of<P>(a, acc[y][x], mb, L.h, fh, fw, z[y]);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = mb + 8 * (r >> 2) + 4 * L.h + (r & 3);
        if (m == t && m < a.cols) a.picked[n] = z[y][r];
        if (m >= a.cols) z[y][r] = -INFINITY;
        top = fmaxf(top, z[y][r]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    float sum = 0.f;
    // nothing but -inf: no sum, whatever -inf - -inf is.  A NaN logit passes fmaxf, and is caught by the sum
#pragma unroll
    for (int y = 0; y < C::TM; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += z[y][r] == -INFINITY ? 0.f : __expf(z[y][r] - top);
    sum += __shfl_xor(sum, 32);
    if (L.h == 0) {
      tops[wm * C::BN + nl] = top;
      sums[wm * C::BN + nl] = sum;
    }
  }
  lds_barrier();
  for (int k = threadIdx.x; k < C::BN; k += C::THREADS) {
    float top = tops[k], sum = sums[k];
#pragma unroll
    for (int w = 1; w < C::WM; ++w) {
      const float t = tops[w * C::BN + k], u = sums[w * C::BN + k], most = fmaxf(top, t);
      sum = (top == -INFINITY ? sum : sum * __expf(top - most)) + (t == -INFINITY ? u : u * __expf(t - most));
      top = most;
    }
    if (n0 + k < a.rows) a.part[(int64_t)im * a.rows + n0 + k] = make_float2(top, sum);
  }
}

struct Finish {
  const float2* part;
  const float* picked;
  const int64_t* target;
  const float* row_weight;
  int64_t ignore;
  int rows, tiles, vocab, blocks;
  float* losses; float* lse;
  double* sums;       // [blocks][2]: weighted loss, rows that count
  float* total; float* count;   // the reduced loss; the number of rows that are not ignored, at least 1
  int reduction;
};

// 32 rows a block, 8 threads a row: the partials of a row, then its loss.
__global__ __launch_bounds__(256) void k_ce_finish(Finish a) {
  __shared__ float tops[8][32], sums[8][32];
  __shared__ double s[32], c[32];
  const int r = threadIdx.x & 31, q = threadIdx.x >> 5, n = blockIdx.x * 32 + r;
  float top = -INFINITY, sum = 0.f;
  if (n < a.rows)
    for (int t = q; t < a.tiles; t += 8) {
      const float2 p = a.part[(int64_t)t * a.rows + n];
      const float most = fmaxf(top, p.x);
      sum = (top == -INFINITY ? sum : sum * __expf(top - most)) + (p.x == -INFINITY ? p.y : p.y * __expf(p.x - most));
      top = most;
    }
  tops[q][r] = top;
  sums[q][r] = sum;
  __syncthreads();
  if (q == 0) {
    for (int k = 1; k < 8; ++k) {
      const float t = tops[k][r], u = sums[k][r], most = fmaxf(top, t);
      sum = (top == -INFINITY ? sum : sum * __expf(top - most)) + (t == -INFINITY ? u : u * __expf(t - most));
      top = most;
    }
    s[r] = c[r] = 0.0;
    if (n < a.rows) {
      const int64_t t = a.target[n];
      const bool kept = t != a.ignore;
      const float w = a.row_weight ? a.row_weight[n] : 1.f;
      const float lse = top + logf(sum);
      // a target outside the vocabulary has no loss: NaN, not a number that looks like one
      float loss = t >= 0 && t < a.vocab ? (lse - a.picked[n]) * w : NAN;
      if (!kept || w == 0.f) loss = 0.f;
      a.lse[n] = lse;
      a.losses[n] = loss;
      s[r] = loss;
      c[r] = kept ? 1.0 : 0.0;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double x = 0.0, y = 0.0;
    for (int k = 0; k < 32; ++k) { x += s[k]; y += c[k]; }
    a.sums[2 * blockIdx.x] = x;
    a.sums[2 * blockIdx.x + 1] = y;
  }
}
__global__ __launch_bounds__(256) void k_ce_total(Finish a) {
  __shared__ double s[256], c[256];
  double x = 0.0, y = 0.0;
  for (int k = threadIdx.x; k < a.blocks; k += 256) { x += a.sums[2 * k]; y += a.sums[2 * k + 1]; }
  s[threadIdx.x] = x;
  c[threadIdx.x] = y;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) { s[threadIdx.x] += s[threadIdx.x + d]; c[threadIdx.x] += c[threadIdx.x + d]; }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double count = c[0] < 1.0 ? 1.0 : c[0];
    *a.total = (float)(a.reduction == GRLHIP_REDUCE_MEAN ? s[0] / count : s[0]);
    *a.count = (float)count;
  }
}

// The gradient of each row's own loss, and the largest of them.
struct Scale {
  const float* grad; int64_t grad_stride;
  const float* row_weight; const float* count;
  const int64_t* target; int64_t ignore;
  int rows, vocab, reduction;
  float* scale; Scalars* s;
};
__global__ __launch_bounds__(256) void k_ce_scale(Scale a) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  float g = 0.f;
  if (n < a.rows) {
    const int64_t t = a.target[n];
    const float w = a.row_weight ? a.row_weight[n] : 1.f;
    if (t != a.ignore && w != 0.f) {
      g = a.grad[n * a.grad_stride] * w;
      if (a.reduction == GRLHIP_REDUCE_MEAN) g /= *a.count;
      if (t < 0 || t >= a.vocab) g = NAN;
    }
    a.scale[n] = g;
  }
  keep_max(&a.s->gmax, g);
}

constexpr float DSCALE = 16384.f;   // fp16 D lies in [-2^14, 2^14]
template <class T> __device__ __forceinline__ float d_scale() { return sizeof(T) == 2 && __is_same(T, __bf16) ? 1.f : DSCALE; }

template <class T, int P, class C>
__global__ __launch_bounds__(C::THREADS, 2) void k_ce_d(Logits a, int tm, int tn) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  int im, in;
  tile_at(xcd_order(blockIdx.x, gridDim.x), tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  f32x16 acc[C::TM][C::TN];
  product<T, P, C>(a.w.p + m0 * a.w.pitch, a.w.pitch, a.cols - m0, a.h.p + n0 * a.h.pitch, a.h.pitch, a.rows - n0, a.nkb, lds, acc);   // KG == 1: every wave goes on
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  const float fh = P == 2 ? 1.f / scale_of(a.s->hmax) : 1.f, fw = P == 2 ? 1.f / scale_of(a.s->wmax) : 1.f;
  const float per = 1.f / ceil_of(a.s->gmax), ds = d_scale<T>();
  unsigned* patch = (unsigned*)(lds + L.wave * PATCH);
  float* bsum = (float*)(lds + C::WAVES * PATCH);   // [WN][BM]
#pragma unroll
  for (int y = 0; y < C::TM; ++y) {
    const int mb = m0 + (wm * C::TM + y) * 32;
    float bs[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) bs[r] = 0.f;
#pragma unroll
    for (int x = 0; x < C::TN; ++x) {
      const int nb = n0 + (wn * C::TN + x) * 32, n = nb + L.j;
      const bool in_rows = n < a.rows;
      const float lse = in_rows ? a.lse[n] : 0.f, g = in_rows ? a.scale[n] : 0.f;
      const int64_t t = in_rows ? a.target[n] - a.v0 : -1;
      float z[16], v[16];
      logits_of<P>(a, acc[y][x], mb, L.h, fh, fw, z);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = mb + 8 * (r >> 2) + 4 * L.h + (r & 3);
        float p = __expf(z[r] - lse) - (m == t ? 1.f : 0.f);
        if (m >= a.cols || g == 0.f) p = 0.f;
        z[r] = p * ds;
        v[r] = p * (g * per) * ds;
        if (m >= a.cols || g == 0.f) v[r] = 0.f;
        bs[r] += m >= a.cols || g == 0.f ? 0.f : p * g;
      }
      if (nb < a.rows && mb < a.d_cols) {
        if constexpr (P == 2) store_t_f16x2((_Float16*)a.d + (int64_t)nb * 2 * a.d_cols + mb * 2, 2 * a.d_cols, patch, L, a.rows - nb, z);
        else store_t_16<T>((T*)a.d + (int64_t)nb * a.d_cols + mb, a.d_cols, patch, L, a.rows - nb, z);
      }
      if (nb < a.dt_cols && mb < a.cols) {
        if constexpr (P == 2) store_n_f16x2((_Float16*)a.dt + (int64_t)mb * 2 * a.dt_cols + nb * 2, 2 * a.dt_cols, patch, L, a.cols - mb, v);
        else store_n_16<T>((T*)a.dt + (int64_t)mb * a.dt_cols + nb, a.dt_cols, patch, L, a.cols - mb, v);
      }
    }
    if (a.bpart) {   // over the 32 columns of the lanes of a half, in one order
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float s = bs[r];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor(s, d);
        if (L.j == 0) bsum[wn * C::BM + (wm * C::TM + y) * 32 + 8 * (r >> 2) + 4 * L.h + (r & 3)] = s;
      }
    }
  }
  if (a.bpart) {
    lds_barrier();
    for (int k = threadIdx.x; k < C::BM; k += C::THREADS) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) s += bsum[w * C::BM + k];
      if (m0 + k < a.cols) a.bpart[(int64_t)in * a.cols + m0 + k] = s;
    }
  }
}

__global__ __launch_bounds__(256) void k_ce_bias(const float* part, int tiles, int cols, float* out) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= cols) return;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t) s += part[(int64_t)t * cols + v];
  out[v] = s;
}

// out[n][m] = f(n) sum_k A[m][k] B[n][k]: dH (A = W^T, B = D; f = the row's gradient) and dW (A = hidden^T, B = D^T).
struct Grad {
  Operand a, b;
  int m, n, nkb, split;     // split: parts of the K blocks
  float* slots;             // fp32 [split][n][m], or null: straight to `out`
  int add;                  // to what the slots hold
  void* out; int64_t o0, o1;   // element strides
  const float* scale;       // per row, or null
  const Scalars* s; int by_w;  // the operands' factors: W's (dH) or hidden's and the gradient's (dW)
};
template <class T>
__device__ __forceinline__ float grad_factor(const Grad& g) {
  float f = 1.f / d_scale<T>();
  if (sizeof(T) == 4) f *= 1.f / scale_of(g.by_w ? g.s->wmax : g.s->hmax);
  return f;
}
template <class T, int P, class C>
__global__ __launch_bounds__(C::THREADS, 2) void k_ce_grad(Grad g, int tm, int tn) {
  typedef typename Piece<T>::type E;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int id = xcd_order(blockIdx.x, gridDim.x), part = id / (tm * tn);
  int im, in;
  tile_at(id - part * tm * tn, tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  const int k0 = (int)((int64_t)g.nkb * part / g.split), k1 = (int)((int64_t)g.nkb * (part + 1) / g.split);
  f32x16 acc[C::TM][C::TN];
  product<E, P, C>(g.a.p + m0 * g.a.pitch + (int64_t)k0 * KBLOCK, g.a.pitch, g.m - m0, g.b.p + n0 * g.b.pitch + (int64_t)k0 * KBLOCK, g.b.pitch,
                   g.n - n0, k1 - k0, lds, acc);
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  const float f = grad_factor<T>(g), f2 = g.by_w ? 1.f : ceil_of(g.s->gmax);
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int n = n0 + (wn * C::TN + x) * 32 + L.j;
    if (n >= g.n) continue;
    const float row = g.scale && !g.slots ? g.scale[n] : 1.f;
    const bool none = g.scale && !g.slots && row == 0.f;
#pragma unroll
    for (int y = 0; y < C::TM; ++y) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = m0 + (wm * C::TM + y) * 32 + 8 * q + 4 * L.h;
        if (m >= g.m) continue;
        if (g.slots) {
          float* o = g.slots + ((int64_t)part * g.n + n) * g.m + m;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (m + i < g.m) o[i] = acc[y][x][4 * q + i] + (g.add ? o[i] : 0.f);
        } else {
          T* o = (T*)g.out + (int64_t)n * g.o0 + (int64_t)m * g.o1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (m + i < g.m) o[i * g.o1] = none ? (T)0.f : (T)(acc[y][x][4 * q + i] * f * f2 * row);
        }
      }
    }
  }
}
template <class T>
__global__ __launch_bounds__(256) void k_ce_join(Grad g) {
  const float f = grad_factor<T>(g), f2 = g.by_w ? 1.f : ceil_of(g.s->gmax);
  const int64_t all = (int64_t)g.n * g.m;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < all; k += (int64_t)gridDim.x * 256) {
    const int64_t n = k / g.m, m = k - n * g.m;
    float s = 0.f;
    for (int p = 0; p < g.split; ++p) s += g.slots[p * all + k];
    const float row = g.scale ? g.scale[n] : 1.f;
    ((T*)g.out)[n * g.o0 + m * g.o1] = g.scale && row == 0.f ? (T)0.f : (T)(s * f * f2 * row);
  }
}

// ------------------------------------------------------------------------------------------------------------- host
struct Shape { int64_t rows, hidden, vocab; int elem; };
int pieces(int elem) { return elem == GRLHIP_ELEM_F32 ? 2 : 1; }

typedef Tile<128, 128, 2, 2, 2> Main;

// How a call goes about it: the same for its workspace and its launches.
struct Layout {
  int64_t kp, np;                   // hidden and rows, padded to whole K blocks
  int64_t piece;                    // vocabulary entries of a piece
  bool pack_h, pack_w;
  int split_h, split_w;             // parts of the sums of dH and dW
  int64_t pieces_n;
  // offsets
  int64_t scalars, hp, wp, ht, wt, d, dt, part, picked, sums, scale, bpart, hslots, wslots, bytes;
};
int split_for(int64_t tiles, int64_t nkb) {   // enough workgroups for the chip, but no part under 8 K blocks
  int64_t s = tiles >= 256 ? 1 : (512 + tiles - 1) / tiles;
  if (s > nkb / 8) s = nkb / 8;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
Layout layout_of(const Shape& c, bool direct_h, bool direct_w, bool backward, bool bias) {
  Layout l = {};
  const int64_t per = pieces(c.elem) * 2;   // bytes of an operand entry
  l.kp = up(c.hidden, 64);
  l.np = up(c.rows, 64);
  l.pack_h = !direct_h;
  l.pack_w = !direct_w;
  int64_t limit = backward ? PIECE / l.np : l.pack_w ? PIECE / l.kp : c.vocab;
  limit = limit < 1024 ? 1024 : limit / 256 * 256;
  if (backward && limit > 1 << 19) limit = 1 << 19;                                       // row offsets inside a tile are 32 bits
  const int64_t most = (1 << 22) / (up(c.rows, Main::BN) / Main::BN) * Main::BM;          // and so is a launch
  if (limit > most) limit = most;
  l.pieces_n = (c.vocab + limit - 1) / limit;
  l.piece = up((c.vocab + l.pieces_n - 1) / l.pieces_n, 256);
  if (l.piece > c.vocab) l.piece = c.vocab;
  l.pieces_n = (c.vocab + l.piece - 1) / l.piece;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += up(bytes, 256); return o; };
  l.scalars = take(sizeof(Scalars));
  if (l.pack_h) l.hp = take(c.rows * l.kp * per);
  if (l.pack_w) l.wp = take(l.piece * l.kp * per);
  if (!backward) {
    l.part = take(up(c.vocab, Main::BM) / Main::BM * c.rows * 8 + l.pieces_n * c.rows * 8);
    l.picked = take(c.rows * 4);
    l.sums = take(up(c.rows, 32) / 32 * 16);
  } else {
    const int64_t vp = up(l.piece, 64);
    l.ht = take(c.hidden * l.np * per);
    l.wt = take(c.hidden * vp * per);
    l.d = take(c.rows * vp * per);
    l.dt = take(l.piece * l.np * per);
    l.scale = take(c.rows * 4);
    if (bias) l.bpart = take(up(c.rows, Main::BN) / Main::BN * l.piece * 4);
    auto tiles = [](int64_t m, int64_t n) { return up(m, Main::BM) / Main::BM * (up(n, Main::BN) / Main::BN); };
    const int64_t kb = pieces(c.elem) == 2 ? 32 : 64;
    l.split_h = split_for(tiles(c.hidden, c.rows), vp / kb);
    l.split_w = split_for(tiles(c.hidden, l.piece), l.np / kb);
    if (l.split_h > 1 || l.pieces_n > 1) l.hslots = take(l.split_h * c.rows * c.hidden * 4);
    if (l.split_w > 1) l.wslots = take(l.split_w * l.piece * c.hidden * 4);
  }
  l.bytes = at;
  return l;
}

struct Call {
  Shape c;
  const void* h; int64_t h0, h1;
  const void* w; int64_t w0, w1;
  const float* bias; const int64_t* target; const float* row_weight;
  int64_t ignore; int reduction;
  float* losses; float* lse; float* total; float* count;
  const float* grad; int64_t grad_stride;
  void* gh; void* gw; float* gb;
  char* ws; size_t ws_bytes; hipStream_t stream;
};
// 16-bit rows that are whole K blocks, 16-byte aligned, are read where they are
bool direct(const void* p, int64_t s0, int64_t s1, const Shape& c) {
  return pieces(c.elem) == 1 && c.hidden % 64 == 0 && s1 == 1 && s0 % 8 == 0 && s0 > 0 && s0 <= MAX_HIDDEN * 32 && ((size_t)p & 15) == 0;
}
int check(const char* who, const Call& a) {
  const Shape& c = a.c;
  const std::string w = std::string(who) + ": ";
  if (c.rows < 1 || c.hidden < 1 || c.vocab < 1) return set_error(GRLHIP_ERR_INVALID, w + "rows, hidden and vocabulary must be at least 1");
  if (c.rows > MAX_ROWS || c.vocab > MAX_VOCAB || c.hidden > MAX_HIDDEN)
    return set_error(GRLHIP_ERR_UNSUPPORTED, w + "over 2^20 rows, 2^21 vocabulary entries or 2^16 features");
  if (c.elem != GRLHIP_ELEM_F32 && c.elem != GRLHIP_ELEM_BF16 && c.elem != GRLHIP_ELEM_F16) return set_error(GRLHIP_ERR_INVALID, w + "unknown element type");
  if (a.reduction < 0 || a.reduction > 2) return set_error(GRLHIP_ERR_INVALID, w + "unknown reduction");
  if (!a.h || !a.w || !a.target || !a.lse || !a.count) return set_error(GRLHIP_ERR_INVALID, w + "null hidden, weight, target, lse or count");
  return 0;
}
template <class K>
int lds_for(K k, int bytes) {
  if (bytes > 65536) LAUNCH_TRY(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return 0;
}

// hidden / weight (a piece of it) as operands, packed where they have to be
template <class T>
int pack(const Call& a, const View& v, void* n, int64_t n_cols, void* t, int64_t t_cols, const unsigned* most, bool mask) {
  if (!n && !t) return 0;
  const dim3 grid((unsigned)(up(v.cols, 64) / 64), (unsigned)(up(v.rows, 64) / 64));
  hipLaunchKernelGGL(k_ce_pack<T>, grid, dim3(256), 0, a.stream, v, n, n_cols, t, t_cols, most, mask ? a.target : nullptr, a.ignore, mask ? a.row_weight : nullptr);
  return 0;
}
template <class T>
View weight_piece(const Call& a, int64_t v0, int64_t cols) {
  return {(const char*)a.w + v0 * a.w0 * (int64_t)sizeof(T), a.w0, a.w1, (int)cols, (int)a.c.hidden};
}
template <class T>
int begin(const Call& a, Scalars* s) {
  hipLaunchKernelGGL(k_ce_clear, dim3(1), dim3(64), 0, a.stream, s);
  if (sizeof(T) == 4) {
    const View h{a.h, a.h0, a.h1, (int)a.c.rows, (int)a.c.hidden}, w{a.w, a.w0, a.w1, (int)a.c.vocab, (int)a.c.hidden};
    auto blocks = [](int64_t n) { n = (n + 4095) / 4096; return (int)(n > 1024 ? 1024 : n); };
    const int hb = blocks((int64_t)h.rows * h.cols), wb = blocks((int64_t)w.rows * w.cols);
    hipLaunchKernelGGL(k_ce_absmax, dim3(hb + wb), dim3(256), 0, a.stream, h, w, hb, s);
  }
  return 0;
}

template <class T>
int forward(const Call& a) {
  typedef typename Piece<T>::type E;
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  typedef Main C;
  const Layout l = layout_of(a.c, direct(a.h, a.h0, a.h1, a.c), direct(a.w, a.w0, a.w1, a.c), false, false);
  if (!a.ws || (int64_t)a.ws_bytes < l.bytes) return set_error(GRLHIP_ERR_WORKSPACE, "linear_ce_forward: workspace too small: need " + std::to_string(l.bytes));
  Scalars* s = (Scalars*)(a.ws + l.scalars);
  begin<T>(a, s);
  const View h{a.h, a.h0, a.h1, (int)a.c.rows, (int)a.c.hidden};
  if (l.pack_h) pack<T>(a, h, a.ws + l.hp, l.kp, nullptr, 0, &s->hmax, false);
  const auto kernel = k_ce_forward<E, P, C>;
  if (const int rc = lds_for(kernel, C::LDS)) return rc;
  int tiles = 0;
  for (int64_t v0 = 0; v0 < a.c.vocab; v0 += l.piece) {
    const int64_t cols = a.c.vocab - v0 < l.piece ? a.c.vocab - v0 : l.piece;
    const View w = weight_piece<T>(a, v0, cols);
    if (l.pack_w) pack<T>(a, w, a.ws + l.wp, l.kp, nullptr, 0, &s->wmax, false);
    Logits g = {};
    g.h = l.pack_h ? Operand{a.ws + l.hp, l.kp * 2 * P} : Operand{(const char*)a.h, a.h0 * 2};
    g.w = l.pack_w ? Operand{a.ws + l.wp, l.kp * 2 * P} : Operand{(const char*)w.p, a.w0 * 2};
    g.bias = a.bias ? a.bias + v0 : nullptr;
    g.target = a.target;
    g.s = s;
    g.rows = (int)a.c.rows;
    g.v0 = (int)v0;
    g.cols = (int)cols;
    g.nkb = (int)(l.kp * 2 * P / KBLOCK);
    g.part = (float2*)(a.ws + l.part) + (int64_t)tiles * a.c.rows;
    g.picked = (float*)(a.ws + l.picked);
    const int tm = (int)(up(cols, C::BM) / C::BM), tn = (int)(up(a.c.rows, C::BN) / C::BN);
    hipLaunchKernelGGL(kernel, dim3(tm * tn), dim3(C::THREADS), C::LDS, a.stream, g, tm, tn);
    tiles += tm;
  }
  Finish f{(float2*)(a.ws + l.part), (float*)(a.ws + l.picked), a.target, a.row_weight, a.ignore, (int)a.c.rows, tiles, (int)a.c.vocab,
           (int)(up(a.c.rows, 32) / 32), a.losses, a.lse, (double*)(a.ws + l.sums), a.total, a.count, a.reduction};
  hipLaunchKernelGGL(k_ce_finish, dim3(f.blocks), dim3(256), 0, a.stream, f);
  hipLaunchKernelGGL(k_ce_total, dim3(1), dim3(256), 0, a.stream, f);
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

template <class T, class C>
int grad_launch(const Call& a, const Grad& g) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  const auto kernel = k_ce_grad<T, P, C>;
  if (const int rc = lds_for(kernel, C::LDS)) return rc;
  const int tm = (int)(up(g.m, C::BM) / C::BM), tn = (int)(up(g.n, C::BN) / C::BN);
  hipLaunchKernelGGL(kernel, dim3(tm * tn * g.split), dim3(C::THREADS), C::LDS, a.stream, g, tm, tn);
  return 0;
}
template <class T>
void join_launch(const Call& a, const Grad& g) {
  const int64_t blocks = ((int64_t)g.n * g.m + 1023) / 1024;
  hipLaunchKernelGGL(k_ce_join<T>, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, a.stream, g);
}

template <class T>
int backward(const Call& a) {
  typedef typename Piece<T>::type E;
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  typedef Main C;
  const Layout l = layout_of(a.c, direct(a.h, a.h0, a.h1, a.c), direct(a.w, a.w0, a.w1, a.c), true, a.gb != nullptr);
  if (!a.ws || (int64_t)a.ws_bytes < l.bytes) return set_error(GRLHIP_ERR_WORKSPACE, "linear_ce_backward: workspace too small: need " + std::to_string(l.bytes));
  Scalars* s = (Scalars*)(a.ws + l.scalars);
  begin<T>(a, s);
  float* scale = (float*)(a.ws + l.scale);
  const Scale sc{a.grad, a.grad_stride, a.row_weight, a.count, a.target, a.ignore, (int)a.c.rows, (int)a.c.vocab, a.reduction, scale, s};
  hipLaunchKernelGGL(k_ce_scale, dim3((unsigned)((a.c.rows + 255) / 256)), dim3(256), 0, a.stream, sc);
  const View h{a.h, a.h0, a.h1, (int)a.c.rows, (int)a.c.hidden};
  pack<T>(a, h, l.pack_h ? a.ws + l.hp : nullptr, l.kp, a.gw ? a.ws + l.ht : nullptr, l.np, &s->hmax, true);
  const auto kernel = k_ce_d<E, P, C>;
  if (const int rc = lds_for(kernel, C::LDS)) return rc;
  Grad gh = {};
  for (int64_t v0 = 0; v0 < a.c.vocab; v0 += l.piece) {
    const int64_t cols = a.c.vocab - v0 < l.piece ? a.c.vocab - v0 : l.piece, vp = up(cols, 64);
    const View w = weight_piece<T>(a, v0, cols);
    pack<T>(a, w, l.pack_w ? a.ws + l.wp : nullptr, l.kp, a.gh ? a.ws + l.wt : nullptr, vp, &s->wmax, false);
    Logits g = {};
    g.h = l.pack_h ? Operand{a.ws + l.hp, l.kp * 2 * P} : Operand{(const char*)a.h, a.h0 * 2};
    g.w = l.pack_w ? Operand{a.ws + l.wp, l.kp * 2 * P} : Operand{(const char*)w.p, a.w0 * 2};
    g.bias = a.bias ? a.bias + v0 : nullptr;
    g.target = a.target;
    g.lse = a.lse;
    g.scale = scale;
    g.s = s;
    g.rows = (int)a.c.rows;
    g.v0 = (int)v0;
    g.cols = (int)cols;
    g.nkb = (int)(l.kp * 2 * P / KBLOCK);
    g.d = a.ws + l.d;
    g.d_cols = vp;
    g.dt = a.ws + l.dt;
    g.dt_cols = l.np;
    g.bpart = a.gb ? (float*)(a.ws + l.bpart) : nullptr;
    const int tm = (int)(up(cols, C::BM) / C::BM), tn = (int)(up(a.c.rows, C::BN) / C::BN);
    hipLaunchKernelGGL(kernel, dim3(tm * tn), dim3(C::THREADS), C::LDS, a.stream, g, tm, tn);
    if (a.gb) hipLaunchKernelGGL(k_ce_bias, dim3((unsigned)((cols + 255) / 256)), dim3(256), 0, a.stream, g.bpart, tn, (int)cols, a.gb + v0);
    if (a.gh) {
      gh = Grad{};
      gh.a = {a.ws + l.wt, vp * 2 * P};
      gh.b = {a.ws + l.d, vp * 2 * P};
      gh.m = (int)a.c.hidden;
      gh.n = (int)a.c.rows;
      gh.nkb = (int)(vp * 2 * P / KBLOCK);
      gh.split = l.split_h;
      gh.slots = l.hslots ? (float*)(a.ws + l.hslots) : nullptr;
      gh.add = v0 > 0;
      gh.out = a.gh;
      gh.o0 = a.c.hidden;
      gh.o1 = 1;
      gh.scale = scale;
      gh.s = s;
      gh.by_w = 1;
      if (const int rc = grad_launch<T, C>(a, gh)) return rc;
    }
    if (a.gw) {
      Grad gw = {};
      gw.a = {a.ws + l.ht, l.np * 2 * P};
      gw.b = {a.ws + l.dt, l.np * 2 * P};
      gw.m = (int)a.c.hidden;
      gw.n = (int)cols;
      gw.nkb = (int)(l.np * 2 * P / KBLOCK);
      gw.split = l.split_w;
      gw.slots = l.wslots ? (float*)(a.ws + l.wslots) : nullptr;
      gw.out = (T*)a.gw + v0 * a.c.hidden;
      gw.o0 = a.c.hidden;
      gw.o1 = 1;
      gw.s = s;
      if (const int rc = grad_launch<T, C>(a, gw)) return rc;
      if (gw.slots) join_launch<T>(a, gw);
    }
  }
  if (a.gh && gh.slots) join_launch<T>(a, gh);
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace grlhip

using namespace grlhip;

extern "C" {

size_t grlhip_linear_ce_workspace_bytes(const void* hidden, const int64_t* hidden_strides, const void* weight, const int64_t* weight_strides,
                                        int64_t rows, int64_t features, int64_t vocab, int elem, int backward_) {
  return guarded_size([&]() -> size_t {
    if (rows < 1 || features < 1 || vocab < 1 || rows > MAX_ROWS || features > MAX_HIDDEN || vocab > MAX_VOCAB || elem < GRLHIP_ELEM_F32 || elem > GRLHIP_ELEM_F16) {
      set_error(GRLHIP_ERR_UNSUPPORTED, "linear_ce: rows, features and vocabulary must be 1 to 2^20, 2^16 and 2^21, and the element type known");
      return 0;
    }
    const Shape c{rows, features, vocab, elem};
    const int64_t dense[2] = {features, 1};
    if (!hidden_strides) hidden_strides = dense;
    if (!weight_strides) weight_strides = dense;
    return (size_t)layout_of(c, direct(hidden, hidden_strides[0], hidden_strides[1], c), direct(weight, weight_strides[0], weight_strides[1], c),
                             backward_ != 0, true).bytes;
  });
}

int grlhip_linear_ce_forward(const void* hidden, const int64_t* hidden_strides, const void* weight, const int64_t* weight_strides, const float* bias,
                             const int64_t* target, int64_t ignore_index, const float* row_weight, int64_t rows, int64_t features, int64_t vocab,
                             int elem, int reduction, float* losses, float* lse, float* total, float* count, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    Call a = {};
    a.c = {rows, features, vocab, elem};
    a.h = hidden;
    a.h0 = hidden_strides ? hidden_strides[0] : features;
    a.h1 = hidden_strides ? hidden_strides[1] : 1;
    a.w = weight;
    a.w0 = weight_strides ? weight_strides[0] : features;
    a.w1 = weight_strides ? weight_strides[1] : 1;
    a.bias = bias;
    a.target = target;
    a.row_weight = row_weight;
    a.ignore = ignore_index;
    a.reduction = reduction;
    a.losses = losses;
    a.lse = lse;
    a.total = total;
    a.count = count;
    a.ws = (char*)workspace;
    a.ws_bytes = workspace_bytes;
    a.stream = (hipStream_t)stream;
    if (const int rc = check("linear_ce_forward", a)) return rc;
    if (!losses || !total) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: null losses or total");
    if ((size_t)workspace & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: the workspace must be aligned to 256 bytes");
    return elem == GRLHIP_ELEM_F32 ? forward<float>(a) : elem == GRLHIP_ELEM_BF16 ? forward<__bf16>(a) : forward<_Float16>(a);
  });
}

int grlhip_linear_ce_backward(const void* hidden, const int64_t* hidden_strides, const void* weight, const int64_t* weight_strides, const float* bias,
                              const int64_t* target, int64_t ignore_index, const float* row_weight, int64_t rows, int64_t features, int64_t vocab,
                              int elem, int reduction, const float* lse, const float* count, const float* grad, int64_t grad_stride,
                              void* grad_hidden, void* grad_weight, float* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    Call a = {};
    a.c = {rows, features, vocab, elem};
    a.h = hidden;
    a.h0 = hidden_strides ? hidden_strides[0] : features;
    a.h1 = hidden_strides ? hidden_strides[1] : 1;
    a.w = weight;
    a.w0 = weight_strides ? weight_strides[0] : features;
    a.w1 = weight_strides ? weight_strides[1] : 1;
    a.bias = bias;
    a.target = target;
    a.row_weight = row_weight;
    a.ignore = ignore_index;
    a.reduction = reduction;
    a.lse = const_cast<float*>(lse);
    a.count = const_cast<float*>(count);
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.gh = grad_hidden;
    a.gw = grad_weight;
    a.gb = grad_bias;
    a.ws = (char*)workspace;
    a.ws_bytes = workspace_bytes;
    a.stream = (hipStream_t)stream;
    if (const int rc = check("linear_ce_backward", a)) return rc;
    if (!grad) return set_error(GRLHIP_ERR_INVALID, "linear_ce_backward: null gradient");
    if ((size_t)workspace & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_backward: the workspace must be aligned to 256 bytes");
    if (!grad_hidden && !grad_weight && !grad_bias) return 0;
    return elem == GRLHIP_ELEM_F32 ? backward<float>(a) : elem == GRLHIP_ELEM_BF16 ? backward<__bf16>(a) : backward<_Float16>(a);
  });
}

}  // extern "C"
