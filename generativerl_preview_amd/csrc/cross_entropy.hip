// Softmax cross entropy of z = hidden W^T + bias over a large vocabulary, and its gradients, without the logits (contract:
// include/grlhip.h, grlhip_linear_ce_forward / grlhip_linear_ce_backward).
//
// Forward: a tile of z lives in accumulators only; its epilogue leaves each row's maximum and sum of exponentials, and the
// target's logit; one pass over these partials gives logsumexp and the loss.  2 N V H flops.
// Backward, one piece of the vocabulary at a time: z again (the same products in the same order), D = softmax - onehot written
// in fp16 both ways round, D as [row][v] for dH += D W and D scaled by the row's gradient as [v][row] for dW = D^T H.  6 N V H
// flops; the workspace holds D of one piece.  Recomputing z costs a third more products than keeping it would.  For that nothing of N V
// entries outlives the forward pass.  At the peak, in the backward pass, it saves memory only where there are several pieces: one of up to
// 2^27 entries holds D in 4 bytes an entry (bf16) or 8, as much as fp32 logits or twice that.
//
// Precision.  z: 16-bit operands are used as they are, fp32 ones as two fp16 pieces a value (gemm_core.hip.inc), each row of hidden and of the
// weight scaled by a power of two of its own that brings its largest entry to 2^13..2^14: what is lost of a value is at most 2^-23 of it or 2^-38
// of the largest of its row.  D lies in [-1, 1] and is held times 2^14 in fp16: one piece for bf16 operands (off by 2^-11 at most, an eighth
// of the gradients' own rounding; held in bf16 it would be off by as much as that), two for fp16 and fp32 (one would be off by as much as an
// fp16 gradient's own rounding; two lose 2^-22 of it or 2^-39).  W^T and hidden^T beside it are fp16 for that: fp16 entries stand as they are, bf16
// ones fit its 11 bits exactly (down to 2^-28 of the tensor's largest, to which they are scaled), fp32 ones are two pieces.  These products sum over
// rows, so that fp32 rows cannot each have their scale there: a row whose largest entry is 2^d below the tensor's stands 2^(d - d/2) below, and D
// beside it is divided by 2^(d/2).  Its entries lose up to 2^(d/2 - 38) of its largest, D up to 2^(d/2 - 39): fp32's 2^-24 for rows up to
// 2^28 apart.  All sums are fp32 or wider and taken in a fixed order: results repeat bit for bit.
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
// entries of D in one piece of the vocabulary: 512 MiB of D both ways round beside bf16 operands.  8192 x 2048 x 65536 in 8.26 ms; with pieces
// of 2^26 8.34, of 2^25 9.14 (each adds to all of dH)
constexpr int64_t PIECE = 1ll << 27;
constexpr int HMAX = 64, WMAX = 512, GMAX = 64;   // blocks of the maxima; k_ce_pack joins WMAX by 2 a thread
__host__ __device__ inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// What the launches of a call share: largest finite magnitudes of hidden and weight, and of the rows' gradients by block.
struct Scalars { float h, w; float gpart[GMAX]; };
// What the pass over the operands' magnitudes leaves: the largest by block, and for fp32 the exponents of the scales of hidden's rows, then
// of the weight's.  In the workspace, or kept by the caller from the forward call to the backward call.
struct Parts { float hpart[HMAX], wpart[WMAX]; };

// 13 - e: the exponent of the power of two that brings the largest magnitude to 2^13..2^14; 0 for nothing but zeros.  Scales are undone by the
// sum of their exponents: a product of one scale's reciprocal with the sum may leave fp32's range where the result does not.
__device__ __forceinline__ int scale_exponent(float most) {
  if (most == 0.f) return 0;
  const int e = __builtin_amdgcn_frexp_expf(most) - 1;
  return 13 - (e < -100 ? -100 : e);
}
__device__ __forceinline__ float scale_of(float most) { return __builtin_ldexpf(1.f, scale_exponent(most)); }
// How far a row's scale is above the largest row's (the common one's exponent; a row of zeros has no scale to speak of)
__device__ __forceinline__ int apart_of(int row, int common) { return row > common ? row - common : 0; }
// of a power of two that no gradient factor passes; not below -112, so that 2^14 over it is a number too
__device__ __forceinline__ int ceil_exponent(float most) {
  if (most == 0.f) return 0;
  const int e = __builtin_amdgcn_frexp_expf(most);
  return e > 127 ? 127 : e < -112 ? -112 : e;
}
__device__ __forceinline__ float finite(float v) { return __builtin_isfinite(v) ? fabsf(v) : 0.f; }
__device__ __forceinline__ float wave_max(float m) {
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  return m;
}
// over a block of 256 threads; all of them get it
__device__ __forceinline__ float block_max(float m, float* sh) {
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}
__device__ __forceinline__ float largest_gradient(const Scalars* s) { return wave_max(s->gpart[threadIdx.x & 63]); }

struct View { const void* p; int64_t s0, s1; int rows, cols; };   // element strides

// What leaves a row of hidden (its target, its weight) or of the weight (a bias of -inf) out of everything.
struct Left { const int64_t* target; const float* row_weight; int64_t ignore; const float* bias; };
__device__ __forceinline__ bool row_counts(const Left& l, int row) { return l.target[row] != l.ignore && !(l.row_weight && l.row_weight[row] == 0.f); }
__device__ __forceinline__ bool masked(const float* bias, int v) { return bias && bias[v] == -INFINITY; }

// The largest finite magnitude of each row of hidden (blocks [0, HMAX)) and of the weight (the others), left behind as the exponent of the
// row's scale (hs, ws, or null), and of all rows of a block.  A row that is left out counts as zeros: padding may hold anything, and a
// scale that follows it would cost the others their bits.  One pass at the rate of the loads: `team` lanes a row, 4 loads of 16 bytes a lane
// in flight, the last one of a row moved back to where the row ends (a maximum may meet an entry twice).
constexpr int MAG_THREADS = 1024, SCALES_END = 256;   // exponents behind the last row: a tile reads its rows' by fours
template <class T>
__global__ __launch_bounds__(MAG_THREADS, 8) void k_ce_magnitudes(View h, View w, Left left, Parts* parts, int* hs, int* ws) {
  __shared__ float sh[MAG_THREADS / 64][64];
  const bool is_h = blockIdx.x < HMAX;
  const View& v = is_h ? h : w;
  int* const out = is_h ? hs : ws;
  const int b = is_h ? blockIdx.x : blockIdx.x - HMAX, n = is_h ? HMAX : WMAX, tid = threadIdx.x, wave = tid >> 6;
  constexpr int E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  float most = 0.f;
  if (out && b == 0 && tid < SCALES_END) out[v.rows + tid] = 0;
  auto done = [&](int row, float m) {   // by one thread a row
    if (!(is_h ? row_counts(left, row) : !masked(left.bias, row))) m = 0.f;
    if (out) out[row] = scale_exponent(m);
    most = fmaxf(most, m);
  };
  if (v.s1 <= v.s0 || v.rows == 1) {
    const bool wide = v.s1 == 1 && v.cols >= E;
    const int chunks = wide ? (v.cols + E - 1) / E : v.cols;
    int team = 1;
    while (team < chunks && team < 64) team *= 2;
    if (chunks > 1024) team = MAG_THREADS;
    const bool few = chunks <= team;   // a load a lane: 4 rows at a time
    const int R = MAG_THREADS / team, lane = tid & (team - 1), mine = tid / team, step = few ? 4 * R : R;
    auto load = [&](int row, int chunk) {
      const T* p = (const T*)v.p + (row < v.rows ? row : v.rows - 1) * v.s0;
      float m = 0.f;
      if (wide) {
        const vec x = *(const vec*)(p + (chunk * E < v.cols - E ? chunk * E : v.cols - E));
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, finite((float)x[e]));
      } else {
        m = finite((float)p[(chunk < v.cols ? chunk : v.cols - 1) * v.s1]);
      }
      return m;
    };
    auto over_team = [&](float m) {
      for (int d = (team < 64 ? team : 64) / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
      return m;
    };
    for (int r0 = b * step; r0 < v.rows; r0 += n * step) {
      float m[4];
      if (few) {
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = load(r0 + u * R + mine, lane);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          m[u] = over_team(m[u]);
          if (lane == 0 && r0 + u * R + mine < v.rows) done(r0 + u * R + mine, m[u]);
        }
        continue;
      }
      float all = 0.f;
      for (int c = lane; c < chunks; c += 4 * team) {
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = load(r0 + mine, c + u * team);
        all = fmaxf(all, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
      }
      all = over_team(all);
      if (team > 64) {   // the block's only row
        if ((tid & 63) == 0) sh[wave][0] = all;
        __syncthreads();
        if (tid == 0)
          for (int k = 1; k < MAG_THREADS / 64; ++k) all = fmaxf(all, sh[k][0]);
        __syncthreads();
      }
      if (lane == 0 && r0 + mine < v.rows) done(r0 + mine, all);
    }
  } else {   // rows closer in memory than columns: a lane a row, the waves take the columns in turn
    const int q = MAG_THREADS / 64, lane = tid & 63;
    for (int r0 = b * 64; r0 < v.rows; r0 += n * 64) {
      const int row = r0 + lane;
      const T* p = (const T*)v.p + (row < v.rows ? row : v.rows - 1) * v.s0;
      float all = 0.f;
      for (int c = wave; c < v.cols; c += 4 * q) {
        float m[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = finite((float)p[(c + u * q < v.cols ? c + u * q : v.cols - 1) * v.s1]);
        all = fmaxf(all, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
      }
      sh[wave][lane] = all;
      __syncthreads();
      if (wave == 0) {
        for (int k = 1; k < q; ++k) all = fmaxf(all, sh[k][lane]);
        if (row < v.rows) done(row, all);
      }
      __syncthreads();
    }
  }
  most = wave_max(most);
  if ((tid & 63) == 0) sh[wave][0] = most;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < MAG_THREADS / 64; ++k) most = fmaxf(most, sh[k][0]);
    (is_h ? parts->hpart : parts->wpart)[b] = most;
  }
}

// A view -> operands: as it stands (n: rows of the view, type E) and transposed (t: its columns, fp16), either may be null; columns
// beyond the view and up to the pitch become zeros.  fp32: two fp16 pieces both ways, each row by its own scale as it stands.  bf16 transposed: scaled.  A row that
// does not count becomes zeros: whatever it holds must not reach a sum over rows; so does a masked row of the weight, whose D is 0.
struct Job {
  View v;
  void* n; int64_t n_cols;
  void* t; int64_t t_cols;
  bool mask; const float* bias;   // leaves out rows: of hidden, of the weight
  const int* scales;              // fp32: the exponents of the rows' scales
  int blocks;
};
// The gradient of each row's own loss, and the largest of them.
struct Scale {
  const float* grad; int64_t grad_stride;
  const float* count;
  int rows, vocab, reduction, blocks;
  float* scale;
};
template <class E, bool TWO, class F>   // 128 bytes of a row by 8 threads
__device__ __forceinline__ void pack_rows(E* out, int64_t cols, int r0, int rows, int c0, F&& value) {
  typedef E e8 __attribute__((ext_vector_type(8)));
  const int chunk = threadIdx.x & 7;
#pragma unroll
  for (int k = 0; k < (TWO ? 4 : 2); ++k) {
    const int line = (threadIdx.x >> 3) + 32 * k, row = TWO ? line >> 1 : line, col = TWO ? (line & 1) * 32 + (chunk & 3) * 8 : chunk * 8;
    e8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = value(row, col + e);
      if constexpr (TWO) {
        _Float16 hi, lo;
        split2(v, hi, lo);
        x[e] = chunk >> 2 ? lo : hi;
      } else {
        x[e] = (E)v;
      }
    }
    if (r0 + row < rows && c0 + col < cols)
      *(e8*)(out + (int64_t)(r0 + row) * (TWO ? 2 : 1) * cols + (TWO ? ((c0 + col) >> 5) * 64 + (chunk >> 2) * 32 + (chunk & 3) * 8 : c0 + col)) = x;
  }
}
// pieces of D and of what it is multiplied by; 3: two, of which the other factor needs one
template <class T> struct GradPieces { static constexpr int P = __is_same(T, float) ? 2 : __is_same(T, _Float16) ? 3 : 1, N = P == 1 ? 1 : 2; };
template <class T>
__global__ __launch_bounds__(256) void k_ce_pack(Job h, Job w, Scale g, Left left, const Parts* parts, Scalars* s, float* largest) {
  constexpr bool TWO = sizeof(T) == 4, SCALED = !__is_same(T, _Float16);
  __shared__ float tile[64][65], sh[4];
  __shared__ int own[64], shared[64];   // fp32: exponents of the rows' scales as they stand, and from there to the common one
  if ((int)blockIdx.x >= h.blocks + w.blocks) {
    const int b = blockIdx.x - h.blocks - w.blocks;
    float most = 0.f;
    for (int n = b * 256 + threadIdx.x; n < g.rows; n += g.blocks * 256) {
      const int64_t t = left.target[n];
      const float rw = left.row_weight ? left.row_weight[n] : 1.f;
      float v = 0.f;
      if (t != left.ignore && rw != 0.f) {
        v = g.grad[n * g.grad_stride] * rw;
        if (g.reduction == GRLHIP_REDUCE_MEAN) v /= *g.count;
        if (t < 0 || t >= g.vocab) v = NAN;
      }
      g.scale[n] = v;
      most = fmaxf(most, finite(v));
    }
    most = block_max(most, sh);
    if (threadIdx.x == 0) s->gpart[b] = most;
    if (b == 0 && (int)threadIdx.x >= g.blocks && threadIdx.x < GMAX) s->gpart[threadIdx.x] = 0.f;
    return;
  }
  const bool is_h = (int)blockIdx.x < h.blocks;
  const Job& a = is_h ? h : w;
  const int b = is_h ? blockIdx.x : blockIdx.x - h.blocks;
  const int across = (a.v.cols + 63) / 64, i0 = b / across * 64, j0 = b % across * 64, tid = threadIdx.x;
  float f = 1.f;
  if (SCALED && (TWO || a.t)) {   // 16-bit operands that stand as they are have no scale
    const float most = block_max(is_h ? (tid < HMAX ? parts->hpart[tid] : 0.f) : fmaxf(parts->wpart[tid], parts->wpart[tid + 256]), sh);
    f = scale_of(most);
    if (b == 0 && tid == 0) {
      (is_h ? s->h : s->w) = most;
      if (TWO && largest) largest[is_h ? 0 : 1] = most;
    }
    if (TWO) {
      if (tid < 64) {
        const int e = a.scales[i0 + tid < a.v.rows ? i0 + tid : a.v.rows - 1], apart = apart_of(e, scale_exponent(most));
        own[tid] = e;
        shared[tid] = (apart >> 1) - apart;
      }
      __syncthreads();
    }
  }
  const bool along = a.v.s1 <= a.v.s0;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int i = along ? (tid >> 6) + 4 * k : tid & 63, j = along ? tid & 63 : (tid >> 6) + 4 * k;
    float x = 0.f;
    if (i0 + i < a.v.rows && j0 + j < a.v.cols) {
      if (!a.mask || row_counts(left, i0 + i)) x = (float)((const T*)a.v.p)[(int64_t)(i0 + i) * a.v.s0 + (int64_t)(j0 + j) * a.v.s1];
      if (masked(a.bias, i0 + i)) x = 0.f;
    }
    tile[i][j] = TWO ? __builtin_ldexpf(x, own[i]) : x;
  }
  __syncthreads();
  if (a.n) {
    if constexpr (TWO) pack_rows<_Float16, true>((_Float16*)a.n, a.n_cols, i0, a.v.rows, j0, [&](int r, int c) { return tile[r][c]; });
    else pack_rows<T, false>((T*)a.n, a.n_cols, i0, a.v.rows, j0, [&](int r, int c) { return tile[r][c]; });
  }
  if (a.t) {
    if constexpr (GradPieces<T>::N == 2)
      pack_rows<_Float16, true>((_Float16*)a.t, a.t_cols, j0, a.v.cols, i0, [&](int r, int c) { return TWO ? __builtin_ldexpf(tile[c][r], shared[c]) : tile[c][r]; });
    else pack_rows<_Float16, false>((_Float16*)a.t, a.t_cols, j0, a.v.cols, i0, [&](int r, int c) { return tile[c][r] * f; });
  }
}

struct Operand { const char* p; int64_t pitch; };   // K-contiguous rows; pitch in bytes

struct Logits {
  Operand w, h;             // rows of the weight piece, rows of hidden
  const float* bias;        // of the piece, or null
  const int64_t* target;
  const float* lse;         // backward
  const float* scale;       // backward: gradient of each row's loss (0: the row does not count)
  const Scalars* s;
  const int *hs, *ws;       // fp32: the exponents of the rows' scales, of hidden and of the piece
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

// The accumulators of 32 rows of the tile (vocabulary entries from mb on) become z, in place.  `hs`: the exponents of the columns' scales; `ws`:
// those of the rows' are left there, 0 behind the piece.
template <int P, int TN>
__device__ __forceinline__ void logits_of(const Logits& a, f32x16 (&acc)[TN], int mb, int h, const int (&hs)[TN], i32x4 (&ws)[4]) {
  if (P == 2) {
#pragma unroll
    for (int q = 0; q < 4; ++q) ws[q] = *(const i32x4*)(a.ws + mb + 8 * q + 4 * h);
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int x = 0; x < TN; ++x) acc[x][r] = __builtin_ldexpf(acc[x][r], -(ws[r >> 2][r & 3] + hs[x]));
  }
  if (a.bias)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = mb + 8 * (r >> 2) + 4 * h + (r & 3);
      const float b = a.bias[m < a.cols ? m : a.cols - 1];
      // a masked entry is -inf whatever its product came to: inf and NaN do not become -inf by adding it
#pragma unroll
      for (int x = 0; x < TN; ++x) acc[x][r] = b == -INFINITY ? b : acc[x][r] + b;
    }
}

// The epilogue is most of a tile's time where the features are few (8 K blocks of 512 features: 15 us of products): ~9 operations an
// entry -- exp counts for 4 -- and what concerns few entries (the end of the vocabulary, the targets) under branches of the whole wave.
template <class T, int P, class C>
__global__ __launch_bounds__(C::THREADS, C::LDS > 81920 ? C::THREADS / 256 : C::THREADS / 128) void k_ce_forward(Logits a, int tm, int tn) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  int im, in;
  tile_at(xcd_order(blockIdx.x, gridDim.x), tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  f32x16 acc[C::TM][C::TN];
  if (!product<T, P, C>(a.w.p + m0 * a.w.pitch, a.w.pitch, a.cols - m0, a.h.p + n0 * a.h.pitch, a.h.pitch, a.rows - n0, a.nkb, lds, acc)) return;
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  int hs[C::TN];
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int n = n0 + (wn * C::TN + x) * 32 + L.j;
    hs[x] = P == 2 ? a.hs[n < a.rows ? n : a.rows - 1] : 0;
  }
  float* tops = (float*)lds;                  // [WM][BN] maxima, then sums
  float* sums = tops + C::WM * C::BN;
#pragma unroll
  for (int y = 0; y < C::TM; ++y) {
    const int mb = m0 + (wm * C::TM + y) * 32;
    i32x4 ws[4];
    logits_of<P>(a, acc[y], mb, L.h, hs, ws);
    if (mb + 32 > a.cols)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (mb + 8 * (r >> 2) + 4 * L.h + (r & 3) >= a.cols)
#pragma unroll
          for (int x = 0; x < C::TN; ++x) acc[y][x][r] = -INFINITY;
  }
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int nl = (wn * C::TN + x) * 32 + L.j, n = n0 + nl;
    const int64_t t = (n < a.rows ? a.target[n] : -1) - a.v0 - m0 - wm * C::TM * 32;
    const int rel = t >= 0 && t < C::TM * 32 && t + m0 + wm * C::TM * 32 < a.cols ? (int)t : -1;   // the target's row of this wave's part
    if (__any(rel >= 0)) {
#pragma unroll
      for (int y = 0; y < C::TM; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (rel == y * 32 + 8 * (r >> 2) + 4 * L.h + (r & 3)) a.picked[n] = acc[y][x][r];
    }
    float top = -INFINITY;
#pragma unroll
    for (int y = 0; y < C::TM; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[y][x][r]);
    top = fmaxf(top, __shfl_xor(top, 32));
    // nothing but -inf: a sum of zeros, not of -inf - -inf.  A NaN passes fmaxf, and is caught by the sum
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < C::TM; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __expf(acc[y][x][r] - ref);
    sum += __shfl_xor(sum, 32);
    if (L.h == 0) {
      tops[wm * C::BN + nl] = top;
      sums[wm * C::BN + nl] = sum;
    }
  }
  lds_barrier();
  for (int k = threadIdx.x; k < C::BN; k += C::ACTIVE) {
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
  double* sums;       // [blocks][2]: weighted loss, rows that count; null: nobody asks for the total
  float* total; float* count;   // the reduced loss; the number of rows that are not ignored, at least 1
  int reduction;
};

// The partials of a row, then its loss: Q threads a row.  8: rows along the lanes, as they lie in memory; 64: a wave a row, where rows
// are few and partials many.
template <int Q>
__global__ __launch_bounds__(256) void k_ce_finish(Finish a) {
  constexpr int R = 256 / Q;
  __shared__ float tops[8][32], sums[8][32];
  __shared__ double s[R], c[R];
  const int r = Q == 64 ? threadIdx.x / 64 : threadIdx.x % R, q = Q == 64 ? threadIdx.x % 64 : threadIdx.x / R, n = blockIdx.x * R + r;
  float top = -INFINITY, sum = 0.f;
  auto add = [&](float t, float u) {
    const float most = fmaxf(top, t);
    sum = (top == -INFINITY ? sum : sum * __expf(top - most)) + (t == -INFINITY ? u : u * __expf(t - most));
    top = most;
  };
  if (n < a.rows)
#pragma unroll 4
    for (int t = q; t < a.tiles; t += Q) {
      const float2 p = a.part[(int64_t)t * a.rows + n];
      add(p.x, p.y);
    }
  if (Q == 64) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const float t = __shfl_xor(top, d), u = __shfl_xor(sum, d);
      add(t, u);
    }
  } else {
    tops[q][r] = top;
    sums[q][r] = sum;
    __syncthreads();
    if (q == 0)
      for (int k = 1; k < Q; ++k) add(tops[k][r], sums[k][r]);
  }
  if (q == 0) {
    s[r] = c[r] = 0.0;
    if (n < a.rows) {
      const int64_t t = a.target[n];
      const bool kept = t != a.ignore;
      const float w = a.row_weight ? a.row_weight[n] : 1.f;
      const float lse = top + logf(sum);
      // a target outside the vocabulary has no loss: NaN, not a number that looks like one
      float loss = t >= 0 && t < a.vocab ? (lse - a.picked[n]) * w : NAN;
      if (!kept || w == 0.f) loss = 0.f;
      if (a.lse) a.lse[n] = lse;
      a.losses[n] = loss;
      s[r] = loss;
      c[r] = kept ? 1.0 : 0.0;
    }
  }
  if (!a.sums) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    double x = 0.0, y = 0.0;
    for (int k = 0; k < R; ++k) { x += s[k]; y += c[k]; }
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

constexpr int DBITS = 14;
constexpr float DSCALE = 1 << DBITS;   // D lies in [-2^14, 2^14]

// N: pieces of D
template <class T, int P, int N, class C>
__global__ __launch_bounds__(C::THREADS, C::LDS > 81920 ? C::THREADS / 256 : C::THREADS / 128) void k_ce_d(Logits a, int tm, int tn) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  int im, in;
  tile_at(xcd_order(blockIdx.x, gridDim.x), tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  f32x16 acc[C::TM][C::TN];
  if (!product<T, P, C>(a.w.p + m0 * a.w.pitch, a.w.pitch, a.cols - m0, a.h.p + n0 * a.h.pitch, a.h.pitch, a.rows - n0, a.nkb, lds, acc)) return;
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  int hs[C::TN];
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int n = n0 + (wn * C::TN + x) * 32 + L.j;
    hs[x] = P == 2 ? a.hs[n < a.rows ? n : a.rows - 1] : 0;
  }
  const float per = __builtin_ldexpf(1.f, DBITS - ceil_exponent(largest_gradient(a.s)));
  const int common_w = P == 2 ? scale_exponent(a.s->w) : 0, common_h = P == 2 ? scale_exponent(a.s->h) : 0;
  unsigned* patch = (unsigned*)(lds + L.wave * PATCH);
  float* bsum = (float*)(lds + C::WAVES * PATCH);   // [WN][BM]
  float lse[C::TN], g[C::TN];
  int64_t t[C::TN];
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
    const int n = n0 + (wn * C::TN + x) * 32 + L.j;
    lse[x] = n < a.rows ? a.lse[n] : 0.f;
    g[x] = n < a.rows ? a.scale[n] : 0.f;
    t[x] = (n < a.rows ? a.target[n] : -1) - a.v0;
  }
#pragma unroll
  for (int y = 0; y < C::TM; ++y) {
    const int mb = m0 + (wm * C::TM + y) * 32;
    i32x4 ws[4];
    logits_of<P>(a, acc[y], mb, L.h, hs, ws);
    float bs[16], scale[16];   // scale: D's for dH
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      bs[r] = 0.f;
      scale[r] = P == 2 ? __builtin_ldexpf(1.f, DBITS - (apart_of(ws[r >> 2][r & 3], common_w) >> 1)) : DSCALE;
    }
#pragma unroll
    for (int x = 0; x < C::TN; ++x) {
      const int nb = n0 + (wn * C::TN + x) * 32;
      const bool dead = g[x] == 0.f;   // a row that does not count, whatever its logits are
      float z[16], v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __expf(acc[y][x][r] - lse[x]);
        z[r] = dead ? 0.f : p;
      }
      const int rel = t[x] >= mb && t[x] < mb + 32 && !dead ? (int)(t[x] - mb) : -1;
      if (__any(rel >= 0)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] -= rel == 8 * (r >> 2) + 4 * L.h + (r & 3) ? 1.f : 0.f;
      }
      if (mb + 32 > a.cols)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (mb + 8 * (r >> 2) + 4 * L.h + (r & 3) >= a.cols) z[r] = 0.f;
      if (a.bpart)
#pragma unroll
        for (int r = 0; r < 16; ++r) bs[r] += z[r] * g[x];
      const float gd = P == 2 ? __builtin_ldexpf(g[x] * per, -(apart_of(hs[x], common_h) >> 1)) : g[x] * per;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        v[r] = z[r] * gd;
        z[r] *= scale[r];
      }
      if (nb < a.rows && mb < a.d_cols) {
        if constexpr (N == 2) store_t_f16x2((_Float16*)a.d + (int64_t)nb * 2 * a.d_cols + mb * 2, 2 * a.d_cols, patch, L, a.rows - nb, z);
        else store_t_16<_Float16>((_Float16*)a.d + (int64_t)nb * a.d_cols + mb, a.d_cols, patch, L, a.rows - nb, z);
      }
      if (nb < a.dt_cols && mb < a.cols) {
        if constexpr (N == 2) store_n_f16x2((_Float16*)a.dt + (int64_t)mb * 2 * a.dt_cols + nb * 2, 2 * a.dt_cols, patch, L, a.cols - mb, v);
        else store_n_16<_Float16>((_Float16*)a.dt + (int64_t)mb * a.dt_cols + nb, a.dt_cols, patch, L, a.cols - mb, v);
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
    for (int k = threadIdx.x; k < C::BM; k += C::ACTIVE) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) s += bsum[w * C::BM + k];
      if (m0 + k < a.cols) a.bpart[(int64_t)in * a.cols + m0 + k] = s;
    }
  }
}

// out[n][m] = f(n) sum_k A[m][k] B[n][k]: dH (A = W^T, B = D; f = the row's gradient) and dW (A = hidden^T, B = D^T).
struct Grad {
  Operand a, b;
  int m, n, nkb, split;     // split: parts of the K blocks
  int tiles;                // of the launch; 0: not asked for
  float* slots;             // fp32 [split][n][m], or null: straight to `out`
  int add;                  // to what the slots hold
  void* out;                // dense rows
  const float* scale;       // per row, or null
  int by_w;                 // the operands' scales: W's (dH) or hidden's and the gradient's (dW)
};
struct Grads { Grad g[2]; const Scalars* s; };   // one launch: dH's tiles, then dW's
template <class T>
__device__ __forceinline__ int undo_of(const Grad& g, const Scalars* s) {
  int e = -DBITS;
  if (!__is_same(T, _Float16)) e -= scale_exponent(g.by_w ? s->w : s->h);
  if (!g.by_w) e += ceil_exponent(largest_gradient(s));
  return e;
}
template <class T, int P, class C>
__global__ __launch_bounds__(C::THREADS, C::LDS > 81920 ? C::THREADS / 256 : C::THREADS / 128) void k_ce_grad(Grads both) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const bool second = (int)blockIdx.x >= both.g[0].tiles;
  const Grad& g = both.g[second];
  const int tm = (g.m + C::BM - 1) / C::BM, tn = (g.n + C::BN - 1) / C::BN;
  const int id = xcd_order(blockIdx.x - (second ? both.g[0].tiles : 0), g.tiles), part = id / (tm * tn);
  int im, in;
  tile_at(id - part * tm * tn, tm, tn, im, in);
  const int m0 = im * C::BM, n0 = in * C::BN;
  const int k0 = (int)((int64_t)g.nkb * part / g.split), k1 = (int)((int64_t)g.nkb * (part + 1) / g.split);
  f32x16 acc[C::TM][C::TN];
  if (!product<_Float16, P, C>(g.a.p + m0 * g.a.pitch + (int64_t)k0 * KBLOCK, g.a.pitch, g.m - m0, g.b.p + n0 * g.b.pitch + (int64_t)k0 * KBLOCK,
                               g.b.pitch, g.n - n0, k1 - k0, lds, acc)) return;
  const Lane L = lane_of();
  const int wm = L.wave / C::WN, wn = L.wave % C::WN;
  const int undo = undo_of<T>(g, both.s);
  float* patch = (float*)(lds + L.wave * PATCH);
  const bool to_slots = g.slots != nullptr;
  // whole 16-byte stores where the rows allow them
  const bool wide = to_slots ? g.m % 4 == 0 : g.m * sizeof(T) % 16 == 0 && ((size_t)g.out & 15) == 0;
#pragma unroll
  for (int x = 0; x < C::TN; ++x) {
#pragma unroll
    for (int y = 0; y < C::TM; ++y) {
      const int mb = m0 + (wm * C::TM + y) * 32, nb = n0 + (wn * C::TN + x) * 32;
      // through LDS: two lanes hold the 32 entries of a row (see store_t_f16x2)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4v*)(patch + L.j * 36 + 8 * q + 4 * L.h) = f32x4v{acc[y][x][4 * q], acc[y][x][4 * q + 1], acc[y][x][4 * q + 2], acc[y][x][4 * q + 3]};
      float v[16];
      const int row = L.lane >> 1, half = L.lane & 1, n = nb + row, m = mb + half * 16;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4v t = *(const f32x4v*)(patch + row * 36 + half * 16 + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
      }
      if (n >= g.n || m >= g.m) continue;
      if (to_slots) {
        float* o = g.slots + ((int64_t)part * g.n + n) * g.m + m;
        if (wide && m + 16 <= g.m) {
          f32x4v old[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) old[q] = g.add ? *(const f32x4v*)(o + 4 * q) : f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; ++q) *(f32x4v*)(o + 4 * q) = old[q] + f32x4v{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        } else {
          for (int i = 0; i < 16 && m + i < g.m; ++i) o[i] = v[i] + (g.add ? o[i] : 0.f);
        }
        continue;
      }
      const float r = g.scale ? g.scale[n] : 1.f;
      T w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = g.scale && r == 0.f ? (T)0.f : (T)(__builtin_ldexpf(v[i], undo) * r);
      T* o = (T*)g.out + (int64_t)n * g.m + m;
      if (wide && m + 16 <= g.m) {
        constexpr int E = 16 / sizeof(T);
        typedef T vec __attribute__((ext_vector_type(E)));
#pragma unroll
        for (int q = 0; q < 16 / E; ++q) {
          vec t;
#pragma unroll
          for (int e = 0; e < E; ++e) t[e] = w[q * E + e];
          *(vec*)(o + q * E) = t;
        }
      } else {
        for (int i = 0; i < 16 && m + i < g.m; ++i) o[i] = w[i];
      }
    }
  }
}
// The parts of the sums, in order: dH's blocks, dW's, the bias' (part [tiles][cols]).
struct Join { Grads both; int blocks[2]; const float* bpart; int btiles, cols; float* gb; };
template <class T>
__global__ __launch_bounds__(256) void k_ce_join(Join a) {
  const int b = blockIdx.x;
  if (b >= a.blocks[0] + a.blocks[1]) {
    const int v = (b - a.blocks[0] - a.blocks[1]) * 256 + threadIdx.x;
    if (v >= a.cols) return;
    float s = 0.f;
#pragma unroll 8
    for (int t = 0; t < a.btiles; ++t) s += a.bpart[(int64_t)t * a.cols + v];
    a.gb[v] = s;
    return;
  }
  const int k = b >= a.blocks[0];
  const Grad& g = a.both.g[k];
  const int undo = undo_of<T>(g, a.both.s);
  const int64_t all = (int64_t)g.n * g.m, step = (int64_t)a.blocks[k] * 256;
  for (int64_t i = (int64_t)(k ? b - a.blocks[0] : b) * 256 + threadIdx.x; i < all; i += step) {
    float s = 0.f;
#pragma unroll 8
    for (int p = 0; p < g.split; ++p) s += g.slots[p * all + i];
    const float row = g.scale ? g.scale[i / g.m] : 1.f;
    ((T*)g.out)[i] = g.scale && row == 0.f ? (T)0.f : (T)(__builtin_ldexpf(s, undo) * row);
  }
}

// ------------------------------------------------------------------------------------------------------------- host
struct Shape { int64_t rows, hidden, vocab; int elem; };
int pieces(int elem) { return elem == GRLHIP_ELEM_F32 ? 2 : 1; }
int grad_pieces(int elem) { return elem == GRLHIP_ELEM_BF16 ? 1 : 2; }

// The shapes of tiles.  Measured per K block (128 bytes a row), one or two pieces: a tile alone on its CU, and the CU's time for one on
// a full chip.  4096 x 4096 x 8192 in bf16: 446, 282, 245 us (616, 976, 1123 TFLOP/s); 1024 x 1024 x 1024: 7.5, 12, 24 us.
typedef Tile<64, 64, 2, 2, 2, 2> Ce64;
typedef Tile<128, 128, 2, 2, 2> Ce128;
typedef Tile<256, 256, 2, 4, 2> Ce256;
constexpr int KINDS = 3, SIDE[KINDS] = {64, 128, 256}, BESIDE[KINDS] = {2, 2, 1};   // workgroups a CU
constexpr double ALONE[2][KINDS] = {{0.30, 0.61, 1.28}, {0.33, 0.67, 1.9}}, FULL[2][KINDS] = {{0.21, 0.55, 1.91}, {0.22, 0.72, 2.73}};
int64_t tiles_of(int64_t m, int64_t n, int k) { return up(m, SIDE[k]) / SIDE[k] * (up(n, SIDE[k]) / SIDE[k]); }
// Time of a launch: its longest tile, or its tiles together on all CUs, in whole tiles a CU; `entry_ns` is a CU's time for one
// entry of the epilogue, 0.8 us what a tile costs besides.
double launch_us(double tiles, double kb, int p, int k, double entry_ns) {
  const double cus = device_cus(), epilogue = SIDE[k] * SIDE[k] * entry_ns * 1e-3 + 0.8;
  return tiles <= cus ? kb * ALONE[p - 1][k] + epilogue : std::ceil(tiles / cus) * (kb * FULL[p - 1][k] + epilogue);
}
int kind_for(int64_t m, int64_t n, int64_t kb, int p, double entry_ns, int from = 0) {
  int best = from;
  for (int k = from + 1; k < KINDS; ++k)
    if (launch_us((double)tiles_of(m, n, k), (double)kb, p, k, entry_ns) < launch_us((double)tiles_of(m, n, best), (double)kb, p, best, entry_ns)) best = k;
  return best;
}
constexpr double FORWARD_NS = 0.1;   // exponentials
double d_ns(int p) { return 0.1 + 4.0 * p / 15; }   // exponentials, and 4 or 8 bytes written at a CU's share of the memory

// How a call goes about it: the same for its workspace and its launches.
struct Layout {
  int64_t kp, np;                   // hidden and rows, padded to whole K blocks
  int64_t piece;                    // vocabulary entries of a piece
  bool pack_h, pack_w;
  int kind_z, kind_g;               // tiles of the logits, of the gradients
  int split_h, split_w;             // parts of the sums of dH and dW
  int64_t pieces_n;
  // offsets
  int64_t scalars, scales, hp, wp, ht, wt, d, dt, part, picked, sums, scale, bpart, hslots, wslots, bytes;
};
// Both gradients are one launch, dH's (long) tiles first: the tiles and the parts of the sums that make it shortest.  A part costs writing
// and reading back fp32 sums and a second launch.  The constants, us by pieces of D as above, are fitted to 70 calls (1 to 20 000 rows, 64
// to 4096 features, 256 to 128 000 entries) with every kind and up to 32 parts of each sum: of 30 calls timed afterwards the rule's
// choice was 2 % over the best on average and 15 % in the worst.
constexpr double GRAD_ALONE[2][KINDS] = {{0.252, 0.684, 1.311}, {0.341, 0.691, 1.758}}, GRAD_FULL[2][KINDS] = {{0.15, 0.373, 1.152}, {0.184, 0.493, 1.645}};
constexpr double GRAD_FIXED = 1.09, GRAD_ENTRY = 0.07e-3, TAIL = 0.74, JOIN = 1.5, JOIN_BYTES = 5.3e6;   // a tile; an entry of it; a join, its bytes a us
void plan_gradients(Layout& l, const Shape& c, int64_t vp, int p) {
  const int64_t kb = p == 2 ? 32 : 64, kh = vp / kb, kw = l.np / kb;
  double best = 0;
  for (int k = 0; k < KINDS; ++k) {
    const int64_t th = tiles_of(c.hidden, c.rows, k), tw = tiles_of(c.hidden, l.piece, k);
    for (int sh = 1; sh <= 32 && (sh == 1 || kh / sh >= 4); sh *= 2)
      for (int sw = 1; sw <= 32 && (sw == 1 || kw / sw >= 4); sw *= 2) {
        const double parts = (sh > 1 ? (double)sh * c.rows * c.hidden : 0) + (sw > 1 ? (double)sw * l.piece * c.hidden : 0);
        const double cus = device_cus(), epilogue = SIDE[k] * SIDE[k] * GRAD_ENTRY + GRAD_FIXED, alone = GRAD_ALONE[p - 1][k], full = GRAD_FULL[p - 1][k];
        const double one_h = (double)kh / sh * full + epilogue, one_w = (double)kw / sw * full + epilogue, tiles = (double)(th * sh + tw * sw);
        // on a full chip the longest tile has others beside it, and the last ones leave some of the chip idle
        const double longest = std::fmax((double)kh / sh, (double)kw / sw) * (tiles <= cus ? alone : std::fmax(alone, full * BESIDE[k])) + epilogue;
        const double us = (tiles <= cus ? longest : std::fmax(longest, (th * sh * one_h + tw * sw * one_w) / cus + TAIL * one_w)) +
                          (parts > 0 ? JOIN + parts * 8 / JOIN_BYTES : 0);
        if ((k == 0 && sh == 1 && sw == 1) || us < best) {
          best = us;
          l.kind_g = k;
          l.split_h = sh;
          l.split_w = sw;
        }
      }
  }
}
// The parts, then the exponents of hidden's rows and of the weight's
int64_t scales_of_hidden() { return up(sizeof(Parts), 256); }
int64_t scales_of_weight(const Shape& c) { return scales_of_hidden() + up((c.rows + SCALES_END) * 4, 256); }
int64_t scales_bytes(const Shape& c) { return scales_of_weight(c) + up((c.vocab + SCALES_END) * 4, 256); }
Layout layout_of(const Shape& c, bool direct_h, bool direct_w, bool backward, bool bias) {
  Layout l = {};
  const int p = pieces(c.elem);
  const int64_t per = p * 2;   // bytes of an operand entry
  l.kp = up(c.hidden, 64);
  l.np = up(c.rows, 64);
  l.pack_h = !direct_h;
  l.pack_w = !direct_w;
  int64_t limit = backward ? PIECE / l.np : l.pack_w ? PIECE / l.kp : up(c.vocab, 256);
  limit = limit < 1024 ? 1024 : limit / 256 * 256;
  if (backward && limit > 1 << 19) limit = 1 << 19;                            // row offsets inside a tile are 32 bits
  const int64_t most = (1 << 20) / (up(c.rows, 64) / 64) * 64;                 // and so is a launch
  if (limit > most) limit = most < 256 ? 256 : most / 256 * 256;
  l.pieces_n = (c.vocab + limit - 1) / limit;
  l.piece = up((c.vocab + l.pieces_n - 1) / l.pieces_n, 256);
  if (l.piece > c.vocab) l.piece = c.vocab;
  l.pieces_n = (c.vocab + l.piece - 1) / l.piece;
  // The backward pass takes its logits' exponentials against the forward pass' logsumexp: both need the same bits (a saturated row of logits of
  // 1e5 has half steps of 2^-8).  The 64-wide tiles add up K in two parts, the others in one: what the forward pass takes decides for both.
  const int64_t kb = l.kp * per / KBLOCK;
  if (!backward) l.kind_z = kind_for(l.piece, c.rows, kb, p, FORWARD_NS);
  else if (layout_of(c, direct_h, direct_w, false, false).kind_z > 0) l.kind_z = kind_for(l.piece, c.rows, kb, p, d_ns(grad_pieces(c.elem)), 1);
  const int side = SIDE[l.kind_z];
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += up(bytes, 256); return o; };
  l.scalars = take(sizeof(Scalars));
  l.scales = take(p == 2 ? scales_bytes(c) : sizeof(Parts));
  if (l.pack_h) l.hp = take(c.rows * l.kp * per);
  if (l.pack_w) l.wp = take(l.piece * l.kp * per);
  if (!backward) {
    l.part = take((up(c.vocab, side) / side + l.pieces_n) * c.rows * 8);
    l.picked = take(c.rows * 4);
    l.sums = take(up(c.rows, 4) / 4 * 16);
  } else {
    const int64_t vp = up(l.piece, 64);
    const int64_t gper = grad_pieces(c.elem) * 2;
    l.ht = take(c.hidden * l.np * gper);
    l.wt = take(c.hidden * vp * gper);
    l.d = take(c.rows * vp * gper);
    l.dt = take(l.piece * l.np * gper);
    l.scale = take(c.rows * 4);
    if (bias) l.bpart = take(up(c.rows, side) / side * l.piece * 4);
    plan_gradients(l, c, vp, grad_pieces(c.elem));
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
  float* losses; float* lse; float* total; float* count; float* largest;
  char* scales;       // fp32: kept by the caller, or null
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
  if (c.rows * c.hidden > 1ll << 34 || c.vocab * c.hidden > 1ll << 34) return set_error(GRLHIP_ERR_UNSUPPORTED, w + "over 2^34 entries of hidden or weight");
  if (c.elem != GRLHIP_ELEM_F32 && c.elem != GRLHIP_ELEM_BF16 && c.elem != GRLHIP_ELEM_F16) return set_error(GRLHIP_ERR_INVALID, w + "unknown element type");
  if (a.reduction < 0 || a.reduction > 2) return set_error(GRLHIP_ERR_INVALID, w + "unknown reduction");
  if (!a.h || !a.w || !a.target) return set_error(GRLHIP_ERR_INVALID, w + "null hidden, weight or target");
  return 0;
}
template <class T>
View weight_piece(const Call& a, int64_t v0, int64_t cols) {
  return {(const char*)a.w + v0 * a.w0 * (int64_t)sizeof(T), a.w0, a.w1, (int)cols, (int)a.c.hidden};
}
View hidden_of(const Call& a) { return {a.h, a.h0, a.h1, (int)a.c.rows, (int)a.c.hidden}; }

Left left_of(const Call& a) { return {a.target, a.row_weight, a.ignore, a.bias}; }

// Where the magnitudes of a call are; hs, ws: fp32
struct Scales { Parts* parts; int *hs, *ws; };
template <class T>
Scales scales_of(const Call& a, const Layout& l) {
  char* at = a.scales ? a.scales : a.ws + l.scales;
  if (sizeof(T) != 4) return {(Parts*)at, nullptr, nullptr};
  return {(Parts*)at, (int*)(at + scales_of_hidden()), (int*)(at + scales_of_weight(a.c))};
}
template <class T>
void magnitudes_launch(const Call& a, const Scales& sc) {
  hipLaunchKernelGGL(k_ce_magnitudes<T>, dim3(HMAX + WMAX), dim3(MAG_THREADS), 0, a.stream, hidden_of(a), weight_piece<T>(a, 0, a.c.vocab), left_of(a), sc.parts,
                     sc.hs, sc.ws);
}
// Packs hidden (h null: not in this launch) and a weight piece, and takes the rows' gradients.
template <class T>
void pack_launch(const Call& a, Job h, Job w, Scale g, const Scales& sc, Scalars* s) {
  auto blocks = [](Job& j) { j.blocks = j.n || j.t ? (int)(up(j.v.cols, 64) / 64 * (up(j.v.rows, 64) / 64)) : 0; };
  blocks(h);
  blocks(w);
  const int all = h.blocks + w.blocks + g.blocks;
  if (all > 0) hipLaunchKernelGGL(k_ce_pack<T>, dim3(all), dim3(256), 0, a.stream, h, w, g, left_of(a), sc.parts, s, a.largest);
}

template <class K, class... A>
int tile_launch(K kernel, int64_t tiles, int threads, int lds, hipStream_t stream, const A&... args) {
  if (lds > 65536) LAUNCH_TRY(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(threads), lds, stream, args...);
  return 0;
}
#define BY_KIND(kind, call)            \
  ((kind) == 0 ? call(Ce64) : (kind) == 1 ? call(Ce128) : call(Ce256))

template <class T>
Logits logits_call(const Call& a, const Layout& l, const View& w, int64_t v0, const Scales& sc, Scalars* s) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  Logits g = {};
  g.h = l.pack_h ? Operand{a.ws + l.hp, l.kp * 2 * P} : Operand{(const char*)a.h, a.h0 * 2};
  g.w = l.pack_w ? Operand{a.ws + l.wp, l.kp * 2 * P} : Operand{(const char*)w.p, a.w0 * 2};
  g.bias = a.bias ? a.bias + v0 : nullptr;
  g.target = a.target;
  g.s = s;
  if (P == 2) {
    g.hs = sc.hs;
    g.ws = sc.ws + v0;
  }
  g.rows = (int)a.c.rows;
  g.v0 = (int)v0;
  g.cols = w.rows;
  g.nkb = (int)(l.kp * 2 * P / KBLOCK);
  return g;
}

template <class T> struct Operands { typedef T type; };
template <> struct Operands<float> { typedef _Float16 type; };

int join_blocks(const Grad& g) {
  const int64_t blocks = ((int64_t)g.n * g.m + 255) / 256;   // an entry a thread while that is few blocks: all parts of all entries in flight
  return (int)(blocks > 4096 ? 4096 : blocks);
}

// From the partials to losses, logsumexps and the total.
template <class T>
int finish(const Call& a, const Layout& l, int tiles) {
  const int64_t q = a.c.rows >= 2048 ? 8 : 64, blocks = (a.c.rows + 256 / q - 1) / (256 / q);   // few rows: more threads for each
  const Finish f{(float2*)(a.ws + l.part), (float*)(a.ws + l.picked), a.target, a.row_weight, a.ignore, (int)a.c.rows, tiles, (int)a.c.vocab, (int)blocks,
                 a.losses, a.lse, a.total ? (double*)(a.ws + l.sums) : nullptr, a.total, a.count, a.reduction};
  if (q == 8) hipLaunchKernelGGL(k_ce_finish<8>, dim3((unsigned)blocks), dim3(256), 0, a.stream, f);
  else hipLaunchKernelGGL(k_ce_finish<64>, dim3((unsigned)blocks), dim3(256), 0, a.stream, f);
  if (a.total) hipLaunchKernelGGL(k_ce_total, dim3(1), dim3(256), 0, a.stream, f);
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

template <class T>
int forward(const Call& a) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;
  const Layout l = layout_of(a.c, direct(a.h, a.h0, a.h1, a.c), direct(a.w, a.w0, a.w1, a.c), false, false);
  if (!a.ws || (int64_t)a.ws_bytes < l.bytes) return set_error(GRLHIP_ERR_WORKSPACE, "linear_ce_forward: workspace too small: need " + std::to_string(l.bytes));
  Scalars* s = (Scalars*)(a.ws + l.scalars);
  const Scales sc = scales_of<T>(a, l);
  if (P == 2) magnitudes_launch<T>(a, sc);
  const int side = SIDE[l.kind_z];
  const int64_t tn = up(a.c.rows, side) / side;
  int tiles = 0;
  for (int64_t v0 = 0; v0 < a.c.vocab; v0 += l.piece) {
    const View w = weight_piece<T>(a, v0, a.c.vocab - v0 < l.piece ? a.c.vocab - v0 : l.piece);
    Job jh{hidden_of(a), v0 == 0 && l.pack_h ? a.ws + l.hp : nullptr, l.kp, nullptr, 0, false, nullptr, sc.hs, 0};
    Job jw{w, l.pack_w ? a.ws + l.wp : nullptr, l.kp, nullptr, 0, false, a.bias ? a.bias + v0 : nullptr, P == 2 ? sc.ws + v0 : nullptr, 0};
    pack_launch<T>(a, jh, jw, Scale{}, sc, s);
    Logits g = logits_call<T>(a, l, w, v0, sc, s);
    g.part = (float2*)(a.ws + l.part) + (int64_t)tiles * a.c.rows;
    g.picked = (float*)(a.ws + l.picked);
    const int tm = (int)(up(w.rows, side) / side);
#define CALL(C) tile_launch(k_ce_forward<typename Operands<T>::type, P, C>, tm * tn, C::THREADS, C::LDS, a.stream, g, tm, (int)tn)
    if (const int rc = BY_KIND(l.kind_z, CALL)) return rc;
#undef CALL
    tiles += tm;
  }
  return finish<T>(a, l, tiles);
}

template <class T>
int backward(const Call& a) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1, N = GradPieces<T>::N;
  const Layout l = layout_of(a.c, direct(a.h, a.h0, a.h1, a.c), direct(a.w, a.w0, a.w1, a.c), true, a.gb != nullptr);
  if (!a.ws || (int64_t)a.ws_bytes < l.bytes) return set_error(GRLHIP_ERR_WORKSPACE, "linear_ce_backward: workspace too small: need " + std::to_string(l.bytes));
  Scalars* s = (Scalars*)(a.ws + l.scalars);
  const Scales sc = scales_of<T>(a, l);
  if (!__is_same(T, _Float16) && !a.scales) magnitudes_launch<T>(a, sc);   // the forward call's, if the caller kept them
  float* scale = (float*)(a.ws + l.scale);
  const int side = SIDE[l.kind_z];
  const int64_t tn = up(a.c.rows, side) / side;
  for (int64_t v0 = 0; v0 < a.c.vocab; v0 += l.piece) {
    const bool first = v0 == 0, last = v0 + l.piece >= a.c.vocab;
    const int64_t cols = last ? a.c.vocab - v0 : l.piece, vp = up(cols, 64);
    const View w = weight_piece<T>(a, v0, cols);
    const Job jh{hidden_of(a), first && l.pack_h ? a.ws + l.hp : nullptr, l.kp, first && a.gw ? a.ws + l.ht : nullptr, l.np, true, nullptr, sc.hs, 0};
    const Job jw{w, l.pack_w ? a.ws + l.wp : nullptr, l.kp, a.gh ? a.ws + l.wt : nullptr, vp, false, a.bias ? a.bias + v0 : nullptr, P == 2 ? sc.ws + v0 : nullptr, 0};
    int64_t gblocks = (a.c.rows + 255) / 256;
    if (gblocks > GMAX) gblocks = GMAX;
    const Scale rows{a.grad, a.grad_stride, a.count, (int)a.c.rows, (int)a.c.vocab, a.reduction, first ? (int)gblocks : 0, scale};
    pack_launch<T>(a, jh, jw, rows, sc, s);

    Logits g = logits_call<T>(a, l, w, v0, sc, s);
    g.lse = a.lse;
    g.scale = scale;
    g.d = a.ws + l.d;
    g.d_cols = vp;
    g.dt = a.ws + l.dt;
    g.dt_cols = l.np;
    g.bpart = a.gb ? (float*)(a.ws + l.bpart) : nullptr;
    const int tm = (int)(up(cols, side) / side);
#define CALL(C) tile_launch(k_ce_d<typename Operands<T>::type, P, N, C>, tm * tn, C::THREADS, C::LDS, a.stream, g, tm, (int)tn)
    if (const int rc = BY_KIND(l.kind_z, CALL)) return rc;
#undef CALL

    Join j = {};
    Grad &gh = j.both.g[0], &gw = j.both.g[1];
    j.both.s = s;
    if (a.gh) {
      gh.a = {a.ws + l.wt, vp * 2 * N};
      gh.b = {a.ws + l.d, vp * 2 * N};
      gh.m = (int)a.c.hidden;
      gh.n = (int)a.c.rows;
      gh.nkb = (int)(vp * 2 * N / KBLOCK);
      gh.split = l.split_h;
      gh.tiles = (int)tiles_of(gh.m, gh.n, l.kind_g) * gh.split;
      gh.slots = l.hslots ? (float*)(a.ws + l.hslots) : nullptr;
      gh.add = !first;
      gh.out = a.gh;
      gh.scale = scale;
      gh.by_w = 1;
      if (gh.slots && last) j.blocks[0] = join_blocks(gh);
    }
    if (a.gw) {
      gw.a = {a.ws + l.ht, l.np * 2 * N};
      gw.b = {a.ws + l.dt, l.np * 2 * N};
      gw.m = (int)a.c.hidden;
      gw.n = (int)cols;
      gw.nkb = (int)(l.np * 2 * N / KBLOCK);
      gw.split = l.split_w;
      gw.tiles = (int)tiles_of(gw.m, gw.n, l.kind_g) * gw.split;
      gw.slots = l.wslots ? (float*)(a.ws + l.wslots) : nullptr;
      gw.out = (T*)a.gw + v0 * a.c.hidden;
      if (gw.slots) j.blocks[1] = join_blocks(gw);
    }
    if (gh.tiles + gw.tiles > 0) {
#define CALL(C) tile_launch(k_ce_grad<T, GradPieces<T>::P, C>, gh.tiles + gw.tiles, C::THREADS, C::LDS, a.stream, j.both)
      if (const int rc = BY_KIND(l.kind_g, CALL)) return rc;
#undef CALL
    }
    int blocks = j.blocks[0] + j.blocks[1];
    if (a.gb) {
      j.bpart = g.bpart;
      j.btiles = (int)tn;
      j.cols = (int)cols;
      j.gb = a.gb + v0;
      blocks += (int)((cols + 255) / 256);
    }
    if (blocks > 0) hipLaunchKernelGGL(k_ce_join<T>, dim3(blocks), dim3(256), 0, a.stream, j);
  }
  LAUNCH_TRY(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace grlhip

using namespace grlhip;

extern "C" {

size_t grlhip_linear_ce_scales_bytes(int64_t rows, int64_t vocab) {
  return guarded_size([&]() -> size_t {
    if (rows < 1 || vocab < 1 || rows > MAX_ROWS || vocab > MAX_VOCAB) {
      set_error(GRLHIP_ERR_UNSUPPORTED, "linear_ce: rows and vocabulary must be 1 to 2^20 and 2^21");
      return 0;
    }
    return (size_t)scales_bytes(Shape{rows, 1, vocab, GRLHIP_ELEM_F32});
  });
}

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

int grlhip_linear_ce_tiles(int64_t rows, int64_t features, int64_t vocab, int elem, int32_t* kinds) {
  return guarded([&]() -> int {
    Call a = {};
    a.c = {rows, features, vocab, elem};
    a.h = a.w = kinds;
    a.target = (const int64_t*)kinds;
    if (const int rc = check("linear_ce_tiles", a)) return rc;
    const bool in_place = direct(nullptr, features, 1, a.c);
    const Layout forward = layout_of(a.c, in_place, in_place, false, false), backward = layout_of(a.c, in_place, in_place, true, true);
    kinds[0] = forward.kind_z;
    kinds[1] = backward.kind_z;
    kinds[2] = backward.kind_g;
    return 0;
  });
}

int grlhip_linear_ce_forward(const void* hidden, const int64_t* hidden_strides, const void* weight, const int64_t* weight_strides, const float* bias,
                             const int64_t* target, int64_t ignore_index, const float* row_weight, int64_t rows, int64_t features, int64_t vocab,
                             int elem, int reduction, float* losses, float* lse, float* total, float* count, float* largest, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    Call a = {};
    const bool kept = (elem & GRLHIP_ELEM_SCALES) && largest;
    if (elem == (GRLHIP_ELEM_F32 | GRLHIP_ELEM_SCALES)) elem = GRLHIP_ELEM_F32;
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
    a.largest = kept ? nullptr : largest;
    a.scales = kept ? (char*)largest : nullptr;
    a.ws = (char*)workspace;
    a.ws_bytes = workspace_bytes;
    a.stream = (hipStream_t)stream;
    if (const int rc = check("linear_ce_forward", a)) return rc;
    if (!losses) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: null losses");
    if (!total != !count || (!total && reduction != GRLHIP_REDUCE_NONE)) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: total and count go together, and may be NULL for GRLHIP_REDUCE_NONE only");
    if ((size_t)a.scales & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: the scales must be aligned to 256 bytes");
    if ((size_t)workspace & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_forward: the workspace must be aligned to 256 bytes");
    return elem == GRLHIP_ELEM_F32 ? forward<float>(a) : elem == GRLHIP_ELEM_BF16 ? forward<__bf16>(a) : forward<_Float16>(a);
  });
}

int grlhip_linear_ce_backward(const void* hidden, const int64_t* hidden_strides, const void* weight, const int64_t* weight_strides, const float* bias,
                              const int64_t* target, int64_t ignore_index, const float* row_weight, int64_t rows, int64_t features, int64_t vocab,
                              int elem, int reduction, const float* lse, const float* count, const float* largest, const float* grad, int64_t grad_stride,
                              void* grad_hidden, void* grad_weight, float* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    Call a = {};
    const bool kept = (elem & GRLHIP_ELEM_SCALES) && largest;
    if (elem == (GRLHIP_ELEM_F32 | GRLHIP_ELEM_SCALES)) elem = GRLHIP_ELEM_F32;
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
    a.scales = kept ? (char*)const_cast<float*>(largest) : nullptr;
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.gh = grad_hidden;
    a.gw = grad_weight;
    a.gb = grad_bias;
    a.ws = (char*)workspace;
    a.ws_bytes = workspace_bytes;
    a.stream = (hipStream_t)stream;
    if (const int rc = check("linear_ce_backward", a)) return rc;
    if (!lse || !grad || (!count && reduction == GRLHIP_REDUCE_MEAN)) return set_error(GRLHIP_ERR_INVALID, "linear_ce_backward: null lse, gradient or count");
    if ((size_t)a.scales & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_backward: the scales must be aligned to 256 bytes");
    if ((size_t)workspace & 255) return set_error(GRLHIP_ERR_INVALID, "linear_ce_backward: the workspace must be aligned to 256 bytes");
    if (!grad_hidden && !grad_weight && !grad_bias) return 0;
    return elem == GRLHIP_ELEM_F32 ? backward<float>(a) : elem == GRLHIP_ELEM_BF16 ? backward<__bf16>(a) : backward<_Float16>(a);
  });
}

}  // extern "C"
