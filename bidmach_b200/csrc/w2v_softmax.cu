// Softmax cross entropy over the whole vocabulary, in pieces, without keeping the logits.
//
//   l_nv = h_n . w_v     lse_n = log sum_v exp l_nv     loss_n = sum_j (lse_n - l_{n, y_nj})
//   d_nv = g_n (k_n exp(l_nv - lse_n) - #{j : y_nj = v})     dH = d W     dW = d^T H
//
// with y_n the targets of row n that lie in the vocabulary and k_n their number (none is fine: loss
// and gradient are zero).  For N rows, V words and D columns the loss costs 2 N V D operations, the
// gradients 4 N V D and, since no logits are kept, the logits' 2 N V D again.
//
// More than kFewRows rows: the tensor cores.  One kernel computes tiles of 128 x 256 of a product
// whose operands TMA brings into shared memory (a producer warp, a warp that issues tcgen05.mma, eight
// warps that read the finished tile from tensor memory while the next one is computed in the other
// half of it).  What the eight warps do with a tile is the difference between its three uses:
//   kLogits  the running maximum and sum of exponentials of each row over the tile's columns: 8
//            bytes a row and half tile go to memory, a small kernel joins them;
//   kProbs   d of a row block and a piece of the vocabulary, in 16 bits, small enough to stay in L2;
//   kGrad    dH and dW from that piece, accumulated in fp32 over the pieces (row blocks).
// fp32 operands are split into two fp16 numbers (after a common power-of-two scale), x = hi + lo, and
// hi hi + hi lo + lo hi computed: 22 bits of each operand.  Products of fp16 or bf16 operands are exact in
// the fp32 accumulators.  d is rounded once to the operands' type (fp32: to hi + lo with lo scaled by
// 2^11, so that small probabilities keep their bits; the operand it meets carries the 2^-11).
//
// Up to kFewRows rows the bound is reading W once: a kernel with the rows in shared memory, W straight
// from memory in its own type, plain fp32 arithmetic.
#include <cuda.h>
#include <math.h>

#include <algorithm>

#include "../../include/bidmach_b200.h"
#include "w2v_device.cuh"
#include "w2v_internal.h"
#include "w2v_tcgen05.cuh"
#include "w2v_types.cuh"

namespace {

using namespace w2v;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFewRows = 8;
constexpr int kMaxDim = 4096;

// A row's sum of exponentials as 2^m * s, with exponents in units of log2 e.
struct Part {
  float m, s;
};
__device__ __forceinline__ Part join(Part a, Part b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return Part{m, a.s + b.s};
  return Part{m, a.s * exp2f(a.m - m) + b.s * exp2f(b.m - m)};
}

// What the gradient needs of a row: d = exp2(l log2e - lse2) * coef - (targets here) * g.
struct RowCoef {
  float lse2, coef, g;
  unsigned hits;   // chunks of 32 columns of the tile at hand that hold a target (only in shared memory)
};

// Found on the device before a product: largest magnitudes (as bits) of H, W and g_n k_n.
struct Scalars {
  unsigned h, w, g;
};

// 2^e such that the largest magnitude times it lies in [2^top, 2^(top+1)); 1 for zero and non-finite.
__device__ __forceinline__ int scale_exp(unsigned bits, int top) {
  if (bits == 0 || bits >= 0x7f800000u) return 0;
  const int e = bits >= 0x800000u ? (int)(bits >> 23) - 127 : -118 - __clz((int)bits);
  return min(100, max(-100, top - e));
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
constexpr int kOperandTop = 13, kProbTop = 14;

// ---------------------------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------------------------
constexpr int kFewThreads = 256;
constexpr int kFewWords = 4;   // words a warp works on at a time

__host__ __device__ __forceinline__ int few_steps(int dim) { return (dim + 255) / 256; }

// Sums each of M totals over the warp; lane l ends with total l / (32 / M).
template <int M>
__device__ __forceinline__ float spread_totals(float (&x)[M]) {
  const int lane = threadIdx.x & 31;
  int step = 16;
#pragma unroll
  for (int cnt = M; cnt > 1; cnt >>= 1, step >>= 1) {
    const bool up = lane & step;
#pragma unroll
    for (int i = 0; i < cnt / 2; i++) {
      const float keep = up ? x[i + cnt / 2] : x[i], give = up ? x[i] : x[i + cnt / 2];
      x[i] = keep + __shfl_xor_sync(kFullMask, give, step);
    }
  }
  float t = x[0];
#pragma unroll
  for (int s = 32 / M / 2; s > 0; s >>= 1) t += __shfl_xor_sync(kFullMask, t, s);
  return t;
}

// The rows of H in shared memory as [row][step][half][lane] float4: both halves of a lane's 8 columns
// are read without bank conflicts.
template <typename T, int RB>
__device__ __forceinline__ void stage_rows(const T *h, int64_t ldh, int rows, int dim, float *sh) {
  const int steps = few_steps(dim);
  for (int i = threadIdx.x; i < RB * steps * 256; i += kFewThreads) {
    const int r = i / (steps * 256), c = i % (steps * 256);
    const int step = c / 256, lane = c % 256 / 8, half = c % 8 / 4, e = c % 4;
    const float x = r < rows && c < dim ? to_float(h[(int64_t)r * ldh + c]) : 0.f;
    sh[((((r * steps + step) * 2 + half) * 32) + lane) * 4 + e] = x;
  }
}
__device__ __forceinline__ void staged8(const float *sh, int steps, int r, int step, int lane, float (&x)[8]) {
  const float4 *p = reinterpret_cast<const float4 *>(sh) + (r * steps + step) * 64 + lane;
  const float4 a = p[0], b = p[32];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// Logits of kFewWords words against RB rows; lane l ends with word l / (32 / M) / RB, row ... % RB.
template <typename T, int RB>
__device__ __forceinline__ float few_logits(const T *w, int64_t ldw, int64_t v0, int64_t vocab, int dim, bool wide,
                                            const float *sh) {
  const int lane = threadIdx.x & 31, steps = few_steps(dim);
  float acc[kFewWords * RB];
#pragma unroll
  for (int i = 0; i < kFewWords * RB; i++) acc[i] = 0.f;
  for (int s = 0; s < steps; s++) {
    const int col = s * 256 + lane * 8, have = min(8, max(0, dim - col));
    float x[kFewWords][8];
#pragma unroll
    for (int q = 0; q < kFewWords; q++) {
      const int n = v0 + q < vocab ? have : 0;
      const T *p = w + (v0 + q) * ldw + col;
      if (wide && n == 8) load8(p, x[q]);
      else load_some(p, n, x[q]);
    }
#pragma unroll
    for (int r = 0; r < RB; r++) {
      float h[8];
      staged8(sh, steps, r, s, lane, h);
#pragma unroll
      for (int q = 0; q < kFewWords; q++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[q * RB + r] = fmaf(x[q][e], h[e], acc[q * RB + r]);
    }
  }
  return spread_totals<kFewWords * RB>(acc);
}

template <typename T, int RB>
__global__ void __launch_bounds__(kFewThreads) few_loss_kernel(const T *h, int64_t ldh, int rows, const T *w, int64_t ldw,
                                                               int64_t vocab, int dim, bool wide, Part *parts) {
  extern __shared__ __align__(16) float sh[];
  __shared__ Part sums[kFewThreads / 32][RB];
  stage_rows<T, RB>(h, ldh, rows, dim, sh);
  __syncthreads();
  constexpr int M = kFewWords * RB, each = 32 / M;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int mine = lane / each, row = mine % RB;
  Part p{-INFINITY, 0.f};
  const int64_t stride = (int64_t)gridDim.x * (kFewThreads / 32) * kFewWords;
  for (int64_t v = ((int64_t)blockIdx.x * (kFewThreads / 32) + warp) * kFewWords; v < vocab; v += stride) {
    const float l = few_logits<T, RB>(w, ldw, v, vocab, dim, wide, sh) * kLog2e;
    if (v + mine / RB < vocab && lane % each == 0) {
      const float m = fmaxf(p.m, l);   // a NaN logit reaches the sum below
      p.s = m == -INFINITY ? p.s : p.s * exp2f(p.m - m) + exp2f(l - m);
      if (isnan(l)) p.s = l;
      p.m = m;
    }
  }
#pragma unroll
  for (int s = 16; s >= RB * each; s >>= 1)
    p = join(p, Part{__shfl_xor_sync(kFullMask, p.m, s), __shfl_xor_sync(kFullMask, p.s, s)});
  if (lane % each == 0 && lane < RB * each) sums[warp][row] = p;
  __syncthreads();
  if (threadIdx.x < rows) {
    Part t = sums[0][threadIdx.x];
    for (int k = 1; k < kFewThreads / 32; k++) t = join(t, sums[k][threadIdx.x]);
    parts[(int64_t)blockIdx.x * rows + threadIdx.x] = t;
  }
}

// dW of a word directly, and d itself (RB floats a word) for the pass that sums dH.
template <typename T, int RB>
__global__ void __launch_bounds__(kFewThreads) few_grad_kernel(const T *h, int64_t ldh, int rows, const T *w, int64_t ldw,
                                                               int64_t vocab, int dim, bool wide, const int *targets,
                                                               int labels, const float *lse, const float *gloss,
                                                               int64_t ldg, T *dw, int64_t lddw, bool wide_out,
                                                               float *d) {
  extern __shared__ __align__(16) float sh[];
  __shared__ float lse_s[RB], g_s[RB], k_s[RB];
  __shared__ __align__(16) float d_s[kFewThreads / 32][RB][kFewWords];
  stage_rows<T, RB>(h, ldh, rows, dim, sh);
  if (threadIdx.x < RB) {
    const int r = threadIdx.x;
    int k = 0;
    if (r < rows)
      for (int j = 0; j < labels; j++) {
        const int y = targets[(int64_t)r * labels + j];
        k += y >= 0 && y < vocab;
      }
    lse_s[r] = r < rows ? lse[r] : 0.f;
    g_s[r] = r < rows ? gloss[r * ldg] : 0.f;
    k_s[r] = (float)k;
  }
  __syncthreads();
  constexpr int M = kFewWords * RB, each = 32 / M;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, steps = few_steps(dim);
  const int mine = lane / each, row = mine % RB, word = mine / RB;
  const int64_t stride = (int64_t)gridDim.x * (kFewThreads / 32) * kFewWords;
  for (int64_t v = ((int64_t)blockIdx.x * (kFewThreads / 32) + warp) * kFewWords; v < vocab; v += stride) {
    const float l = few_logits<T, RB>(w, ldw, v, vocab, dim, wide, sh);
    float x = 0.f;
    if (k_s[row] > 0.f) {
      x = k_s[row] * expf(l - lse_s[row]);
      for (int j = 0; j < labels; j++) x -= targets[(int64_t)row * labels + j] == v + word ? 1.f : 0.f;
      x *= g_s[row];
    }
    if (lane % each == 0) {
      d_s[warp][row][word] = x;
      if (v + word < vocab) d[(v + word) * RB + row] = x;
    }
    __syncwarp();
    for (int s = 0; s < steps; s++) {
      const int col = s * 256 + lane * 8, have = min(8, max(0, dim - col));
      float acc[kFewWords][8] = {};
#pragma unroll
      for (int r = 0; r < RB; r++) {
        float hx[8];
        staged8(sh, steps, r, s, lane, hx);
        const float4 dv = *reinterpret_cast<const float4 *>(d_s[warp][r]);
        const float dq[4] = {dv.x, dv.y, dv.z, dv.w};
#pragma unroll
        for (int q = 0; q < kFewWords; q++)
#pragma unroll
          for (int e = 0; e < 8; e++) acc[q][e] = fmaf(dq[q], hx[e], acc[q][e]);
      }
#pragma unroll
      for (int q = 0; q < kFewWords; q++) {
        if (v + q >= vocab) break;
        T *p = dw + (v + q) * lddw + col;
        if (wide_out && have == 8) store8(p, acc[q]);
        else store_some(p, have, acc[q]);
      }
    }
    __syncwarp();
  }
}

// dH of few rows: a block sums d_nv w_v over a range of words, a thread a column.
template <typename T, int RB>
__global__ void __launch_bounds__(kFewThreads) few_dh_kernel(const T *w, int64_t ldw, int64_t vocab, int dim,
                                                             const float *d, float *parts) {
  const int64_t each = (vocab + gridDim.x - 1) / gridDim.x;
  const int64_t lo = blockIdx.x * each, hi = min(vocab, lo + each);
  for (int c = blockIdx.y * kFewThreads + threadIdx.x; c < dim; c += gridDim.y * kFewThreads) {
    float acc[RB] = {};
    int64_t v = lo;
    for (; v + 4 <= hi; v += 4) {
      float x[4];
#pragma unroll
      for (int q = 0; q < 4; q++) x[q] = to_float(w[(v + q) * ldw + c]);
#pragma unroll
      for (int q = 0; q < 4; q++)
#pragma unroll
        for (int r = 0; r < RB; r++) acc[r] = fmaf(d[(v + q) * RB + r], x[q], acc[r]);
    }
    for (; v < hi; v++) {
      const float x = to_float(w[v * ldw + c]);
#pragma unroll
      for (int r = 0; r < RB; r++) acc[r] = fmaf(d[v * RB + r], x, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < RB; r++) parts[((int64_t)blockIdx.x * RB + r) * dim + c] = acc[r];
  }
}

// What a gradient's sums have to be multiplied with: the powers of two that d and the other operand
// were scaled by, and the one factor for all rows where there is one.
struct Rescale {
  const Scalars *sc;   // null: 1
  const float *gloss;  // null: 1
  int operand;         // 0: none scaled, 1: W, 2: H
};
__device__ __forceinline__ float rescale_of(const Rescale &r) {
  float x = r.gloss ? *r.gloss : 1.f;
  if (r.sc) {
    x *= pow2(-scale_exp(r.sc->g, kProbTop));
    if (r.operand) x *= pow2(-scale_exp(r.operand == 1 ? r.sc->w : r.sc->h, kOperandTop));
  }
  return x;
}

// out[r][c] = factor * sum over slabs, in their order; a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) slabs_kernel(const float *slabs, int count, int64_t slab, int64_t lds, int64_t rows,
                                                    int dim, T *out, int64_t ldo, bool wide, const Rescale rescale) {
  const float f = rescale_of(rescale);
  const int lane = threadIdx.x & 31;
  const int cols = (dim + 255) / 256;
  const int64_t stride = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; i < rows * cols; i += stride) {
    const int64_t r = cols == 1 ? i : i / cols;
    const int c = (int)(i - r * cols) * 256 + lane * 8, have = min(8, dim - c);
    if (have <= 0) continue;
    const float *p = slabs + r * lds + c;
    float x[8];
    if (wide) load8(p, x);
    else load_some(p, have, x);
    for (int k = 1; k < count; k += 4) {
      float y[4][8];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (wide && k + j < count) load8(p + (k + j) * slab, y[j]);
        else load_some(p + (k + j) * slab, k + j < count ? have : 0, y[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] += y[j][e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= f;
    T *to = out + r * ldo + c;
    if (have == 8 && reinterpret_cast<uintptr_t>(to) % (8 * sizeof(T)) == 0) store8(to, x);
    else store_some(to, have, x);
  }
}

// ---------------------------------------------------------------------------------------------
// Joining the parts of a row and the targets' logits
// ---------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 8;

// parts[k][row], row < ldp.  While the parts are read a warp is eight rows times four parts (the rows
// of a part lie side by side); then a warp is a row, two targets' dot products at a time.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) loss_join_kernel(const Part *parts, int count, int64_t ldp, int rows,
                                                                 const T *h, int64_t ldh, const T *w, int64_t ldw,
                                                                 int64_t vocab, int dim, bool wide, const int *targets,
                                                                 int labels, float *loss, float *lse) {
  __shared__ Part sums[kJoinThreads / 32][kJoinRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, warps = kJoinThreads / 32;
  const int r0 = blockIdx.x * kJoinRows, here = min(kJoinRows, rows - r0);
  Part p{-INFINITY, 0.f};
  const int row = lane % kJoinRows;
  constexpr int step = kJoinThreads / kJoinRows;
  if (row < here)
    for (int k = threadIdx.x / kJoinRows; k < count; k += step * 4) {
      Part x[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        x[j] = k + j * step < count ? parts[(int64_t)(k + j * step) * ldp + r0 + row] : Part{-INFINITY, 0.f};
#pragma unroll
      for (int j = 0; j < 4; j++) p = join(p, x[j]);
    }
#pragma unroll
  for (int s = 16; s >= kJoinRows; s >>= 1)
    p = join(p, Part{__shfl_xor_sync(kFullMask, p.m, s), __shfl_xor_sync(kFullMask, p.s, s)});
  if (lane < kJoinRows) sums[warp][lane] = p;
  __syncthreads();
  if (warp >= here) return;
  p = sums[0][warp];
#pragma unroll
  for (int k = 1; k < warps; k++) p = join(p, sums[k][warp]);
  const float z = (p.m + log2f(p.s)) / kLog2e;
  const int64_t n = r0 + warp;
  const int *y = targets + n * labels;
  const T *hr = h + n * ldh;
  float sum = 0.f;
  for (int j = 0; j < labels; j += 2) {
    int at[2];
    float x[2] = {0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 2; q++) at[q] = j + q < labels ? y[j + q] : -1;
    for (int c = lane * 8; c < dim; c += 256) {
      const int have = min(8, dim - c);
      float a[8], b[2][8];
      if (wide && have == 8) load8(hr + c, a);
      else load_some(hr + c, have, a);
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const bool there = at[q] >= 0 && at[q] < vocab;
        const T *wr = w + (there ? (int64_t)at[q] : 0) * ldw + c;
        if (wide && there && have == 8) load8(wr, b[q]);
        else load_some(wr, there ? have : 0, b[q]);
      }
#pragma unroll
      for (int q = 0; q < 2; q++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[q] = fmaf(a[e], b[q][e], x[q]);
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const float l = warp_sum(x[q]);
      if (at[q] >= 0 && at[q] < vocab) sum += z - l;
    }
  }
  if (lane == 0) {
    lse[n] = z;
    loss[n] = sum;
  }
}

// ---------------------------------------------------------------------------------------------
// Preparing operands
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int valid_targets(const int *y, int labels, int64_t vocab) {
  int k = 0;
  for (int j = 0; j < labels; j++) k += y[j] >= 0 && y[j] < vocab;
  return k;
}

struct Source {
  const void *p;
  int64_t ld, rows;
};

__device__ __forceinline__ void block_max(unsigned top, unsigned *to) {
  top = __reduce_max_sync(kFullMask, top);
  if ((threadIdx.x & 31) == 0 && top) atomicMax(to, top);
}

// Largest magnitudes of fp32 operands (z = 0: H, 1: W) and of the rows' g_n k_n (z = 2).
__global__ void __launch_bounds__(256) amax_kernel(Source h, Source w, int dim, const float *gloss, int64_t ldg,
                                                   const int *targets, int labels, int64_t vocab, Scalars *sc) {
  unsigned top = 0;
  if (blockIdx.z < 2) {
    const Source s = blockIdx.z == 0 ? h : w;
    if (!s.p) return;
    const float *a = static_cast<const float *>(s.p);
    const int lane = threadIdx.x & 31;
    const bool wide = reinterpret_cast<uintptr_t>(a) % 32 == 0 && s.ld % 8 == 0;
    for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < s.rows; r += (int64_t)gridDim.x * 8)
      for (int c = lane * 8; c < dim; c += 256) {
        const int have = min(8, dim - c);
        float x[8];
        if (wide && have == 8) load8(a + r * s.ld + c, x);
        else load_some(a + r * s.ld + c, have, x);
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      }
    block_max(top, blockIdx.z == 0 ? &sc->h : &sc->w);
  } else if (gloss) {
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < h.rows; n += (int64_t)gridDim.x * 256) {
      const int k = valid_targets(targets + n * labels, labels, vocab);
      if (k) top = max(top, __float_as_uint((ldg ? gloss[n] : 1.f) * (float)k) & 0x7fffffffu);
    }
    block_max(top, &sc->g);
  }
}

// Rows of T as rows of `width` (a multiple of 64) 16-bit elements, zeros behind the last column;
// fp32 as `parts` of them: hi, lo, and hi 2^-11.
template <typename T>
__device__ __forceinline__ void stage_row(const T *src, int dim, T *dst, int width, int, float) {
  for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    float x[8];
    load_some(src + c, min(8, max(0, dim - c)), x);
    store8(dst + c, x);
  }
}
template <>
__device__ __forceinline__ void stage_row<float>(const float *src, int dim, float *to, int width, int parts,
                                                 float scale) {
  __half *dst = reinterpret_cast<__half *>(to);
  for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    const int have = min(8, max(0, dim - c));
    float x[8], lo[8], small[8];
    if (have == 8 && reinterpret_cast<uintptr_t>(src + c) % 32 == 0) load8(src + c, x);
    else load_some(src + c, have, x);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float y = x[e] * scale;
      x[e] = __half2float(__float2half_rn(y));
      lo[e] = isfinite(x[e]) ? y - x[e] : 0.f;
      small[e] = x[e] * 0x1p-11f;
    }
    store8(dst + c, x);
    store8(dst + width + c, lo);
    if (parts == 3) store8(dst + 2 * width + c, small);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) stage_kernel(Source h, Source w, int dim, void *hs, void *ws, int width, int parts,
                                                    const Scalars *sc) {
  const Source s = blockIdx.z == 0 ? h : w;
  void *to = blockIdx.z == 0 ? hs : ws;
  if (!to) return;
  constexpr bool split = sizeof(T) == 4;
  const float scale = split ? pow2(scale_exp(blockIdx.z == 0 ? sc->h : sc->w, kOperandTop)) : 1.f;
  for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < s.rows; r += (int64_t)gridDim.x * 8) {
    char *dst = static_cast<char *>(to) + r * width * parts * 2;
    stage_row<T>(static_cast<const T *>(s.p) + r * s.ld, dim, reinterpret_cast<T *>(dst), width, parts, scale);
  }
}

__global__ void __launch_bounds__(256) row_coef_kernel(const float *lse, const float *gloss, int64_t ldg,
                                                       const int *targets, int labels, int64_t vocab, int64_t rows,
                                                       const Scalars *sc, RowCoef *out) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= rows) return;
  // one factor for all rows is left to the end: the targets' -1 then has no rounding in d
  const float g = (ldg ? gloss[n] : 1.f) * pow2(scale_exp(sc->g, kProbTop));
  const int k = valid_targets(targets + n * labels, labels, vocab);
  // lse log2e to twice the precision: what the rounded exponent lacks goes into the factor
  const float hi = lse[n] * kLog2e, lo = fmaf(lse[n], kLog2e, -hi);
  // a row without targets: exp2(l - inf) = 0, times 0
  out[n] = k ? RowCoef{hi, g * (float)k * exp2f(-lo), g, 0u} : RowCoef{INFINITY, 0.f, 0.f, 0u};
}

// ---------------------------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------------------------
constexpr int kM = 128, kN = 256, kK = 64, kStages = 6;   // rows of each of a pair's CTAs, columns of both
constexpr int kPairM = 2 * kM;
constexpr int kBytesA = kM * kK * 2, kBytesB = kN / 2 * kK * 2;
constexpr int kMmaThreads = 384;   // producer, issuer, two idle warps, eight that read the tiles
constexpr int kSmem = kStages * (kBytesA + kBytesB) + 1024;

enum Use { kLogits, kProbs, kGrad, kGradSegments };
__host__ __device__ constexpr bool is_grad(Use u) { return u == kGrad || u == kGradSegments; }

struct Product {
  CUtensorMap a, b;
  int mt, nt, ntile;      // tiles of kPairM rows, columns a tile (a multiple of 32)
  int splits, kblocks;    // of 64, over all splits, for one pair of parts
  int pairs, pa[3], pb[3];// offsets of the parts that are multiplied, the smaller products first
  int k16;                // steps of 16 in the last block of K
  int a_mn, b_mn;         // operands whose rows run along K
  int a_y, b_y;           // first row of each in its matrix
  int bf16;
  // logits and probabilities
  const Scalars *sc;
  int split_scale;        // operands carry the scales of sc
  int64_t vocab;
  int word0;              // word of the first column
  int rows;               // rows that exist
  Part *parts;
  int64_t ldparts;
  const RowCoef *coef;
  const int *targets;
  int labels;
  uint16_t *probs;        // d in strips of 64 columns: [part][strip][row][64]
  int strip;              // rows of a strip
  int64_t prob_lo;        // offset of the second part, 0 for none
  // gradients
  int segment;            // blocks of K that are accumulated in tensor memory at a time
  float *scratch;         // kM x kN for each block
  float *acc;             // [splits][acc_rows][ldacc]
  int64_t acc_slab, ldacc;
  int add;                // to what is there already
  void *out;              // not null: the finished gradient goes here, not to acc
  int64_t ldout;
  int out_type, out_wide, dim;
  Rescale rescale;
};

__device__ __forceinline__ void store32(void *a, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t halves(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
  }
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}

// 32 values to 16 bits at `to` (32-byte aligned), and what that lacks, times 2^11, `lo` elements on.
template <bool BF16, bool LO>
__device__ __forceinline__ void store_probs(uint16_t *to, int64_t lo, const float (&x)[32]) {
#pragma unroll
  for (int b = 0; b < 2; b++) {
    uint32_t r[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float u = x[b * 16 + 2 * i], v = x[b * 16 + 2 * i + 1];
      r[i] = halves<BF16>(u, v);
      if (LO) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
        s[i] = halves<false>((u - f.x) * 2048.f, (v - f.y) * 2048.f);
      }
    }
    store32(to + b * 16, r);
    if (LO) store32(to + lo + b * 16, s);
  }
}

template <Use USE>
__device__ __forceinline__ void tile_of(const Product &p, int t, int &m, int &n, int &k) {
  if (is_grad(USE)) {   // blocks that run together share a strip of d
    n = t % p.nt;
    m = t / p.nt % p.mt;
    k = t / (p.nt * p.mt);
  } else {              // ... and a few tiles of W, against all rows
    m = t % p.mt;
    n = t / p.mt;
    k = 0;
  }
}

template <typename T>
__device__ __forceinline__ void put_typed(T *to, bool wide, int have, const float (&v)[8]) {
  if (wide && have == 8) store8(to, v);
  else store_some(to, have, v);
}

// Eight columns of a gradient's tile, from column `col` of it.
__device__ __forceinline__ void put_grad(const Product &p, int64_t r, int n, int k, int col, const float *x, float factor) {
  const int at = n * p.ntile + col;
  if (r >= p.rows || col >= p.ntile || at >= p.dim) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = x[e];
  if (p.out) {
    const int have = min(8, p.dim - at);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] *= factor;
    const int64_t to = r * p.ldout + at;
    if (p.out_type == W2V_F32) put_typed(static_cast<float *>(p.out) + to, p.out_wide, have, v);
    else if (p.out_type == W2V_BF16) put_typed(static_cast<__nv_bfloat16 *>(p.out) + to, p.out_wide, have, v);
    else put_typed(static_cast<__half *>(p.out) + to, p.out_wide, have, v);
    return;
  }
  float *to = p.acc + k * p.acc_slab + r * p.ldacc + at;
  if (p.add) {
    float old[8];
    load8(to, old);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += old[e];
  }
  store8(to, v);
}

template <Use USE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmaThreads, 1) product_kernel(const __grid_constant__ Product p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  __shared__ u64 full[kStages], empty[kStages], tfull[2], tempty[2], done, hfull[2], hempty[2];
  __shared__ RowCoef coef_s[2][USE == kProbs ? kM : 1];
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up_s;
  volatile int *gave_up = &gave_up_s;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 16);   // the warps that read tiles, of both CTAs
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&hfull[i], 2);
      mbar_init(&hempty[i], 8);
    }
    mbar_init(&done, 1);
    gave_up_s = 0;
    mbar_init_fence();
    async_proxy_fence();
  }
  if (warp == 2) tmem_alloc(&tmem_at, 512);
  tmem_before_sync();
  cluster_sync();
  tmem_after_sync();
  const uint32_t tmem = tmem_at;
  const int rank = (int)cluster_rank(), pair = blockIdx.x / 2, npairs = gridDim.x / 2;
  const int tiles = p.mt * p.nt * p.splits;
  // blocks of K that a split starts with: every split has one at least (splits <= kblocks)
  auto first_k = [&](int k) { return (int)((int64_t)k * p.kblocks / p.splits); };

  if (warp == 0) {
    if (elected()) {
      int it = 0;
      bool ok = true;
      // each CTA brings its own rows of A and half of the columns of B; the leader counts both
      const int half_n = p.ntile / 2, groups_b = (half_n + 63) / 64;
      const unsigned bytes = 2 * (kBytesA + (is_grad(USE) ? groups_b * 8192 : kBytesB));
      for (int t = pair; ok && t < tiles; t += npairs) {
        int m, n, k;
        tile_of<USE>(p, t, m, n, k);
        const int kend = first_k(k + 1);
        for (int k0 = first_k(k); ok && k0 < kend; k0 += p.segment)
        for (int q = 0; ok && q < p.pairs; q++)
          for (int kb = k0; kb < min(kend, k0 + p.segment); kb++, it++) {
            const int s = it % kStages;
            if (!mbar_wait(&empty[s], (it / kStages + 1) & 1, gave_up)) {
              ok = false;
              break;
            }
            const uint32_t bar = in_leader(&full[s]);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
            unsigned char *sa = smem + s * (kBytesA + kBytesB), *sb = sa + kBytesA;
            const int mrow = m * kPairM + rank * kM;
            if (!is_grad(USE)) {
              tma_load_2d(sa, &p.a, p.pa[q] + kb * kK, p.a_y + mrow, bar);
              tma_load_2d(sb, &p.b, p.pb[q] + kb * kK, p.b_y + n * kN + rank * (kN / 2), bar);
            } else {
              if (p.a_mn) {   // d transposed: 64 rows of two strips
                for (int g = 0; g < 2; g++)
                  tma_load_2d(sa + g * 8192, &p.a, 0, p.pa[q] + (mrow / 64 + g) * p.strip + kb * kK, bar);
              } else {        // 128 rows of a strip
                tma_load_2d(sa, &p.a, 0, p.pa[q] + kb * p.strip + mrow, bar);
              }
              for (int g = 0; g < groups_b; g++)
                tma_load_2d(sb + g * 8192, &p.b, p.pb[q] + n * p.ntile + rank * half_n + g * 64, p.b_y + kb * kK, bar);
            }
          }
      }
      if (!ok) {   // copies in flight still write into this block's shared memory
        int none = 0;
        if (rank == 0)
          for (int i = max(0, it - kStages); i < it; i++) mbar_wait(&full[i % kStages], (i / kStages) & 1, &none);
        else   // they are counted in the other CTA: a millisecond is long enough for any copy
          for (int i = 0; i < 1000; i++) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elected()) {
      int stage = 0, phase = 0, local = 0;
      bool ok = true;
      const uint32_t idesc = mma_desc(p.bf16, p.a_mn, p.b_mn, kPairM, p.ntile);
      const uint32_t step_a = p.a_mn ? 2048 >> 4 : 32 >> 4, step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;
      const uint64_t da0 = smem_desc(smem_addr(smem), p.a_mn ? 8192 : 16, 1024);
      const uint64_t db0 = smem_desc(smem_addr(smem) + kBytesA, p.b_mn ? 8192 : 16, 1024);
      for (int t = pair; ok && t < tiles; t += npairs) {
        int m, n, k;
        tile_of<USE>(p, t, m, n, k);
        const int kend = first_k(k + 1);
        for (int k0 = first_k(k); ok && k0 < kend; k0 += p.segment, local++) {
          const int buf = local & 1, k1 = min(kend, k0 + p.segment);
          if (!mbar_wait(&tempty[buf], (local / 2 + 1) & 1, gave_up)) {
            ok = false;
            break;
          }
          tmem_after_sync();
          const uint32_t d = tmem + buf * 256;
          bool add = false;
          for (int q = 0; ok && q < p.pairs; q++)
            for (int kb = k0; kb < k1; kb++) {
              if (!mbar_wait(&full[stage], phase, gave_up)) {
                ok = false;
                break;
              }
              tmem_after_sync();
              const uint64_t da = da0 + stage * ((kBytesA + kBytesB) >> 4), db = db0 + stage * ((kBytesA + kBytesB) >> 4);
              mma_f16(d, da, db, idesc, add);
              if (is_grad(USE) || kb != p.kblocks - 1 || p.k16 == kK / 16) {
#pragma unroll
                for (int i = 1; i < kK / 16; i++) mma_f16(d, da + i * step_a, db + i * step_b, idesc, true);
              } else {
                for (int i = 1; i < p.k16; i++) mma_f16(d, da + i * step_a, db + i * step_b, idesc, true);
              }
              add = true;
              mma_commit(&empty[stage]);
              if (++stage == kStages) {
                stage = 0;
                phase ^= 1;
              }
            }
          if (ok) mma_commit(&tfull[buf]);
        }
      }
      if (!ok) {   // products in flight still read shared memory
        int none = 0;
        mma_commit(&done);
        mbar_wait(&done, 0, &none);
      }
    }
    __syncwarp();
  } else if (USE == kProbs && warp < 4) {
    // one tile ahead of the warps that read it: what they need of each row, so that they never wait
    // for global memory (ten targets a row cost as much as the tile itself)
    bool ok = true;
    int local = 0;
    for (int t = pair; ok && t < tiles; t += npairs, local++) {
      int m, n, k;
      tile_of<USE>(p, t, m, n, k);
      const int buf = local & 1;
      ok = __all_sync(kFullMask, mbar_wait(&hempty[buf], (local / 2 + 1) & 1, gave_up));
      const int64_t first = p.word0 + (int64_t)n * kN;
      for (int i = (warp - 2) * 32 + lane; ok && i < kM; i += 64) {
        const int64_t r = (int64_t)m * kPairM + rank * kM + i;
        RowCoef rc{INFINITY, 0.f, 0.f, 0u};
        if (r < p.rows) {
          rc = p.coef[r];
          const int *y = p.targets + r * p.labels;
          for (int j = 0; j < p.labels; j += 8) {
            int at[8];
#pragma unroll
            for (int q = 0; q < 8; q++) at[q] = j + q < p.labels ? y[j + q] : -1;
#pragma unroll
            for (int q = 0; q < 8; q++) {
              const int64_t c = at[q] - first;
              if (at[q] >= 0 && c >= 0 && c < kN) rc.hits |= 1u << (c >> 5);
            }
          }
          if (rc.g == 0.f) rc.hits = 0;
        }
        coef_s[buf][i] = rc;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(smem_addr(&hfull[buf]));
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) / 4;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t tempty_at[2] = {in_leader(&tempty[0]), in_leader(&tempty[1])};
    float c = kLog2e;
    if (!is_grad(USE) && p.split_scale)
      c = kLog2e * pow2(-scale_exp(p.sc->h, kOperandTop)) * pow2(-scale_exp(p.sc->w, kOperandTop));
    const float factor = is_grad(USE) ? rescale_of(p.rescale) : 1.f;
    int local = 0;
    bool ok = true;
    // a block that gave up fills its tiles with NaN: nothing it did not compute passes for a result
    auto begin = [&](int buf) {
      ok = ok && mbar_wait(&tfull[buf], (local / 2) & 1, gave_up);
      ok = __all_sync(kFullMask, ok);
      tmem_after_sync();
    };
    auto end = [&](int buf) {
      tmem_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(tempty_at[buf]);
      local++;
    };
    const int chunks = (p.ntile + 31) / 32;
    for (int t = pair; t < tiles; t += npairs) {
      int m, n, k;
      tile_of<USE>(p, t, m, n, k);
      const int64_t r = (int64_t)m * kPairM + rank * kM + row;
      auto fetch = [&](int ch, float (&x)[32]) {
        if (ok) {
          tmem_load32(lanes + (local & 1) * 256 + ch * 32, x);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) x[i] = __int_as_float(0x7fffffff);
        }
      };
      if (USE == kLogits) {
        const int buf = local & 1;
        begin(buf);
        Part part{-INFINITY, 0.f};
        const int64_t left = p.vocab - (int64_t)n * kN;   // columns of the tile that are words
        for (int ch = half; ch < chunks; ch += 2) {
          float x[32];
          fetch(ch, x);
          if (left < kN) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (ch * 32 + i >= left) x[i] = -INFINITY;
          }
          float top = x[0];
#pragma unroll
          for (int i = 1; i < 32; i++) top = fmaxf(top, x[i]);
          const float m2 = fmaxf(part.m, top * c);
          if (m2 > part.m) {
            part.s *= exp2_fast(part.m - m2);
            part.m = m2;
          }
          const float base = part.m == -INFINITY ? 0.f : part.m;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            s0 += exp2_fast(fmaf(x[i], c, -base));
            s1 += exp2_fast(fmaf(x[i + 1], c, -base));
          }
          part.s += s0 + s1;
        }
        if (r < p.rows) p.parts[(int64_t)(2 * n + half) * p.ldparts + r] = part;
        end(buf);
      } else if (USE == kProbs) {
        const int buf = local & 1;
        ok = ok && mbar_wait(&hfull[buf], (local / 2) & 1, gave_up);
        ok = __all_sync(kFullMask, ok);
        const RowCoef rc = ok ? coef_s[buf][row] : RowCoef{INFINITY, 0.f, 0.f, 0u};
        const unsigned hits = rc.hits;
        const int64_t left = p.vocab - p.word0 - (int64_t)n * kN;
        const int64_t first = p.word0 + (int64_t)n * kN;
        const int *y = p.targets + r * p.labels;
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(smem_addr(&hempty[buf]));
        begin(buf);
        for (int ch = half; ch < chunks; ch += 2) {
          float x[32];
          fetch(ch, x);
#pragma unroll
          for (int i = 0; i < 32; i++) x[i] = exp2_fast(fmaf(x[i], c, -rc.lse2)) * rc.coef;
          if (left < kN) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (ch * 32 + i >= left) x[i] = 0.f;
          }
          if (__any_sync(kFullMask, hits >> ch & 1)) {
            if (hits >> ch & 1)
              for (int j = 0; j < p.labels; j++) {
                const int64_t at = y[j] - first - ch * 32;
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] -= at == i ? rc.g : 0.f;
              }
            __syncwarp();
          }
          uint16_t *to = p.probs + ((int64_t)(n * (kN / 64) + ch / 2) * p.strip + r) * 64 + ch % 2 * 32;
          if (p.bf16) store_probs<true, false>(to, 0, x);
          else if (p.prob_lo) store_probs<false, true>(to, p.prob_lo, x);
          else store_probs<false, false>(to, 0, x);
        }
        end(buf);
      } else if (USE == kGrad) {
        const int buf = local & 1;
        begin(buf);
        for (int ch = half; ch < chunks; ch += 2) {
          float x[32];
          fetch(ch, x);
#pragma unroll
          for (int b = 0; b < 4; b++) put_grad(p, r, n, k, ch * 32 + b * 8, &x[b * 8], factor);
        }
        end(buf);
      } else {
        // the tensor cores truncate what they accumulate: after `segment` blocks of K the sum goes on in
        // fp32 with rounding, in a scratch of the block's own that stays in L2 (a thread's eight values
        // side by side, a warp's in one piece); registers for it would spill
        float *mine = p.scratch + (int64_t)blockIdx.x * kM * kN + (threadIdx.x - 128) * 8;
        const int kstart = first_k(k), kend = first_k(k + 1);
        for (int k0 = kstart; k0 < kend; k0 += p.segment) {
          const int buf = local & 1;
          begin(buf);
          for (int ch = half; ch < chunks; ch += 2) {
            float x[32];
            float *at = mine + ch / 2 * (4 * 256 * 8);
            float old[4][8];
            if (k0 > kstart) {
#pragma unroll
              for (int b = 0; b < 4; b++) load8(at + b * (256 * 8), old[b]);
            }
            fetch(ch, x);
#pragma unroll
            for (int b = 0; b < 4; b++) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; e++) v[e] = k0 > kstart ? x[b * 8 + e] + old[b][e] : x[b * 8 + e];
              if (k0 + p.segment < kend) store8(at + b * (256 * 8), v);
              else put_grad(p, r, n, k, ch * 32 + b * 8, v, factor);
            }
          }
          end(buf);
        }
      }
    }
  }
  // neither CTA leaves while the other's products read its shared memory or its barriers are arrived on
  tmem_before_sync();
  __syncwarp();
  cluster_sync();
  tmem_after_sync();
  if (warp == 2) tmem_free(tmem, 512);
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
bool aligned(const void *a, size_t to) { return reinterpret_cast<uintptr_t>(a) % to == 0; }
int64_t up(int64_t a, int64_t to) { return (a + to - 1) / to * to; }

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// A matrix of 16-bit elements, `inner` a row, rows `ld` elements apart; boxes of 64 x box_rows.
int tensor_map(CUtensorMap *map, const void *base, int64_t inner, int64_t rows, int64_t ld, int box_rows) {
  const EncodeTiled encode = encoder();
  if (!encode) return (int)cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult e = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return e == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// An operand as the products read it.
struct Operand {
  const void *p;
  int64_t ld, inner, rows;
  int width;   // offset between parts
};

template <Use USE>
int launch_product(Product &p, const Operand &a, const Operand &b, cudaStream_t s) {
  int err = tensor_map(&p.a, a.p, a.inner, a.rows, a.ld, p.a_mn ? 64 : kM);
  if (!err) err = tensor_map(&p.b, b.p, b.inner, b.rows, b.ld, p.b_mn ? 64 : kN / 2);
  if (err) return err;
  // an attribute of the function on the current device, so it is set on every device that gets here
  const cudaError_t e = cudaFuncSetAttribute(product_kernel<USE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return (int)e;
  const int tiles = p.mt * p.nt * p.splits;
  product_kernel<USE><<<2 * std::max(1, std::min(tiles, device_sm_count() / 2)), kMmaThreads, kSmem, s>>>(p);
  count_launch(1);
  return (int)cudaGetLastError();
}

struct Shape {
  int64_t n, vocab;
  int dim, labels, type;
};

bool good_shape(const Shape &x) {
  return x.n >= 0 && x.n < ((int64_t)1 << 31) - 1024 && x.vocab >= 1 && x.vocab < ((int64_t)1 << 31) - 512 && x.dim >= 1 &&
         x.dim <= kMaxDim && x.labels >= 1 && x.labels <= 1024 &&
         (x.type == W2V_F32 || x.type == W2V_BF16 || x.type == W2V_F16);
}

constexpr int64_t kLossRows = 16384;            // rows whose parts are kept at a time
constexpr int64_t kGradRows = 8192;             // rows of a piece of d
constexpr int64_t kProbBytes = (int64_t)512 << 20;
constexpr int kSegment = 8;                     // fp32 gradients: blocks of K between two roundings

int few_blocks(int64_t vocab) {
  const int64_t need = (vocab + kFewThreads / 32 * kFewWords - 1) / (kFewThreads / 32 * kFewWords);
  return (int)std::min<int64_t>(need, (int64_t)device_sm_count() * 2);
}
int few_dh_blocks(int64_t vocab) {
  return (int)std::min<int64_t>((vocab + 31) / 32, (int64_t)device_sm_count() * 4);
}
int few_rows_of(int64_t n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8; }

struct Layout {
  int64_t scalars, coef, hs, ws, parts, probs, scratch, acc_h, acc_w, total;
  int width, nparts;         // staged operands
  int64_t rows, words;       // of a piece of d
  int nt, ntile, hsplits, wsplits;
  bool direct_h, direct_w;   // sums are complete in one go: no slabs
};

// Column tiles of a gradient: as few as hold dim, equally wide.
void column_tiles(int dim, int *nt, int *ntile) {
  *nt = (dim + kN - 1) / kN;
  *ntile = (int)up((dim + *nt - 1) / *nt, 32);
}
// In how many parts K is cut, each with a slab of sums of its own, by an estimate in microseconds: the
// rounds of tiles over the pairs of SMs, a block of K taking 512 clocks for 256 columns, against
// writing the slabs and reading them again at about 5 TB/s.  With one part and `whole` there is no slab.
int splits_for(int64_t tiles, int64_t kblocks, int pairs, int ntile, int64_t slab_bytes, bool whole) {
  const int sms = std::max(1, device_sm_count() / 2);
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 32 && (s == 1 || kblocks / s >= 4); s++) {
    const double rounds = (double)((tiles * s + sms - 1) / sms);
    const double product = rounds * ((double)kblocks / s * pairs * 512 * ntile / kN + 1500) / 1700;
    const double slabs = s == 1 && whole ? 0 : 2.0 * s * slab_bytes / 5e6;
    if (product + slabs < cost) {
      cost = product + slabs;
      best = s;
    }
  }
  return best;
}

Layout plan(const Shape &x, bool grad) {
  Layout l{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(std::max<int64_t>(bytes, 1), 1024);
    return here;
  };
  l.scalars = take(sizeof(Scalars));
  if (x.n <= kFewRows) {
    const int rb = few_rows_of(x.n);
    if (!grad) {
      l.parts = take((int64_t)few_blocks(x.vocab) * x.n * sizeof(Part));
    } else {
      l.probs = take(x.vocab * rb * 4);
      l.acc_h = take((int64_t)few_dh_blocks(x.vocab) * rb * x.dim * 4);
    }
    l.total = at;
    return l;
  }
  l.width = (int)up(x.dim, 64);
  l.nparts = x.type == W2V_F32 ? (grad ? 3 : 2) : 1;
  l.hs = take(x.n * l.width * l.nparts * 2);
  l.ws = take(x.vocab * l.width * l.nparts * 2);
  if (!grad) {
    l.parts = take(2 * ((x.vocab + kN - 1) / kN) * std::min(x.n, kLossRows) * sizeof(Part));
  } else {
    const int bytes = x.type == W2V_F32 ? 4 : 2;
    l.rows = up(std::min(x.n, kGradRows), kPairM);
    // pieces of the vocabulary of equal width, up to a quarter more than kProbBytes
    const int64_t most = std::max<int64_t>(kN, kProbBytes / (l.rows * bytes));
    const int64_t pieces = std::max<int64_t>(1, (x.vocab + most * 5 / 4 - 1) / (most * 5 / 4));
    l.words = up((x.vocab + pieces - 1) / pieces, kN);
    column_tiles(x.dim, &l.nt, &l.ntile);
    const int pairs = x.type == W2V_F32 ? 3 : 1;
    const int64_t cols = (int64_t)l.nt * l.ntile * 4;
    l.hsplits = splits_for(l.rows / kPairM * l.nt, l.words / kK, pairs, l.ntile, l.rows * cols, l.words >= x.vocab && x.dim % 8 == 0);
    l.wsplits = splits_for(l.words / kPairM * l.nt, l.rows / kK, pairs, l.ntile, l.words * cols,
                           l.rows >= x.n && x.dim % 8 == 0);
    l.coef = take(x.n * sizeof(RowCoef));
    l.probs = take(l.rows * l.words * bytes);
    if (x.type == W2V_F32) l.scratch = take((int64_t)device_sm_count() * kM * kN * 4);
    // rows that are not a multiple of eight elements are better written by a warp each than by a thread each
    l.direct_h = l.hsplits == 1 && l.words >= x.vocab && x.dim % 8 == 0;
    l.direct_w = l.wsplits == 1 && l.rows >= x.n && x.dim % 8 == 0;
    if (!l.direct_h) l.acc_h = take((int64_t)l.hsplits * l.rows * l.nt * l.ntile * 4);
    if (!l.direct_w) l.acc_w = take((int64_t)l.wsplits * up(x.vocab, kM) * l.nt * l.ntile * 4);
  }
  l.total = at;
  return l;
}

template <typename T>
bool direct(const void *p, int64_t ld) {   // TMA can read the caller's matrix
  return sizeof(T) == 2 && aligned(p, 16) && ld * sizeof(T) % 16 == 0;
}

// Operands for the products: the caller's own where TMA can read them, else staged ones.
template <typename T>
int stage(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const float *gloss,
          int64_t ldg, const int *targets, char *ws, Operand *oh, Operand *ow, cudaStream_t s) {
  constexpr bool split = sizeof(T) == 4;
  Scalars *sc = reinterpret_cast<Scalars *>(ws + l.scalars);
  const Source sh{h, ldh, x.n}, sw{w, ldw, x.vocab};
  cudaError_t e = cudaMemsetAsync(sc, 0, sizeof(Scalars), s);
  if (e != cudaSuccess) return (int)e;
  const int blocks = device_sm_count() * 8;
  if (split || gloss) {
    const Source none{nullptr, 0, x.n};
    amax_kernel<<<dim3(split ? blocks : 64, 1, 3), 256, 0, s>>>(split ? sh : none, split ? sw : Source{nullptr, 0, 0},
                                                                 x.dim, gloss, ldg, targets, x.labels, x.vocab, sc);
    count_launch(1);
  }
  void *hs = direct<T>(h, ldh) ? nullptr : ws + l.hs, *wst = direct<T>(w, ldw) ? nullptr : ws + l.ws;
  if (hs || wst) {
    stage_kernel<T><<<dim3(blocks, 1, 2), 256, 0, s>>>(sh, sw, x.dim, hs, wst, l.width, l.nparts, sc);
    count_launch(1);
  }
  const int64_t staged = (int64_t)l.width * l.nparts;
  *oh = hs ? Operand{hs, staged, staged, x.n, l.width} : Operand{h, ldh, x.dim, x.n, 0};
  *ow = wst ? Operand{wst, staged, staged, x.vocab, l.width} : Operand{w, ldw, x.dim, x.vocab, 0};
  return (int)cudaGetLastError();
}

template <typename T>
Product logits_product(const Shape &x, const Operand &oh, const Operand &ow, const Scalars *sc) {
  Product p{};
  constexpr bool split = sizeof(T) == 4;
  p.ntile = kN;
  p.splits = 1;
  p.kblocks = (x.dim + kK - 1) / kK;
  p.pairs = split ? 3 : 1;
  if (split) {   // lo hi, hi lo, hi hi
    p.pa[0] = oh.width;
    p.pb[1] = ow.width;
  }
  p.segment = p.kblocks;
  p.k16 = (x.dim - (p.kblocks - 1) * kK + 15) / 16;
  p.bf16 = x.type == W2V_BF16;
  p.sc = sc;
  p.split_scale = split;
  p.vocab = x.vocab;
  return p;
}

template <typename T, int RB>
int few_loss(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, char *ws,
             int *count, cudaStream_t s) {
  const size_t smem = (size_t)RB * few_steps(x.dim) * 1024;
  auto k = few_loss_kernel<T, RB>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  const bool wide = aligned(w, 8 * sizeof(T)) && ldw % 8 == 0;
  *count = few_blocks(x.vocab);
  k<<<*count, kFewThreads, smem, s>>>(static_cast<const T *>(h), ldh, (int)x.n, static_cast<const T *>(w), ldw, x.vocab,
                                      x.dim, wide, reinterpret_cast<Part *>(ws + l.parts));
  count_launch(1);
  return (int)cudaGetLastError();
}

template <typename T>
int run_loss(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const int *targets,
             float *loss, float *lse, char *ws, cudaStream_t s) {
  Part *parts = reinterpret_cast<Part *>(ws + l.parts);
  const bool wide = aligned(h, 8 * sizeof(T)) && ldh % 8 == 0 && aligned(w, 8 * sizeof(T)) && ldw % 8 == 0;
  auto join_rows = [&](int count, int64_t ldp, int64_t r0, int rows) {
    loss_join_kernel<T><<<(rows + kJoinRows - 1) / kJoinRows, kJoinThreads, 0, s>>>(
        parts, count, ldp, rows, static_cast<const T *>(h) + r0 * ldh, ldh, static_cast<const T *>(w), ldw, x.vocab,
        x.dim, wide, targets + r0 * x.labels, x.labels, loss + r0, lse + r0);
    count_launch(1);
    return (int)cudaGetLastError();
  };
  if (x.n <= kFewRows) {
    int count = 0, err = 0;
    switch (few_rows_of(x.n)) {
      case 1: err = few_loss<T, 1>(x, l, h, ldh, w, ldw, ws, &count, s); break;
      case 2: err = few_loss<T, 2>(x, l, h, ldh, w, ldw, ws, &count, s); break;
      case 4: err = few_loss<T, 4>(x, l, h, ldh, w, ldw, ws, &count, s); break;
      default: err = few_loss<T, 8>(x, l, h, ldh, w, ldw, ws, &count, s);
    }
    return err ? err : join_rows(count, x.n, 0, (int)x.n);
  }
  Operand oh, ow;
  int err = stage<T>(x, l, h, ldh, w, ldw, nullptr, 0, nullptr, ws, &oh, &ow, s);
  if (err) return err;
  Product p = logits_product<T>(x, oh, ow, reinterpret_cast<const Scalars *>(ws + l.scalars));
  p.nt = (int)((x.vocab + kN - 1) / kN);
  p.parts = parts;
  for (int64_t r0 = 0; r0 < x.n; r0 += kLossRows) {
    p.rows = (int)std::min(kLossRows, x.n - r0);
    p.mt = (p.rows + kPairM - 1) / kPairM;
    p.a_y = (int)r0;
    p.ldparts = p.rows;
    err = launch_product<kLogits>(p, oh, ow, s);
    if (!err) err = join_rows(2 * p.nt, p.ldparts, r0, p.rows);
    if (err) return err;
  }
  return 0;
}

template <typename T, int RB>
int few_grad(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const int *targets,
             const float *lse, const float *gloss, int64_t ldg, void *dh, int64_t lddh, void *dw, int64_t lddw, char *ws,
             cudaStream_t s) {
  const size_t smem = (size_t)RB * few_steps(x.dim) * 1024;
  auto k = few_grad_kernel<T, RB>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  const bool wide = aligned(w, 8 * sizeof(T)) && ldw % 8 == 0, wout = aligned(dw, 8 * sizeof(T)) && lddw % 8 == 0;
  float *d = reinterpret_cast<float *>(ws + l.probs), *acc = reinterpret_cast<float *>(ws + l.acc_h);
  const T *wt = static_cast<const T *>(w);
  k<<<few_blocks(x.vocab), kFewThreads, smem, s>>>(static_cast<const T *>(h), ldh, (int)x.n, wt, ldw, x.vocab, x.dim, wide,
                                                   targets, x.labels, lse, gloss, ldg, static_cast<T *>(dw), lddw, wout, d);
  const int blocks = few_dh_blocks(x.vocab);
  few_dh_kernel<T, RB><<<dim3(blocks, (x.dim + kFewThreads - 1) / kFewThreads), kFewThreads, 0, s>>>(wt, ldw, x.vocab,
                                                                                                    x.dim, d, acc);
  slabs_kernel<T><<<(int)std::min<int64_t>((x.n * ((x.dim + 255) / 256) + 7) / 8, 1024), 256, 0, s>>>(
      acc, blocks, (int64_t)RB * x.dim, x.dim, x.n, x.dim, static_cast<T *>(dh), lddh, false, Rescale{nullptr, nullptr, 0});
  count_launch(3);
  return (int)cudaGetLastError();
}

template <typename T>
int run_grad(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const int *targets,
             const float *lse, const float *gloss, int64_t ldg, void *dh, int64_t lddh, void *dw, int64_t lddw, char *ws,
             cudaStream_t s) {
  if (x.n == 0) return (int)cudaMemset2DAsync(dw, lddw * sizeof(T), 0, x.dim * sizeof(T), x.vocab, s);
  if (x.n <= kFewRows) {
    switch (few_rows_of(x.n)) {
      case 1: return few_grad<T, 1>(x, l, h, ldh, w, ldw, targets, lse, gloss, ldg, dh, lddh, dw, lddw, ws, s);
      case 2: return few_grad<T, 2>(x, l, h, ldh, w, ldw, targets, lse, gloss, ldg, dh, lddh, dw, lddw, ws, s);
      case 4: return few_grad<T, 4>(x, l, h, ldh, w, ldw, targets, lse, gloss, ldg, dh, lddh, dw, lddw, ws, s);
      default: return few_grad<T, 8>(x, l, h, ldh, w, ldw, targets, lse, gloss, ldg, dh, lddh, dw, lddw, ws, s);
    }
  }
  constexpr bool split = sizeof(T) == 4;
  Operand oh, ow;
  int err = stage<T>(x, l, h, ldh, w, ldw, gloss, ldg, targets, ws, &oh, &ow, s);
  if (err) return err;
  const Scalars *sc = reinterpret_cast<const Scalars *>(ws + l.scalars);
  RowCoef *coef = reinterpret_cast<RowCoef *>(ws + l.coef);
  row_coef_kernel<<<(int)((x.n + 255) / 256), 256, 0, s>>>(lse, gloss, ldg, targets, x.labels, x.vocab, x.n, sc, coef);
  count_launch(1);
  const int64_t ldacc = (int64_t)l.nt * l.ntile;
  // d lies in strips of 64 columns, 128 bytes a row: what a warp writes of a tile, and what a load of
  // either gradient's operand reads, is one piece of memory
  const int strips = (int)(l.words / 64) * (split ? 2 : 1);
  const Operand probs{ws + l.probs, 64, 64, strips * l.rows, (int)(l.words / 64 * l.rows)};
  float *acc_h = reinterpret_cast<float *>(ws + l.acc_h), *acc_w = reinterpret_cast<float *>(ws + l.acc_w);
  const int64_t acc_w_rows = up(x.vocab, kM);
  const int sums = device_sm_count() * 8;
  const float *one_gloss = ldg ? nullptr : gloss;
  const Rescale rescale_h{sc, one_gloss, split ? 1 : 0}, rescale_w{sc, one_gloss, split ? 2 : 0};
  for (int64_t r0 = 0; r0 < x.n; r0 += l.rows) {
    const int rows = (int)std::min(l.rows, x.n - r0);
    for (int64_t v0 = 0; v0 < x.vocab; v0 += l.words) {
      const int words = (int)std::min(l.words, x.vocab - v0);
      Product p = logits_product<T>(x, oh, ow, sc);
      p.mt = (rows + kPairM - 1) / kPairM;
      p.nt = (words + kN - 1) / kN;
      p.a_y = (int)r0;
      p.b_y = p.word0 = (int)v0;
      p.rows = rows;
      p.coef = coef + r0;
      p.targets = targets + r0 * x.labels;
      p.labels = x.labels;
      p.probs = static_cast<uint16_t *>(const_cast<void *>(probs.p));
      p.strip = (int)l.rows;
      p.prob_lo = split ? (int64_t)probs.width * 64 : 0;
      err = launch_product<kProbs>(p, oh, ow, s);
      if (err) return err;
      for (int which = 0; which < 2; which++) {   // dH, then dW
        const Operand &o = which == 0 ? ow : oh;
        Product q{};
        q.nt = l.nt;
        q.ntile = l.ntile;
        q.mt = which == 0 ? p.mt : (words + kPairM - 1) / kPairM;
        q.kblocks = which == 0 ? (words + kK - 1) / kK : (rows + kK - 1) / kK;
        // the last piece may be too short for all splits: it adds to some of the slabs, which the
        // first piece, never the shorter one, has filled
        q.splits = std::min(which == 0 ? l.hsplits : l.wsplits, q.kblocks);
        q.pairs = split ? 3 : 1;
        if (split) {   // (lo 2^11) (hi 2^-11), hi lo, hi hi
          q.pa[0] = probs.width;
          q.pb[0] = 2 * o.width;
          q.pb[1] = o.width;
        }
        q.segment = split ? kSegment : q.kblocks;
        q.k16 = kK / 16;
        q.scratch = reinterpret_cast<float *>(ws + l.scratch);
        q.strip = (int)l.rows;
        q.a_mn = which;
        q.b_mn = 1;
        q.b_y = (int)(which == 0 ? v0 : r0);
        q.bf16 = x.type == W2V_BF16;
        q.rows = which == 0 ? rows : words;
        q.dim = x.dim;
        q.ldacc = ldacc;
        q.acc = which == 0 ? acc_h : acc_w + v0 * ldacc;
        q.acc_slab = (which == 0 ? l.rows : acc_w_rows) * ldacc;
        q.add = which == 0 ? v0 > 0 : r0 > 0;
        q.rescale = which == 0 ? rescale_h : rescale_w;
        if (which == 0 ? l.direct_h : l.direct_w) {
          q.out = which == 0 ? static_cast<T *>(dh) + r0 * lddh : static_cast<T *>(dw) + v0 * lddw;
          q.ldout = which == 0 ? lddh : lddw;
          q.out_type = x.type;
          q.out_wide = aligned(q.out, 8 * sizeof(T)) && q.ldout % 8 == 0;
        }
        err = split ? launch_product<kGradSegments>(q, probs, o, s) : launch_product<kGrad>(q, probs, o, s);
        if (err) return err;
      }
    }
    if (!l.direct_h) {
      slabs_kernel<T><<<sums, 256, 0, s>>>(acc_h, l.hsplits, l.rows * ldacc, ldacc, rows, x.dim,
                                           static_cast<T *>(dh) + r0 * lddh, lddh, true, rescale_h);
      count_launch(1);
    }
  }
  if (!l.direct_w) {
    slabs_kernel<T><<<sums, 256, 0, s>>>(acc_w, l.wsplits, acc_w_rows * ldacc, ldacc, x.vocab, x.dim,
                                         static_cast<T *>(dw), lddw, true, rescale_w);
    count_launch(1);
  }
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" int64_t w2v_softmax_workspace(int64_t n, int64_t vocab, int dim, int labels, int type, int grad) {
  const Shape x{n, vocab, dim, labels, type};
  return good_shape(x) ? plan(x, grad != 0).total : -1;
}

extern "C" int w2v_softmax_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const int *targets,
                                int64_t n, int64_t vocab, int dim, int labels, int type, float *loss, float *lse,
                                void *workspace, int64_t workspace_bytes, void *stream) {
  const Shape x{n, vocab, dim, labels, type};
  if (!good_shape(x) || ldh < dim || ldw < dim || !weight || !workspace || !aligned(workspace, 256)) return 1;
  if (n == 0) return 0;
  if (!hidden || !targets || !loss || !lse) return 1;
  const Layout l = plan(x, false);
  if (workspace_bytes < l.total) return 1;
  char *ws = static_cast<char *>(workspace);
  const auto s = static_cast<cudaStream_t>(stream);
  if (type == W2V_F32) return run_loss<float>(x, l, hidden, ldh, weight, ldw, targets, loss, lse, ws, s);
  if (type == W2V_BF16) return run_loss<__nv_bfloat16>(x, l, hidden, ldh, weight, ldw, targets, loss, lse, ws, s);
  return run_loss<__half>(x, l, hidden, ldh, weight, ldw, targets, loss, lse, ws, s);
}

extern "C" int w2v_softmax_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const int *targets,
                                int64_t n, int64_t vocab, int dim, int labels, int type, const float *lse,
                                const float *gloss, int64_t ldg, void *dhidden, int64_t lddh, void *dweight,
                                int64_t lddw, void *workspace, int64_t workspace_bytes, void *stream) {
  const Shape x{n, vocab, dim, labels, type};
  if (!good_shape(x) || ldh < dim || ldw < dim || lddh < dim || lddw < dim || !weight || !dweight || !workspace ||
      !aligned(workspace, 256) || (ldg != 0 && ldg != 1))
    return 1;
  if (n > 0 && (!hidden || !targets || !lse || !gloss || !dhidden)) return 1;
  const Layout l = plan(x, true);
  if (workspace_bytes < l.total) return 1;
  char *ws = static_cast<char *>(workspace);
  const auto s = static_cast<cudaStream_t>(stream);
  if (type == W2V_F32)
    return run_grad<float>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw, ws, s);
  if (type == W2V_BF16)
    return run_grad<__nv_bfloat16>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw,
                                   ws, s);
  return run_grad<__half>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw, ws, s);
}
