// Softmax cross entropy over the whole vocabulary, in pieces, without keeping the logits.
//
//   l_nv = h_n . w_v     lse_n = log sum_v exp l_nv     loss_n = sum_j (lse_n - l_{n, y_nj})
//   d_nv = g_n (k_n exp(l_nv - lse_n) - #{j : y_nj = v})     dH = d W     dW = d^T H
//
// with y_n the targets of row n that lie in the vocabulary and k_n their number (none is fine: loss
// and gradient are zero).  For N rows, V words and D columns the loss costs 2 N V D operations, the
// gradients 4 N V D and, since no logits are kept, the logits' 2 N V D again.
//
// More than a few rows (few_rows): the tensor cores.  Pairs of CTAs compute tiles of 256 x 256 of a product
// whose operands TMA brings into shared memory: a producer warp in each, one thread of the pair that
// issues tcgen05.mma, eight warps in each that read the finished tile from tensor memory while the next
// one is computed in the other half of it.
//   product_kernel<kLogits>  the maximum and sum of exponentials of each row over half a tile's columns:
//            8 bytes a row go to memory, a small kernel joins them;
//   product_kernel<kProbs>   d of a row block and a piece of the vocabulary, in 16 bits;
//   grad_kernel              dH and dW from that piece, added up in fp32 over the pieces (row blocks).
// The products are bound by the issue of the matrix instructions and, over long times, by the power cap:
// 8192 x 131072 x 1024 logits in bf16 take 1.39 ms in a single run (1.58 PFLOP/s, 0.93 of the measured burst
// rate) and 1.5 in a row (1.40 GHz); d and both gradients of the same sizes 5.5 to 5.7 ms (1.2 PFLOP/s).
// fp32 operands are split into two fp16 numbers (after a common power-of-two scale), x = hi + lo, and
// hi hi + hi lo + lo hi computed: 22 bits of each operand.  Products of fp16 or bf16 operands are exact in
// the fp32 accumulators.  d is rounded once to the operands' type (fp32: to hi + lo with lo scaled by
// 2^11, so that small probabilities keep their bits; the operand it meets carries the 2^-11).
// One scale serves a matrix whose rows' largest magnitudes lie within 2^kRowSpan of each other.  Where they
// do not (an outlier in one row), two fp16 numbers would lose the bits of the others: the operands are
// then split into three bf16 numbers, which keep their own exponents, and six products computed.  The
// device decides, from magnitudes that it has to find for the scale anyway (find_wide).  4096 x 100000 x 256:
// loss 0.47 ms, with an outlier 0.96; gradients 2.08 ms, with one 3.78.
//
// For few rows the bound is reading W once: a kernel with eight rows in shared memory, W straight from
// memory in its own type, plain fp32 arithmetic.  fp32 goes that way up to 16 rows, in two passes: the
// tensor cores would need W in two parts, three more passes over it (100000 x 256, loss / gradients: 8 rows
// 30 / 78 us, 16 rows 60 / 156, against 107 / 223 for 9 or more).  16-bit types go that way up to four
// rows.  The loss does so where W would have to be copied (100000 x 300, 4 rows: 44 us against 66) or has at most
// 256 columns, a step of the kernel's (128: 27 against 26, 256: 24 against 28, 384: 54 against 31, 1024: 138
// against 82).  The gradients always do: here d stays in fp32 and is not rounded to 16 bits, for a
// tenth more time, a quarter at most (100000 x 256, 4 rows: 98 us against 88, x 768 231 against 187; x 300, where
// W would be copied, 163 against 180).
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/bidmach_b200.h"
#include "w2v_chain.cuh"
#include "w2v_device.cuh"
#include "w2v_internal.h"
#include "w2v_tcgen05.cuh"
#include "w2v_types.cuh"

namespace {

using namespace w2v;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFewRows = 8;   // of a pass, fp32
constexpr int kFewRows16 = 4;
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

// Found on the device before a product: largest finite magnitudes (as bits) of H, W and g_n k_n, and the
// smallest ones of a row that are not zero, as kInfBits less them (0: no row), so that all are maxima.
constexpr unsigned kInfBits = 0x7f800000u;
struct Scalars {
  unsigned h, w, g, h_low, w_low, g_low;
  unsigned wide;   // three bf16 parts rather than two fp16 ones, set by stage_kernel
};

// With row maxima within 2^14 the last row's lies above 2^-1 after scaling, and the steps of its fp16 parts,
// 2^-24 and more, are its 22nd bits or better.  Factors g_n k_n: d = g k p has 2^-36 as its smallest half
// step; beyond 2^12 the probabilities of a row would be off by 2^-20 of their sum in a vocabulary of 2^17.
constexpr int kRowSpan = 14, kFactorSpan = 12;
__device__ __forceinline__ bool apart(unsigned top, unsigned low, int span) {
  return low && (int)(top >> 23) - (int)((kInfBits - low) >> 23) > span;
}
__device__ __forceinline__ bool find_wide(const Scalars *sc) {
  return apart(sc->h, sc->h_low, kRowSpan) || apart(sc->w, sc->w_low, kRowSpan) || apart(sc->g, sc->g_low, kFactorSpan);
}

// 2^e such that the largest magnitude times it lies in [2^top, 2^(top+1)); 1 for zero.
__device__ __forceinline__ int scale_exp(unsigned bits, int top) {
  if (bits == 0) return 0;
  const int e = bits >= 0x800000u ? (int)(bits >> 23) - 127 : -118 - __clz((int)bits);
  return min(126, max(-126, top - e));
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
  chain_wait();
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
                                                               int64_t ldg, T *dw, int64_t lddw, bool wide_out, bool add,
                                                               float *d) {
  extern __shared__ __align__(16) float sh[];
  __shared__ float lse_s[RB], g_s[RB], k_s[RB];
  __shared__ __align__(16) float d_s[kFewThreads / 32][RB][kFewWords];
  chain_wait();
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
        if (add) {   // fp32 only: a second pass
          float old[8];
          load_some(p, have, old);
#pragma unroll
          for (int e = 0; e < 8; e++) acc[q][e] += old[e];
        }
        if (wide_out && have == 8) store8(p, acc[q]);
        else store_some(p, have, acc[q]);
      }
    }
    __syncwarp();
  }
}

// dH of few rows: a warp sums d_nv w_v over a range of words, 256 columns (8 a lane) of all rows at a
// time, four words in flight; the block adds its warps' sums.  parts is [block][RB][dim].
template <typename T, int RB>
__global__ void __launch_bounds__(kFewThreads) few_dh_kernel(const T *w, int64_t ldw, int64_t vocab, int dim, bool wide,
                                                             const float *d, float *parts) {
  constexpr int warps = kFewThreads / 32;
  __shared__ __align__(16) float sums[warps][256];
  chain_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t all = (int64_t)gridDim.x * warps, me = (int64_t)blockIdx.x * warps + warp;
  const int64_t lo = me * vocab / all, hi = (me + 1) * vocab / all;
  const int col = blockIdx.y * 256 + lane * 8, have = min(8, max(0, dim - col));
  float acc[RB][8] = {};
  for (int64_t v = lo; v < hi; v += 4) {
    float x[4][8], dv[4][RB];
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const bool there = v + q < hi;
      const T *p = w + (v + q) * ldw + col;
      if (wide && there && have == 8) load8(p, x[q]);
      else load_some(p, there ? have : 0, x[q]);
#pragma unroll
      for (int r = 0; r < RB; r++) dv[q][r] = there ? d[(v + q) * RB + r] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int r = 0; r < RB; r++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[r][e] = fmaf(dv[q][r], x[q][e], acc[r][e]);
  }
  const int c = blockIdx.y * 256 + threadIdx.x;
#pragma unroll
  for (int r = 0; r < RB; r++) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      *reinterpret_cast<float4 *>(&sums[warp][lane * 8 + e]) =
          make_float4(acc[r][e], acc[r][e + 1], acc[r][e + 2], acc[r][e + 3]);
    __syncthreads();
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < warps; k++) x += sums[k][threadIdx.x];
    if (c < dim) parts[((int64_t)blockIdx.x * RB + r) * dim + c] = x;
  }
}

// Power of two that d is stored with, so that fp16 holds it: `given`, where one factor for all rows is
// left to the end and d is at most the number of targets, else from the largest |g_n k_n|.
constexpr int kFromRows = 1 << 20;
__device__ __forceinline__ int prob_exp(const Scalars *sc, int given) {
  return given == kFromRows ? scale_exp(sc->g, kProbTop) : given;
}

// What a gradient's sums have to be multiplied with: the powers of two that d and the other operand
// were scaled by, and the one factor for all rows where there is one.
struct Rescale {
  const Scalars *sc;
  const float *gloss;  // null: 1
  int given;           // of prob_exp
  int operand;         // 0: not scaled, 1: W, 2: H
};
__device__ __forceinline__ float rescale_of(const Rescale &r) {
  const float x = (r.gloss ? *r.gloss : 1.f) * pow2(-prob_exp(r.sc, r.given));
  return r.operand ? x * pow2(-scale_exp(r.operand == 1 ? r.sc->w : r.sc->h, kOperandTop)) : x;
}

// out[r][c] = sum over slabs: eight warps take an eighth of them each, for 32 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) slabs_kernel(const float *slabs, int count, int64_t slab, int dim, T *out,
                                                    int64_t ldo) {
  __shared__ float sums[8][32];
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  const int each = (count + 7) / 8, a = min(count, warp * each), b = min(count, a + each);
  const float *p = slabs + (int64_t)blockIdx.y * dim + c;
  float x = 0.f;
  for (int k = a; k < b; k += 8) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = k + j < b && c < dim ? p[(k + j) * slab] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) x += y[j];
  }
  sums[warp][lane] = x;
  __syncthreads();
  if (warp > 0 || c >= dim) return;
#pragma unroll
  for (int k = 1; k < 8; k++) x += sums[k][lane];
  out[(int64_t)blockIdx.y * ldo + c] = from_float<T>(x);
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
  chain_wait();
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
      // z and l are sums of their own, each with its own rounding: for a row that is sure of its target their
      // difference may come out below zero, which it never is (a NaN stays)
      const float term = z - warp_sum(x[q]);
      if (at[q] >= 0 && at[q] < vocab) sum += term < 0.f ? 0.f : term;
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

__device__ __forceinline__ void warp_max(unsigned top, unsigned *to) {
  top = __reduce_max_sync(kFullMask, top);
  if ((threadIdx.x & 31) == 0 && top) atomicMax(to, top);
}

// Bits of a magnitude; an infinity or a NaN counts as zero: it spoils its own row, not the others' scale.
__device__ __forceinline__ unsigned magnitude(float x) {
  const unsigned bits = __float_as_uint(x) & 0x7fffffffu;
  return bits < kInfBits ? bits : 0u;
}

// Largest finite magnitudes of fp32 operands (z = 0: H, 1: W) and of the rows' g_n k_n (z = 2), and the smallest row's.
__global__ void __launch_bounds__(256) amax_kernel(Source h, Source w, int dim, const float *gloss,
                                                   const int *targets, int labels, int64_t vocab, Scalars *sc) {
  chain_wait();
  unsigned top = 0, low = 0;
  if (blockIdx.z < 2) {
    const Source s = blockIdx.z == 0 ? h : w;
    if (!s.p) return;
    const float *a = static_cast<const float *>(s.p);
    const int lane = threadIdx.x & 31;
    const bool wide = reinterpret_cast<uintptr_t>(a) % 32 == 0 && s.ld % 8 == 0;
    for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < s.rows; r += (int64_t)gridDim.x * 8) {
      unsigned most = 0;
      for (int c = lane * 8; c < dim; c += 256) {
        const int have = min(8, dim - c);
        float x[8];
        if (wide && have == 8) load8(a + r * s.ld + c, x);
        else load_some(a + r * s.ld + c, have, x);
#pragma unroll
        for (int e = 0; e < 8; e++) most = max(most, magnitude(x[e]));
      }
      most = __reduce_max_sync(kFullMask, most);
      top = max(top, most);
      if (most) low = max(low, kInfBits - most);
    }
    warp_max(top, blockIdx.z == 0 ? &sc->h : &sc->w);
    warp_max(low, blockIdx.z == 0 ? &sc->h_low : &sc->w_low);
  } else if (gloss) {
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < h.rows; n += (int64_t)gridDim.x * 256) {
      const int k = valid_targets(targets + n * labels, labels, vocab);
      const unsigned m = k ? magnitude(gloss[n] * (float)k) : 0u;
      top = max(top, m);
      if (m) low = max(low, kInfBits - m);
    }
    warp_max(top, &sc->g);
    warp_max(low, &sc->g_low);
  }
}

// Rows of T as rows of `width` (a multiple of 64) 16-bit elements, zeros behind the last column.
template <typename T>
__device__ __forceinline__ void stage_row(const T *src, int dim, T *dst, int width) {
  for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    float x[8];
    load_some(src + c, min(8, max(0, dim - c)), x);
    store8(dst + c, x);
  }
}

// x as T, and in its place what that lacks (nothing where it is not finite).
template <typename T>
__device__ __forceinline__ float take_part(float &x) {
  float hi = to_float(from_float<T>(x));
  if (isinf(hi) && isfinite(x)) hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);   // bf16 rounds up to infinity
  x = isfinite(hi) ? x - hi : 0.f;
  return hi;
}

// fp32 as `parts` of them: fp16 hi, lo and hi 2^-11, or, WIDE, three bf16 ones that add up to it.
template <bool WIDE>
__device__ __forceinline__ void stage_split(const float *src, int dim, uint16_t *to, int width, int parts, float scale) {
  using P = typename std::conditional<WIDE, __nv_bfloat16, __half>::type;
  P *dst = reinterpret_cast<P *>(to);
  for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    const int have = min(8, max(0, dim - c));
    float x[8], hi[8], lo[8], small[8];
    if (have == 8 && reinterpret_cast<uintptr_t>(src + c) % 32 == 0) load8(src + c, x);
    else load_some(src + c, have, x);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[e] *= scale;
      hi[e] = take_part<P>(x[e]);
      if (WIDE) {
        lo[e] = take_part<P>(x[e]);
        small[e] = x[e];
      } else {
        lo[e] = x[e];
        small[e] = hi[e] * 0x1p-11f;
      }
    }
    store8(dst + c, hi);
    store8(dst + width + c, lo);
    if (WIDE || parts == 3) store8(dst + 2 * width + c, small);
  }
}

// Rows lie `pitch` elements apart; `parts` of fp32 are needed (three where they are bf16).
template <typename T>
__global__ void __launch_bounds__(256) stage_kernel(Source h, Source w, int dim, uint16_t *hs, uint16_t *ws, int width,
                                                    int64_t pitch, int parts, Scalars *sc) {
  chain_wait();
  const Source s = blockIdx.z == 0 ? h : w;
  uint16_t *to = blockIdx.z == 0 ? hs : ws;
  if (!to) return;
  constexpr bool split = sizeof(T) == 4;
  const float scale = split ? pow2(scale_exp(blockIdx.z == 0 ? sc->h : sc->w, kOperandTop)) : 1.f;
  const bool wide = split && find_wide(sc);
  if (wide && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) sc->wide = 1;
  for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < s.rows; r += (int64_t)gridDim.x * 8) {
    const T *src = static_cast<const T *>(s.p) + r * s.ld;
    uint16_t *dst = to + r * pitch;
    if constexpr (!split) stage_row<T>(src, dim, reinterpret_cast<T *>(dst), width);
    else if (wide) stage_split<true>(src, dim, dst, width, parts, scale);
    else stage_split<false>(src, dim, dst, width, parts, scale);
  }
}

// ---------------------------------------------------------------------------------------------
// The products
// ---------------------------------------------------------------------------------------------
constexpr int kM = 128, kN = 256, kK = 64;   // rows of each of a pair's CTAs, columns of both
constexpr int kPairM = 2 * kM;
constexpr int kBytesA = kM * kK * 2, kBytesB = kN / 2 * kK * 2, kBytesStage = kBytesA + kBytesB;
constexpr int kMmaThreads = 384;   // producer, issuer, two helpers, eight that read the tiles
constexpr int kMostStages = 6;
constexpr int smem_bytes(int stages, int more) { return stages * kBytesStage + more + 1024; }

// What the roles of a CTA share.
struct Pipe {
  u64 full[kMostStages], empty[kMostStages];   // operands: in the leader, counting both CTAs' bytes; read by the products
  u64 tfull[2], tempty[2];             // halves of tensor memory: finished; read (in the leader, by both CTAs)
  u64 hfull[2], hempty[2];             // rows' coefficients: there; read
  u64 done;
  uint32_t tmem;
  int gave_up;
};

// Returns the address of the pair's tensor memory, which `readers` warps of each CTA read.
__device__ __forceinline__ uint32_t pair_begin(Pipe &s, int readers) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMostStages; i++) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s.tfull[i], 1);
      mbar_init(&s.tempty[i], 2 * readers);
      mbar_init(&s.hfull[i], 2);
      mbar_init(&s.hempty[i], 8);
    }
    mbar_init(&s.done, 1);
    s.gave_up = 0;
    mbar_init_fence();
    async_proxy_fence();
  }
  if (threadIdx.x / 32 == 2) tmem_alloc(&s.tmem, 512);
  tmem_before_sync();
  cluster_sync();
  tmem_after_sync();
  return s.tmem;
}
// Neither CTA leaves while the other's products read its shared memory or its barriers are arrived on.  What
// arrives without a thread behind it is waited for before: copies (`full`) by the issuer, finished
// tiles (`tfull`) by both CTAs' readers, stages that were read (`empty`) by both CTAs' producers
// (Ring::drain).  Where a wait ran out that chain is broken: a millisecond is long enough for any of them.
// The host is told by `fault`.
__device__ __forceinline__ void pair_end(Pipe &s, uint32_t tmem, int *fault) {
  if (*const_cast<volatile int *>(&s.gave_up)) {
    if (fault) {
      *const_cast<volatile int *>(fault) = 1;
      __threadfence_system();
    }
    for (int i = 0; i < 1000; i++) __nanosleep(1000);
  }
  tmem_before_sync();
  __syncwarp();
  cluster_sync();
  tmem_after_sync();
  if (threadIdx.x / 32 == 2) tmem_free(tmem, 512);
}

// The producer's place in the ring of stages.
template <int STAGES>
struct Ring {
  Pipe &s;
  unsigned char *smem;
  volatile int *gave_up;
  int it = 0;

  // The next stage's operands and the leader's barrier for them; false when the wait ran out.
  __device__ __forceinline__ bool next(unsigned bytes, unsigned char *&a, unsigned char *&b, uint32_t &bar) {
    const int i = it % STAGES;
    if (!mbar_wait(&s.empty[i], (it / STAGES + 1) & 1, gave_up)) return false;
    it++;
    bar = in_leader(&s.full[i]);
    if (cluster_rank() == 0) mbar_arrive_expect_tx(&s.full[i], bytes);
    a = smem + i * kBytesStage;
    b = a + kBytesA;
    return true;
  }
  // The products tell both CTAs of each stage that they have read, the last ones too: a CTA that left before
  // would have them arrive in the shared memory of the next one on its SM.
  __device__ __forceinline__ bool drain() {
    bool ok = true;
    for (int i = max(0, it - STAGES); ok && i < it; i++) ok = mbar_wait(&s.empty[i % STAGES], (i / STAGES) & 1, gave_up);
    return ok;
  }
  // Copies in flight still write into this CTA's shared memory.
  __device__ __forceinline__ void settle() {
    int none = 0;
    if (cluster_rank() == 0)
      for (int i = max(0, it - STAGES); i < it; i++) mbar_wait(&s.full[i % STAGES], (i / STAGES) & 1, &none);
    else   // they are counted in the other CTA: a millisecond is long enough for any copy
      for (int i = 0; i < 1000; i++) __nanosleep(1000);
  }
};

// The issuing thread's place: products of the stages in their order.
template <int STAGES>
struct Issue {
  Pipe &s;
  volatile int *gave_up;
  uint32_t tmem;
  uint32_t smem;
  int stage = 0, phase = 0, local = 0;

  // A half of tensor memory to accumulate in; false when the wait ran out.
  __device__ __forceinline__ bool begin(uint32_t &d) {
    const int buf = local & 1;
    if (!mbar_wait(&s.tempty[buf], (local / 2 + 1) & 1, gave_up)) return false;
    tmem_after_sync();
    d = tmem + buf * 256;
    return true;
  }
  __device__ __forceinline__ void end() { mma_commit(&s.tfull[local++ & 1]); }
  // Descriptors of a stage whose rows run along K (`mn`) or across it.
  __device__ __forceinline__ uint64_t desc(int offset, bool mn) const { return smem_desc(smem + offset, mn ? 8192 : 16, 1024); }
  // One block of K: `steps` products of 16.
  template <bool WHOLE>
  __device__ __forceinline__ bool block(uint32_t d, uint64_t da0, uint64_t db0, uint32_t step_a, uint32_t step_b,
                                        uint32_t idesc, bool add, int steps) {
    if (!mbar_wait(&s.full[stage], phase, gave_up)) return false;
    tmem_after_sync();
    const uint64_t da = da0 + stage * (kBytesStage >> 4), db = db0 + stage * (kBytesStage >> 4);
    mma_f16(d, da, db, idesc, add);
    if (WHOLE || steps == kK / 16) {
#pragma unroll
      for (int i = 1; i < kK / 16; i++) mma_f16(d, da + i * step_a, db + i * step_b, idesc, true);
    } else {
      for (int i = 1; i < steps; i++) mma_f16(d, da + i * step_a, db + i * step_b, idesc, true);
    }
    mma_commit(&s.empty[stage]);
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
    return true;
  }
  // Products in flight still read shared memory.
  __device__ __forceinline__ void settle() {
    int none = 0;
    mma_commit(&s.done);
    mbar_wait(&s.done, 0, &none);
  }
};

// A reading warp's place: 32 rows of the halves of tensor memory, one after the other.
struct Reader {
  Pipe &s;
  volatile int *gave_up;
  uint32_t lanes, release[2];
  int local = 0;
  bool ok = true;

  __device__ __forceinline__ Reader(Pipe &pipe, volatile int *g, uint32_t tmem) : s(pipe), gave_up(g) {
    lanes = tmem + ((uint32_t)(threadIdx.x / 32 % 4 * 32) << 16);
    release[0] = in_leader(&s.tempty[0]);
    release[1] = in_leader(&s.tempty[1]);
  }
  __device__ __forceinline__ bool wait(u64 *bars) {
    ok = ok && mbar_wait(&bars[local & 1], (local / 2) & 1, gave_up);
    ok = __all_sync(kFullMask, ok);
    return ok;
  }
  __device__ __forceinline__ void begin() {
    wait(s.tfull);
    tmem_after_sync();
  }
  // A warp that gave up reads NaN: nothing that was not computed passes for a result.
  template <int N>
  __device__ __forceinline__ void fetch(int col, float (&x)[N]) const {
    if (ok) {
      if constexpr (N == 32) tmem_load32(lanes + (local & 1) * 256 + col, x);
      else tmem_load16(lanes + (local & 1) * 256 + col, x);
      tmem_wait_load();
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = __int_as_float(0x7fffffff);
    }
  }
  __device__ __forceinline__ void end() {
    tmem_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive_leader(release[local & 1]);
    local++;
  }
};

// The products of parts, the smaller ones first (the tensor cores truncate what they accumulate): the parts
// of A and of B in product q at bits 2 q.
struct Parts {
  int count;
  unsigned a, b;
  __device__ __forceinline__ int of_a(int q) const { return a >> 2 * q & 3; }
  __device__ __forceinline__ int of_b(int q) const { return b >> 2 * q & 3; }
};
__host__ __device__ constexpr unsigned part_list(int a, int b, int c, int d = 0, int e = 0, int f = 0) {
  return a | b << 2 | c << 4 | d << 6 | e << 8 | f << 10;
}
template <bool SPLIT, bool GRADIENTS>
__device__ __forceinline__ Parts parts_of(bool wide) {
  if (!SPLIT) return Parts{1, 0, 0};
  if (wide) return Parts{6, part_list(1, 2, 0, 1, 0, 0), part_list(1, 0, 2, 0, 1, 0)};
  // lo hi, hi lo, hi hi; of gradients (lo 2^11) (hi 2^-11), hi lo, hi hi
  return Parts{3, part_list(1, 0, 0), GRADIENTS ? part_list(2, 1, 0) : part_list(0, 1, 0)};
}

// ---- logits, and d ---------------------------------------------------------------------------
enum Use { kLogits, kProbs };

struct Product {
  CUtensorMap a, b;         // H and W
  int mt, nt;               // tiles
  int kblocks, k16;         // of 64 for one pair of parts; steps of 16 in the last one
  int a_part, b_part;       // from one part of an operand to the next
  int a_y, b_y;             // first row of each
  int bf16;
  const Scalars *sc;        // operands in parts carry its scales
  int64_t vocab;
  int rows;                 // rows that exist
  Part *parts;
  int64_t ldparts;
  const float *lse, *gloss;   // gloss: null where one factor is left to the end
  int given;                  // of prob_exp
  const int *targets;
  int labels;
  uint16_t *probs;          // d in strips of 64 columns: [part][strip][row][64], see put_strip
  int strip;                // rows of a strip
  int64_t prob_part;        // from one part to the next
  int *fault;               // of pair_end
};

template <bool BF16>
__device__ __forceinline__ uint32_t halves(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
  }
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}

// 32 values as 16 bits.
template <bool BF16>
__device__ __forceinline__ void pack32(const float *x, uint32_t *to) {
#pragma unroll
  for (int i = 0; i < 16; i++) to[i] = halves<BF16>(x[2 * i], x[2 * i + 1]);
}
// What 16-bit values lack of the 64 they were made from, times 2^11 for fp16, in their place.
template <bool BF16>
__device__ __forceinline__ void leave_rest(float (&x)[64], const uint32_t (&taken)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i++) {
    float a, b;
    if (BF16) unpack2(taken[i], a, b, __nv_bfloat16());
    else unpack2(taken[i], a, b, __half());
    x[2 * i] = (x[2 * i] - a) * (BF16 ? 1.f : 2048.f);
    x[2 * i + 1] = (x[2 * i + 1] - b) * (BF16 ? 1.f : 2048.f);
  }
}

// A warp's 32 rows of a strip, a row a lane, through shared memory to memory in one bulk copy of 4 KB.
// Each row's eight 16-byte pieces are put in the order that the operands of a product have in shared
// memory (piece j of row r at j ^ (r & 7)): no two lanes meet in a bank, and the loads need not swizzle.
// A row a lane straight to memory would take 62 passes of the L1 for 1 KB, as many as the tensor cores'
// own reads.
__device__ __forceinline__ void put_strip(unsigned char *buffer, uint16_t *to, const uint32_t (&x)[32]) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) bulk_wait_group_read<0>();   // the copy before this one has read the buffer
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; j++)
    *reinterpret_cast<uint4 *>(buffer + lane * 128 + ((j ^ (lane & 7)) * 16)) =
        make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
  async_proxy_fence();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], 4096;" ::"l"(to), "r"(smem_addr(buffer))
                 : "memory");
    bulk_commit_group();
  }
}

// Stages, and shared memory behind them: a strip's buffer for each warp that writes d.
template <Use USE>
constexpr int kProductStages = USE == kProbs ? 5 : 6;
template <Use USE>
constexpr int kProductSmem = smem_bytes(kProductStages<USE>, USE == kProbs ? 8 * 4096 : 0);

// SPLIT: fp32 operands in parts.
template <Use USE, bool SPLIT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmaThreads, 1) product_kernel(const __grid_constant__ Product p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  __shared__ Pipe pipe;
  __shared__ RowCoef coef_s[2][USE == kProbs ? kM : 1];
  volatile int *gave_up = &pipe.gave_up;
  constexpr int STAGES = kProductStages<USE>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t tmem = pair_begin(pipe, 8);
  const int rank = (int)cluster_rank(), pair = blockIdx.x / 2, npairs = gridDim.x / 2;
  const int tiles = p.mt * p.nt;
  const bool wide = SPLIT && p.sc->wide;
  const Parts parts = parts_of<SPLIT, false>(wide);
  // pairs that run together share a few tiles of W, against all rows
  auto first_row = [&](int t) { return t % p.mt * kPairM + rank * kM; };
  auto column_tile = [&](int t) { return t / p.mt; };

  if (warp == 0) {
    if (elected()) {
      Ring<STAGES> ring{pipe, smem, gave_up};
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += npairs) {
        const int row = p.a_y + first_row(t), col = p.b_y + column_tile(t) * kN + rank * (kN / 2);
        for (int q = 0; ok && q < parts.count; q++)
          for (int kb = 0; kb < p.kblocks; kb++) {
            unsigned char *a, *b;
            uint32_t bar;
            if (!(ok = ring.next(2 * kBytesStage, a, b, bar))) break;
            tma_load_2d(a, &p.a, parts.of_a(q) * p.a_part + kb * kK, row, bar);
            tma_load_2d(b, &p.b, parts.of_b(q) * p.b_part + kb * kK, col, bar);
          }
      }
      if (!ok || !ring.drain()) ring.settle();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elected()) {
      Issue<STAGES> issue{pipe, gave_up, tmem, smem_addr(smem)};
      bool ok = true;
      const uint32_t idesc = mma_desc(SPLIT ? wide : p.bf16, false, false, kPairM, kN);
      const uint64_t da = issue.desc(0, false), db = issue.desc(kBytesA, false);
      for (int t = pair; ok && t < tiles; t += npairs) {
        uint32_t d;
        if (!(ok = issue.begin(d))) break;
        bool add = false;
        for (int q = 0; ok && q < parts.count; q++)
          for (int kb = 0; ok && kb < p.kblocks; kb++) {
            ok = issue.template block<false>(d, da, db, 2, 2, idesc, add, kb == p.kblocks - 1 ? p.k16 : kK / 16);
            add = true;
          }
        if (ok) issue.end();
      }
      if (!ok) issue.settle();
    }
    __syncwarp();
  } else if (USE == kProbs && warp < 4) {
    // one tile ahead of the warps that read it: what they need of each row, so that they never wait
    // for global memory (ten targets a row cost as much as the tile itself)
    const float scale = pow2(prob_exp(p.sc, p.given));
    bool ok = true;
    int local = 0;
    for (int t = pair; ok && t < tiles; t += npairs, local++) {
      const int buf = local & 1;
      ok = __all_sync(kFullMask, mbar_wait(&pipe.hempty[buf], (local / 2 + 1) & 1, gave_up));
      const int64_t first = p.b_y + (int64_t)column_tile(t) * kN;
      for (int i = (warp - 2) * 32 + lane; ok && i < kM; i += 64) {
        const int64_t r = first_row(t) + i;
        RowCoef rc{INFINITY, 0.f, 0.f, 0u};   // a row without targets: exp2(l - inf) = 0, times 0
        if (r < p.rows) {
          const float lse = p.lse[r], g = (p.gloss ? p.gloss[r] : 1.f) * scale;
          const int *y = p.targets + r * p.labels;
          int k = 0;
          for (int j = 0; j < p.labels; j += 8) {
            int at[8];
#pragma unroll
            for (int q = 0; q < 8; q++) at[q] = j + q < p.labels ? y[j + q] : -1;
#pragma unroll
            for (int q = 0; q < 8; q++) {
              if (at[q] < 0 || at[q] >= p.vocab) continue;
              const int64_t c = at[q] - first;
              k++;
              if (c >= 0 && c < kN) rc.hits |= 1u << (c >> 5);
            }
          }
          if (k) {
            // lse log2e to twice the precision: what the rounded exponent lacks goes into the factor
            rc.lse2 = lse * kLog2e;
            rc.coef = g * (float)k * exp2f(-fmaf(lse, kLog2e, -rc.lse2));
            rc.g = g;
          }
        }
        coef_s[buf][i] = rc;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(smem_addr(&pipe.hfull[buf]));
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int half = (warp - 4) / 4, row = (warp & 3) * 32 + lane;
    float c = kLog2e;
    if (SPLIT) c = kLog2e * pow2(-scale_exp(p.sc->h, kOperandTop)) * pow2(-scale_exp(p.sc->w, kOperandTop));
    Reader reader(pipe, gave_up, tmem);
    for (int t = pair; t < tiles; t += npairs) {
      const int n = column_tile(t);
      const int64_t r = first_row(t) + row;
      const int64_t first = p.b_y + (int64_t)n * kN, left = p.vocab - first;   // columns of the tile that are words
      if (USE == kLogits) {
        reader.begin();
        Part part{-INFINITY, 0.f};
        for (int ch = half; ch < kN / 32; ch += 2) {
          float x[32];
          reader.fetch(ch * 32, x);
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
      } else {
        const bool there = reader.wait(pipe.hfull);
        const RowCoef rc = there ? coef_s[reader.local & 1][row] : RowCoef{INFINITY, 0.f, 0.f, 0u};
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(smem_addr(&pipe.hempty[reader.local & 1]));
        reader.begin();
        const int *y = p.targets + r * p.labels;
        unsigned char *buffer = smem + STAGES * kBytesStage + (warp - 4) * 4096;
        for (int strip = 2 * half; strip < 2 * half + 2; strip++) {
          uint32_t taken[32];
          float all[64];   // both halves of the strip, while parts of them are taken
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const int ch = 2 * strip + b;
            float x[32];
            reader.fetch(ch * 32, x);
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = exp2_fast(fmaf(x[i], c, -rc.lse2)) * rc.coef;
            if (left < kN) {
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (ch * 32 + i >= left) x[i] = 0.f;
            }
            if (__any_sync(kFullMask, rc.hits >> ch & 1)) {
              if (rc.hits >> ch & 1)
                for (int j = 0; j < p.labels; j++) {
                  const int64_t at = y[j] - first - ch * 32;
#pragma unroll
                  for (int i = 0; i < 32; i++) x[i] -= at == i ? rc.g : 0.f;
                }
              __syncwarp();
            }
            if (SPLIT) {
#pragma unroll
              for (int i = 0; i < 32; i++) all[32 * b + i] = x[i];
            } else if (p.bf16) {
              pack32<true>(x, taken + 16 * b);
            } else {
              pack32<false>(x, taken + 16 * b);
            }
          }
          uint16_t *to = p.probs + ((int64_t)(n * (kN / 64) + strip) * p.strip + r - lane) * 64;
          if (!SPLIT) {
            put_strip(buffer, to, taken);
          } else if (!wide) {
#pragma unroll
            for (int part = 0; part < 2; part++) {
              pack32<false>(all, taken);
              pack32<false>(all + 32, taken + 16);
              if (part == 0) leave_rest<false>(all, taken);
              put_strip(buffer, to + part * p.prob_part, taken);
            }
          } else {
#pragma unroll 1
            for (int part = 0; part < 3; part++) {
              pack32<true>(all, taken);
              pack32<true>(all + 32, taken + 16);
              leave_rest<true>(all, taken);
              put_strip(buffer, to + part * p.prob_part, taken);
            }
          }
        }
      }
      reader.end();
    }
    if (USE == kProbs && lane == 0) bulk_wait_group_all();
  }
  pair_end(pipe, tmem, p.fault);
}

// ---- gradients from a piece of d -------------------------------------------------------------
//
// One launch computes the tiles of both gradients.  The pairs take whole tiles in turn (those that run
// together share a strip of d) as long as there is one for each; what is left of both is cut into equal
// shares of blocks of K, so that all pairs finish together, whatever the sizes.  A tile that was cut
// leaves its pieces in memory, at most two a pair, and pieces_kernel adds them in their order.
struct Side {
  CUtensorMap a, b;         // d or its transpose, and the operand
  int kblocks, tiles, whole;// of 64; tiles, and how many each pair takes whole
  int a_mn;                 // d transposed
  int b_y;                  // first row of the operand
  int a_part, b_part;       // from one part of d and of the operand to the next
  int rows;
  float *acc;               // sums of earlier launches, or of this one for later ones
  int add, last;
  void *out;
  int64_t ldout;
  int out_wide;
  Rescale rescale;
  __host__ __device__ __forceinline__ int rest(int npairs) const { return tiles > whole * npairs ? tiles - whole * npairs : 0; }
};

struct Gradients {
  Side side[2];             // dW, dH
  int nt, ntile, nlast;     // column tiles, their width and the last one's (multiples of 32)
  int npairs, sharers;      // pairs of CTAs; how many of them share what is left
  int64_t left;             // its blocks of K
  int bf16, strip, dim, out_type;
  int64_t ldacc;
  float *pieces;            // [pair][2][kPairM][ntile]
  int *fault;               // of pair_end
  __device__ __forceinline__ int width(int n) const { return n == nt - 1 ? nlast : ntile; }
};

struct Piece {
  int side, tile, k0, k1, slot;   // slot -1: a whole tile; 0: it was begun by another pair; 1: begun here
};

__host__ __device__ __forceinline__ int64_t share_begin(const Gradients &g, int pair) { return pair * g.left / g.sharers; }

// The side, tile and block of K at a place in what is left.  A tile counts for kReading blocks more than
// it has: what reading it from tensor memory takes.
constexpr int kReading = 8;
__device__ __forceinline__ void place(const Gradients &g, int64_t at, int &side, int &tile, int &k) {
  const int64_t first = (int64_t)g.side[0].rest(g.npairs) * (g.side[0].kblocks + kReading);
  side = at >= first;
  const int64_t q = side ? at - first : at;
  const Side &s = g.side[side];
  tile = s.whole * g.npairs + (int)(q / (s.kblocks + kReading));
  k = (int)(q % (s.kblocks + kReading));
}

struct Walk {
  const Gradients &g;
  int pair, i = 0;
  int64_t at, end;

  __device__ __forceinline__ Walk(const Gradients &grads, int p) : g(grads), pair(p) {
    at = p < g.sharers ? share_begin(g, p) : 0;
    end = p < g.sharers ? share_begin(g, p + 1) : 0;
  }
  __device__ __forceinline__ bool next(Piece &p) {
    const int w0 = g.side[0].whole, w1 = g.side[1].whole;
    while (i < w0 + w1) {
      p.side = i >= w0;
      p.tile = (i - (p.side ? w0 : 0)) * g.npairs + pair;
      p.k0 = 0;
      p.k1 = g.side[p.side].kblocks;
      p.slot = -1;
      i++;
      if (p.tile < g.side[p.side].tiles) return true;
    }
    while (at < end) {
      place(g, at, p.side, p.tile, p.k0);
      const int all = g.side[p.side].kblocks, to = (int)min((int64_t)(all + kReading), p.k0 + (end - at));
      at += to - p.k0;
      p.k1 = min(all, to);
      p.slot = p.k0 == 0 ? (p.k1 == all ? -1 : 1) : 0;
      if (p.k0 < p.k1) return true;
    }
    return false;
  }
};

template <typename T>
__device__ __forceinline__ void put16(T *to, const float (&v)[16]) {
#pragma unroll
  for (int b = 0; b < 2; b++) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = v[b * 8 + e];
    store8(to + b * 8, x);
  }
}

// A column of every other row, from row `first`, of the `rows` that exist.
template <typename T>
__device__ __forceinline__ void put_rows(T *to, int64_t step, const float *from, int first, int rows) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = from[i * 34];
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (first + 2 * i < rows) to[i * step] = from_float<T>(x[i]);
}

// 32 rows x 16 columns of a finished tile, a row a lane (row0: lane 0's).  Rows that no wide store fits
// go through `stage`, 32 x 17 floats of this warp's, so that half a warp writes a row's 16 in one piece.
__device__ __forceinline__ void put_tile(const Gradients &g, const Side &s, int64_t row0, int at, const float *x, float factor,
                                         float *stage) {
  if (at >= g.dim) return;
  const int lane = threadIdx.x & 31;
  const int64_t r = row0 + lane;
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; e++) v[e] = x[e];
  float *acc = s.acc + r * g.ldacc + at;
  if (s.add && r < s.rows) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      float old[8];
      load8(acc + b * 8, old);
#pragma unroll
      for (int e = 0; e < 8; e++) v[b * 8 + e] += old[e];
    }
  }
  if (!s.last) {
    if (r < s.rows) put16(acc, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; e++) v[e] *= factor;
  if (s.out_wide && at + 16 <= g.dim) {
    if (r >= s.rows) return;
    const int64_t to = r * s.ldout + at;
    if (g.out_type == W2V_F32) put16(static_cast<float *>(s.out) + to, v);
    else if (g.out_type == W2V_BF16) put16(static_cast<__nv_bfloat16 *>(s.out) + to, v);
    else put16(static_cast<__half *>(s.out) + to, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; e++) stage[lane * 17 + e] = v[e];
  __syncwarp();
  const int c = lane % 16, first = lane / 16;
  const int rows = at + c < g.dim ? (int)max((int64_t)0, min((int64_t)32, s.rows - row0)) : 0;
  const int64_t to = (row0 + first) * s.ldout + at + c;
  const float *from = stage + first * 17 + c;
  if (g.out_type == W2V_F32) put_rows(static_cast<float *>(s.out) + to, 2 * s.ldout, from, first, rows);
  else if (g.out_type == W2V_BF16) put_rows(static_cast<__nv_bfloat16 *>(s.out) + to, 2 * s.ldout, from, first, rows);
  else put_rows(static_cast<__half *>(s.out) + to, 2 * s.ldout, from, first, rows);
  __syncwarp();
}

// Blocks of K that are accumulated in tensor memory at a time: all, or for SEGMENTS (fp32) as many as have
// six products.
template <bool SEGMENTS>
__device__ __forceinline__ int segment_of(bool wide) { return !SEGMENTS ? 1 << 30 : wide ? 1 : 2; }

constexpr int kGradStages = 5, kGradSmem = smem_bytes(kGradStages, 0);

// SEGMENTS (fp32): the tensor cores truncate what they accumulate, so after `segment` blocks of K the sum
// moves to registers, where it is rounded: sixteen warps, 64 columns of a row a lane.  dH of 4096 x 100000
// x 256 is then 1.2e-6 off in norm (2 blocks; 4: 2.7e-6, 8: 5.8e-6; an fp32 product: 6.5e-6), dW 1.6e-7 (fp32
// product 5.4e-7), and takes 2.26 ms (4 blocks: 2.20).
template <bool SEGMENTS>
constexpr int kGradReaders = SEGMENTS ? 16 : 8;
template <bool SEGMENTS>
constexpr int kGradThreads = 128 + 32 * kGradReaders<SEGMENTS>;

template <bool SEGMENTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGradThreads<SEGMENTS>, 1) grad_kernel(const __grid_constant__ Gradients g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  __shared__ Pipe pipe;
  __shared__ float stage_s[kGradReaders<SEGMENTS>][32 * 17];
  volatile int *gave_up = &pipe.gave_up;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const uint32_t tmem = pair_begin(pipe, kGradReaders<SEGMENTS>);
  const int rank = (int)cluster_rank();
  const bool wide = SEGMENTS && g.side[0].rescale.sc->wide;
  const Parts parts = parts_of<SEGMENTS, true>(wide);
  const int segment = segment_of<SEGMENTS>(wide);
  Walk walk(g, blockIdx.x / 2);
  Piece p;

  if (warp == 0) {
    if (elected()) {
      Ring<kGradStages> ring{pipe, smem, gave_up};
      bool ok = true;
      // each CTA brings its own rows of d and half of the operand's columns
      while (ok && walk.next(p)) {
        const Side &s = g.side[p.side];
        const int half_n = g.width(p.tile % g.nt) / 2, groups = (half_n + 63) / 64;
        const unsigned bytes = 2 * (kBytesA + groups * 8192);
        const int row = p.tile / g.nt * kPairM + rank * kM, col = p.tile % g.nt * g.ntile + rank * half_n;
        for (int k0 = p.k0; ok && k0 < p.k1; k0 += segment)
          for (int q = 0; ok && q < parts.count; q++)
            for (int kb = k0; kb < min(p.k1, k0 + segment); kb++) {
              unsigned char *a, *b;
              uint32_t bar;
              if (!(ok = ring.next(bytes, a, b, bar))) break;
              const int a_at = parts.of_a(q) * s.a_part;
              if (s.a_mn) {   // 64 rows of two strips
                for (int i = 0; i < 2; i++)
                  tma_load_2d(a + i * 8192, &s.a, 0, a_at + (row / 64 + i) * g.strip + kb * kK, bar);
              } else {        // 128 rows of a strip
                tma_load_2d(a, &s.a, 0, a_at + kb * g.strip + row, bar);
              }
              for (int i = 0; i < groups; i++)
                tma_load_2d(b + i * 8192, &s.b, parts.of_b(q) * s.b_part + col + i * 64, s.b_y + kb * kK, bar);
            }
      }
      if (!ok || !ring.drain()) ring.settle();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elected()) {
      Issue<kGradStages> issue{pipe, gave_up, tmem, smem_addr(smem)};
      bool ok = true;
      while (ok && walk.next(p)) {
        const bool mn = g.side[p.side].a_mn;
        const uint32_t idesc = mma_desc(SEGMENTS ? wide : g.bf16, mn, true, kPairM, g.width(p.tile % g.nt));
        const uint64_t da = issue.desc(0, mn), db = issue.desc(kBytesA, true);
        const uint32_t step_a = mn ? 2048 >> 4 : 32 >> 4;
        for (int k0 = p.k0; ok && k0 < p.k1; k0 += segment) {
          uint32_t d;
          if (!(ok = issue.begin(d))) break;
          const int blocks = parts.count * (min(p.k1, k0 + segment) - k0);
          for (int b = 0; ok && b < blocks; b++) ok = issue.template block<true>(d, da, db, step_a, 2048 >> 4, idesc, b > 0, kK / 16);
          if (ok) issue.end();
        }
      }
      if (!ok) issue.settle();
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int part = (warp - 4) / 4, row = (warp & 3) * 32;
    float *stage = stage_s[warp - 4];
    const float factor[2] = {rescale_of(g.side[0].rescale), rescale_of(g.side[1].rescale)};
    Reader reader(pipe, gave_up, tmem);
    while (walk.next(p)) {
      const Side &s = g.side[p.side];
      const int n = p.tile % g.nt, width = g.width(n);
      const int64_t row0 = (int64_t)(p.tile / g.nt) * kPairM + rank * kM + row;
      float *piece = g.pieces + ((int64_t)(walk.pair * 2 + max(p.slot, 0)) * kPairM + rank * kM + row + lane) * g.ntile;
      // 16 columns of the sum over the piece
      auto finish = [&](int col, const float *x) {
        if (p.slot < 0) {
          put_tile(g, s, row0, n * g.ntile + col, x, factor[p.side], stage);
        } else {
#pragma unroll
          for (int b = 0; b < 2; b++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = x[b * 8 + e];
            store8(piece + col + b * 8, v);
          }
        }
      };
      if (!SEGMENTS) {
        reader.begin();
        for (int ch = part; ch < width / 32; ch += 2) {
          float x[32];
          reader.fetch(ch * 32, x);
          finish(ch * 32, x);
          finish(ch * 32 + 16, x + 16);
        }
        reader.end();
      } else {
        float acc[4][16];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int e = 0; e < 16; e++) acc[i][e] = 0.f;
        for (int k0 = p.k0; k0 < p.k1; k0 += segment) {
          reader.begin();
          if (part * 64 < width) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              float x[16];
              reader.fetch(part * 64 + i * 16, x);
#pragma unroll
              for (int e = 0; e < 16; e++) acc[i][e] += x[e];
            }
          }
          reader.end();
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (part * 64 + i * 16 < width) finish(part * 64 + i * 16, acc[i]);
      }
    }
  }
  pair_end(pipe, tmem, g.fault);
}

// The tiles that were cut: blockIdx.x is the tile in what is left, a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) pieces_kernel(const __grid_constant__ Gradients g) {
  chain_wait();
  const int t = blockIdx.x, rest0 = g.side[0].rest(g.npairs);
  const Side &s = g.side[t >= rest0];
  const int64_t begin = t < rest0 ? (int64_t)t * (g.side[0].kblocks + kReading)
                                  : (int64_t)rest0 * (g.side[0].kblocks + kReading) +
                                        (int64_t)(t - rest0) * (g.side[1].kblocks + kReading);
  // the pair whose share holds a place: the last one that begins at or before it
  auto pair_at = [&](int64_t at) { return (int)(((at + 1) * g.sharers - 1) / g.left); };
  const int first = pair_at(begin), last = pair_at(begin + s.kblocks - 1);
  if (first == last) return;
  const int tile = s.whole * g.npairs + (t < rest0 ? t : t - rest0);
  const int row = blockIdx.y * 8 + threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)(tile / g.nt) * kPairM + row;
  if (r >= s.rows) return;
  const float factor = rescale_of(s.rescale);
  const int col = lane * 8, at = tile % g.nt * g.ntile + col;
  if (col >= g.width(tile % g.nt) || at >= g.dim) return;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int q = first; q <= last; q += 4) {
    float x[4][8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int pair = min(q + j, last);
      load8(g.pieces + ((int64_t)(pair * 2 + (pair == first)) * kPairM + row) * g.ntile + col, x[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (q + j <= last) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += x[j][e];
      }
  }
  float *acc = s.acc + r * g.ldacc + at;
  if (s.add) {
    float old[8];
    load8(acc, old);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += old[e];
  }
  if (!s.last) {
    store8(acc, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] *= factor;
  T *to = static_cast<T *>(s.out) + r * s.ldout + at;
  const int have = min(8, g.dim - at);
  if (s.out_wide && have == 8) store8(to, v);
  else store_some(to, have, v);
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

// A matrix of 16-bit elements, `inner` a row, rows `ld` elements apart; boxes of 64 x box_rows, which arrive with the
// 128-byte swizzle of a product's operands unless they are `swizzled` in memory.
int tensor_map(CUtensorMap *map, const void *base, int64_t inner, int64_t rows, int64_t ld, int box_rows,
               bool swizzled = false) {
  const EncodeTiled encode = encoder();
  if (!encode) return (int)cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult e = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return e == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// An operand as the products read it.
struct Operand {
  const void *p;
  int64_t ld, inner, rows;
  int width;   // offset between parts
};

// The kernels that work in pairs of CTAs with tensor memory are launched in the ordinary way, each after
// its predecessor has ended; started early like the others (w2v_chain.cuh), short ones in a row were seen
// to stop now and then, from a cause that reading has not shown.  Every wait of theirs on a barrier in shared
// memory is bounded.  What is not: tcgen05.alloc, which never waits (a CTA's shared memory leaves no room
// for a second one with tensor memory on its SM), the barriers of the pair, which all threads of both CTAs
// reach, and the wait for the predecessor, of which no two kernels can form a circle.

// An attribute of the function on the current device, set once for each (a call costs a microsecond).
template <auto KERNEL>
int allow_smem(size_t bytes) {
  constexpr int kDevices = 64;
  static std::atomic<size_t> allowed[kDevices];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  if (device < kDevices && allowed[device].load() >= bytes) return 0;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && device < kDevices) allowed[device].store(bytes);
  return (int)e;
}
// Raised by a kernel that gave up waiting: pinned host memory that every device can write, null where there
// is none.
int *fault_flag() {
  static int *flag = [] {
    int *f = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // the first call may be captured
    cudaThreadExchangeStreamCaptureMode(&mode);
    const cudaError_t e = cudaHostAlloc(&f, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return (int *)nullptr;
    }
    *f = 0;
    return f;
  }();
  return flag;
}
// Reported once, by the first call that finds the flag raised.
int take_fault() {
  int *flag = fault_flag();
  if (!flag || !*const_cast<volatile int *>(flag)) return 0;
  *flag = 0;
  return (int)cudaErrorLaunchTimeout;
}

int sm_pairs() { return std::max(1, device_sm_count() / 2); }

template <Use USE, typename T>
int launch_product(const Product &p, cudaStream_t s) {
  constexpr bool split = sizeof(T) == 4;
  const int err = allow_smem<product_kernel<USE, split>>(kProductSmem<USE>);
  if (err) return err;
  product_kernel<USE, split><<<2 * std::min(p.mt * p.nt, sm_pairs()), kMmaThreads, kProductSmem<USE>, s>>>(p);
  count_launch(1);
  return (int)cudaGetLastError();
}

template <typename T>
int launch_gradients(const Gradients &g, cudaStream_t s) {
  constexpr bool split = sizeof(T) == 4;
  int err = allow_smem<grad_kernel<split>>(kGradSmem);
  if (err) return err;
  const bool whole = g.side[0].whole || g.side[1].whole;
  grad_kernel<split><<<2 * (whole ? g.npairs : g.sharers), kGradThreads<split>, kGradSmem, s>>>(g);
  count_launch(1);
  err = (int)cudaGetLastError();
  const int rest = g.side[0].rest(g.npairs) + g.side[1].rest(g.npairs);
  if (!err && rest > 0 && g.sharers > 1) err = launch_chained(pieces_kernel<T>, dim3(rest, kPairM / 8), 256, 0, s, g);
  return err;
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
constexpr int64_t kProbBytes = (int64_t)256 << 20;

int few_blocks(int64_t vocab) {
  const int64_t need = (vocab + kFewThreads / 32 * kFewWords - 1) / (kFewThreads / 32 * kFewWords);
  return (int)std::min<int64_t>(need, (int64_t)device_sm_count() * 2);
}
int few_dh_blocks(int64_t vocab) {
  return (int)std::min<int64_t>((vocab + 31) / 32, (int64_t)device_sm_count());
}
int few_rows_of(int64_t n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8; }
bool few_rows(const Shape &x, bool grad, bool direct_w) {
  if (x.type == W2V_F32) return x.n <= 2 * kFewRows;
  return x.n <= kFewRows16 && (grad || !direct_w || x.dim <= 256);
}

struct Layout {
  int64_t scalars, hs, ws, parts, probs, pieces, acc_h, acc_w, total;
  int width, nparts;         // staged operands
  int64_t rows, words;       // of a piece of d
  int nt, ntile, nlast;
  bool few;
};

// Column tiles of a gradient: as wide as they can be, the rest in a last one.  A block of K of any width up
// to 128 + 128 columns costs at least the time that d's part of it takes to arrive, so two of 160 take
// as long as two of 256 (301 columns at 1023 x 50021: 94 us as 160 + 160, 87 as 256 + 64).
void column_tiles(int dim, int *nt, int *ntile, int *nlast) {
  *nt = (dim + kN - 1) / kN;
  *nlast = (int)up(dim - (*nt - 1) * kN, 32);
  *ntile = *nt > 1 ? kN : *nlast;
}

bool direct(int type, const void *p, int64_t ld) {   // TMA can read the caller's matrix
  return type != W2V_F32 && aligned(p, 16) && ld % 8 == 0;
}

// `direct_h`, `direct_w`: operands that TMA reads where they lie, so that no copy of them is made.
Layout plan(const Shape &x, bool grad, bool direct_h, bool direct_w) {
  Layout l{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(std::max<int64_t>(bytes, 1), 1024);
    return here;
  };
  l.scalars = take(sizeof(Scalars));
  l.few = few_rows(x, grad, direct_w);
  if (l.few) {
    const int rb = few_rows_of(x.n);
    if (!grad) {
      l.parts = take((int64_t)few_blocks(x.vocab) * rb * sizeof(Part));
    } else {
      l.probs = take(x.vocab * rb * 4);
      l.acc_h = take((int64_t)few_dh_blocks(x.vocab) * rb * x.dim * 4);
    }
    l.total = at;
    return l;
  }
  l.width = (int)up(x.dim, 64);
  l.nparts = x.type == W2V_F32 ? 3 : 1;
  l.hs = take(direct_h ? 0 : x.n * l.width * l.nparts * 2);
  l.ws = take(direct_w ? 0 : x.vocab * l.width * l.nparts * 2);
  if (!grad) {
    l.parts = take(2 * ((x.vocab + kN - 1) / kN) * std::min(x.n, kLossRows) * sizeof(Part));
  } else {
    const int bytes = x.type == W2V_F32 ? 4 : 2;
    l.rows = up(std::min(x.n, kGradRows), kPairM);
    // pieces of the vocabulary of equal width, up to a quarter more than kProbBytes
    const int64_t most = std::max<int64_t>(kN, kProbBytes / (l.rows * bytes));
    const int64_t pieces = std::max<int64_t>(1, (x.vocab + most * 5 / 4 - 1) / (most * 5 / 4));
    l.words = up((x.vocab + pieces - 1) / pieces, kN);
    column_tiles(x.dim, &l.nt, &l.ntile, &l.nlast);
    const int64_t cols = (int64_t)l.nt * l.ntile * 4;
    l.probs = take(l.rows * l.words * 2 * l.nparts);
    l.pieces = take((int64_t)sm_pairs() * 2 * kPairM * l.ntile * 4);
    if (l.words < x.vocab) l.acc_h = take(l.rows * cols);
    if (l.rows < x.n) l.acc_w = take(up(x.vocab, kPairM) * cols);
  }
  l.total = at;
  return l;
}

// Operands for the products: the caller's own where TMA can read them, else staged ones.
template <typename T>
int stage(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const float *gloss,
          const int *targets, int parts, char *ws, Operand *oh, Operand *ow, cudaStream_t s) {
  constexpr bool split = sizeof(T) == 4;
  Scalars *sc = reinterpret_cast<Scalars *>(ws + l.scalars);
  const Source sh{h, ldh, x.n}, sw{w, ldw, x.vocab};
  const int blocks = device_sm_count() * 8;
  if (split || gloss) {
    const cudaError_t e = cudaMemsetAsync(sc, 0, sizeof(Scalars), s);
    if (e != cudaSuccess) return (int)e;
    const Source none{nullptr, 0, x.n};
    const int err = launch_chained(amax_kernel, dim3(split ? blocks : 64, 1, 3), 256, 0, s, split ? sh : none,
                                   split ? sw : Source{nullptr, 0, 0}, x.dim, gloss, targets, x.labels, x.vocab, sc);
    if (err) return err;
  }
  uint16_t *hs = direct(x.type, h, ldh) ? nullptr : reinterpret_cast<uint16_t *>(ws + l.hs);
  uint16_t *wst = direct(x.type, w, ldw) ? nullptr : reinterpret_cast<uint16_t *>(ws + l.ws);
  const int64_t staged = (int64_t)l.width * l.nparts;
  if (hs || wst) {
    const int err = launch_chained(stage_kernel<T>, dim3(blocks, 1, 2), 256, 0, s, sh, sw, x.dim, hs, wst, l.width, staged, parts, sc);
    if (err) return err;
  }
  *oh = hs ? Operand{hs, staged, staged, x.n, l.width} : Operand{h, ldh, x.dim, x.n, 0};
  *ow = wst ? Operand{wst, staged, staged, x.vocab, l.width} : Operand{w, ldw, x.dim, x.vocab, 0};
  return 0;
}

template <typename T>
int logits_product(const Shape &x, const Operand &oh, const Operand &ow, const Scalars *sc, Product *to) {
  Product p{};
  int err = tensor_map(&p.a, oh.p, oh.inner, oh.rows, oh.ld, kM);
  if (!err) err = tensor_map(&p.b, ow.p, ow.inner, ow.rows, ow.ld, kN / 2);
  p.kblocks = (x.dim + kK - 1) / kK;
  p.k16 = (x.dim - (p.kblocks - 1) * kK + 15) / 16;
  p.a_part = oh.width;
  p.b_part = ow.width;
  p.bf16 = x.type == W2V_BF16;
  p.fault = fault_flag();
  p.sc = sc;
  p.vocab = x.vocab;
  *to = p;
  return err;
}

template <typename T, int RB>
int few_loss(const Shape &x, const Layout &l, const T *h, int64_t ldh, int rows, const void *w, int64_t ldw, char *ws,
             int *count, cudaStream_t s) {
  const size_t smem = (size_t)RB * few_steps(x.dim) * 1024;
  const auto k = few_loss_kernel<T, RB>;
  const int refused = allow_smem<few_loss_kernel<T, RB>>((size_t)RB * few_steps(kMaxDim) * 1024);
  if (refused) return refused;
  const bool wide = aligned(w, 8 * sizeof(T)) && ldw % 8 == 0;
  *count = few_blocks(x.vocab);
  return launch_chained(k, *count, kFewThreads, smem, s, h, ldh, rows,
                        static_cast<const T *>(w), ldw, x.vocab, x.dim, wide, reinterpret_cast<Part *>(ws + l.parts));
}

template <typename T>
int run_loss(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const int *targets,
             float *loss, float *lse, char *ws, cudaStream_t s) {
  Part *parts = reinterpret_cast<Part *>(ws + l.parts);
  const bool wide = aligned(h, 8 * sizeof(T)) && ldh % 8 == 0 && aligned(w, 8 * sizeof(T)) && ldw % 8 == 0;
  auto join_rows = [&](int count, int64_t ldp, int64_t r0, int rows) {
    return launch_chained(loss_join_kernel<T>, (rows + kJoinRows - 1) / kJoinRows, kJoinThreads, 0, s, parts, count, ldp,
                          rows, static_cast<const T *>(h) + r0 * ldh, ldh, static_cast<const T *>(w), ldw, x.vocab, x.dim,
                          wide, targets + r0 * x.labels, x.labels, loss + r0, lse + r0);
  };
  if (l.few) {
    int err = 0;
    for (int64_t r0 = 0; r0 < x.n && !err; r0 += kFewRows) {
      const int rows = (int)std::min<int64_t>(kFewRows, x.n - r0);
      const T *hr = static_cast<const T *>(h) + r0 * ldh;
      int count = 0;
      switch (few_rows_of(rows)) {
        case 1: err = few_loss<T, 1>(x, l, hr, ldh, rows, w, ldw, ws, &count, s); break;
        case 2: err = few_loss<T, 2>(x, l, hr, ldh, rows, w, ldw, ws, &count, s); break;
        case 4: err = few_loss<T, 4>(x, l, hr, ldh, rows, w, ldw, ws, &count, s); break;
        default:
          if constexpr (sizeof(T) == 4) err = few_loss<T, 8>(x, l, hr, ldh, rows, w, ldw, ws, &count, s);
      }
      if (!err) err = join_rows(count, rows, r0, rows);
    }
    return err;
  }
  Operand oh, ow;
  int err = stage<T>(x, l, h, ldh, w, ldw, nullptr, nullptr, 2, ws, &oh, &ow, s);
  if (err) return err;
  Product p;
  err = logits_product<T>(x, oh, ow, reinterpret_cast<const Scalars *>(ws + l.scalars), &p);
  if (err) return err;
  p.nt = (int)((x.vocab + kN - 1) / kN);
  p.parts = parts;
  for (int64_t r0 = 0; r0 < x.n; r0 += kLossRows) {
    p.rows = (int)std::min(kLossRows, x.n - r0);
    p.mt = (p.rows + kPairM - 1) / kPairM;
    p.a_y = (int)r0;
    p.ldparts = p.rows;
    err = launch_product<kLogits, T>(p, s);
    if (!err) err = join_rows(2 * p.nt, p.ldparts, r0, p.rows);
    if (err) return err;
  }
  return 0;
}

template <typename T, int RB>
int few_grad(const Shape &x, const Layout &l, const void *h, int64_t ldh, int64_t r0, int rows, const void *w, int64_t ldw,
             const int *targets, const float *lse, const float *gloss, int64_t ldg, void *dh, int64_t lddh, void *dw,
             int64_t lddw, char *ws, cudaStream_t s) {
  const size_t smem = (size_t)RB * few_steps(x.dim) * 1024;
  const auto k = few_grad_kernel<T, RB>;
  const int refused = allow_smem<few_grad_kernel<T, RB>>((size_t)RB * few_steps(kMaxDim) * 1024);
  if (refused) return refused;
  const bool wide = aligned(w, 8 * sizeof(T)) && ldw % 8 == 0, wout = aligned(dw, 8 * sizeof(T)) && lddw % 8 == 0;
  float *d = reinterpret_cast<float *>(ws + l.probs), *acc = reinterpret_cast<float *>(ws + l.acc_h);
  const T *wt = static_cast<const T *>(w);
  int err = launch_chained(k, few_blocks(x.vocab), kFewThreads, smem, s, static_cast<const T *>(h) + r0 * ldh, ldh, rows,
                           wt, ldw, x.vocab, x.dim, wide, targets + r0 * x.labels, x.labels, lse + r0, gloss + r0 * ldg, ldg,
                           static_cast<T *>(dw), lddw, wout, r0 > 0, d);
  const int blocks = few_dh_blocks(x.vocab);
  if (!err)
    err = launch_chained(few_dh_kernel<T, RB>, dim3(blocks, (x.dim + 255) / 256), kFewThreads, 0, s, wt, ldw, x.vocab, x.dim,
                         wide, d, acc);
  if (!err)
    err = launch_chained(slabs_kernel<T>, dim3((x.dim + 31) / 32, rows), 256, 0, s, acc, blocks, (int64_t)RB * x.dim, x.dim,
                         static_cast<T *>(dh) + r0 * lddh, lddh);
  return err;
}

template <typename T>
int run_grad(const Shape &x, const Layout &l, const void *h, int64_t ldh, const void *w, int64_t ldw, const int *targets,
             const float *lse, const float *gloss, int64_t ldg, void *dh, int64_t lddh, void *dw, int64_t lddw, char *ws,
             cudaStream_t s) {
  if (x.n == 0) return (int)cudaMemset2DAsync(dw, lddw * sizeof(T), 0, x.dim * sizeof(T), x.vocab, s);
  if (l.few) {
    int err = 0;
    for (int64_t r0 = 0; r0 < x.n && !err; r0 += kFewRows) {
      const int rows = (int)std::min<int64_t>(kFewRows, x.n - r0);
      auto go = [&](auto rb) {
        return few_grad<T, decltype(rb)::value>(x, l, h, ldh, r0, rows, w, ldw, targets, lse, gloss, ldg, dh, lddh, dw, lddw,
                                                ws, s);
      };
      switch (few_rows_of(rows)) {
        case 1: err = go(std::integral_constant<int, 1>()); break;
        case 2: err = go(std::integral_constant<int, 2>()); break;
        case 4: err = go(std::integral_constant<int, 4>()); break;
        default:
          if constexpr (sizeof(T) == 4) err = go(std::integral_constant<int, 8>());
      }
    }
    return err;
  }
  constexpr bool split = sizeof(T) == 4;
  const float *each_gloss = ldg ? gloss : nullptr, *one_gloss = ldg ? nullptr : gloss;
  Operand oh, ow;
  int err = stage<T>(x, l, h, ldh, w, ldw, each_gloss, targets, 3, ws, &oh, &ow, s);
  if (err) return err;
  const Scalars *sc = reinterpret_cast<const Scalars *>(ws + l.scalars);
  // one factor for all rows is left to the end: the targets' -1 then has no rounding in d
  int given = kFromRows;
  if (one_gloss)
    for (given = kProbTop; (1 << (kProbTop - given)) < x.labels;) given--;
  // d lies in strips of 64 columns, 128 bytes a row: what a warp writes of a tile, and what a load of
  // either gradient's operand reads, is one piece of memory
  const int strip_rows = (int)(l.words / 64 * l.rows);
  Product p;
  err = logits_product<T>(x, oh, ow, sc, &p);
  p.labels = x.labels;
  p.given = given;
  p.probs = reinterpret_cast<uint16_t *>(ws + l.probs);
  p.strip = (int)l.rows;
  p.prob_part = (int64_t)strip_rows * 64;

  Gradients g{};
  g.nt = l.nt;
  g.ntile = l.ntile;
  g.nlast = l.nlast;
  g.npairs = sm_pairs();
  g.bf16 = x.type == W2V_BF16;
  g.strip = (int)l.rows;
  g.dim = x.dim;
  g.out_type = x.type;
  g.ldacc = (int64_t)l.nt * l.ntile;
  g.pieces = reinterpret_cast<float *>(ws + l.pieces);
  g.fault = p.fault;
  for (int i = 0; i < 2 && !err; i++) {
    Side &side = g.side[i];
    const Operand &o = i == 0 ? oh : ow;
    side.a_mn = i == 0;
    err = tensor_map(&side.a, ws + l.probs, 64, (int64_t)strip_rows * l.nparts, 64, side.a_mn ? 64 : kM, true);
    if (!err) err = tensor_map(&side.b, o.p, o.inner, o.rows, o.ld, 64);
    side.a_part = strip_rows;
    side.b_part = o.width;
    side.rescale = Rescale{sc, one_gloss, given, split ? (i == 0 ? 2 : 1) : 0};
    side.ldout = i == 0 ? lddw : lddh;
  }
  if (err) return err;
  float *acc_h = reinterpret_cast<float *>(ws + l.acc_h), *acc_w = reinterpret_cast<float *>(ws + l.acc_w);
  for (int64_t r0 = 0; r0 < x.n; r0 += l.rows) {
    const int rows = (int)std::min(l.rows, x.n - r0);
    for (int64_t v0 = 0; v0 < x.vocab; v0 += l.words) {
      const int words = (int)std::min(l.words, x.vocab - v0);
      p.mt = (rows + kPairM - 1) / kPairM;
      p.nt = (words + kN - 1) / kN;
      p.a_y = (int)r0;
      p.b_y = (int)v0;
      p.rows = rows;
      p.lse = lse + r0;
      p.gloss = each_gloss ? each_gloss + r0 : nullptr;
      p.targets = targets + r0 * x.labels;
      err = launch_product<kProbs, T>(p, s);
      if (err) return err;
      g.left = 0;
      for (int i = 0; i < 2; i++) {
        Side &side = g.side[i];
        side.rows = i == 0 ? words : rows;
        side.kblocks = ((i == 0 ? rows : words) + kK - 1) / kK;
        side.tiles = (i == 0 ? (words + kPairM - 1) / kPairM : p.mt) * l.nt;
        // tiles of few blocks of K are not worth cutting: reading one costs as much
        side.whole = side.kblocks < 16 ? (side.tiles + g.npairs - 1) / g.npairs : side.tiles / g.npairs;
        side.b_y = (int)(i == 0 ? r0 : v0);
        side.acc = i == 0 ? acc_w + v0 * g.ldacc : acc_h;
        side.add = i == 0 ? r0 > 0 : v0 > 0;
        side.last = i == 0 ? r0 + l.rows >= x.n : v0 + l.words >= x.vocab;
        side.out = i == 0 ? static_cast<T *>(dw) + v0 * lddw : static_cast<T *>(dh) + r0 * lddh;
        side.out_wide = aligned(side.out, 8 * sizeof(T)) && side.ldout % 8 == 0;
        g.left += (int64_t)side.rest(g.npairs) * (side.kblocks + kReading);
      }
      // a share of fewer than sixteen blocks of K would not pay for a piece
      g.sharers = (int)std::max<int64_t>(1, std::min<int64_t>(g.npairs, (g.left + 15) / 16));
      err = launch_gradients<T>(g, s);
      if (err) return err;
    }
  }
  return 0;
}

}  // namespace

extern "C" int *w2v_softmax_fault(void) { return fault_flag(); }

extern "C" int64_t w2v_softmax_workspace(int64_t n, int64_t vocab, int dim, int labels, int type, int flags) {
  const Shape x{n, vocab, dim, labels, type};
  const bool h = flags & W2V_HIDDEN_IN_PLACE, w = flags & W2V_WEIGHT_IN_PLACE;
  const bool grad = flags & W2V_SOFTMAX_GRAD, half = type != W2V_F32;
  if (!good_shape(x)) return -1;
  // without its flag, W may be read in place all the same, and another path taken for it
  return std::max(plan(x, grad, half && h, half && w).total, plan(x, grad, half && h, half).total);
}

extern "C" int w2v_softmax_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const int *targets,
                                int64_t n, int64_t vocab, int dim, int labels, int type, float *loss, float *lse,
                                void *workspace, int64_t workspace_bytes, void *stream) {
  const Shape x{n, vocab, dim, labels, type};
  if (!good_shape(x) || ldh < dim || ldw < dim || !weight || !workspace || !aligned(workspace, 256)) return 1;
  if (n == 0) return 0;
  if (!hidden || !targets || !loss || !lse) return 1;
  const Layout l = plan(x, false, direct(type, hidden, ldh), direct(type, weight, ldw));
  if (workspace_bytes < l.total) return 1;
  if (const int fault = take_fault()) return fault;
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
  const Layout l = plan(x, true, direct(type, hidden, ldh), direct(type, weight, ldw));
  if (workspace_bytes < l.total) return 1;
  if (const int fault = take_fault()) return fault;
  char *ws = static_cast<char *>(workspace);
  const auto s = static_cast<cudaStream_t>(stream);
  if (type == W2V_F32)
    return run_grad<float>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw, ws, s);
  if (type == W2V_BF16)
    return run_grad<__nv_bfloat16>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw,
                                   ws, s);
  return run_grad<__half>(x, l, hidden, ldh, weight, ldw, targets, lse, gloss, ldg, dhidden, lddh, dweight, lddw, ws, s);
}
