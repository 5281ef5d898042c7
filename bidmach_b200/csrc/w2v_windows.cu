// The rows of a minibatch for the softmax over the whole vocabulary: for each position whose word is
// somebody's context, the word, and the centre words that have it in their window.  These are the pairs
// of the positive update (Word2Vec.scala:283-302, 309-330), grouped by the context's position: its
// logits are then computed once for all of its up to 2 * nskip centres (a word that stands at several positions has a
// row for each).  Positions without a pair are left out (subsampling drops about half of a text), in the
// order of the text.
//
// Three passes over 12 bytes a position: count rows in blocks of 256, add the counts up, write.
#include "../../include/bidmach_b200.h"
#include "w2v_chain.cuh"
#include "w2v_device.cuh"

namespace {

using w2v::chain_wait;
using w2v::kFullMask;

constexpr int kBlock = 256;

// Calls use(word) for the centres that have position k in their window, in the order of the text.
template <typename F>
__device__ __forceinline__ void centres_of(const int *words, const int *lb, const int *ub, int n, int nskip, int k, F use) {
  if (words[k] < 0) return;
  for (int i = max(0, k - nskip); i <= min(n - 1, k + nskip); i++)
    if (i != k && words[i] >= 0 && lb[i] <= k - i && k - i <= ub[i]) use(words[i]);
}

__device__ __forceinline__ int row_count(const int *words, const int *lb, const int *ub, int n, int nskip, int k) {
  int c = 0;
  if (k < n) centres_of(words, lb, ub, n, nskip, k, [&](int) { c++; });
  return c;
}

__global__ void __launch_bounds__(kBlock) count_kernel(const int *words, const int *lb, const int *ub, int n, int nskip,
                                                       int *counts) {
  chain_wait();
  const int rows = __syncthreads_count(row_count(words, lb, ub, n, nskip, blockIdx.x * kBlock + threadIdx.x) > 0);
  if (threadIdx.x == 0) counts[blockIdx.x] = rows;
}

// Exclusive sums in place, and the total behind them.
__global__ void __launch_bounds__(1024) offsets_kernel(int *counts, int blocks, int *nrows) {
  __shared__ int sums[32];
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  int base = 0;
  for (int b = 0; b < blocks; b += 1024) {
    const int i = b + threadIdx.x, x = i < blocks ? counts[i] : 0;
    int s = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(kFullMask, s, d);
      if (lane >= d) s += y;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 32; w++) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (i < blocks) counts[i] = base + before + s - x;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *nrows = base;
}

__global__ void __launch_bounds__(kBlock) fill_kernel(const int *words, const int *lb, const int *ub, int n, int nskip,
                                                      const int *offsets, int *ids, int *targets) {
  __shared__ int sums[kBlock / 32];
  chain_wait();
  const int k = blockIdx.x * kBlock + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const bool row = row_count(words, lb, ub, n, nskip, k) > 0;
  const unsigned votes = __ballot_sync(kFullMask, row);
  if (lane == 0) sums[warp] = __popc(votes);
  __syncthreads();
  if (!row) return;
  int at = offsets[blockIdx.x] + __popc(votes & ((1u << lane) - 1));
  for (int w = 0; w < warp; w++) at += sums[w];
  ids[at] = words[k];
  int *to = targets + (int64_t)at * 2 * nskip;
  int c = 0;
  centres_of(words, lb, ub, n, nskip, k, [&](int w) { to[c++] = w; });
  for (; c < 2 * nskip; c++) to[c] = -1;
}

}  // namespace

extern "C" int64_t w2v_window_rows_workspace(int n) { return n < 0 ? -1 : ((int64_t)n + kBlock - 1) / kBlock * 4 + 4; }

extern "C" int w2v_window_rows(const int *words, const int *lb, const int *ub, int n, int nskip, int *ids, int *targets,
                               int *nrows, void *workspace, int64_t workspace_bytes, void *stream) {
  if (n < 0 || nskip < 1 || nskip > 512 || !nrows || !workspace || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 ||
      workspace_bytes < w2v_window_rows_workspace(n) || (n > 0 && (!words || !lb || !ub || !ids || !targets)))
    return 1;
  const auto s = static_cast<cudaStream_t>(stream);
  int *counts = static_cast<int *>(workspace);
  const int blocks = (n + kBlock - 1) / kBlock;
  int err = 0;
  if (blocks) err = w2v::launch_chained(count_kernel, blocks, kBlock, 0, s, words, lb, ub, n, nskip, counts);
  if (!err) err = w2v::launch_chained(offsets_kernel, 1, 1024, 0, s, counts, blocks, nrows);
  if (!err && blocks) err = w2v::launch_chained(fill_kernel, blocks, kBlock, 0, s, words, lb, ub, n, nskip, counts, ids, targets);
  return err;
}
