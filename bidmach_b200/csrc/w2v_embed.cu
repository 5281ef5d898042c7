// Rows of a matrix picked by ids, and the gradient of that: grad of row v = sum of the gradients of
// the tokens whose id is v, in the order of the tokens (no atomics on the sums: the same call gives
// the same bits).
//
// The forward pass copies N rows, and the backward reads N rows and writes the whole gradient
// matrix; both are bound by the memory.  The backward needs the tokens grouped by id.  They are
// sorted stably, and the sorted list is cut into chunks of 32, a warp each: the warp walks its
// chunk, adding rows in registers, and writes a row whenever the id changes.  Ids are Zipf
// distributed (the most frequent word is every tenth token), so a run may cover thousands of
// chunks: what a chunk has of a run that crosses its border goes to a workspace of one row per
// border, and a second kernel adds those, one block a run, in the order of the chunks.
#include <cub/device/device_radix_sort.cuh>

#include <algorithm>

#include "../../include/bidmach_b200.h"
#include "w2v_device.cuh"
#include "w2v_internal.h"
#include "w2v_types.cuh"

namespace {

using w2v::from_float;
using w2v::kFullMask;
using w2v::load8;
using w2v::load_some;
using w2v::store8;
using w2v::store_some;

constexpr int kThreads = 256;
constexpr int kChunk = 32;          // sorted tokens a warp walks
constexpr int kWide = 256;          // columns a warp holds: 8 a lane
constexpr int kJoinThreads = 512;   // 16 warps share the partial rows of one run

template <typename T>
__global__ void __launch_bounds__(kThreads) rows_kernel(const int *ids, int64_t n, const T *m, int64_t ldm,
                                                        int64_t vocab, int dim, T *out, int64_t ldo, bool wide) {
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; i < n; i += stride) {
    const int id = ids[i];
    const bool there = id >= 0 && id < vocab;
    const T *src = m + (there ? (int64_t)id : 0) * ldm;
    T *dst = out + i * ldo;
    if (wide) {
      constexpr int per = 16 / sizeof(T);
      for (int c = lane * per; c < dim; c += 32 * per) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (there) x = *reinterpret_cast<const uint4 *>(src + c);
        *reinterpret_cast<uint4 *>(dst + c) = x;
      }
    } else {
      for (int c = lane; c < dim; c += 32) dst[c] = there ? src[c] : from_float<T>(0.f);
    }
  }
}

// Keys of the sort: an id that is not in the matrix goes behind all others.
__global__ void __launch_bounds__(kThreads) keys_kernel(const int *ids, int n, int vocab, int *keys, int *order) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  const int id = ids[i];
  keys[i] = id >= 0 && id < vocab ? id : vocab;
  order[i] = i;
}

template <typename T>
__device__ __forceinline__ void get8(const T *a, bool wide, int n, float (&x)[8]) {
  if (wide && n >= 8) load8(a, x);
  else load_some(a, n, x);
}
template <typename T>
__device__ __forceinline__ void put8(T *a, bool wide, int n, const float (&x)[8]) {
  if (wide && n >= 8) store8(a, x);
  else store_some(a, n, x);
}

struct Runs {
  const int *keys;    // sorted
  const int *order;   // token of each
  int n, vocab, dim, chunks, padded;
  float *part;        // [2 * chunks][padded]: the part before the first border of a chunk, and after the last
  int *owners;        // chunks in which a run starts that crosses their end
  int *nowners;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) runs_kernel(const Runs r, const T *grad, int64_t ldg, T *out, int64_t ldo,
                                                        bool wide) {
  const int chunk = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (chunk >= r.chunks) return;
  const int lo = chunk * kChunk, cnt = min(kChunk, r.n - lo);
  const int my_key = lane < cnt ? r.keys[lo + lane] : -1;
  const int my_row = lane < cnt ? r.order[lo + lane] : 0;
  const int first = __shfl_sync(kFullMask, my_key, 0);
  if (first >= r.vocab) return;
  const int before = lo > 0 ? r.keys[lo - 1] : -1;
  const int after = lo + cnt < r.n ? r.keys[lo + cnt] : -1;
  const int col = blockIdx.y * kWide + lane * 8, have = min(8, max(0, r.dim - col));
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  int cur = first;
  auto flush = [&](bool last) {
    if (cur >= r.vocab) return;
    const bool head = cur == first && before == cur, tail = last && after == cur;
    if (!head && !tail) {
      put8(out + (int64_t)cur * ldo + col, wide, have, acc);
    } else {
      float *to = r.part + (int64_t)(2 * chunk + (head ? 0 : 1)) * r.padded + col;
      if (col < r.padded) store8(to, acc);
      if (!head && lane == 0 && blockIdx.y == 0) r.owners[atomicAdd(r.nowners, 1)] = chunk;
    }
  };
  // four rows in flight
  for (int i = 0; i < cnt; i += 4) {
    float x[4][8];
    int key[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      key[j] = __shfl_sync(kFullMask, my_key, (i + j) & 31);
      const int row = __shfl_sync(kFullMask, my_row, (i + j) & 31);
      const bool use = i + j < cnt && key[j] < r.vocab;
      get8(grad + (int64_t)row * ldg + col, wide, use ? have : 0, x[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (i + j >= cnt) break;
      if (key[j] != cur) {
        flush(false);
        cur = key[j];
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] += x[j][e];
    }
  }
  flush(true);
}

// The runs that cross chunks: the part behind the last border of the chunk they start in, then the
// first part of every chunk up to the one they end in.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Runs r, T *out, int64_t ldo, bool wide) {
  __shared__ float parts[kJoinThreads / 32][kWide];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = kJoinThreads / 32;
  const int owners = *r.nowners;
  const int col = blockIdx.y * kWide + lane * 8, have = min(8, max(0, r.dim - col));
  for (int k = blockIdx.x; k < owners; k += gridDim.x) {
    const int chunk = r.owners[k];
    const int key = r.keys[min(r.n, (chunk + 1) * kChunk) - 1];
    // the last position of the run, by bisection
    int lo = (chunk + 1) * kChunk, hi = r.n - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (r.keys[mid] == key) lo = mid;
      else hi = mid - 1;
    }
    const int count = lo / kChunk - chunk + 1;   // parts: the owner's and one of each following chunk
    const int each = (count + warps - 1) / warps;
    const int a = min(count, warp * each), b = min(count, a + each);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (col < r.padded) {
      for (int i = a; i < b; i += 4) {
        float x[4][8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int c = min(i + j, b - 1);
          load8(r.part + (int64_t)(c == 0 ? 2 * chunk + 1 : 2 * (chunk + c)) * r.padded + col, x[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (i + j < b) {
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] += x[j][e];
          }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) parts[warp][lane * 8 + e] = acc[e];
    __syncthreads();
    if (warp == 0) {
      const int used = (count + each - 1) / each;
      for (int w = 1; w < used; w++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += parts[w][lane * 8 + e];
      put8(out + (int64_t)key * ldo + col, wide, have, acc);
    }
    __syncthreads();
  }
}

bool good_type(int type) { return type == W2V_F32 || type == W2V_BF16 || type == W2V_F16; }
bool aligned(const void *a, size_t to) { return reinterpret_cast<uintptr_t>(a) % to == 0; }
int64_t up(int64_t a, int64_t to) { return (a + to - 1) / to * to; }

// Workspace of the backward pass, in this order: partial rows, sorted keys and order, keys and
// order, owners, their count, the sort's own.
struct Layout {
  int64_t part, keys, order, keys_in, order_in, owners, nowners, sort, total;
  size_t sort_bytes;
  int padded, chunks, bits;
};

int plan(int64_t n, int64_t vocab, int dim, Layout *l) {
  l->padded = (int)up(dim, 8);
  l->chunks = (int)((n + kChunk - 1) / kChunk);
  l->bits = 1;
  while (l->bits < 31 && ((int64_t)1 << l->bits) <= vocab) l->bits++;
  l->sort_bytes = 0;
  const cudaError_t e = cub::DeviceRadixSort::SortPairs(nullptr, l->sort_bytes, (const int *)nullptr, (int *)nullptr,
                                                        (const int *)nullptr, (int *)nullptr, (int)n, 0, l->bits);
  if (e != cudaSuccess) return (int)e;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(std::max<int64_t>(bytes, 1), 256);
    return here;
  };
  l->part = take((int64_t)2 * l->chunks * l->padded * 4);
  l->keys = take(n * 4);
  l->order = take(n * 4);
  l->keys_in = take(n * 4);
  l->order_in = take(n * 4);
  l->owners = take((int64_t)l->chunks * 4);
  l->nowners = take(4);
  l->sort = take((int64_t)l->sort_bytes);
  l->total = at;
  return 0;
}

bool good_shape(int64_t n, int64_t vocab, int dim, int type) {
  return n >= 0 && n < ((int64_t)1 << 30) && vocab >= 1 && vocab < ((int64_t)1 << 31) - 1 && dim >= 1 &&
         dim <= (1 << 16) && good_type(type);
}

template <typename T>
int run_rows(const int *ids, int64_t n, const void *m, int64_t ldm, int64_t vocab, int dim, void *out, int64_t ldo,
             cudaStream_t s) {
  const bool wide = aligned(m, 16) && aligned(out, 16) && ldm * sizeof(T) % 16 == 0 && ldo * sizeof(T) % 16 == 0 &&
                    dim * sizeof(T) % 16 == 0;
  const int64_t need = (n + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = (int)std::min<int64_t>(need, (int64_t)w2v::device_sm_count() * 32);
  rows_kernel<T><<<grid, kThreads, 0, s>>>(ids, n, static_cast<const T *>(m), ldm, vocab, dim, static_cast<T *>(out),
                                           ldo, wide);
  w2v::count_launch(1);
  return (int)cudaGetLastError();
}

template <typename T>
int run_grad(const Layout &l, const int *ids, int n, const void *grad, int64_t ldg, int vocab, int dim, void *out,
             int64_t ldo, char *ws, cudaStream_t s) {
  int *keys = reinterpret_cast<int *>(ws + l.keys), *order = reinterpret_cast<int *>(ws + l.order);
  int *keys_in = reinterpret_cast<int *>(ws + l.keys_in), *order_in = reinterpret_cast<int *>(ws + l.order_in);
  Runs r{keys, order, n, vocab, dim, l.chunks, l.padded, reinterpret_cast<float *>(ws + l.part),
         reinterpret_cast<int *>(ws + l.owners), reinterpret_cast<int *>(ws + l.nowners)};
  cudaError_t e = cudaMemsetAsync(r.nowners, 0, 4, s);
  if (e == cudaSuccess)
    e = ldo == dim ? cudaMemsetAsync(out, 0, (size_t)vocab * dim * sizeof(T), s)
                   : cudaMemset2DAsync(out, ldo * sizeof(T), 0, dim * sizeof(T), vocab, s);
  if (e != cudaSuccess) return (int)e;
  if (n == 0) return 0;
  keys_kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, s>>>(ids, n, vocab, keys_in, order_in);
  size_t bytes = l.sort_bytes;
  e = cub::DeviceRadixSort::SortPairs(ws + l.sort, bytes, keys_in, keys, order_in, order, n, 0, l.bits, s);
  if (e != cudaSuccess) return (int)e;
  const T *g = static_cast<const T *>(grad);
  T *o = static_cast<T *>(out);
  const bool gw = aligned(g, 8 * sizeof(T)) && ldg % 8 == 0, ow = aligned(o, 8 * sizeof(T)) && ldo % 8 == 0;
  const int cols = (dim + kWide - 1) / kWide;
  runs_kernel<T><<<dim3((l.chunks + kThreads / 32 - 1) / (kThreads / 32), cols), kThreads, 0, s>>>(r, g, ldg, o, ldo,
                                                                                                   gw && ow);
  join_kernel<T><<<dim3(std::min(l.chunks, w2v::device_sm_count() * 4), cols), kJoinThreads, 0, s>>>(r, o, ldo, ow);
  w2v::count_launch(3);
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" int w2v_embed_rows(const int *ids, int64_t n, const void *matrix, int64_t ldm, int64_t vocab, int dim,
                              int type, void *out, int64_t ldo, void *stream) {
  if (!good_shape(n, vocab, dim, type) || ldm < dim || ldo < dim) return 1;
  if (n == 0) return 0;
  if (!ids || !matrix || !out) return 1;
  const auto s = static_cast<cudaStream_t>(stream);
  if (type == W2V_F32) return run_rows<float>(ids, n, matrix, ldm, vocab, dim, out, ldo, s);
  if (type == W2V_BF16) return run_rows<__nv_bfloat16>(ids, n, matrix, ldm, vocab, dim, out, ldo, s);
  return run_rows<__half>(ids, n, matrix, ldm, vocab, dim, out, ldo, s);
}

extern "C" int64_t w2v_embed_grad_workspace(int64_t n, int64_t vocab, int dim, int type) {
  Layout l;
  if (!good_shape(n, vocab, dim, type) || plan(n, vocab, dim, &l)) return -1;
  return l.total;
}

extern "C" int w2v_embed_grad(const int *ids, int64_t n, const void *grad, int64_t ldg, int64_t vocab, int dim,
                              int type, void *out, int64_t ldo, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  Layout l;
  if (!good_shape(n, vocab, dim, type) || ldg < dim || ldo < dim || !out || (n > 0 && (!ids || !grad)) ||
      !workspace || !aligned(workspace, 256))
    return 1;
  const int err = plan(n, vocab, dim, &l);
  if (err) return err;
  if (workspace_bytes < l.total) return 1;
  const auto s = static_cast<cudaStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  if (type == W2V_F32) return run_grad<float>(l, ids, (int)n, grad, ldg, (int)vocab, dim, out, ldo, ws, s);
  if (type == W2V_BF16) return run_grad<__nv_bfloat16>(l, ids, (int)n, grad, ldg, (int)vocab, dim, out, ldo, ws, s);
  return run_grad<__half>(l, ids, (int)n, grad, ldg, (int)vocab, dim, out, ldo, ws, s);
}
