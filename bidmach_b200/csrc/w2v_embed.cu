// Rows of a matrix picked by ids, and the gradient of that: grad of row v = sum of the gradients of
// the tokens whose id is v, in the order of the tokens (no atomics on the sums: the same call gives
// the same bits).
//
// The forward pass copies N rows, and the backward reads N rows and writes the whole gradient
// matrix; both are bound by the memory.  The backward needs the tokens grouped by id.  They are
// sorted stably, and the sorted list is cut into chunks of up to 32, a warp each: the warp walks its
// chunk, adding rows in registers, and writes a row whenever the id changes.  Ids are Zipf
// distributed (the most frequent word is every tenth token), so a run may cover thousands of
// chunks: what a chunk has of a run that crosses its border goes to a workspace of one row per
// border, and those are added in the order of the chunks, by a warp or, for a long run, a block.
//
// Measured: a million Zipf tokens of 100000 x 300 fp32: rows 242 us (1.2 GB written, 5.0 TB/s), sums 260 us
// (1.14 GB of rows of 1200 bytes gathered, 4.4 TB/s) after a sort of 70 us, joining 30 us.
#include <cub/block/block_radix_sort.cuh>
#include <cub/device/device_radix_sort.cuh>

#include <algorithm>

#include "../../include/bidmach_b200.h"
#include "w2v_chain.cuh"
#include "w2v_device.cuh"
#include "w2v_internal.h"
#include "w2v_types.cuh"

namespace {

using w2v::chain_wait;
using w2v::from_float;
using w2v::kFullMask;
using w2v::launch_chained;

constexpr int kThreads = 256;
constexpr int kMostChunk = 32;      // sorted tokens a warp walks, one a lane while their ids are looked up
constexpr int kShortRun = 16;       // parts that one warp adds
constexpr int kJoinThreads = 1024;  // 32 warps share the parts of a longer run

__device__ __forceinline__ uint4 load_once(const void *a) {
  return __ldcs(reinterpret_cast<const uint4 *>(a));
}

// A warp copies `each` rows (up to 32, an even number), two at a time and each whole before its first store: up to G pieces of 16 bytes
// a lane and row.  The copy is written past L2 (it is read by another kernel, if at all), the matrix,
// whose frequent rows come again and again, is not.
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) rows_kernel(const int *ids, int64_t n, const T *m, int64_t ldm,
                                                        int64_t vocab, int dim, T *out, int64_t ldo, int each) {
  chain_wait();
  constexpr int per = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t r0 = ((int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * each;
  if (r0 >= n) return;
  const int cnt = (int)min((int64_t)each, n - r0);
  const int id = lane < cnt ? ids[r0 + lane] : -1;
  const int c0 = blockIdx.y * G * 32 * per + lane * per;
  for (int i = 0; i < cnt; i += 2) {
    uint4 x[2][G];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int v = __shfl_sync(kFullMask, id, (i + j) & 31);
      const bool there = i + j < cnt && v >= 0 && v < vocab;
      const T *src = m + (there ? (int64_t)v : 0) * ldm;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int c = c0 + g * 32 * per;
        x[j][g] = make_uint4(0, 0, 0, 0);
        if (there && c < dim) x[j][g] = __ldg(reinterpret_cast<const uint4 *>(src + c));
      }
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int c = c0 + g * 32 * per;
        if (i + j < cnt && c < dim) __stcs(reinterpret_cast<uint4 *>(out + (r0 + i + j) * ldo + c), x[j][g]);
      }
  }
}

// Rows that no 16-byte access fits.
template <typename T>
__global__ void __launch_bounds__(kThreads) rows_any_kernel(const int *ids, int64_t n, const T *m, int64_t ldm,
                                                            int64_t vocab, int dim, T *out, int64_t ldo) {
  chain_wait();
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; i < n; i += stride) {
    const int id = ids[i];
    const bool there = id >= 0 && id < vocab;
    const T *src = m + (there ? (int64_t)id : 0) * ldm;
    T *dst = out + i * ldo;
#pragma unroll 4
    for (int c = lane; c < dim; c += 32) dst[c] = there ? src[c] : from_float<T>(0.f);
  }
}

// Keys of the sort: an id that is not in the matrix goes behind all others.
__device__ __forceinline__ int key_of(int id, int vocab) { return id >= 0 && id < vocab ? id : vocab; }

__global__ void __launch_bounds__(kThreads) keys_kernel(const int *ids, int n, int vocab, int *keys, int *order,
                                                        int *nowners) {
  chain_wait();
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i == 0) *nowners = 0;
  if (i >= n) return;
  keys[i] = key_of(ids[i], vocab);
  order[i] = i;
}

// Up to THREADS * 8 tokens: keys and sort in one block.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) small_sort_kernel(const int *ids, int n, int vocab, int bits, int *keys, int *order,
                                                             int *nowners) {
  using Sort = cub::BlockRadixSort<int, THREADS, 8, int, 5>;
  __shared__ typename Sort::TempStorage temp;
  int key[8], at[8];
  chain_wait();
#pragma unroll
  for (int j = 0; j < 8; j++) {
    at[j] = threadIdx.x * 8 + j;
    key[j] = at[j] < n ? key_of(ids[at[j]], vocab) : vocab;   // those behind the last come last: the sort is stable
  }
  Sort(temp).Sort(key, at, 0, bits);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int i = threadIdx.x * 8 + j;
    if (i < n) {
      keys[i] = key[j];
      order[i] = at[j];
    }
  }
  if (threadIdx.x == 0) *nowners = 0;
}
constexpr int kSmallSort = 512 * 8;

struct Runs {
  const int *keys;    // sorted
  const int *order;   // token of each
  int n, vocab, dim, chunk, chunks, padded;
  float *part;        // [2 * chunks][padded]: the part before the first border of a chunk, and after the last
  int *owners;        // chunks in which a run starts that crosses their end
  int *nowners;
};

// VEC columns of a lane, in the G groups of 32 * VEC that a warp holds.
template <typename T, int VEC>
__device__ __forceinline__ void get(const T *a, bool there, float (&x)[VEC]) {
  if (VEC == 1) {
    x[0] = there ? w2v::to_float(*a) : 0.f;
  } else {
    const uint4 raw = there ? load_once(a) : make_uint4(0, 0, 0, 0);
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = w2v::to_float(e[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void put(T *a, const float (&x)[VEC]) {
  if (VEC == 1) {
    *a = from_float<T>(x[0]);
  } else {
    uint4 raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i++) e[i] = from_float<T>(x[i]);
    *reinterpret_cast<uint4 *>(a) = raw;
  }
}
template <int VEC>
__device__ __forceinline__ void put_part(float *a, const float (&x)[VEC]) {
  if (VEC == 1) a[0] = x[0];
  else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4 *>(a + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
}
template <int VEC>
__device__ __forceinline__ void get_part(const float *a, float (&x)[VEC]) {
  if (VEC == 1) x[0] = a[0];
  else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 f = *reinterpret_cast<const float4 *>(a + i);
      x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
    }
  }
}

template <typename T, int VEC, int G>
__global__ void __launch_bounds__(kThreads) runs_kernel(const Runs r, const T *grad, int64_t ldg, T *out, int64_t ldo) {
  const int chunk = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  chain_wait();
  if (chunk >= r.chunks) return;
  const int lo = chunk * r.chunk, cnt = min(r.chunk, r.n - lo);
  const int my_key = lane < cnt ? r.keys[lo + lane] : -1;
  const int my_row = lane < cnt ? r.order[lo + lane] : 0;
  const int before = lo > 0 ? r.keys[lo - 1] : -1;
  const int after = lo + cnt < r.n ? r.keys[lo + cnt] : -1;
  const int first = __shfl_sync(kFullMask, my_key, 0);
  if (first >= r.vocab) return;
  const int c0 = blockIdx.y * G * 32 * VEC + lane * VEC;
  float acc[G][VEC];
  int cur = first;
  auto clear = [&] {
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[g][e] = 0.f;
  };
  auto flush = [&](bool last) {
    if (cur >= r.vocab) return;
    const bool head = cur == first && before == cur, tail = last && after == cur;
    float *to = r.part + (int64_t)(2 * chunk + (head ? 0 : 1)) * r.padded;
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int c = c0 + g * 32 * VEC;
      if (c >= r.dim) continue;
      if (!head && !tail) put<T, VEC>(out + (int64_t)cur * ldo + c, acc[g]);
      else put_part<VEC>(to + c, acc[g]);
    }
    if (!head && tail && lane == 0 && blockIdx.y == 0) r.owners[atomicAdd(r.nowners, 1)] = chunk;
  };
  clear();
  constexpr int U = G * VEC > 16 ? 2 : 4;   // rows in flight
  for (int i = 0; i < cnt; i += U) {
    float x[U][G][VEC];
    int key[U];
#pragma unroll
    for (int j = 0; j < U; j++) {
      key[j] = __shfl_sync(kFullMask, my_key, (i + j) & 31);
      const int row = __shfl_sync(kFullMask, my_row, (i + j) & 31);
      const bool use = i + j < cnt && key[j] < r.vocab;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int c = c0 + g * 32 * VEC;
        get<T, VEC>(grad + (int64_t)row * ldg + c, use && c < r.dim, x[j][g]);
      }
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
      if (i + j >= cnt) break;
      if (key[j] != cur) {
        flush(false);
        cur = key[j];
        clear();
      }
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[g][e] += x[j][g][e];
    }
  }
  flush(true);
}

// Adds the parts a .. b - 1 of the run that starts in `chunk`: its own, then the first part of each
// following chunk.
template <int VEC>
__device__ __forceinline__ void add_parts(const Runs &r, int chunk, int a, int b, int c, float (&acc)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; e++) acc[e] = 0.f;
  constexpr int U = VEC == 8 ? 4 : 8;
  for (int i = a; i < b; i += U) {
    float x[U][VEC];
#pragma unroll
    for (int j = 0; j < U; j++) {
      const int k = min(i + j, b - 1);
      get_part<VEC>(r.part + (int64_t)(k == 0 ? 2 * chunk + 1 : 2 * (chunk + k)) * r.padded + c, x[j]);
    }
#pragma unroll
    for (int j = 0; j < U; j++)
      if (i + j < b) {
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] += x[j][e];
      }
  }
}

// The runs that cross chunks: a warp each where there are few parts, then the whole block for each of
// its longer ones.  Block b takes the runs b, b + gridDim.x, ... of the list, a warp one of every 32.
template <typename T, int VEC>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Runs r, T *out, int64_t ldo) {
  constexpr int warps = kJoinThreads / 32;
  __shared__ float sums[warps][32 * VEC + 1];
  __shared__ int longer[warps], nlonger, count_s;
  chain_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, owners = *r.nowners;
  const int c = blockIdx.y * 32 * VEC + lane * VEC;
  for (int64_t k0 = blockIdx.x; k0 < owners; k0 += (int64_t)gridDim.x * warps) {
    if (threadIdx.x == 0) nlonger = 0;
    __syncthreads();
    const int64_t k = k0 + (int64_t)warp * gridDim.x;
    if (k < owners) {
      const int chunk = r.owners[k], key = r.keys[(chunk + 1) * r.chunk - 1];
      // does the run reach into chunk + 1 + lane?
      const int64_t at = (int64_t)(chunk + 1 + lane) * r.chunk;
      const unsigned in = __ballot_sync(kFullMask, lane < kShortRun && at < r.n && r.keys[at < r.n ? at : 0] == key);
      const int parts = 1 + __popc(in);
      if (parts > kShortRun) {
        if (lane == 0) longer[atomicAdd(&nlonger, 1)] = chunk;
      } else if (c < r.dim) {
        float acc[VEC];
        add_parts<VEC>(r, chunk, 0, parts, c, acc);
        put<T, VEC>(out + (int64_t)key * ldo + c, acc);
      }
    }
    __syncthreads();
    for (int i = 0; i < nlonger; i++) {
      const int chunk = longer[i], key = r.keys[(chunk + 1) * r.chunk - 1];
      if (warp == 0) {
        // the chunk that the run ends in: 32 places at a time
        int lo = chunk + 1, hi = r.chunks;   // keys at the start of `lo` belong to the run, at `hi` not
        while (hi - lo > 1) {
          const int step = (hi - lo + 31) / 32, at = lo + lane * step;
          const unsigned in = __ballot_sync(kFullMask, at < hi && r.keys[(int64_t)min(at, hi - 1) * r.chunk] == key);
          const int top = 31 - __clz(in);    // lane 0 is always in
          lo += top * step;
          hi = min(hi, lo + step);
        }
        if (lane == 0) count_s = lo - chunk + 1;
      }
      __syncthreads();
      const int count = count_s, each = (count + warps - 1) / warps;
      const int a = min(count, warp * each), b = min(count, a + each);
      float acc[VEC];
      add_parts<VEC>(r, chunk, a, c < r.dim ? b : a, c, acc);
#pragma unroll
      for (int e = 0; e < VEC; e++) sums[warp][lane * VEC + e] = acc[e];
      __syncthreads();
      // warps in their order, a column a thread
      if (threadIdx.x < 32 * VEC) {
        float x = 0.f;
#pragma unroll 8
        for (int w = 0; w < warps; w++) x += sums[w][threadIdx.x];
        const int col = blockIdx.y * 32 * VEC + threadIdx.x;
        if (col < r.dim) out[(int64_t)key * ldo + col] = from_float<T>(x);
      }
      __syncthreads();
    }
  }
}

bool good_type(int type) { return type == W2V_F32 || type == W2V_BF16 || type == W2V_F16; }
bool aligned(const void *a, size_t to) { return reinterpret_cast<uintptr_t>(a) % to == 0; }
int64_t up(int64_t a, int64_t to) { return (a + to - 1) / to * to; }

// Workspace of the backward pass, in this order: partial rows, sorted keys and order, keys and
// order, the runs to join and their counts, the sort's own.
struct Layout {
  int64_t part, keys, order, keys_in, order_in, owners, nowners, sort, total;
  size_t sort_bytes;
  int padded, chunk, chunks, bits;
};

int plan(int64_t n, int64_t vocab, int dim, Layout *l) {
  l->padded = (int)up(dim, 8);
  // few tokens: more warps with less to walk (4096 tokens in 512 warps rather than 128)
  l->chunk = n <= 16384 ? 8 : n <= 131072 ? 16 : kMostChunk;
  l->chunks = (int)((n + l->chunk - 1) / l->chunk);
  l->bits = 1;
  while (l->bits < 31 && ((int64_t)1 << l->bits) <= vocab) l->bits++;
  l->sort_bytes = 0;
  if (n > kSmallSort) {
    const cudaError_t e = cub::DeviceRadixSort::SortPairs(nullptr, l->sort_bytes, (const int *)nullptr, (int *)nullptr,
                                                          (const int *)nullptr, (int *)nullptr, (int)n, 0, l->bits);
    if (e != cudaSuccess) return (int)e;
  }
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

// Rows of 16-byte pieces: base and leading dimension allow them, and the last piece ends with the row.
template <typename T>
bool pieces(const void *a, int64_t ld, int dim) {
  return aligned(a, 16) && ld * sizeof(T) % 16 == 0 && dim * sizeof(T) % 16 == 0;
}

template <typename T>
int run_rows(const int *ids, int64_t n, const void *m, int64_t ldm, int64_t vocab, int dim, void *out, int64_t ldo,
             cudaStream_t s) {
  const T *src = static_cast<const T *>(m);
  T *dst = static_cast<T *>(out);
  if (pieces<T>(m, ldm, dim) && pieces<T>(out, ldo, dim)) {
    const int groups = (int)((dim * sizeof(T) / 16 + 31) / 32);
    // enough warps to fill the SMs first, then rows for each of them
    const int each = (int)std::max<int64_t>(2, std::min<int64_t>(32, n / (w2v::device_sm_count() * 64) / 2 * 2));
    const int64_t block = (int64_t)each * (kThreads / 32);
    const dim3 grid((unsigned)((n + block - 1) / block), (groups + 3) / 4);
    const auto k = groups == 1 ? rows_kernel<T, 1> : groups == 2 ? rows_kernel<T, 2> : groups == 3 ? rows_kernel<T, 3>
                                                                                           : rows_kernel<T, 4>;
    return launch_chained(k, grid, kThreads, 0, s, ids, n, src, ldm, vocab, dim, dst, ldo, each);
  }
  const int64_t need = (n + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = (int)std::min<int64_t>(need, (int64_t)w2v::device_sm_count() * 32);
  return launch_chained(rows_any_kernel<T>, grid, kThreads, 0, s, ids, n, src, ldm, vocab, dim, dst, ldo);
}

template <typename T, int VEC>
int run_runs(const Runs &r, const T *g, int64_t ldg, T *o, int64_t ldo, cudaStream_t s) {
  const int groups = (r.dim + 32 * VEC - 1) / (32 * VEC);
  constexpr int most = VEC == 8 ? 2 : 4;
  const dim3 grid((r.chunks + kThreads / 32 - 1) / (kThreads / 32), (groups + most - 1) / most);
  const auto k = groups == 1   ? runs_kernel<T, VEC, 1>
                 : groups == 2 ? runs_kernel<T, VEC, 2>
                 : groups == 3 ? runs_kernel<T, VEC, most == 2 ? 2 : 3>
                               : runs_kernel<T, VEC, most>;
  const int err = launch_chained(k, grid, kThreads, 0, s, r, g, ldg, o, ldo);
  if (err || r.chunks < 2) return err;
  return launch_chained(join_kernel<T, VEC>, dim3(std::min(r.chunks / 2, w2v::device_sm_count() * 2), groups), kJoinThreads,
                        0, s, r, o, ldo);
}

template <typename T>
int run_grad(const Layout &l, const int *ids, int n, const void *grad, int64_t ldg, int vocab, int dim, void *out,
             int64_t ldo, char *ws, cudaStream_t s) {
  int *keys = reinterpret_cast<int *>(ws + l.keys), *order = reinterpret_cast<int *>(ws + l.order);
  int *keys_in = reinterpret_cast<int *>(ws + l.keys_in), *order_in = reinterpret_cast<int *>(ws + l.order_in);
  const Runs r{keys, order, n, vocab, dim, l.chunk, l.chunks, l.padded, reinterpret_cast<float *>(ws + l.part),
               reinterpret_cast<int *>(ws + l.owners), reinterpret_cast<int *>(ws + l.nowners)};
  cudaError_t e = ldo == dim ? cudaMemsetAsync(out, 0, (size_t)vocab * dim * sizeof(T), s)
                             : cudaMemset2DAsync(out, ldo * sizeof(T), 0, dim * sizeof(T), vocab, s);
  if (e != cudaSuccess || n == 0) return (int)e;
  int err = 0;
  if (n <= 128 * 8) {
    err = launch_chained(small_sort_kernel<128>, 1, 128, 0, s, ids, n, vocab, l.bits, keys, order, r.nowners);
  } else if (n <= kSmallSort) {
    err = launch_chained(small_sort_kernel<512>, 1, 512, 0, s, ids, n, vocab, l.bits, keys, order, r.nowners);
  } else {
    err = launch_chained(keys_kernel, (n + kThreads - 1) / kThreads, kThreads, 0, s, ids, n, vocab, keys_in, order_in, r.nowners);
    size_t bytes = l.sort_bytes;
    if (!err)
      err = (int)cub::DeviceRadixSort::SortPairs(ws + l.sort, bytes, keys_in, keys, order_in, order, n, 0, l.bits, s);
  }
  if (err) return err;
  const T *g = static_cast<const T *>(grad);
  T *o = static_cast<T *>(out);
  if (pieces<T>(g, ldg, dim) && pieces<T>(o, ldo, dim)) return run_runs<T, 16 / sizeof(T)>(r, g, ldg, o, ldo, s);
  return run_runs<T, 1>(r, g, ldg, o, ldo, s);
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
