// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps),   c = 1 - b^t
//
// Every element is read and written once and nothing else moves: 28 bytes an element with fp32
// moments, 16 with 8-bit ones (fp32 parameters and gradients), so the bound is the memory.  The
// work is cut into units of 256 elements, a warp each, 8 consecutive elements a lane (32 bytes of
// fp32: one 256-bit access).  The tensors' addresses travel as kernel arguments, not through a
// table in device memory: nothing has to be uploaded before a step, and a captured step holds
// its own.
//
// Measured: 51 million elements with fp32 moments 217 us (6.6 TB/s); 300 million with 8-bit moments, and
// their values as fp32, 1.41 ms (5.1 TB/s; the codes take more than half of the instructions, the values alone
// 491 us).  Telling lanes without a code of zero apart, to spare them the selects, cost 7 %.
//
// Each operation on the moments is rounded on its own (no contraction to fused multiply-adds), so the
// result does not depend on how a compiler groups them: next to the border of two 8-bit codes that
// would change a stored moment by a whole step.
//
// 8-bit moments.  A unit is also the block that shares a scale, the largest magnitude in it.  A
// code is the leading bits of the fp32 number y = x / scale (0 < |y| <= 1), rounded to nearest
// even: for m a sign and 7 bits (3 of mantissa), for sqrt(v) 8 bits (4 of mantissa), the topmost
// code meaning 1.  Both span about 16 octaves; what is below rounds to zero for m and to the
// smallest code for sqrt(v), so that no step divides by eps alone.  The root of v is stored, not v:
// it needs half the octaves.  The step itself uses the moments before they are rounded.
//
// Neighbouring codes of sqrt(v) are 3 to 6 % apart and a step with beta2 = 0.999 lowers it by 0.05 %: rounded to
// nearest such a moment never falls, and rises only where a gradient is several times its root.  Over more than
// a few steps the codes have to be rounded at random (RANDOM): up with the probability that makes the
// mean of the stored m and of the stored v (the square, not the root) the values before rounding.  The
// random bits are a hash of seed, step and element, so equal calls give equal bits.  They cost instructions:
// a step of 300 million fp32 elements takes 1.18 ms (nearest 0.82), of 40 million bf16 175 us (132).
#include <math.h>

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
using w2v::to_float;

constexpr int kUnit = 256;
constexpr int kThreads = 256;

// Running products b1^t and b2^t, the blocks that have finished the step, and the steps done.
struct Clock {
  double b1t, b2t;
  unsigned arrived, t;
};

template <int CAP>
struct Table {
  void *p[CAP];
  const void *g[CAP];
  void *m[CAP];
  void *v[CAP];
  float *ms[CAP];
  float *vs[CAP];
  int64_t n[CAP];
  int64_t first[CAP + 1];   // unit at which the tensor starts
  unsigned char wide[CAP];  // all addresses allow the 8-element accesses
  int count;
};

struct Rates {
  double lrate, beta1, beta2, eps, wdecay;
  const float *lrate_dev;
  Clock *clock;
  int advance;
  unsigned seed;   // of the random rounding, this launch's own
};

constexpr float kSmallest = 1.17549435e-38f;   // 2^-126: its reciprocal is still finite

// What a step computes once, each rounded to fp32 from its value in 64 bits; eps is at least 2^-126, so
// that an element without a gradient is not divided by zero (a root of v that is not zero is above 2^-75).
struct Consts {
  float b1, ob1, b2, ob2, lrc1, rc2, eps, keep;
};

__device__ __forceinline__ Consts constants(const Rates &r) {
  const double c1 = 1.0 - r.clock->b1t * r.beta1, c2 = 1.0 - r.clock->b2t * r.beta2;
  const double lr = r.lrate_dev ? (double)*r.lrate_dev : r.lrate;
  return Consts{(float)r.beta1, (float)(1.0 - r.beta1), (float)r.beta2, (float)(1.0 - r.beta2),
                (float)(lr / c1), (float)(1.0 / sqrt(c2)), fmaxf((float)r.eps, kSmallest), (float)(1.0 - lr * r.wdecay)};
}

// One unit in the last place off; zero from 2^126 on.
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void step8(float (&p)[8], const float (&g)[8], float (&m)[8], float (&v)[8],
                                      float (&root)[8], const Consts &c) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    m[i] = __fadd_rn(__fmul_rn(m[i], c.b1), __fmul_rn(g[i], c.ob1));
    v[i] = __fadd_rn(__fmul_rn(v[i], c.b2), __fmul_rn(__fmul_rn(g[i], g[i]), c.ob2));
    root[i] = __fsqrt_rn(v[i]);
    const float d = __fadd_rn(__fmul_rn(root[i], c.rc2), c.eps);
    // the quotient reaches the parameter only, not a stored moment: two units in its last place will do
    p[i] = __fsub_rn(__fmul_rn(p[i], c.keep), __fmul_rn(__fmul_rn(m[i], c.lrc1), reciprocal(d)));
  }
}

constexpr int kOne = 0x3F800000;

// NaN where a or b is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Scale of a unit, the largest of |x|; bits of non-negative floats order as unsigned numbers, NaN last.
__device__ __forceinline__ float unit_scale(const float (&x)[8]) {
  float most = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; i++) most = max_nan(most, fabsf(x[i]));
  const unsigned top = __reduce_max_sync(kFullMask, __float_as_uint(most));
  if (top >= 0x7f800000u) return __uint_as_float(0x7fffffffu);   // infinity or NaN: the unit reads as NaN
  const float s = __uint_as_float(top);
  return s >= kSmallest ? s : 0.f;
}

// The finalizer of MurmurHash3 (Appleby): every bit of the result depends on every bit of x.
__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {
  x = (x ^ x >> 16) * 0x85ebca6bu;
  x = (x ^ x >> 13) * 0xc2b2ae35u;
  return x ^ x >> 16;
}

// Code of |y| (as bits, at most 2 of 32 above 1) rounded up with a probability, `random` deciding.  Of m the place
// between the two codes; of sqrt(v), f of the way from M to M + 1 in units of the last mantissa bit, the
// place of its square: f (2 M + f) / (2 M + 1).
template <bool SIGNED>
__device__ __forceinline__ int random_code(unsigned bits, unsigned random) {
  if (SIGNED) return min((int)((bits + (random & 0xfffffu)) >> 20), kOne >> 20) - ((kOne >> 20) - 127);
  constexpr unsigned low = (1u << 19) - 1u;
  const float f = __fmul_rn((float)(bits & low), 0x1p-19f), m = (float)(32u + (bits >> 18 & 30u));   // 2 M
  const float up = __fmul_rn(__fmul_rn(f, __fadd_rn(m, f)), __frcp_rn(__fadd_rn(m, 1.f)));
  const unsigned place = (unsigned)__fmul_rn(up, 0x1p19f);
  return min((int)((bits >> 19) + ((place + (random >> 13)) >> 19)), kOne >> 19) - ((kOne >> 19) - 255);
}

// `first`: place of x[0] among the random bits, for RANDOM.
template <bool SIGNED, bool RANDOM = false>
__device__ __forceinline__ void encode8(const float (&x)[8], float scale, unsigned (&code)[2], unsigned key = 0,
                                        unsigned first = 0) {
  constexpr int shift = SIGNED ? 20 : 19, top = SIGNED ? 127 : 255, offset = (kOne >> shift) - top;
  code[0] = code[1] = 0;
  if (!(scale > 0.f)) return;   // all zero, or not finite: the scale says which
  const float r = __fdiv_rn(1.f, scale);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // |y| <= 1 and a little more, which rounds to 1: the topmost code needs no clamp
    const unsigned y = __float_as_uint(__fmul_rn(x[i], r));
    const unsigned bits = SIGNED ? y & 0x7fffffffu : y;
    int c;
    if (RANDOM) c = random_code<SIGNED>(bits, mix32(first + i ^ key));
    else c = (int)((bits + ((1u << (shift - 1)) - 1u) + ((bits >> shift) & 1u)) >> shift) - offset;
    if (SIGNED) {
      c = c > 0 ? (int)((y >> 24 & 0x80u) | (unsigned)c) : 0;
    } else {
      c = max(c, bits != 0 ? 1 : 0);
    }
    code[i >> 2] |= (unsigned)c << (8 * (i & 3));
  }
}

template <bool SIGNED>
__device__ __forceinline__ void decode8(const unsigned (&code)[2], float scale, float (&x)[8]) {
  constexpr int shift = SIGNED ? 20 : 19, top = SIGNED ? 127 : 255, offset = (kOne >> shift) - top;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const unsigned c = __byte_perm(code[i >> 2], 0, 0x4440u | (unsigned)(i & 3));
    const unsigned low = SIGNED ? c & 127u : c;
    unsigned bits = (low << shift) + ((unsigned)offset << shift);
    if (SIGNED) bits |= (c & 128u) << 24;
    x[i] = low ? __fmul_rn(__uint_as_float(bits), scale) : __fmul_rn(0.f, scale);
  }
}

__device__ __forceinline__ void load_codes(const unsigned char *a, bool wide, int n, unsigned (&c)[2]) {
  if (wide && n >= 8) {
    const uint2 r = *reinterpret_cast<const uint2 *>(a);
    c[0] = r.x;
    c[1] = r.y;
    return;
  }
  c[0] = c[1] = 0;
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) c[i >> 2] |= (unsigned)a[i] << (8 * (i & 3));
}
__device__ __forceinline__ void store_codes(unsigned char *a, bool wide, int n, const unsigned (&c)[2]) {
  if (wide && n >= 8) {
    *reinterpret_cast<uint2 *>(a) = make_uint2(c[0], c[1]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) a[i] = (unsigned char)(c[i >> 2] >> (8 * (i & 3)));
}

template <typename T>
__device__ __forceinline__ void fetch8(const T *a, bool wide, int n, float (&x)[8]) {
  if (wide && n >= 8) load8(a, x);
  else load_some(a, n, x);
}
template <typename T>
__device__ __forceinline__ void put8(T *a, bool wide, int n, const float (&x)[8]) {
  if (wide && n >= 8) store8(a, x);
  else store_some(a, n, x);
}

// A warp works on consecutive units, so that it looks its tensor up once and again only at its end.
struct Span {
  int64_t begin, end;
};
__device__ __forceinline__ Span span_of(int64_t units) {
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32), w = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  return Span{w * units / warps, (w + 1) * units / warps};
}

// The tensor that unit `u` belongs to.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP> &t, int64_t u) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename PT, typename GT, int BITS, bool RANDOM, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> t,
                                                         const __grid_constant__ Rates rates) {
  __shared__ Consts shared_consts;
  __shared__ unsigned shared_key;
  if (threadIdx.x == 0) {
    shared_consts = constants(rates);
    if (RANDOM) shared_key = mix32(rates.seed + rates.clock->t * 0x9e3779b9u);
  }
  __syncthreads();
  const Consts c = shared_consts;
  const unsigned key = RANDOM ? shared_key : 0u;
  const int lane = threadIdx.x & 31;
  const int64_t units = t.first[t.count];
  const Span span = span_of(units);
  int k = span.begin < span.end ? tensor_of(t, span.begin) : 0;
  for (int64_t u = span.begin; u < span.end; u++) {
    while (u >= t.first[k + 1]) k++;
    const int64_t block = u - t.first[k];
    const int64_t at = block * kUnit + lane * 8;
    const int n = (int)min((int64_t)8, max((int64_t)0, t.n[k] - at));
    const bool wide = t.wide[k];
    PT *pp = static_cast<PT *>(t.p[k]) + at;
    const GT *gp = static_cast<const GT *>(t.g[k]) + at;
    float p[8], g[8], m[8], v[8], root[8];
    if (BITS == 32) {
      float *mp = static_cast<float *>(t.m[k]) + at, *vp = static_cast<float *>(t.v[k]) + at;
      fetch8(pp, wide, n, p);
      fetch8(gp, wide, n, g);
      fetch8(mp, wide, n, m);
      fetch8(vp, wide, n, v);
      step8(p, g, m, v, root, c);
      put8(pp, wide, n, p);
      put8(mp, wide, n, m);
      put8(vp, wide, n, v);
    } else {
      unsigned char *mp = static_cast<unsigned char *>(t.m[k]) + at, *vp = static_cast<unsigned char *>(t.v[k]) + at;
      unsigned mc[2], vc[2];
      fetch8(pp, wide, n, p);
      fetch8(gp, wide, n, g);
      load_codes(mp, wide, n, mc);
      load_codes(vp, wide, n, vc);
      decode8<true>(mc, t.ms[k][block], m);
      decode8<false>(vc, t.vs[k][block], v);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = __fmul_rn(v[i], v[i]);
      step8(p, g, m, v, root, c);
      const float ms = unit_scale(m), vs = unit_scale(root);
      const unsigned first = (unsigned)u * kUnit + lane * 8;
      encode8<true, RANDOM>(m, ms, mc, key, first);
      encode8<false, RANDOM>(root, vs, vc, key, first);
      put8(pp, wide, n, p);
      store_codes(mp, wide, n, mc);
      store_codes(vp, wide, n, vc);
      if (lane == 0) {
        t.ms[k][block] = ms;
        t.vs[k][block] = vs;
      }
    }
  }
  // The block that finishes last moves the clock on: every block has read it by then.
  if (rates.advance) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      if (atomicAdd(&rates.clock->arrived, 1u) == gridDim.x - 1) {
        rates.clock->b1t *= rates.beta1;
        rates.clock->b2t *= rates.beta2;
        rates.clock->t++;
        rates.clock->arrived = 0;
      }
    }
  }
}

// 8-bit moments as the values they stand for: p and g of the table are the two fp32 outputs.
template <int CAP>
__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ Table<CAP> t) {
  const int lane = threadIdx.x & 31;
  const int64_t units = t.first[t.count];
  const Span span = span_of(units);
  int k = span.begin < span.end ? tensor_of(t, span.begin) : 0;
  for (int64_t u = span.begin; u < span.end; u++) {
    while (u >= t.first[k + 1]) k++;
    const int64_t block = u - t.first[k];
    const int64_t at = block * kUnit + lane * 8;
    const int n = (int)min((int64_t)8, max((int64_t)0, t.n[k] - at));
    const bool wide = t.wide[k];
    unsigned mc[2], vc[2];
    float m[8], v[8];
    load_codes(static_cast<const unsigned char *>(t.m[k]) + at, wide, n, mc);
    load_codes(static_cast<const unsigned char *>(t.v[k]) + at, wide, n, vc);
    decode8<true>(mc, t.ms[k][block], m);
    decode8<false>(vc, t.vs[k][block], v);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __fmul_rn(v[i], v[i]);
    put8(static_cast<float *>(t.p[k]) + at, wide, n, m);
    put8(static_cast<float *>(const_cast<void *>(t.g[k])) + at, wide, n, v);
  }
}

__global__ void clock_kernel(Clock *c, double b1t, double b2t, unsigned t) { *c = Clock{b1t, b2t, 0, t}; }

bool aligned(const void *a, size_t to) { return reinterpret_cast<uintptr_t>(a) % to == 0; }
size_t type_size(int type) { return type == W2V_F32 ? 4 : 2; }

// Blocks: as many as fit on the SMs, and up to eight times that as long as each warp has eight units left
// (each block begins with a few hundred clocks of constants in 64 bits, but many short ones use the
// memory better than few long ones: 51 million elements in 224 us against 245).
int grid_for(int64_t units) {
  constexpr int warps = kThreads / 32;
  const int64_t fit = (int64_t)w2v::device_sm_count() * 4, need = (units + warps - 1) / warps;
  const int64_t most = std::min<int64_t>(fit * 8, units / (warps * 8));
  return (int)std::max<int64_t>(1, std::min(need, std::max(fit, most)));
}

enum Moments { kFp32, kNearest, kRandom };

template <typename PT, typename GT, int CAP>
int launch_typed(const Table<CAP> &t, const Rates &r, Moments moments, cudaStream_t s) {
  const int grid = grid_for(t.first[t.count]);
  if (moments == kFp32) adamw_kernel<PT, GT, 32, false, CAP><<<grid, kThreads, 0, s>>>(t, r);
  else if (moments == kNearest) adamw_kernel<PT, GT, 8, false, CAP><<<grid, kThreads, 0, s>>>(t, r);
  else adamw_kernel<PT, GT, 8, true, CAP><<<grid, kThreads, 0, s>>>(t, r);
  w2v::count_launch(1);
  return (int)cudaGetLastError();
}

template <int CAP>
int launch(const Table<CAP> &t, const Rates &r, int ptype, int gtype, Moments m, cudaStream_t s) {
  if (ptype == W2V_F32) return launch_typed<float, float>(t, r, m, s);
  if (ptype == W2V_BF16)
    return gtype == W2V_F32 ? launch_typed<__nv_bfloat16, float>(t, r, m, s)
                            : launch_typed<__nv_bfloat16, __nv_bfloat16>(t, r, m, s);
  return gtype == W2V_F32 ? launch_typed<__half, float>(t, r, m, s)
                          : launch_typed<__half, __half>(t, r, m, s);
}

template <int CAP>
void add(Table<CAP> &t, const w2v_adamw_tensor &x, const void *g, size_t psize, size_t gsize, int bits) {
  const int k = t.count++;
  if (k == 0) t.first[0] = 0;
  t.p[k] = x.p;
  t.g[k] = g;
  t.m[k] = x.m;
  t.v[k] = x.v;
  t.ms[k] = x.mscale;
  t.vs[k] = x.vscale;
  t.n[k] = x.n;
  t.first[k + 1] = t.first[k] + (x.n + kUnit - 1) / kUnit;
  const size_t state = bits == 32 ? 32 : 8;
  t.wide[k] = aligned(x.p, 8 * psize) && aligned(g, 8 * gsize) && aligned(x.m, state) && aligned(x.v, state);
}

constexpr int kFew = 16, kSome = 64, kMany = 256;

// Calls `go` with tables of at most `kMany` of the `n` chosen tensors (small tables for few: the
// arguments of a launch are copied with it, 16 KB in 8 us and 4 KB in 5).
template <typename ADD, typename GO>
int in_tables(int n, ADD put, GO go) {
  auto once = [&](auto &t) {
    t.count = 0;
    t.first[0] = 0;
    for (int i = 0; i < n; i++) put(t, i);
    return go(t, true);
  };
  if (n <= kFew) {
    Table<kFew> t;
    return once(t);
  }
  if (n <= kSome) {
    Table<kSome> t;
    return once(t);
  }
  for (int a = 0; a < n; a += kMany) {
    Table<kMany> t;
    t.count = 0;
    t.first[0] = 0;
    const int b = std::min(n, a + kMany);
    for (int i = a; i < b; i++) put(t, i);
    const int err = go(t, b == n);
    if (err) return err;
  }
  return 0;
}

bool good_state(const w2v_adamw_tensor &x, int bits) {
  if (x.n < 0 || x.n > ((int64_t)1 << 42)) return false;
  if (x.n == 0) return true;
  if (!x.m || !x.v) return false;
  return bits == 32 || (x.mscale && x.vscale);
}

int step(const w2v_adamw_tensor *tensors, const void *const *grads, const int *gtypes, int ntensors, Moments moments,
         const w2v_adamw_opts *o, const float *lrate_dev, uint64_t seed, void *clock, void *stream) {
  const int bits = moments == kFp32 ? 32 : 8;
  if (ntensors < 0 || (ntensors > 0 && (!tensors || !grads || !gtypes)) || !o || !clock || !aligned(clock, 8)) return 1;
  if (!(o->beta1 >= 0 && o->beta1 < 1) || !(o->beta2 >= 0 && o->beta2 < 1) || !(o->eps > 0)) return 1;
  // the tensors of each pair of types go together; the last launch of all moves the clock on
  constexpr int kPairs = 5;
  const int pairs[kPairs][2] = {{W2V_F32, W2V_F32}, {W2V_BF16, W2V_F32}, {W2V_BF16, W2V_BF16},
                                {W2V_F16, W2V_F32}, {W2V_F16, W2V_F16}};
  int counts[kPairs] = {0, 0, 0, 0, 0};
  auto pair_of = [&](int i) {
    for (int q = 0; q < kPairs; q++)
      if (tensors[i].ptype == pairs[q][0] && gtypes[i] == pairs[q][1]) return q;
    return -1;
  };
  for (int i = 0; i < ntensors; i++) {
    const int q = pair_of(i);
    if (q < 0 || !good_state(tensors[i], bits)) return 1;
    if (tensors[i].n > 0 && (!tensors[i].p || !grads[i])) return 1;
    if (tensors[i].n > 0) counts[q]++;
  }
  int last = 0;
  for (int q = 0; q < kPairs; q++)
    if (counts[q]) last = q;
  const auto s = static_cast<cudaStream_t>(stream);
  Rates r{o->lrate, o->beta1, o->beta2, o->eps, o->wdecay, lrate_dev, static_cast<Clock *>(clock), 0, 0};
  unsigned launches = 0;
  for (int q = 0; q <= last; q++) {
    if (!counts[q] && q != last) continue;
    int next = 0;   // walks the tensors of this pair in order
    const int err = in_tables(
        counts[q],
        [&](auto &t, int) {
          while (tensors[next].n == 0 || pair_of(next) != q) next++;
          add(t, tensors[next], grads[next], type_size(pairs[q][0]), type_size(pairs[q][1]), bits);
          next++;
        },
        [&](const auto &t, bool end) {
          r.advance = end && q == last;
          // launches number their elements from zero: random bits of their own
          r.seed = mix32((unsigned)seed + mix32((unsigned)(seed >> 32) + launches++ * 0x9e3779b9u));
          return launch(t, r, pairs[q][0], pairs[q][1], moments, s);
        });
    if (err) return err;
  }
  return 0;
}

}  // namespace

extern "C" int w2v_adamw_clock(void *clock, double beta1, double beta2, int64_t t, void *stream) {
  if (!clock || !aligned(clock, 8) || t < 0 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1)) return 1;
  clock_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<Clock *>(clock), pow(beta1, (double)t),
                                                               pow(beta2, (double)t), (unsigned)t);
  w2v::count_launch(1);
  return (int)cudaGetLastError();
}

extern "C" int w2v_adamw_step(const w2v_adamw_tensor *tensors, const void *const *grads, const int *gtypes,
                              int ntensors, int bits, const w2v_adamw_opts *o, const float *lrate_dev, void *clock,
                              void *stream) {
  if (bits != 32 && bits != 8) return 1;
  return step(tensors, grads, gtypes, ntensors, bits == 32 ? kFp32 : kNearest, o, lrate_dev, 0, clock, stream);
}

extern "C" int w2v_adamw_step_random(const w2v_adamw_tensor *tensors, const void *const *grads, const int *gtypes,
                                     int ntensors, const w2v_adamw_opts *o, const float *lrate_dev, uint64_t seed,
                                     void *clock, void *stream) {
  return step(tensors, grads, gtypes, ntensors, kRandom, o, lrate_dev, seed, clock, stream);
}

extern "C" int w2v_adamw_moments(const w2v_adamw_tensor *tensors, float *const *mout, float *const *vout, int ntensors,
                                 void *stream) {
  if (ntensors < 0 || (ntensors > 0 && (!tensors || !mout || !vout))) return 1;
  int count = 0;
  for (int i = 0; i < ntensors; i++) {
    if (!good_state(tensors[i], 8) || (tensors[i].n > 0 && (!mout[i] || !vout[i]))) return 1;
    count += tensors[i].n > 0;
  }
  if (!count) return 0;
  const auto s = static_cast<cudaStream_t>(stream);
  int next = 0;
  return in_tables(
      count,
      [&](auto &t, int) {
        while (tensors[next].n == 0) next++;
        w2v_adamw_tensor x = tensors[next];
        x.p = mout[next];
        add(t, x, vout[next], 4, 4, 8);
        next++;
      },
      [&](const auto &t, bool) {
        moments_kernel<<<grid_for(t.first[t.count]), kThreads, 0, s>>>(t);
        w2v::count_launch(1);
        return (int)cudaGetLastError();
      });
}
