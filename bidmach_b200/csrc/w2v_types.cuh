// Element types of the training operators: 8 consecutive elements in the registers of one lane.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace w2v {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// 8 elements at an address aligned to their size (32 bytes of fp32, 16 of a 16-bit type): one load.
__device__ __forceinline__ void load8(const float *a, float (&x)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(a)
               : "memory");
}
__device__ __forceinline__ void store8(float *a, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a), "f"(x[0]), "f"(x[1]),
               "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
// Two 16-bit values in a word.
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b, __nv_bfloat16) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ uint32_t packed2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t packed2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}
template <typename T>
__device__ __forceinline__ void load8(const T *a, float (&x)[8]) {
  static_assert(sizeof(T) == 2, "a 16-bit type");
  const uint4 raw = *reinterpret_cast<const uint4 *>(a);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; i++) unpack2(w[i], x[2 * i], x[2 * i + 1], T());
}
template <typename T>
__device__ __forceinline__ void store8(T *a, const float (&x)[8]) {
  static_assert(sizeof(T) == 2, "a 16-bit type");
  *reinterpret_cast<uint4 *>(a) = make_uint4(packed2(x[0], x[1], T()), packed2(x[2], x[3], T()), packed2(x[4], x[5], T()),
                                             packed2(x[6], x[7], T()));
}

// The first `n` of 8 elements, one at a time: any alignment; the others read as zero.
template <typename T>
__device__ __forceinline__ void load_some(const T *a, int n, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = i < n ? to_float(a[i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_some(T *a, int n, const float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) a[i] = from_float<T>(x[i]);
}

}  // namespace w2v
