// Element types and vectors of the layer operators: fp16, bf16 and fp32
// values, computed in fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace exl3 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// V elements loaded and stored at once (one 16-byte access where they fill it)
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// Two elements at a time: one conversion instruction per pair on the way back
__device__ __forceinline__ float2 to_f32x2(const Vec<__half, 2>& v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float2 to_f32x2(const Vec<__nv_bfloat16, 2>& v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ float2 to_f32x2(const Vec<float, 2>& v) {
  return make_float2(v.e[0], v.e[1]);
}
template <typename T>
__device__ __forceinline__ Vec<T, 2> from_f32x2(float2 f);
template <>
__device__ __forceinline__ Vec<__half, 2> from_f32x2<__half>(float2 f) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const Vec<__half, 2>*>(&h);
}
template <>
__device__ __forceinline__ Vec<__nv_bfloat16, 2> from_f32x2<__nv_bfloat16>(float2 f) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const Vec<__nv_bfloat16, 2>*>(&h);
}
template <>
__device__ __forceinline__ Vec<float, 2> from_f32x2<float>(float2 f) {
  return {{f.x, f.y}};
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f32(v.e[0]);
  } else {
    const Vec<T, 2>* p = reinterpret_cast<const Vec<T, 2>*>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 x = to_f32x2(p[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> pack(const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (V == 1) {
    v.e[0] = from_f32<T>(f[0]);
  } else {
    Vec<T, 2>* p = reinterpret_cast<Vec<T, 2>*>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = from_f32x2<T>(make_float2(f[2 * i], f[2 * i + 1]));
  }
  return v;
}

inline bool aligned_to(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace exl3
