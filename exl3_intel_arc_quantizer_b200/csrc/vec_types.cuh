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

// V elements as 32-bit words, the way they are loaded, selected and stored (a
// struct of 16-bit elements makes the compiler move each element by itself)
template <typename T, int V>
struct Raw {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  static_assert(V * sizeof(T) % 4 == 0, "whole words");
  uint32_t w[kWords];
};

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  Raw<T, V> r;
  constexpr int n = Raw<T, V>::kWords;
  if constexpr (n % 4 == 0) {
#pragma unroll
    for (int i = 0; i < n; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
      r.w[i] = x.x;
      r.w[i + 1] = x.y;
      r.w[i + 2] = x.z;
      r.w[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, V>& r) {
  constexpr int n = Raw<T, V>::kWords;
  if constexpr (n % 4 == 0) {
#pragma unroll
    for (int i = 0; i < n; i += 4)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) =
          make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) reinterpret_cast<uint32_t*>(p)[i] = r.w[i];
  }
}

// a word of two 16-bit elements
template <typename T>
__device__ __forceinline__ float2 word_to_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 word_to_f32<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 word_to_f32<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t f32_to_word(float2 f);
template <>
__device__ __forceinline__ uint32_t f32_to_word<__half>(float2 f) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t f32_to_word<__nv_bfloat16>(float2 f) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 x = word_to_f32<T>(r.w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&f)[V]) {
  Raw<T, V> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.w[i] = f32_to_word<T>(make_float2(f[2 * i], f[2 * i + 1]));
  }
  return r;
}

// The same for single elements, which have no words of their own
template <typename T, int V>
struct Pieces {
  using type = Raw<T, V>;
};
template <typename T>
struct Pieces<T, 1> {
  using type = float;
};
template <typename T, int V>
__device__ __forceinline__ typename Pieces<T, V>::type load_piece(const T* p) {
  if constexpr (V == 1)
    return to_f32(*p);
  else
    return load_raw<T, V>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[V]) {
  if constexpr (V == 1)
    *p = from_f32<T>(f[0]);
  else
    store_raw<T, V>(p, pack<T, V>(f));
}
__device__ __forceinline__ void unpack(float x, float (&f)[1]) { f[0] = x; }

// Arithmetic on V floats, two at a time where there are two (packed f32x2:
// each lane rounds like the scalar operation)
__device__ __forceinline__ float2 pair_of(float s) { return make_float2(s, s); }
#define EXL3_PAIRWISE(a, pair_expr, one_expr)                              \
  if constexpr (V % 2 == 0) {                                              \
    _Pragma("unroll") for (int i = 0; i < V; i += 2) {                     \
      const float2 x = make_float2((a)[i], (a)[i + 1]);                    \
      const float2 r = pair_expr;                                          \
      (a)[i] = r.x;                                                        \
      (a)[i + 1] = r.y;                                                    \
    }                                                                      \
  } else {                                                                 \
    _Pragma("unroll") for (int i = 0; i < V; ++i) {                        \
      const float x = (a)[i];                                              \
      (a)[i] = one_expr;                                                   \
    }                                                                      \
  }
// a s
template <int V>
__device__ __forceinline__ void vec_scale(float (&a)[V], float s) {
  EXL3_PAIRWISE(a, __fmul2_rn(x, pair_of(s)), x * s)
}
// a + s
template <int V>
__device__ __forceinline__ void vec_add(float (&a)[V], float s) {
  EXL3_PAIRWISE(a, __fadd2_rn(x, pair_of(s)), x + s)
}
// a b
template <int V>
__device__ __forceinline__ void vec_mul(float (&a)[V], const float (&b)[V]) {
  EXL3_PAIRWISE(a, __fmul2_rn(x, make_float2(b[i], b[i + 1])), x * b[i])
}
// s a + c
template <int V>
__device__ __forceinline__ void vec_axpy(float (&a)[V], float s, const float (&c)[V]) {
  EXL3_PAIRWISE(a, __ffma2_rn(pair_of(s), x, make_float2(c[i], c[i + 1])), fmaf(s, x, c[i]))
}
// b a + c
template <int V>
__device__ __forceinline__ void vec_fma(float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  EXL3_PAIRWISE(a, __ffma2_rn(make_float2(b[i], b[i + 1]), x, make_float2(c[i], c[i + 1])),
                fmaf(b[i], x, c[i]))
}
#undef EXL3_PAIRWISE
// acc + a^2, two sums
template <int V>
__device__ __forceinline__ void vec_squares(const float (&a)[V], float2& acc) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = make_float2(a[i], a[i + 1]);
      acc = __ffma2_rn(x, x, acc);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) acc.x = fmaf(a[i], a[i], acc.x);
  }
}

inline bool aligned_to(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace exl3
