// What the token-by-token and the chunked gated delta rule share.
#pragma once

#include "common.cuh"
#include "vec_types.cuh"

namespace exl3 {

constexpr float kNormEps = 1e-6f;  // added to a sum of squares of q or k

// The chunked form (delta_chunk.cu); dk <= 128.
size_t delta_chunk_ws_bytes(const exl3_delta_args& a);
int delta_chunks(const exl3_delta_args& a, void* ws, cudaStream_t stream);

// Tokens [t0, t1) of sequence s. The offsets are device data that the host
// has not seen: they are clamped into [0, tokens], and a sequence that would
// end before it begins is empty.
__device__ __forceinline__ void seq_bounds(const exl3_delta_args& a, int64_t s, int64_t& t0,
                                           int64_t& t1) {
  const int64_t b = a.cu_seqlens[s], e = a.cu_seqlens[s + 1];
  t0 = b < 0 ? 0 : b > a.tokens ? a.tokens : b;
  t1 = e < t0 ? t0 : e > a.tokens ? a.tokens : e;
}

// Outputs of the tokens before the first and after the last sequence: n
// columns from col of head h, written by the threads of those sequences.
template <typename T>
__device__ __forceinline__ void zero_outside(const exl3_delta_args& a, int64_t s, int64_t t0,
                                             int64_t t1, int h, int col, int n) {
  T* o = static_cast<T*>(a.out);
  if (s == 0)
    for (int64_t t = 0; t < t0; ++t)
      for (int c = 0; c < n; ++c) o[(t * a.heads + h) * a.dv + col + c] = from_f32<T>(0.f);
  if (s == a.seqs - 1)
    for (int64_t t = t1; t < a.tokens; ++t)
      for (int c = 0; c < n; ++c) o[(t * a.heads + h) * a.dv + col + c] = from_f32<T>(0.f);
}

}  // namespace exl3
