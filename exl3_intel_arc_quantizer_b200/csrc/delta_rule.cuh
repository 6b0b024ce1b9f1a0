// What the token-by-token and the chunked gated delta rule share.
#pragma once

#include "common.cuh"
#include "vec_types.cuh"

namespace exl3 {

constexpr float kNormEps = 1e-6f;  // added to a sum of squares of q or k

// The chunked form (delta_chunk.cu), dk <= 128, of the sequences of more than
// `above` tokens (-1: of all).
size_t delta_chunk_ws_bytes(const exl3_delta_args& a);
int delta_chunks(const exl3_delta_args& a, void* ws, int above, cudaStream_t stream);

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

// N consecutive elements of a row of k or q, zero past its end
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_row(const T* p, int at, int d, bool vec) {
  Raw<T, N> r;
  if (vec && N == 4) {
    if (at < d) {
      const uint2 x = *reinterpret_cast<const uint2*>(p + at);
      r.w[0] = x.x;
      r.w[1] = x.y;
    } else {
      r.w[0] = r.w[1] = 0u;
    }
  } else if (vec) {
#pragma unroll
    for (int c = 0; c < N; c += 8) {
      Raw<T, 8> x = {{0, 0, 0, 0}};
      if (at + c < d) x = load_raw<T, 8>(p + at + c);  // d is a multiple of 8
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[c / 2 + i] = x.w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      r.w[i / 2] = at + i < d ? f32_to_word<T>(make_float2(to_f32(p[at + i]), to_f32(p[at + i + 1]))) : 0u;
  }
  return r;
}

// Tokens t0 .. t1 - 1 of one sequence and head, by one warp: four columns from
// `col` per lane, CL lanes side by side, the state's rows over the others
// (ROWS each, dk <= ROWS * 32 / CL). The state is number `slot`. vec: bit 0
// for rows of k and q that can be read in 16-byte words, bit 1 for v in
// 8-byte words. Two rows of the state stand in a float2, so that the packed
// arithmetic takes k and q as they are loaded; the loads of a token are
// issued before the sums of the one before it.
template <typename T, int ROWS, int CL>
__device__ __forceinline__ void token_steps(const exl3_delta_args& a, int64_t slot, int h, int col, int64_t t0,
                                            int64_t t1, int lane, int vec) {
  const bool in = col < a.dv;  // dv is a multiple of 8: four columns are all in or all out
  const int row0 = (lane / CL) * ROWS, kh = h / (a.heads / a.key_heads);
  const int64_t state_at = (slot * a.heads + h) * (int64_t)a.dk * a.dv + (int64_t)row0 * a.dv + col;
  float2 S[ROWS / 2][4];
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (a.state_in && in && row0 + 2 * i < a.dk) {  // dk is even
      x = *reinterpret_cast<const float4*>(a.state_in + state_at + (int64_t)(2 * i) * a.dv);
      y = *reinterpret_cast<const float4*>(a.state_in + state_at + (int64_t)(2 * i + 1) * a.dv);
    }
    S[i][0] = make_float2(x.x, y.x);
    S[i][1] = make_float2(x.y, y.y);
    S[i][2] = make_float2(x.z, y.z);
    S[i][3] = make_float2(x.w, y.w);
  }
  const T* q = static_cast<const T*>(a.q) + kh * a.q_strides[1];
  const T* k = static_cast<const T*>(a.k) + kh * a.k_strides[1];
  const T* v = static_cast<const T*>(a.v) + h * a.v_strides[1];
  Raw<T, ROWS> kw, qw;
  Raw<T, 4> vw = {{0, 0}};
  float gt = 0.f, bt = 0.f;
  const auto load = [&](int64_t t) {
    kw = load_row<T, ROWS>(k + t * a.k_strides[0], row0, a.dk, vec & 1);
    qw = load_row<T, ROWS>(q + t * a.q_strides[0], row0, a.dk, vec & 1);
    if (in) {
      const T* p = v + t * a.v_strides[0] + col;
      if (vec & 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        vw = {{x.x, x.y}};
      } else {
        const float f[4] = {to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3])};
        vw = pack<T, 4>(f);
      }
    }
    gt = a.g[t * a.g_stride + h];
    bt = a.beta[t * a.beta_stride + h];
  };
  if (t0 < t1) load(t0);
  for (int64_t t = t0; t < t1; ++t) {
    float2 kr[ROWS / 2], qr[ROWS / 2];
    float vr[4];
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i) {
      kr[i] = word_to_f32<T>(kw.w[i]);
      qr[i] = word_to_f32<T>(qw.w[i]);
    }
    unpack(vw, vr);
    const float G = expf(gt), beta = bt;
    if (t + 1 < t1) load(t + 1);
    // kk, qq, qk, then the four columns of S^T k and S^T q
    float2 pair[11];
#pragma unroll
    for (int j = 0; j < 11; ++j) pair[j] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i) {
      pair[0] = __ffma2_rn(kr[i], kr[i], pair[0]);
      pair[1] = __ffma2_rn(qr[i], qr[i], pair[1]);
      pair[2] = __ffma2_rn(qr[i], kr[i], pair[2]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        pair[3 + c] = __ffma2_rn(S[i][c], kr[i], pair[3 + c]);
        pair[7 + c] = __ffma2_rn(S[i][c], qr[i], pair[7 + c]);
      }
    }
    float r[11];
#pragma unroll
    for (int j = 0; j < 11; ++j) r[j] = pair[j].x + pair[j].y;
#pragma unroll
    for (int o = CL; o < 32; o <<= 1)
#pragma unroll
      for (int j = 0; j < 11; ++j) r[j] += __shfl_xor_sync(0xFFFFFFFFu, r[j], o);
    const float rk = a.normalize_qk ? rsqrtf(r[0] + kNormEps) : 1.f;
    const float rq = (a.normalize_qk ? rsqrtf(r[1] + kNormEps) : 1.f) * a.scale;
    float o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float u = beta * (vr[c] - G * rk * r[3 + c]);
      o[c] = rq * (G * r[7 + c] + r[2] * rk * u);
#pragma unroll
      for (int i = 0; i < ROWS / 2; ++i)
        S[i][c] = __ffma2_rn(kr[i], pair_of(rk * u), __fmul2_rn(pair_of(G), S[i][c]));
    }
    if (in && lane < CL)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (t * a.heads + h) * a.dv + col) =
          make_uint2(f32_to_word<T>(make_float2(o[0], o[1])), f32_to_word<T>(make_float2(o[2], o[3])));
  }
  if (in)
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i)
      if (row0 + 2 * i < a.dk) {
        *reinterpret_cast<float4*>(a.state_out + state_at + (int64_t)(2 * i) * a.dv) =
            make_float4(S[i][0].x, S[i][1].x, S[i][2].x, S[i][3].x);
        *reinterpret_cast<float4*>(a.state_out + state_at + (int64_t)(2 * i + 1) * a.dv) =
            make_float4(S[i][0].y, S[i][1].y, S[i][2].y, S[i][3].y);
      }
}

}  // namespace exl3
