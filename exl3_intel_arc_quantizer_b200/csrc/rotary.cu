// Rotary positions on the queries and keys of a layer, one launch for both.
//
// phi = position * inv_freq[j]; a pair (a, b) of a head turns to
// f (a cos phi - b sin phi), f (b cos phi + a sin phi); the elements past
// rotary_dim are copied. In fp32 the product position * inv_freq is off by
// up to 2^-24 of its size (0.008 rad at position 131,072), so the angle is
// taken as a fraction of a turn in 64-bit fixed point: inv_freq / 2 pi
// within 2^-62, times the position, wraps exactly at whole turns.
//
// Bound: HBM (each element is read and written once). A CTA holds the
// cosines and sines of its tokens in shared memory, computed once and used
// by every head; a thread then turns 16-byte vectors (one from each half of
// the head, or one vector of four neighbouring pairs), kUnroll of them
// loaded before the first is turned.
#include "common.cuh"
#include "vec_types.cuh"

namespace exl3 {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

struct RotaryLaunch {
  exl3_rotary_args a;
  int tokens_per_cta;   // a CTA's tokens (of one batch entry)
  int heads_per_cta;    // its q and k heads
  int lanes;            // threads that share a head (a power of two <= 32)
};

// inv_freq / 2 pi as a fraction of a turn in units of 2^-64. 1 / 2 pi is a
// 28-bit head, whose product with a 24-bit frequency is exact in a double,
// and a tail of 2^-30 of its size.
__device__ __forceinline__ uint64_t turn_step(float inv_freq) {
  const double f = (double)inv_freq;
  double head = f * 0x1.45f306cp-3, tail = f * 0x1.c9c882a53f84fp-31;
  head -= floor(head);
  tail -= floor(tail);
  return __double2ull_rz(head * 0x1p64) + __double2ull_rz(tail * 0x1p64);
}

// An item is what a thread turns at once: V pairs (two vectors of the half
// layout, or 2V neighbouring elements = two vectors, interleaved), or two
// vectors of the part that is copied.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryLaunch p) {
  extern __shared__ float2 cs[];  // [tokens][rotary_dim / 2]: factor * (cos, sin)
  const exl3_rotary_args& a = p.a;
  const int half = a.rotary_dim / 2, tid = threadIdx.x;
  const int64_t blocks = (a.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  const int64_t b = blockIdx.x / blocks, t0 = (blockIdx.x - b * blocks) * p.tokens_per_cta;
  const int nt = (int)(a.tokens - t0 < p.tokens_per_cta ? a.tokens - t0 : p.tokens_per_cta);
  const int h0 = blockIdx.y * p.heads_per_cta;
  const int heads = a.q_heads + a.k_heads;
  const int nh = heads - h0 < p.heads_per_cta ? heads - h0 : p.heads_per_cta;

  for (int i = tid; i < nt * half; i += kThreads) {
    const int t = i / half, j = i - t * half;
    const int64_t at = b * a.position_strides[0] + (t0 + t) * a.position_strides[1];
    const int64_t pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[at]
                                       : static_cast<const int32_t*>(a.positions)[at];
    const uint64_t step = turn_step(a.inv_freq[j]);
    const int64_t phase = (int64_t)((uint64_t)pos * step);
    float s, c;
    sincospif(__ll2float_rn(phase) * 1.0842021724855044e-19f, &s, &c);  // 2^-63: half turns
    if (a.transposed) s = -s;
    cs[i] = make_float2(a.factor * c, a.factor * s);
  }
  __syncthreads();

  const int turned = half / V;                                   // items that turn, per head
  const int copied = (a.dim - a.rotary_dim) / V;                 // vectors that are copied
  const int items = turned + (copied + 1) / 2;
  const int lane = tid & (p.lanes - 1), groups = kThreads / p.lanes;
  const int pairs = nt * nh;
  using Ve = Vec<T, V>;
  for (int i0 = lane; i0 < items; i0 += p.lanes) {
    const bool turn = i0 < turned;
    const int e0 = turn ? (INTER ? 2 * V * i0 : V * i0) : a.rotary_dim + 2 * V * (i0 - turned);
    const int e1 = turn ? (INTER ? e0 + V : e0 + half) : e0 + V;
    const bool second = e1 < a.dim;
    for (int p0 = tid / p.lanes; p0 < pairs; p0 += groups * kUnroll) {
      Ve x0[kUnroll], x1[kUnroll];
      T* dst[kUnroll];
      const float2* tab[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int pr = p0 + u * groups;
        if (pr >= pairs) break;
        const int t = pr / nh, h = h0 + pr - t * nh;
        const bool isq = h < a.q_heads;
        const int hh = isq ? h : h - a.q_heads;
        const int64_t* si = isq ? a.q_strides : a.k_strides;
        const int64_t* so = isq ? a.q_out_strides : a.k_out_strides;
        const T* src = static_cast<const T*>(isq ? a.q : a.k) + b * si[0] + (t0 + t) * si[1] + hh * si[2];
        dst[u] = static_cast<T*>(isq ? a.q_out : a.k_out) + b * so[0] + (t0 + t) * so[1] + hh * so[2];
        tab[u] = cs + t * half + V * i0;
        x0[u] = *reinterpret_cast<const Ve*>(src + e0);
        if (second) x1[u] = *reinterpret_cast<const Ve*>(src + e1);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (p0 + u * groups >= pairs) break;
        if (turn) {
          if constexpr (INTER) {
            T* y0 = x0[u].e;
            T* y1 = x1[u].e;
#pragma unroll
            for (int m = 0; m < V; ++m) {
              // pair m holds elements 2m and 2m + 1 of the two vectors
              T& ea = (2 * m < V) ? y0[(2 * m) % V] : y1[(2 * m) % V];
              T& eb = (2 * m + 1 < V) ? y0[(2 * m + 1) % V] : y1[(2 * m + 1) % V];
              const float2 w = tab[u][m];
              const float va = to_f32(ea), vb = to_f32(eb);
              ea = from_f32<T>(va * w.x - vb * w.y);
              eb = from_f32<T>(vb * w.x + va * w.y);
            }
          } else {
#pragma unroll
            for (int m = 0; m < V; ++m) {
              const float2 w = tab[u][m];
              const float va = to_f32(x0[u].e[m]), vb = to_f32(x1[u].e[m]);
              x0[u].e[m] = from_f32<T>(va * w.x - vb * w.y);
              x1[u].e[m] = from_f32<T>(vb * w.x + va * w.y);
            }
          }
        }
        *reinterpret_cast<Ve*>(dst[u] + e0) = x0[u];
        if (second) *reinterpret_cast<Ve*>(dst[u] + e1) = x1[u];
      }
    }
  }
}

template <typename T, int V>
int launch(const exl3_rotary_args& a, cudaStream_t stream) {
  RotaryLaunch p;
  p.a = a;
  const int heads = a.q_heads + a.k_heads, half = a.rotary_dim / 2;
  const int items = half / V + ((a.dim - a.rotary_dim) / V + 1) / 2;
  p.lanes = 1;
  while (p.lanes < items && p.lanes < 32) p.lanes *= 2;
  // few tokens: a CTA takes one token and as many heads as its threads hold
  // at once; many tokens: all heads, and tokens for four rounds of loads
  const int groups = kThreads / p.lanes;
  int tokens = 1;
  while (tokens * heads < groups * kUnroll && tokens * 2 * half * 8 <= 32768 &&
         a.batch * ((a.tokens + 2 * tokens - 1) / (2 * tokens)) >= 4 * sm_count())
    tokens *= 2;
  p.tokens_per_cta = tokens;
  p.heads_per_cta = a.batch * a.tokens >= 4 * sm_count() ? heads : (groups < heads ? groups : heads);
  const int64_t bx = a.batch * ((a.tokens + tokens - 1) / tokens);
  const int by = (heads + p.heads_per_cta - 1) / p.heads_per_cta;
  EXL3_REQUIRE(bx < (1ll << 31) && by < 65536, "too many tokens or heads");
  const dim3 grid((unsigned)bx, (unsigned)by);
  const size_t smem = (size_t)tokens * half * sizeof(float2);
  if (a.interleaved)
    rotary_kernel<T, V, true><<<grid, kThreads, smem, stream>>>(p);
  else
    rotary_kernel<T, V, false><<<grid, kThreads, smem, stream>>>(p);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

bool vectors_fit(const void* ptr, const int64_t* strides, int64_t v, size_t bytes) {
  return aligned_to(ptr, bytes) && strides[0] % v == 0 &&
         strides[1] % v == 0 && strides[2] % v == 0;
}

template <typename T>
int launch_t(const exl3_rotary_args& a, cudaStream_t stream) {
  // 16-byte vectors where every head starts on one and both halves are whole
  // vectors; else element by element
  constexpr int V = 16 / sizeof(T);
  const bool wide = (a.rotary_dim / 2) % V == 0 && a.dim % V == 0 &&
                    vectors_fit(a.q, a.q_strides, V, 16) && vectors_fit(a.q_out, a.q_out_strides, V, 16) &&
                    (a.k_heads == 0 || (vectors_fit(a.k, a.k_strides, V, 16) &&
                                        vectors_fit(a.k_out, a.k_out_strides, V, 16)));
  return wide ? launch<T, V>(a, stream) : launch<T, 1>(a, stream);
}

}  // namespace
}  // namespace exl3

using namespace exl3;

extern "C" int exl3_rotary(const exl3_rotary_args* args, exl3_stream_t stream) {
  EXL3_REQUIRE(args != nullptr, "args is NULL");
  const exl3_rotary_args& a = *args;
  EXL3_REQUIRE(a.dtype >= EXL3_F16 && a.dtype <= EXL3_F32, "dtype must be 0..2, got %d", a.dtype);
  EXL3_REQUIRE(a.batch >= 0 && a.tokens >= 0, "batch and tokens must be non-negative");
  EXL3_REQUIRE(a.q_heads >= 1 && a.k_heads >= 0, "q_heads must be positive and k_heads non-negative");
  EXL3_REQUIRE(a.rotary_dim >= 2 && a.rotary_dim % 2 == 0 && a.rotary_dim <= a.dim && a.dim <= 8192,
               "rotary_dim must be even, in 2..dim, and dim at most 8192, got %d of %d",
               a.rotary_dim, a.dim);
  if (a.batch == 0 || a.tokens == 0) return EXL3_OK;
  EXL3_REQUIRE(a.q && a.q_out && a.positions && a.inv_freq && (a.k_heads == 0 || (a.k && a.k_out)),
               "NULL pointer argument");
  cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == EXL3_F16) return launch_t<__half>(a, s);
  if (a.dtype == EXL3_BF16) return launch_t<__nv_bfloat16>(a, s);
  return launch_t<float>(a, s);
}
