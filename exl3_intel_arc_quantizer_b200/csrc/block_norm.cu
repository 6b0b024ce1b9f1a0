// The norm after a block, its gate, the scaled residual sum and the norm
// before the next block in one pass over the rows.
//
//   y = x / sqrt(mean(x^2) + eps) * (offset + weight)     (or x)
//   y = y * act(gate)                                      (or y)
//   h = residual + s * y                      (or y)       -> hidden
//   n = h / sqrt(mean(h^2) + eps) * (offset + next_weight) -> normed
//
// The second norm takes h before its rounding. Bound: HBM, each tensor moved
// once: a row stays in registers as fp32 between its two sums. Rows of up to
// 1,024 elements belong to part of a warp or a warp (sums by shuffles), longer
// ones to a CTA (one barrier per sum); rows past the registers of a CTA are
// read again for each sum.
#include "common.cuh"
#include "vec_types.cuh"

namespace exl3 {
namespace {

constexpr int kMaxThreads = 512;  // of a CTA that owns a row: 128 registers each

__device__ __forceinline__ float act_sigmoid(float z) {
  // exp(-z) = inf gives 0
  return __frcp_rn(1.0f + __expf(-z));
}

__device__ __forceinline__ float gated(float y, float z, int act) {
  return y * (act == 1 ? act_sigmoid(z) : z * act_sigmoid(z));
}

// Sum over the threads of a row: `lanes` neighbouring threads of a warp, or
// the CTA. red: 2 x 32 floats; the slot alternates, so that one barrier per
// sum is enough (a slot is written again only after the next sum's barrier).
template <bool CTA_ROW>
__device__ __forceinline__ float row_sum(float v, int lanes, float (*red)[32], int& slot) {
  if (CTA_ROW) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < warps; ++w) v += red[slot][w];
    slot ^= 1;
    return v;
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

template <typename T, typename P, int V, int NV, bool CTA_ROW>
__global__ void __launch_bounds__(CTA_ROW ? kMaxThreads : 128)
block_norm_kernel(const __grid_constant__ exl3_block_norm_args a, int lanes) {
  __shared__ float red[2][32];
  int slot = 0;
  const int per_cta = CTA_ROW ? 1 : blockDim.x / lanes;
  const int lane = CTA_ROW ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int width = CTA_ROW ? blockDim.x : lanes;
  const int sub = CTA_ROW ? 0 : threadIdx.x / lanes;
  const int nvec = (int)((a.d + V - 1) / V);
  const float inv_d = 1.0f / (float)a.d;
  using Vt = Vec<T, V>;
  using Vp = Vec<P, V>;
  const T* x = static_cast<const T*>(a.x);
  const T* gate = static_cast<const T*>(a.gate);
  const T* residual = static_cast<const T*>(a.residual);
  const P* weight = static_cast<const P*>(a.weight);
  const P* next_weight = static_cast<const P*>(a.next_weight);
  const P* scale = static_cast<const P*>(a.scale);
  T* hidden = static_cast<T*>(a.hidden);
  T* normed = static_cast<T*>(a.normed);

  for (int64_t r0 = (int64_t)blockIdx.x * per_cta; r0 < a.rows; r0 += (int64_t)gridDim.x * per_cta) {
    // every thread of the warp takes part in the sums; rows past the end
    // compute on zeros and store nothing
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    float y[NV][V];
    Vt gv[NV], rv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + i * width;
      const bool in = live && c < nvec;
      Vt xv = {};
      gv[i] = {};
      rv[i] = {};
      if (in) {
        xv = *reinterpret_cast<const Vt*>(x + row * a.x_stride + (int64_t)c * V);
        if (gate) gv[i] = *reinterpret_cast<const Vt*>(gate + row * a.gate_stride + (int64_t)c * V);
        if (residual)
          rv[i] = *reinterpret_cast<const Vt*>(residual + row * a.residual_stride + (int64_t)c * V);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) y[i][e] = to_f32(xv.e[e]);
    }
    if (weight) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(y[i][e], y[i][e], ss);
      ss = row_sum<CTA_ROW>(ss, lanes, red, slot);
      const float r = rsqrtf(ss * inv_d + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = lane + i * width;
        if (c >= nvec) break;
        const Vp wv = *reinterpret_cast<const Vp*>(weight + (int64_t)c * V);
#pragma unroll
        for (int e = 0; e < V; ++e) y[i][e] = y[i][e] * r * (a.weight_offset + to_f32(wv.e[e]));
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + i * width;
      if (c >= nvec) break;
      Vp sv = {};
      if (scale) sv = *reinterpret_cast<const Vp*>(scale + (int64_t)c * V);
      Vt hv;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float h = y[i][e];
        if (gate) h = gated(h, to_f32(gv[i].e[e]), a.gate_activation);
        if (residual)
          h = fmaf(scale ? a.residual_scale * to_f32(sv.e[e]) : a.residual_scale, h,
                   to_f32(rv[i].e[e]));
        y[i][e] = h;
        ss = fmaf(h, h, ss);
        hv.e[e] = from_f32<T>(h);
      }
      if (hidden && live)
        *reinterpret_cast<Vt*>(hidden + row * a.hidden_stride + (int64_t)c * V) = hv;
    }
    if (next_weight) {
      ss = row_sum<CTA_ROW>(ss, lanes, red, slot);
      const float r = rsqrtf(ss * inv_d + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = lane + i * width;
        if (c >= nvec) break;
        const Vp wv = *reinterpret_cast<const Vp*>(next_weight + (int64_t)c * V);
        Vt nv;
#pragma unroll
        for (int e = 0; e < V; ++e)
          nv.e[e] = from_f32<T>(y[i][e] * r * (a.weight_offset + to_f32(wv.e[e])));
        if (live) *reinterpret_cast<Vt*>(normed + row * a.normed_stride + (int64_t)c * V) = nv;
      }
    }
  }
}

// Rows of any length, element by element, read again for each sum.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
block_norm_long_kernel(const __grid_constant__ exl3_block_norm_args a) {
  __shared__ float red[2][32];
  int slot = 0;
  const T* x = static_cast<const T*>(a.x);
  const T* gate = static_cast<const T*>(a.gate);
  const T* residual = static_cast<const T*>(a.residual);
  const P* weight = static_cast<const P*>(a.weight);
  const P* next_weight = static_cast<const P*>(a.next_weight);
  const P* scale = static_cast<const P*>(a.scale);
  T* hidden = static_cast<T*>(a.hidden);
  T* normed = static_cast<T*>(a.normed);
  const float inv_d = 1.0f / (float)a.d;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float r = 1.f;
    if (weight) {
      float ss = 0.f;
      for (int64_t c = threadIdx.x; c < a.d; c += blockDim.x) {
        const float v = to_f32(x[row * a.x_stride + c]);
        ss = fmaf(v, v, ss);
      }
      r = rsqrtf(row_sum<true>(ss, 32, red, slot) * inv_d + a.eps);
    }
    const auto value = [&](int64_t c) {
      float h = to_f32(x[row * a.x_stride + c]);
      if (weight) h = h * r * (a.weight_offset + to_f32(weight[c]));
      if (gate) h = gated(h, to_f32(gate[row * a.gate_stride + c]), a.gate_activation);
      if (residual)
        h = fmaf(scale ? a.residual_scale * to_f32(scale[c]) : a.residual_scale, h,
                 to_f32(residual[row * a.residual_stride + c]));
      return h;
    };
    float ss = 0.f, r2 = 0.f;
    if (next_weight) {
      for (int64_t c = threadIdx.x; c < a.d; c += blockDim.x) {
        const float h = value(c);
        ss = fmaf(h, h, ss);
      }
      r2 = rsqrtf(row_sum<true>(ss, 32, red, slot) * inv_d + a.eps);
    }
    for (int64_t c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float h = value(c);
      if (hidden) hidden[row * a.hidden_stride + c] = from_f32<T>(h);
      if (next_weight)
        normed[row * a.normed_stride + c] =
            from_f32<T>(h * r2 * (a.weight_offset + to_f32(next_weight[c])));
    }
  }
}

template <typename T, typename P, int V, int NV, bool CTA_ROW>
int launch(const exl3_block_norm_args& a, int threads, int lanes, cudaStream_t stream) {
  const int per_cta = CTA_ROW ? 1 : threads / lanes;
  const int64_t ctas = (a.rows + per_cta - 1) / per_cta;
  const int64_t most = (int64_t)sm_count() * 64;
  block_norm_kernel<T, P, V, NV, CTA_ROW>
      <<<(unsigned)(ctas < most ? ctas : most), threads, 0, stream>>>(a, lanes);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

template <typename T, typename P, int V>
int launch_v(const exl3_block_norm_args& a, cudaStream_t stream) {
  const int64_t nvec = (a.d + V - 1) / V;
  if (nvec <= 128) {
    int lanes = 1;
    while (lanes < nvec && lanes < 32) lanes *= 2;
    if (nvec <= lanes) return launch<T, P, V, 1, false>(a, 128, lanes, stream);
    if (nvec <= 2 * lanes) return launch<T, P, V, 2, false>(a, 128, lanes, stream);
    return launch<T, P, V, 4, false>(a, 128, lanes, stream);
  }
  const auto threads = [&](int nv) { return (int)((nvec + 32 * nv - 1) / (32 * nv)) * 32; };
  // few rows: as many threads as there are vectors; else two vectors each
  if (nvec <= kMaxThreads && a.rows <= sm_count())
    return launch<T, P, V, 1, true>(a, threads(1), 32, stream);
  if (nvec <= 2 * kMaxThreads) return launch<T, P, V, 2, true>(a, threads(2), 32, stream);
  if (nvec <= 4 * kMaxThreads) return launch<T, P, V, 4, true>(a, threads(4), 32, stream);
  const int64_t most = (int64_t)sm_count() * 16;
  block_norm_long_kernel<T, P>
      <<<(unsigned)(a.rows < most ? a.rows : most), 1024, 0, stream>>>(a);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

template <typename T, typename P>
int launch_t(const exl3_block_norm_args& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const auto row_ok = [](const void* p, int64_t stride) {
    return !p || (aligned_to(p, 16) && stride % V == 0);
  };
  const auto vec_ok = [](const void* p) { return !p || aligned_to(p, V * sizeof(P)); };
  const bool wide = a.d % V == 0 && row_ok(a.x, a.x_stride) && row_ok(a.gate, a.gate_stride) &&
                    row_ok(a.residual, a.residual_stride) && row_ok(a.hidden, a.hidden_stride) &&
                    row_ok(a.normed, a.normed_stride) && vec_ok(a.weight) &&
                    vec_ok(a.next_weight) && vec_ok(a.scale);
  return wide ? launch_v<T, P, V>(a, stream) : launch_v<T, P, 1>(a, stream);
}

}  // namespace
}  // namespace exl3

using namespace exl3;

extern "C" int exl3_block_norm(const exl3_block_norm_args* args, exl3_stream_t stream) {
  EXL3_REQUIRE(args != nullptr, "args is NULL");
  exl3_block_norm_args a = *args;
  EXL3_REQUIRE(a.dtype >= EXL3_F16 && a.dtype <= EXL3_F32, "dtype must be 0..2, got %d", a.dtype);
  EXL3_REQUIRE(a.param_dtype == a.dtype || a.param_dtype == EXL3_F32,
               "param_dtype must be dtype or fp32, got %d", a.param_dtype);
  EXL3_REQUIRE(a.gate_activation >= 0 && a.gate_activation <= 2,
               "gate_activation must be 0 (none), 1 (sigmoid) or 2 (silu), got %d",
               a.gate_activation);
  EXL3_REQUIRE(a.rows >= 0 && a.d >= 1 && a.d < (1ll << 31), "rows must be >= 0 and d positive");
  EXL3_REQUIRE(!a.gate || a.gate_activation != 0, "a gate needs an activation");
  if (a.rows == 0) return EXL3_OK;
  EXL3_REQUIRE(a.x, "NULL pointer argument");
  EXL3_REQUIRE(!a.next_weight == !a.normed, "normed and next_weight go together");
  EXL3_REQUIRE(a.hidden || a.normed, "no output");
  cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == EXL3_F32) return launch_t<float, float>(a, s);
  if (a.dtype == EXL3_F16)
    return a.param_dtype == EXL3_F32 ? launch_t<__half, float>(a, s) : launch_t<__half, __half>(a, s);
  return a.param_dtype == EXL3_F32 ? launch_t<__nv_bfloat16, float>(a, s)
                                   : launch_t<__nv_bfloat16, __nv_bfloat16>(a, s);
}
