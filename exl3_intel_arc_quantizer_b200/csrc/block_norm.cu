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
// 128 vectors belong to part of a warp or a warp (sums by shuffles), longer
// ones to a CTA (one barrier per sum). CTAs walk over the rows and load the
// next row's vectors before they work on this one's, so that loads are in
// flight across the sums; rows past the registers of a CTA are read again for
// each sum.
#include <algorithm>

#include "common.cuh"
#include "pipeline.cuh"
#include "vec_types.cuh"

namespace exl3 {

__device__ unsigned int g_norm_faults = 0;

namespace {

constexpr int kMaxThreads = 512;  // of a CTA that owns a row

__device__ __forceinline__ float act_sigmoid(float z) {
  float r;  // 2^-22; exp(-z) = inf gives 0
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-z)));
  return r;
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

// What a thread holds of a row as it was loaded.
template <typename T, int V, int NV, bool GATE>
struct Held {
  typename Pieces<T, V>::type x[NV], r[NV], g[GATE ? NV : 1];
};

// SHIFT: rows do not start on 16 bytes, but every tensor's row is as far past
// a boundary as the others': vector c of a row is the aligned one that holds
// its elements c V - off .. c V - off + V - 1, the first and the last of them
// moved element by element.
template <typename T, typename P, int V, int NV, bool CTA_ROW, bool GATE, bool SHIFT>
__global__ void __launch_bounds__(CTA_ROW ? kMaxThreads : 128)
block_norm_kernel(const __grid_constant__ exl3_block_norm_args a, int lanes) {
  __shared__ float red[2][32];
  int slot = 0;
  const int per_cta = CTA_ROW ? 1 : blockDim.x / lanes;
  const int lane = CTA_ROW ? threadIdx.x : threadIdx.x & (lanes - 1);
  const int width = CTA_ROW ? blockDim.x : lanes;
  const int sub = CTA_ROW ? 0 : threadIdx.x / lanes;
  const int d = (int)a.d;
  const float inv_d = 1.0f / (float)d;
  using Vt = typename Pieces<T, V>::type;
  const T* const x = static_cast<const T*>(a.x);
  const T* const gate = static_cast<const T*>(a.gate);
  const T* const residual = static_cast<const T*>(a.residual);
  const P* const weight = static_cast<const P*>(a.weight);
  const P* const next_weight = static_cast<const P*>(a.next_weight);
  const P* const scale = static_cast<const P*>(a.scale);
  T* const hidden = static_cast<T*>(a.hidden);
  T* const normed = static_cast<T*>(a.normed);

  const auto offset = [&](int64_t row) {
    return SHIFT ? (int)(reinterpret_cast<uintptr_t>(x + row * a.x_stride) / sizeof(T) % V) : 0;
  };
  // vector c of a row that starts at p: elements e0 .. e0 + V - 1
  const auto load = [&](const T* p, int e0) {
    if constexpr (SHIFT)
      if (e0 < 0 || e0 + V > d) {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = e0 + e >= 0 && e0 + e < d ? to_f32(p[e0 + e]) : 0.f;
        return pack<T, V>(f);  // the elements' own values again
      }
    return load_piece<T, V>(p + e0);
  };
  const auto store = [&](T* p, int e0, const float (&f)[V]) {
    if (!SHIFT || (e0 >= 0 && e0 + V <= d)) {
      store_piece<T, V>(p + e0, f);
      return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e0 + e >= 0 && e0 + e < d) p[e0 + e] = from_f32<T>(f[e]);
  };
  const auto param = [&](const P* p, int e0, float (&w)[V]) {
    if constexpr (SHIFT) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int at = e0 + e < 0 ? 0 : e0 + e < d ? e0 + e : d - 1;
        w[e] = to_f32(p[at]);
      }
    } else {
      unpack(load_piece<P, V>(p + e0), w);
    }
  };
  const auto fetch = [&](int64_t row, Held<T, V, NV, GATE>& raw) {
    const int off = offset(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (lane + i * width) * V - off;
      raw.x[i] = {};
      raw.r[i] = {};
      if (GATE) raw.g[i] = {};
      if (row < a.rows && e0 < d) {
        raw.x[i] = load(x + row * a.x_stride, e0);
        if (GATE) raw.g[i] = load(gate + row * a.gate_stride, e0);
        if (residual) raw.r[i] = load(residual + row * a.residual_stride, e0);
      }
    }
  };

  const int64_t step = (int64_t)gridDim.x * per_cta;
  Held<T, V, NV, GATE> ahead;
  fetch((int64_t)blockIdx.x * per_cta + sub, ahead);
  for (int64_t r0 = (int64_t)blockIdx.x * per_cta; r0 < a.rows; r0 += step) {
    // every thread of the warp takes part in the sums; rows past the end
    // compute on zeros and store nothing
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    const int off = offset(row);
    const Held<T, V, NV, GATE> raw = ahead;
    if (r0 + step < a.rows) fetch(row + step, ahead);
    float y[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack(raw.x[i], y[i]);
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
        const int e0 = (lane + i * width) * V - off;
        if (e0 >= d) break;
        float w[V];
        param(weight, e0, w);
#pragma unroll
        for (int e = 0; e < V; ++e) y[i][e] = y[i][e] * r * (a.weight_offset + w[e]);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (lane + i * width) * V - off;
      if (e0 >= d) break;
      float g[V], res[V], w[V];
      if (GATE) unpack(raw.g[i], g);
      unpack(raw.r[i], res);
      if (scale) param(scale, e0, w);
      float h[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[e] = y[i][e];
        if (GATE) h[e] = gated(h[e], g[e], a.gate_activation);
        if (residual) h[e] = fmaf(scale ? a.residual_scale * w[e] : a.residual_scale, h[e], res[e]);
        // elements outside the row were loaded as zeros, but a zero gate's or
        // sum's exact zero is not relied on
        y[i][e] = SHIFT && (e0 + e < 0 || e0 + e >= d) ? 0.f : h[e];
        ss = fmaf(y[i][e], y[i][e], ss);
      }
      if (hidden && live) store(hidden + row * a.hidden_stride, e0, h);
    }
    if (next_weight) {
      ss = row_sum<CTA_ROW>(ss, lanes, red, slot);
      const float r = rsqrtf(ss * inv_d + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e0 = (lane + i * width) * V - off;
        if (e0 >= d) break;
        float w[V];
        param(next_weight, e0, w);
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = y[i][e] * r * (a.weight_offset + w[e]);
        if (live) store(normed + row * a.normed_stride, e0, w);
      }
    }
  }
}

// Many rows: bulk copies bring tiles of rows into a ring in shared memory, far
// enough ahead to keep HBM busy (64 to 100 KB in flight per CTA, two CTAs per
// SM; with loads into registers the kernel above holds a third of that), and
// eight warps work on them, `lanes` threads or `warps` warps to a row.
constexpr int kRingWarps = 8;
constexpr int kRingThreads = 32 * (kRingWarps + 1);

struct RingPlan {
  int64_t tiles;
  int rows;            // of a tile
  int lanes;           // threads of a row, up to 32
  int warps;           // of a row
  int stages;
  int slot_bytes;      // of one tensor's rows in a stage
  int contiguous;      // rows follow one another without gaps in every tensor read
  int weight_pitch;    // SHIFT: floats per residue class of the weights in shared memory
};

template <typename T, typename P, int V, int NV, bool GATE, bool SHIFT>
__global__ void __launch_bounds__(kRingThreads, 2)
block_norm_ring_kernel(const __grid_constant__ exl3_block_norm_args a,
                       const __grid_constant__ RingPlan plan) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t bars[2 * 16 + 2 * kRingWarps];
  __shared__ float red[kRingWarps][2][kRingWarps];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int d = (int)a.d;
  using Vt = Raw<T, V>;
  const int tensors = 1 + (GATE ? 1 : 0) + (a.residual ? 1 : 0);
  const auto full = [&](int s) { return smem_u32(&bars[s]); };
  const auto empty = [&](int s) { return smem_u32(&bars[16 + s]); };
  const auto slot = [&](int s, int t) { return ring + (size_t)(s * tensors + t) * plan.slot_bytes; };
  // SHIFT: the weights as floats, element e at (e % V) pitch + e / V, so that
  // neighbouring threads' elements are neighbours whatever the row's offset
  float* const wts = reinterpret_cast<float*>(ring + (size_t)plan.stages * tensors * plan.slot_bytes);
  const P* const params[3] = {static_cast<const P*>(a.weight), static_cast<const P*>(a.next_weight),
                              static_cast<const P*>(a.scale)};
  if (tid == 0) {
    for (int s = 0; s < plan.stages; ++s) {
      bar_init(full(s), 1);
      bar_init(empty(s), kRingWarps);
    }
    for (int i = 0; i < 2 * kRingWarps; ++i) bar_init(smem_u32(&bars[32 + i]), plan.warps);
    abort_word = 0;
    bar_init_fence();
  }
  if (SHIFT)
    for (int k = 0; k < 3; ++k)
      if (params[k])
        for (int e = tid; e < d; e += kRingThreads)
          wts[(k * V + e % V) * plan.weight_pitch + e / V] = to_f32(params[k][e]);
  __syncthreads();

  if (warp == kRingWarps) {
    // ---------------- copies ----------------
    const T* src[3] = {static_cast<const T*>(a.x), nullptr, nullptr};
    int64_t stride[3] = {a.x_stride, 0, 0};
    int k = 1;
    if (GATE) {
      src[k] = static_cast<const T*>(a.gate);
      stride[k++] = a.gate_stride;
    }
    if (a.residual) {
      src[k] = static_cast<const T*>(a.residual);
      stride[k] = a.residual_stride;
    }
    int issued = 0;
    for (int64_t tile = blockIdx.x; tile < plan.tiles; tile += gridDim.x, ++issued) {
      const int s = issued % plan.stages, round = issued / plan.stages;
      bool ok = true;
      if (round > 0) ok = bar_wait(empty(s), (round - 1) & 1, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      const int64_t r0 = tile * plan.rows;
      const int rows = (int)(a.rows - r0 < plan.rows ? a.rows - r0 : plan.rows);
      if (SHIFT) {
        // one run of bytes per tensor, from the 16-byte boundary before it to
        // the one after it where those are inside the tensor; the last few
        // bytes at the tensor's own ends are copied by hand
        uint32_t bytes[3], skip[3], total = 0;
        for (int t = 0; t < tensors; ++t) {
          const uintptr_t base = reinterpret_cast<uintptr_t>(src[t]);
          const uintptr_t begin = base + r0 * d * sizeof(T), end = begin + (uintptr_t)rows * d * sizeof(T);
          const uintptr_t last = base + a.rows * d * sizeof(T), origin = begin & ~(uintptr_t)15;
          uintptr_t lo = origin, hi = (end + 15) & ~(uintptr_t)15;
          if (lo < base) lo += 16;
          if (hi > last) hi -= 16;
          skip[t] = (uint32_t)(lo - origin);
          bytes[t] = hi > lo ? (uint32_t)(hi - lo) : 0;
          total += bytes[t];
          T* dst = reinterpret_cast<T*>(slot(s, t));
          for (uintptr_t p = begin + lane * sizeof(T); p < end; p += 32 * sizeof(T)) {
            if (p >= lo && p < hi) {
              // on to the bytes behind the run
              if (hi >= end) break;
              p = hi + lane * sizeof(T);
              if (p >= end) break;
            }
            dst[(p - origin) / sizeof(T)] = *reinterpret_cast<const T*>(p);
          }
        }
        __syncwarp();
        if (lane == 0) {
          bar_expect(full(s), total);
          for (int t = 0; t < tensors; ++t) {
            const uintptr_t origin =
                (reinterpret_cast<uintptr_t>(src[t]) + r0 * d * sizeof(T)) & ~(uintptr_t)15;
            if (bytes[t])
              bulk_load(slot(s, t) + skip[t], reinterpret_cast<const void*>(origin + skip[t]), bytes[t],
                        full(s));
          }
        }
      } else {
        const uint32_t row_bytes = (uint32_t)(d * sizeof(T));
        if (lane == 0) bar_expect(full(s), row_bytes * rows * tensors);
        __syncwarp();
        if (plan.contiguous) {
          if (lane < tensors)
            bulk_load(slot(s, lane), src[lane] + r0 * d, row_bytes * rows, full(s));
        } else {
          for (int i = lane; i < rows * tensors; i += 32) {
            const int t = i / rows, r = i - t * rows;
            bulk_load(slot(s, t) + (size_t)r * row_bytes, src[t] + (r0 + r) * stride[t], row_bytes, full(s));
          }
        }
      }
      __syncwarp();
    }
    // copies in flight land before the CTA ends
    for (int i = issued > plan.stages ? issued - plan.stages : 0; i < issued; ++i)
      bar_drain(full(i % plan.stages), (i / plan.stages) & 1);
  } else {
    // ---------------- rows ----------------
    const int group = warp / plan.warps, per_warp = 32 / plan.lanes;
    const int width = plan.warps > 1 ? 32 * plan.warps : plan.lanes;
    const int at = plan.warps > 1 ? tid - group * 32 * plan.warps : lane & (plan.lanes - 1);
    const int sub = plan.warps > 1 ? 0 : lane / plan.lanes;
    const int step = plan.warps > 1 ? kRingWarps / plan.warps : kRingWarps * per_warp;
    const int first = plan.warps > 1 ? group : warp * per_warp;
    const float inv_d = 1.0f / (float)d;
    int sums = 0;
    const auto sum = [&](float v) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < plan.lanes) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
      if (plan.warps > 1) {
        // two sides in turn: one is written again only after all have passed
        // the other's barrier
        const int side = sums & 1;
        const uint32_t bar = smem_u32(&bars[32 + 2 * group + side]);
        if (lane == 0) {
          red[group][side][warp - group * plan.warps] = v;
          bar_arrive(bar);
        }
        bar_wait(bar, (sums >> 1) & 1, abort_flag);
        v = 0.f;
        for (int w = 0; w < plan.warps; ++w) v += red[group][side][w];
        ++sums;
      }
      return v;
    };
    // parameter k of elements e0 .. e0 + V - 1
    const auto param = [&](int k, int e0, float (&w)[V]) {
      if constexpr (SHIFT) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int i = e0 + e < 0 ? 0 : e0 + e < d ? e0 + e : d - 1;
          w[e] = wts[(k * V + i % V) * plan.weight_pitch + i / V];
        }
      } else {
        unpack(load_raw<P, V>(params[k] + e0), w);
      }
    };
    int it = 0;
    for (int64_t tile = blockIdx.x; tile < plan.tiles; tile += gridDim.x, ++it) {
      const int s = it % plan.stages;
      const bool ok = bar_wait(full(s), (it / plan.stages) & 1, abort_flag);
      // a CTA whose copies do not come ends without results: every warp finds
      // the same barrier incomplete
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      const int64_t r0 = tile * plan.rows;
      const int rows = (int)(a.rows - r0 < plan.rows ? a.rows - r0 : plan.rows);
      for (int base = first; base < rows; base += step) {
        const int rr = base + sub;
        const bool live = rr < rows;
        const int64_t row = r0 + rr;
        // byte of the row in its slot, and its elements past a boundary
        int begin = rr * d * (int)sizeof(T);
        if (SHIFT) begin += (int)((reinterpret_cast<uintptr_t>(a.x) + r0 * d * sizeof(T)) & 15);
        const int off = SHIFT ? (begin & 15) / (int)sizeof(T) : 0;
        const auto load = [&](int t, int e0) {
          Vt v = {};
          if (live && e0 < d)
            v = load_raw<T, V>(reinterpret_cast<const T*>(slot(s, t) + begin + e0 * (int)sizeof(T)));
          return v;
        };
        float y[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e0 = (at + i * width) * V - off;
          unpack(load(0, e0), y[i]);
          if (SHIFT)
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (e0 + e < 0 || e0 + e >= d) y[i][e] = 0.f;
        }
        if (params[0]) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(y[i][e], y[i][e], ss);
          const float r = rsqrtf(sum(ss) * inv_d + a.eps);
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int e0 = (at + i * width) * V - off;
            if (e0 >= d) break;
            float w[V];
            param(0, e0, w);
#pragma unroll
            for (int e = 0; e < V; ++e) y[i][e] = y[i][e] * r * (a.weight_offset + w[e]);
          }
        }
        const auto store = [&](T* p, int e0, const float (&f)[V]) {
          if (!SHIFT || (e0 >= 0 && e0 + V <= d)) {
            store_raw<T, V>(p + e0, pack<T, V>(f));
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (e0 + e >= 0 && e0 + e < d) p[e0 + e] = from_f32<T>(f[e]);
          }
        };
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e0 = (at + i * width) * V - off;
          if (e0 >= d) break;
          float g[V], res[V], w[V];
          if (GATE) {
            unpack(load(1, e0), g);
#pragma unroll
            for (int e = 0; e < V; ++e) y[i][e] = gated(y[i][e], g[e], a.gate_activation);
          }
          if (a.residual) {
            unpack(load(GATE ? 2 : 1, e0), res);
            if (params[2]) {
              param(2, e0, w);
#pragma unroll
              for (int e = 0; e < V; ++e) y[i][e] = fmaf(a.residual_scale * w[e], y[i][e], res[e]);
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) y[i][e] = fmaf(a.residual_scale, y[i][e], res[e]);
            }
          }
          if (SHIFT)
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (e0 + e < 0 || e0 + e >= d) y[i][e] = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) ss = fmaf(y[i][e], y[i][e], ss);
        }
        // the slot is read: its next tile may come
        if (base + step >= rows) {
          __syncwarp();
          if (lane == 0) bar_arrive(empty(s));
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e0 = (at + i * width) * V - off;
          if (a.hidden && live && e0 < d) store(static_cast<T*>(a.hidden) + row * a.hidden_stride, e0, y[i]);
        }
        if (params[1]) {
          const float r = rsqrtf(sum(ss) * inv_d + a.eps);
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int e0 = (at + i * width) * V - off;
            if (e0 >= d) break;
            float w[V];
            param(1, e0, w);
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = y[i][e] * r * (a.weight_offset + w[e]);
            if (live) store(static_cast<T*>(a.normed) + row * a.normed_stride, e0, w);
          }
        }
      }
      if (first >= rows && lane == 0) bar_arrive(empty(s));
    }
  }
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicAdd(&g_norm_faults, 1u);
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

template <typename T, typename P, int V, int NV, bool CTA_ROW, bool GATE, bool SHIFT>
int launch(const exl3_block_norm_args& a, int threads, int lanes, cudaStream_t stream) {
  const auto kernel = block_norm_kernel<T, P, V, NV, CTA_ROW, GATE, SHIFT>;
  const int per_cta = CTA_ROW ? 1 : threads / lanes;
  const int64_t ctas = (a.rows + per_cta - 1) / per_cta;
  // as many CTAs as run at once: each has a next row to load
  static std::atomic<int> known[kMaxThreads / 32 + 1];  // by warps of a CTA
  int resident = known[threads / 32].load(std::memory_order_relaxed);
  if (resident == 0) {
    EXL3_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, threads, 0));
    if (resident < 1) resident = 1;
    known[threads / 32].store(resident, std::memory_order_relaxed);
  }
  const int64_t most = (int64_t)sm_count() * resident;
  kernel<<<(unsigned)(ctas < most ? ctas : most), threads, 0, stream>>>(a, lanes);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

// The ring's plan; false where the rows are too few or too long for it.
template <typename T, int V, bool GATE, bool SHIFT>
bool plan_ring(const exl3_block_norm_args& a, RingPlan& p, size_t& smem) {
  constexpr size_t kBudget = 100 * 1024;  // two CTAs per SM
  const int64_t row_bytes = a.d * (int64_t)sizeof(T);
  const int64_t nvec = (a.d + V - 1) / V + (SHIFT ? 1 : 0);
  if (nvec > 4 * 32 * kRingWarps || a.rows < 4 * sm_count()) return false;
  p.contiguous = a.x_stride == a.d && (!a.gate || a.gate_stride == a.d) &&
                 (!a.residual || a.residual_stride == a.d);
  if (SHIFT && !p.contiguous) return false;
  // up to two vectors per thread, then more warps per row
  p.lanes = 32;
  p.warps = 1;
  if (nvec <= 32) {
    while (p.lanes > 1 && p.lanes / 2 >= nvec) p.lanes /= 2;
  } else {
    while (p.warps < kRingWarps && nvec > 64 * p.warps) p.warps *= 2;
  }
  const int per_pass = p.warps > 1 ? kRingWarps / p.warps : kRingWarps * (32 / p.lanes);
  // tiles of about 8 KB per tensor, whole passes of the warps, rows for all
  int64_t rows = std::max<int64_t>(1, 8192 / row_bytes);
  rows = rows < per_pass ? per_pass : rows / per_pass * per_pass;
  rows = std::max<int64_t>(1, std::min<int64_t>(rows, (a.rows + 2 * sm_count() - 1) / (2 * sm_count())));
  const int tensors = 1 + (GATE ? 1 : 0) + (a.residual ? 1 : 0);
  p.rows = (int)rows;
  p.tiles = (a.rows + rows - 1) / rows;
  p.slot_bytes = (int)((rows * row_bytes + 32 + 127) / 128 * 128);
  p.weight_pitch = SHIFT ? (int)((a.d + V - 1) / V) | 1 : 0;
  const size_t weights = SHIFT ? (size_t)3 * V * p.weight_pitch * sizeof(float) : 0;
  if (weights + 2 * (size_t)tensors * p.slot_bytes > kBudget) return false;
  p.stages = (int)std::min<size_t>(16, (kBudget - weights) / ((size_t)tensors * p.slot_bytes));
  smem = (size_t)p.stages * tensors * p.slot_bytes + weights;
  return true;
}

template <typename T, typename P, int V, int NV, bool GATE, bool SHIFT>
int launch_ring(const exl3_block_norm_args& a, const RingPlan& p, size_t smem, cudaStream_t stream) {
  const auto kernel = block_norm_ring_kernel<T, P, V, NV, GATE, SHIFT>;
  static DeviceBits attr_done;
  int dev = 0;
  EXL3_CUDA(cudaGetDevice(&dev));
  if (!attr_done.has(dev)) {
    EXL3_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024));
    attr_done.set(dev);
  }
  const int64_t most = 2 * (int64_t)sm_count();
  kernel<<<(unsigned)std::min(p.tiles, most), kRingThreads, smem, stream>>>(a, p);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

template <typename T, typename P, int V, bool GATE, bool SHIFT>
int launch_v(const exl3_block_norm_args& a, cudaStream_t stream) {
  if constexpr (V > 1) {
    RingPlan p;
    size_t smem;
    if (plan_ring<T, V, GATE, SHIFT>(a, p, smem)) {
      const int64_t width = p.warps > 1 ? 32 * p.warps : p.lanes;
      const int64_t nvec = (a.d + V - 1) / V + (SHIFT ? 1 : 0);
      if (nvec <= width) return launch_ring<T, P, V, 1, GATE, SHIFT>(a, p, smem, stream);
      if (nvec <= 2 * width) return launch_ring<T, P, V, 2, GATE, SHIFT>(a, p, smem, stream);
      return launch_ring<T, P, V, 4, GATE, SHIFT>(a, p, smem, stream);
    }
  }
  // a shifted row may reach into one vector more
  const int64_t nvec = (a.d + V - 1) / V + (SHIFT ? 1 : 0);
  if (nvec <= 128) {
    int lanes = 1;
    while (lanes < nvec && lanes < 32) lanes *= 2;
    if (nvec <= lanes) return launch<T, P, V, 1, false, GATE, SHIFT>(a, 128, lanes, stream);
    if (nvec <= 2 * lanes) return launch<T, P, V, 2, false, GATE, SHIFT>(a, 128, lanes, stream);
    return launch<T, P, V, 4, false, GATE, SHIFT>(a, 128, lanes, stream);
  }
  const auto threads = [&](int nv) { return (int)((nvec + 32 * nv - 1) / (32 * nv)) * 32; };
  // few rows: as many threads as there are vectors; else two vectors each
  if (nvec <= kMaxThreads && a.rows <= sm_count())
    return launch<T, P, V, 1, true, GATE, SHIFT>(a, threads(1), 32, stream);
  if (nvec <= 2 * kMaxThreads) return launch<T, P, V, 2, true, GATE, SHIFT>(a, threads(2), 32, stream);
  if (nvec <= 4 * kMaxThreads) return launch<T, P, V, 4, true, GATE, SHIFT>(a, threads(4), 32, stream);
  const int64_t most = (int64_t)sm_count() * 2;
  block_norm_long_kernel<T, P>
      <<<(unsigned)(a.rows < most ? a.rows : most), 1024, 0, stream>>>(a);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

template <typename T, typename P, int V, bool SHIFT>
int launch_g(const exl3_block_norm_args& a, cudaStream_t stream) {
  return a.gate ? launch_v<T, P, V, true, SHIFT>(a, stream) : launch_v<T, P, V, false, SHIFT>(a, stream);
}

template <typename T, typename P>
int launch_t(const exl3_block_norm_args& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const struct { const void* p; int64_t stride; } rows[] = {
      {a.x, a.x_stride}, {a.gate, a.gate_stride}, {a.residual, a.residual_stride},
      {a.hidden, a.hidden_stride}, {a.normed, a.normed_stride}};
  bool wide = a.d % V == 0, alike = true;
  for (const auto& r : rows) {
    if (!r.p) continue;
    wide = wide && aligned_to(r.p, 16) && r.stride % V == 0;
    alike = alike && reinterpret_cast<uintptr_t>(r.p) % sizeof(T) == 0 &&
            (reinterpret_cast<uintptr_t>(r.p) - reinterpret_cast<uintptr_t>(a.x)) % 16 == 0 &&
            (r.stride - a.x_stride) % V == 0;
  }
  for (const void* p : {a.weight, a.next_weight, a.scale}) wide = wide && (!p || aligned_to(p, V * sizeof(P)));
  // vectors, vectors from each row's boundary on, or element by element
  if (wide) return launch_g<T, P, V, false>(a, stream);
  if (alike && a.d >= 4 * V) return launch_g<T, P, V, true>(a, stream);
  return launch_g<T, P, 1, false>(a, stream);
}

}  // namespace

int norm_fault_count(unsigned int* count) {
  EXL3_CUDA(cudaMemcpyFromSymbol(count, g_norm_faults, sizeof(unsigned int)));
  return EXL3_OK;
}

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
