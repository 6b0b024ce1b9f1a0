// The gated delta rule over whole sequences, in chunks of 64 tokens.
//
// Within a chunk, with G_i = g_0 + .. + g_i and S the state before it,
//   (I + M) U = beta (V - e^G K S),   M_ij = beta_i e^{G_i - G_j} k_i . k_j  (j < i)
//   O = scale (e^G Q S + P U),        P_ij = e^{G_i - G_j} q_i . k_j         (j <= i)
//   S' = e^{G_63} S + K^T (e^{G_63 - G} U)
// so the tokens of a chunk are matrix products, and only S passes from chunk
// to chunk. Two kernels:
//
//  * delta_prep_kernel, parallel over chunks and key heads: K K^T and Q K^T
//    (mma.sync), per value head the inverse of I + M in fp32 (16x16 diagonal
//    blocks by substitution, then twice by halves), T = (I + M)^-1 beta and
//    P T, written as the tensor-core operand the second kernel reads.
//  * delta_chain_kernel, one CTA per sequence, head and slice of columns of
//    the state (columns do not interact): three tcgen05 products per chunk,
//      [K; Q] S            -> K S and Q S
//      [T; P T] R          -> U and P U,     R = V - e^G K S
//      K^T (e^{G_63 - G} U) -> the state's update,
//    the two halves of each stacked to M = 128. S stays in fp32 registers of
//    the epilogue warps.
//
// Precision: the states are fp32, so no product that reaches them may round
// its operands to 11 bits. S, R, U, T and P T are split into two fp16 parts,
// x = hi + lo, 22 bits; the product of two low parts (2^-24 of a term) is left
// out. fp16 q and k are one part as they are, bf16 ones after a scaling of
// each row by a power of two (8 bits fit 11; what lies 2^-14 below a row's
// largest element loses bits of 2^-25 of it). Two bf16 parts (16 bits) for
// the same number of products left the final states off by 3e-6 to 4e-5.
//
// Range: fp16 ends at 65,504, so S, R and U are scaled by powers of two from
// bounds that hold for any input: with smax the largest |S| before the chunk
// (exact, from the registers) and vmax that of its v,
//   |R| <= BR = vmax + A smax,      A = sqrt(dk) max_i a_i |k_i|
//   |c U| <= max_j c_j t BR,        t = the largest row sum of |T|
//   |S'| <= e^{G_63} smax + t (sum_j c_j |k_j|) BR
// A bound is put at 2^14 to 2^15. It may lie far above the values: at 2^-12
// of it two parts still resolve 2^-28 of it.
//
// Decays are e^{G_i - G_j} <= 1 from prefix sums in fp64, so that a token
// with e^g = 0 (g = -inf, taken as -200: e^-200 is 0 in fp32) leaves the
// differences behind it exact.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "delta_rule.cuh"

namespace exl3 {

__device__ unsigned int g_delta_faults = 0;

namespace {

constexpr int kChunk = 64;
constexpr int kImageBytes = 128 * 128 * 2;  // [T; P T]: 128 rows x 64, high and low parts
// per chunk and head: a (64), b (64), c (64), the scalars, and the factors of
// the 64 k and 64 q rows on their way to fp16
constexpr int kVecFloats = 384;
constexpr int kGamma = 192, kBoundA = 193, kBoundU = 194, kBoundS = 195, kScaleT = 196,
              kScalePT = 197, kRowScale = 256;
constexpr int64_t kSlotBytes = kImageBytes + kVecFloats * 4;

// Chunk c of a sequence that begins at token t0 has workspace slot
// t0 / 64 + s + c: sequences never share one, and there are tokens / 64 +
// seqs of them, whatever the lengths.
__device__ __forceinline__ int64_t slot_base(int64_t t0, int64_t s) { return t0 / kChunk + s; }

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Byte of 16-byte piece q of row r in a 128-byte-swizzled operand tile
// (rows of 128 bytes, groups of 8 rows; the tile starts on 1,024 bytes).
__device__ __forceinline__ uint32_t swz(int r, int q) {
  return (uint32_t)(r * 128 + ((q ^ (r & 7)) << 4));
}

// x = hi + lo, two fp16 parts each
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void split8(const float* x, uint4& hi, uint4& lo) {
  split2(x[0], x[1], hi.x, lo.x);
  split2(x[2], x[3], hi.y, lo.y);
  split2(x[4], x[5], hi.z, lo.z);
  split2(x[6], x[7], hi.w, lo.w);
}

// The power of two that puts a bound (>= 0) into [2^14, 2^15), and its
// inverse. Bounds below 2^-97 are taken as that; infinities and NaN keep the
// factor finite (the values stay what they are).
__device__ __forceinline__ void pow2_scale(float bound, float& scale, float& inverse) {
  uint32_t e = (__float_as_uint(bound) >> 23) & 255u;
  e = e < 30u ? 30u : e;
  scale = __uint_as_float((268u - e) << 23);    // 2^(141 - e)
  inverse = __uint_as_float((e - 14u) << 23);   // 2^(e - 141)
}

// 8 elements of type T from p as 16 bytes; zero where n is 0
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  Vec<T, 8> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.e[i] = p[i];
  return *reinterpret_cast<const uint4*>(&v);
}

// ---------------------------------------------------------------------------
// Chunk preparation
// ---------------------------------------------------------------------------

constexpr int kPrepThreads = 256;
constexpr int kLdk = 136;  // elements per row of the staged q and k (17 x 16 bytes)
constexpr int kLds = 68;   // floats per row of the 64 x 64 matrices
constexpr int kLdd = 65;

struct PrepSmem {
  union {
    uint16_t kq[2][kChunk][kLdk];
    struct {
      float M[kChunk][kLds];
      float X[kChunk][kLds];
    } m;
  } u;
  float dot[2][kChunk][kLdd];  // k_i . k_j and q_i . k_j, j <= i
  float P[kChunk][kLds];
  float tmp[32][36];
  double G[kChunk];
  float beta[kChunk], rk[kChunk], rq[kChunk];
  float rowscale[2 * kChunk];   // power of two that brings a k or q row into fp16
  uint32_t peak[3];             // bits of max |T|, max |P T|, largest row sum of |T|
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T>
__global__ void __launch_bounds__(kPrepThreads)
delta_prep_kernel(const __grid_constant__ exl3_delta_args a, uint8_t* __restrict__ ws, int vec) {
  extern __shared__ __align__(16) uint8_t dsm[];
  PrepSmem& sm = *reinterpret_cast<PrepSmem*>(dsm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t slot = blockIdx.x;
  const int kh = blockIdx.y;

  // the last sequence whose first slot is not past this one
  int64_t s = 0;
  for (int64_t hi = a.seqs; hi - s > 1;) {
    const int64_t mid = (s + hi) / 2;
    int64_t b0, b1;
    seq_bounds(a, mid, b0, b1);
    if (slot_base(b0, mid) <= slot) s = mid; else hi = mid;
  }
  int64_t t0, t1;
  seq_bounds(a, s, t0, t1);
  t0 += (slot - slot_base(t0, s)) * kChunk;
  if (t0 >= t1) return;
  const int n = (int)(t1 - t0 < kChunk ? t1 - t0 : kChunk);

  // q and k of the chunk, zeros past its end and up to a multiple of 16
  const int pieces = a.dk / 8, padded = (a.dk + 15) / 16 * 2;
  for (int i = tid; i < 2 * kChunk * padded; i += kPrepThreads) {
    const int r = i / padded, q = i - r * padded, row = r & (kChunk - 1), isq = r >> 6;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < n && q < pieces) {
      const int64_t* st = isq ? a.q_strides : a.k_strides;
      v = load8(static_cast<const T*>(isq ? a.q : a.k) + (t0 + row) * st[0] + kh * st[1] + 8 * q, vec);
    }
    *reinterpret_cast<uint4*>(&sm.u.kq[isq][row][8 * q]) = v;
  }
  __syncthreads();

  // warps 0-3: rows 16 w of K K^T; warps 4-7: of Q K^T; columns up to the
  // diagonal tile
  {
    const int mt = warp & 3, which = warp >> 2;
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    for (int k0 = 0; k0 < a.dk; k0 += 16) {
      uint32_t fa[4];
      ldsm4(fa, smem_u32(&sm.u.kq[which][16 * mt + (lane & 15)][k0 + 8 * (lane >> 4)]));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > mt) break;
        uint32_t fb[4];  // columns 16 j .. 16 j + 15: two n-tiles, two k halves
        ldsm4(fb, smem_u32(&sm.u.kq[0][16 * j + (lane & 7) + 8 * (lane >> 4)]
                                   [k0 + 8 * ((lane >> 3) & 1)]));
        mma16816<T>(acc[2 * j], fa, fb[0], fb[1]);
        mma16816<T>(acc[2 * j + 1], fa, fb[2], fb[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j > 2 * mt + 1) break;
      const int r = 16 * mt + (lane >> 2), c = 8 * j + 2 * (lane & 3);
      sm.dot[which][r][c] = acc[j][0];
      sm.dot[which][r][c + 1] = acc[j][1];
      sm.dot[which][r + 8][c] = acc[j][2];
      sm.dot[which][r + 8][c + 1] = acc[j][3];
    }
    // |q|^2, and the largest |k| and |q|: four threads per row
    const int row = tid >> 2;
    float ss = 0.f, big[2] = {0.f, 0.f};
    for (int c = tid & 3; c < a.dk; c += 4) {
      const uint16_t bk = sm.u.kq[0][row][c], bq = sm.u.kq[1][row][c];
      const float v = to_f32(*reinterpret_cast<const T*>(&bq));
      ss = fmaf(v, v, ss);
      big[0] = fmaxf(big[0], fabsf(to_f32(*reinterpret_cast<const T*>(&bk))));
      big[1] = fmaxf(big[1], fabsf(v));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      big[0] = fmaxf(big[0], __shfl_xor_sync(0xFFFFFFFFu, big[0], o));
      big[1] = fmaxf(big[1], __shfl_xor_sync(0xFFFFFFFFu, big[1], o));
    }
    if ((tid & 3) == 0) {
      sm.rq[row] = a.normalize_qk ? rsqrtf(ss + kNormEps) : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // the row's largest element goes to [1, 2); fp16 rows stay
        uint32_t e = (__float_as_uint(big[i]) >> 23) & 255u;
        e = e < 2u ? 2u : e > 252u ? 252u : e;
        sm.rowscale[64 * i + row] =
            std::is_same<T, __half>::value || big[i] == 0.f ? 1.f : __uint_as_float((254u - e) << 23);
      }
    }
  }
  __syncthreads();
  if (tid < kChunk) sm.rk[tid] = a.normalize_qk ? rsqrtf(sm.dot[0][tid][tid] + kNormEps) : 1.f;
  float knorm[2] = {0.f, 0.f};  // |k| of rows 2 lane and 2 lane + 1
  if (warp == 0) {
    knorm[0] = sqrtf(sm.dot[0][2 * lane][2 * lane]);
    knorm[1] = sqrtf(sm.dot[0][2 * lane + 1][2 * lane + 1]);
  }

  const int rep = a.heads / a.key_heads;
  for (int h = kh * rep; h < (kh + 1) * rep; ++h) {
    __syncthreads();  // rk, and the last head's matrices read
    if (tid < 3) sm.peak[tid] = 0;
    if (warp == 0) {
      double g[2], run;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        float v = r < n ? a.g[(t0 + r) * a.g_stride + h] : 0.f;
        v = v < -200.f ? -200.f : v;
        g[i] = (double)v;
        sm.beta[r] = r < n ? a.beta[(t0 + r) * a.beta_stride + h] : 0.f;
      }
      run = g[0] + g[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += up;
      }
      sm.G[2 * lane] = run - g[1];
      sm.G[2 * lane + 1] = run;
    }
    __syncthreads();
    float(&M)[kChunk][kLds] = sm.u.m.M;
    float(&X)[kChunk][kLds] = sm.u.m.X;
    for (int i = tid; i < kChunk * kChunk; i += kPrepThreads) {
      const int r = i >> 6, c = i & 63;
      float m = 0.f, p = 0.f;
      if (c <= r) {
        const float d = expf((float)(sm.G[r] - sm.G[c])) * sm.rk[c];
        p = a.scale * sm.rq[r] * d * sm.dot[1][r][c];
        if (c < r) m = sm.beta[r] * sm.rk[r] * d * sm.dot[0][r][c];
      }
      M[r][c] = m;
      sm.P[r][c] = p;
      X[r][c] = 0.f;
    }
    __syncthreads();
    // (I + M)^-1: the 16x16 diagonal blocks, a thread per column
    if (tid < 64) {
      const int b = tid & ~15, c = tid & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) v = fmaf(-M[b + i][b + j], x[j], v);
        x[i] = v;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) X[b + i][b + c] = x[i];
    }
    __syncthreads();
    // halves of 32: X21 = -X22 (M21 X11), two pairs of blocks at once
    {
      const int p = tid >> 7, r = (tid >> 3) & 15, c = 2 * (tid & 7), b = 32 * p;
      float v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float m = M[b + 16 + r][b + k];
        v0 = fmaf(m, X[b + k][b + c], v0);
        v1 = fmaf(m, X[b + k][b + c + 1], v1);
      }
      sm.tmp[16 * p + r][c] = v0;
      sm.tmp[16 * p + r][c + 1] = v1;
      __syncthreads();
      v0 = v1 = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float m = X[b + 16 + r][b + 16 + k];
        v0 = fmaf(m, sm.tmp[16 * p + k][c], v0);
        v1 = fmaf(m, sm.tmp[16 * p + k][c + 1], v1);
      }
      X[b + 16 + r][b + c] = -v0;
      X[b + 16 + r][b + c + 1] = -v1;
    }
    __syncthreads();
    // the whole: the same with blocks of 32
    {
      const int r = tid >> 3, c = 4 * (tid & 7);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float m = M[32 + r][k];
        const float4 x = *reinterpret_cast<const float4*>(&X[k][c]);
        v[0] = fmaf(m, x.x, v[0]);
        v[1] = fmaf(m, x.y, v[1]);
        v[2] = fmaf(m, x.z, v[2]);
        v[3] = fmaf(m, x.w, v[3]);
      }
      *reinterpret_cast<float4*>(&sm.tmp[r][c]) = make_float4(v[0], v[1], v[2], v[3]);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float m = X[32 + r][32 + k];
        const float4 x = *reinterpret_cast<const float4*>(&sm.tmp[k][c]);
        v[0] = fmaf(m, x.x, v[0]);
        v[1] = fmaf(m, x.y, v[1]);
        v[2] = fmaf(m, x.z, v[2]);
        v[3] = fmaf(m, x.w, v[3]);
      }
      *reinterpret_cast<float4*>(&X[32 + r][c]) = make_float4(-v[0], -v[1], -v[2], -v[3]);
    }
    __syncthreads();
    // T = X beta into M's place, P T into tmp-free registers: a 4x4 tile each
    uint8_t* img = ws + (slot * a.heads + h) * kSlotBytes;
    {
      const int r = 4 * (tid >> 4), c = 4 * (tid & 15);
      float v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = 0.f;
      if (c <= r) {
        for (int k = c; k < r + 4; k += 4) {  // P is zero past the diagonal, X before it
          float p[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 t = *reinterpret_cast<const float4*>(&sm.P[r + i][k]);
            p[i][0] = t.x;
            p[i][1] = t.y;
            p[i][2] = t.z;
            p[i][3] = t.w;
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const float4 x = *reinterpret_cast<const float4*>(&X[k + kk][c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i][0] = fmaf(p[i][kk], x.x, v[i][0]);
              v[i][1] = fmaf(p[i][kk], x.y, v[i][1]);
              v[i][2] = fmaf(p[i][kk], x.z, v[i][2]);
              v[i][3] = fmaf(p[i][kk], x.w, v[i][3]);
            }
          }
        }
      }
      const float4 bt = *reinterpret_cast<const float4*>(&sm.beta[c]);
      float x[4][4];
      float most = 0.f, most_p = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 t = *reinterpret_cast<const float4*>(&X[r + i][c]);
        x[i][0] = t.x * bt.x;
        x[i][1] = t.y * bt.y;
        x[i][2] = t.z * bt.z;
        x[i][3] = t.w * bt.w;
        v[i][0] *= bt.x;
        v[i][1] *= bt.y;
        v[i][2] *= bt.z;
        v[i][3] *= bt.w;
        float row = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          row += fabsf(x[i][e]);
          most = fmaxf(most, fabsf(x[i][e]));
          most_p = fmaxf(most_p, fabsf(v[i][e]));
        }
        // the row's 16 threads are neighbours
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) row += __shfl_xor_sync(0xFFFFFFFFu, row, o);
        sum = fmaxf(sum, row);
      }
      // the order of these maxima (of bits of non-negative floats) does not matter
      const uint32_t m0 = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most));
      const uint32_t m1 = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most_p));
      const uint32_t m2 = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(sum));
      if (lane == 0) {
        atomicMax(&sm.peak[0], m0);
        atomicMax(&sm.peak[1], m1);
        atomicMax(&sm.peak[2], m2);
      }
      __syncthreads();
      float st, sp, inv;
      pow2_scale(__uint_as_float(sm.peak[0]), st, inv);
      pow2_scale(__uint_as_float(sm.peak[1]), sp, inv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 hi, lo;
        split2(x[i][0] * st, x[i][1] * st, hi.x, lo.x);
        split2(x[i][2] * st, x[i][3] * st, hi.y, lo.y);
        const uint32_t at = swz(r + i, c >> 3) + 2 * (c & 7);
        *reinterpret_cast<uint2*>(img + at) = hi;
        *reinterpret_cast<uint2*>(img + kImageBytes / 2 + at) = lo;
        split2(v[i][0] * sp, v[i][1] * sp, hi.x, lo.x);
        split2(v[i][2] * sp, v[i][3] * sp, hi.y, lo.y);
        const uint32_t at2 = swz(64 + r + i, c >> 3) + 2 * (c & 7);
        *reinterpret_cast<uint2*>(img + at2) = hi;
        *reinterpret_cast<uint2*>(img + kImageBytes / 2 + at2) = lo;
      }
    }
    float* vout = reinterpret_cast<float*>(img + kImageBytes);
    if (tid >= 64 && tid < 192) vout[kRowScale + tid - 64] = sm.rowscale[tid - 64];
    if (warp == 0) {
      float ba = 0.f, bu = 0.f, bs = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float up = 1.f / sm.rowscale[r], eg = expf((float)sm.G[r]);
        const float c = sm.rk[r] * expf((float)(sm.G[63] - sm.G[r]));
        vout[r] = eg * sm.rk[r] * up;
        vout[64 + r] = a.scale * sm.rq[r] * eg / sm.rowscale[64 + r];
        vout[128 + r] = c * up;
        ba = fmaxf(ba, eg * sm.rk[r] * knorm[i]);
        bu = fmaxf(bu, c * up);
        bs += c * knorm[i];
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        ba = fmaxf(ba, __shfl_xor_sync(0xFFFFFFFFu, ba, o));
        bu = fmaxf(bu, __shfl_xor_sync(0xFFFFFFFFu, bu, o));
        bs += __shfl_xor_sync(0xFFFFFFFFu, bs, o);
      }
      if (lane == 0) {
        const float t = __uint_as_float(sm.peak[2]);
        float scale, inv;
        vout[kGamma] = expf((float)sm.G[63]);
        vout[kBoundA] = ba * sqrtf((float)a.dk);
        vout[kBoundU] = bu * t;
        vout[kBoundS] = bs * t;
        pow2_scale(__uint_as_float(sm.peak[0]), scale, inv);
        vout[kScaleT] = inv;
        pow2_scale(__uint_as_float(sm.peak[1]), scale, inv);
        vout[kScalePT] = inv;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The chain of states
// ---------------------------------------------------------------------------

constexpr uint64_t kWaitNs = 2000000000ull;  // 2 s per wait

// GROUPS column groups of NV columns, each with its own barriers, tensor
// memory and issuing thread (one group's products run under the other's
// elementwise steps); CT columns per epilogue thread. NV = 32 keeps the high
// and low parts of an operand side by side as 64 columns (their products
// land in separate columns and are added in the epilogue); NV = 64 keeps two
// operands, whose products accumulate.
template <typename T, int GROUPS, int NV, int CT>
struct Geo {
  static constexpr bool kPacked = NV == 32;
  static constexpr int kWG = NV / CT;                    // epilogue warpgroups of a group
  static constexpr int kEpiWarps = 4 * kWG * GROUPS;
  static constexpr int kProducers = GROUPS == 2 ? 2 : 4;  // warps
  static constexpr int kThreads = 32 * (kEpiWarps + GROUPS + kProducers);
  static constexpr int kBox = 128 * 128;                 // [K; Q]: 128 rows x 64 of dk
  static constexpr int kKQ = 2 * kBox;
  static constexpr int kKQStages = 2;
  static constexpr int kTStages = 2;
  static constexpr int kPartsB = kPacked ? 1 : 2;        // operand tiles of S, R, U
  static constexpr int kSBytes = 128 * 128 * kPartsB;
  static constexpr int kRBytes = 64 * 128 * kPartsB;
  static constexpr int kCols = 3 * 64;                   // tensor memory of a group
  static constexpr int kAlloc = GROUPS == 2 ? 512 : 256;
  static constexpr int kBars = 2 * kKQStages + 2 * kTStages + 7 * GROUPS;
  static constexpr size_t kSmem = 1024 + (size_t)kKQStages * kKQ + kTStages * kImageBytes +
                                  GROUPS * (kSBytes + kRBytes) + kBars * 8 + 16 + 32;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ uint64_t gtimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// true when the phase completed; false on timeout (which raises the abort
// flag) or when another role has aborted
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (bar_try(bar, parity)) return true;
  const uint64_t start = gtimer();
  for (uint32_t it = 0;; ++it) {
    if (bar_try(bar, parity)) return true;
    if ((it & 31u) == 31u) {
      if (*abort_flag) return false;
      if (gtimer() - start > kWaitNs) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
// the shutdown path's wait: bounded, whatever the abort flag says
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  const uint64_t start = gtimer();
  while (!bar_try(bar, parity))
    if (gtimer() - start > kWaitNs) return;
}

// 128-byte-swizzled operand: 8-row groups 1,024 bytes apart; lbo is the
// distance of the next 64 rows or columns of an operand whose M or N runs
// along the 128 bytes (not used along K)
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 x fp16 -> fp32, M = 128; B's N along the 128 bytes, A's K or M
__host__ __device__ constexpr uint32_t idesc(int n, bool a_m_major) {
  return (1u << 4) | ((a_m_major ? 1u : 0u) << 15) | (1u << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(id), "r"((uint32_t)add));
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&f)[16]) {
  uint32_t v[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

template <typename T, int GROUPS, int NV, int CT>
__global__ void __launch_bounds__(Geo<T, GROUPS, NV, CT>::kThreads, 1)
delta_chain_kernel(const __grid_constant__ exl3_delta_args a, const uint8_t* __restrict__ ws,
                   int vec) {
  using L = Geo<T, GROUPS, NV, CT>;
  constexpr bool kPacked = L::kPacked;
  extern __shared__ uint8_t dsm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slices = (a.dv + GROUPS * NV - 1) / (GROUPS * NV);
  const int slice = blockIdx.x % slices;
  const int64_t sh = blockIdx.x / slices;
  const int64_t s = sh / a.heads;
  const int h = (int)(sh - s * a.heads), kh = h / (a.heads / a.key_heads);
  const int64_t state_at = (s * a.heads + h) * (int64_t)a.dk * a.dv;
  int64_t t0, t1;
  seq_bounds(a, s, t0, t1);
  const int col_base = slice * GROUPS * NV;
  const int col_end = col_base + GROUPS * NV < a.dv ? col_base + GROUPS * NV : a.dv;

  // tokens outside every sequence, and sequences without tokens
  if (s == 0 || s == a.seqs - 1) {
    const int per = (col_end - col_base) / 8;
    T* o = static_cast<T*>(a.out);
    const int64_t before = s == 0 ? t0 : 0, after = s == a.seqs - 1 ? a.tokens - t1 : 0;
    for (int64_t i = tid; i < (before + after) * per; i += L::kThreads) {
      const int64_t t = i / per;
      const int64_t at = t < before ? t : t1 + (t - before);
      *reinterpret_cast<uint4*>(o + (at * a.heads + h) * a.dv + col_base + 8 * (i - t * per)) =
          make_uint4(0, 0, 0, 0);
    }
  }
  if (t0 == t1) {
    const int per = (col_end - col_base) / 4;
    for (int i = tid; i < a.dk * per; i += L::kThreads) {
      const int64_t at = state_at + (int64_t)(i / per) * a.dv + col_base + 4 * (i % per);
      *reinterpret_cast<float4*>(a.state_out + at) =
          a.state_in ? *reinterpret_cast<const float4*>(a.state_in + at) : make_float4(0, 0, 0, 0);
    }
    return;
  }
  const int chunks = (int)((t1 - t0 + kChunk - 1) / kChunk);
  const uint8_t* img = ws + (slot_base(t0, s) * a.heads + h) * kSlotBytes;
  const int64_t img_step = (int64_t)a.heads * kSlotBytes;

  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(dsm) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* kq_base = smem;
  uint8_t* t_base = kq_base + L::kKQStages * L::kKQ;
  uint8_t* s_base = t_base + L::kTStages * kImageBytes;
  uint8_t* r_base = s_base + GROUPS * L::kSBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(r_base + GROUPS * L::kRBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // per group: bits of max |S| before step ch and of max |v| of it, by ch & 1
  uint32_t(*peak)[2][2] = reinterpret_cast<uint32_t(*)[2][2]>(tmem_slot + 4);
  const auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const auto kq_full = [&](int st) { return bar(st); };
  const auto kq_empty = [&](int st) { return bar(L::kKQStages + st); };
  const auto t_full = [&](int st) { return bar(2 * L::kKQStages + st); };
  const auto t_empty = [&](int st) { return bar(2 * L::kKQStages + L::kTStages + st); };
  constexpr int kG0 = 2 * L::kKQStages + 2 * L::kTStages;
  // per group: s, r, u ready (epilogue -> issuer), d1, d2, d3 (products), done
  const auto gbar = [&](int g, int i) { return bar(kG0 + 7 * g + i); };

  if (tid == 0) {
    for (int i = 0; i < L::kKQStages; ++i) {
      bar_init(kq_full(i), 32 * L::kProducers);
      bar_init(kq_empty(i), GROUPS);
    }
    for (int i = 0; i < L::kTStages; ++i) {
      bar_init(t_full(i), 1);
      bar_init(t_empty(i), GROUPS);
    }
    for (int g = 0; g < GROUPS; ++g) {
      bar_init(gbar(g, 0), 4 * L::kWG);
      bar_init(gbar(g, 1), 2 * L::kWG);
      bar_init(gbar(g, 2), 2 * L::kWG);
      for (int i = 3; i < 7; ++i) bar_init(gbar(g, i), 1);
    }
    *abort_flag = 0;
    for (int i = 0; i < 4 * GROUPS; ++i) (&peak[0][0][0])[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // columns past dk are read by the products and never written again
  for (int i = tid; i < L::kKQStages * L::kKQ / 16; i += L::kThreads)
    reinterpret_cast<uint4*>(kq_base)[i] = make_uint4(0, 0, 0, 0);
  fence_async();
  if (warp == L::kEpiWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(L::kAlloc));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < L::kEpiWarps) {
    // ---------------- epilogue ----------------
    const int g = warp / (4 * L::kWG), quarter = warp & 3;
    const int c0 = ((warp >> 2) % L::kWG) * CT;       // first column in the group
    const int col = col_base + g * NV + c0;           // in the state
    const int row = 32 * quarter + lane;              // of dk; of [K; Q]
    const bool lower = quarter < 2;                   // K S, U rows; the others Q S, O rows
    uint8_t* s_op = s_base + g * L::kSBytes;
    uint8_t* r_op = r_base + g * L::kRBytes;
    const uint32_t d1 = tmem + (uint32_t)(g * L::kCols) + ((uint32_t)(32 * quarter) << 16) + c0;
    const uint32_t d2 = d1 + 64, d3 = d1 + 128;
    // a product's columns c .. c + 15 of this thread's row
    const auto product = [&](uint32_t d, int c, float (&f)[16]) {
      tmem_ld(d + c, f);
      if constexpr (kPacked) {
        float l[16];
        tmem_ld(d + 32 + c, l);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] += l[i];
      } else {
        tmem_ld_wait();
      }
    };
    // 16 values into columns c .. c + 15 of row r of an operand, both parts
    const auto store_op = [&](uint8_t* op, int tile, int r, int c, const float (&f)[16]) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint4 hi, lo;
        split8(f + 8 * e, hi, lo);
        const int q = (c0 + c) / 8 + e;
        *reinterpret_cast<uint4*>(op + swz(r, q)) = hi;
        *reinterpret_cast<uint4*>(kPacked ? op + swz(r, q + 4) : op + tile + swz(r, q)) = lo;
      }
    };
    const auto ready = [&](int i) {
      fence_async();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(gbar(g, i));
    };
    float S[CT];
    uint4 vr[CT / 8];
    const T* v = static_cast<const T*>(a.v) + h * a.v_strides[1] + col;
    T* out = static_cast<T*>(a.out) + (int64_t)h * a.dv + col;
    const auto load_v = [&](int ch) {
      const int64_t t = t0 + (int64_t)ch * kChunk + row;
#pragma unroll
      for (int c = 0; c < CT / 8; ++c)
        vr[c] = lower && t < t1 && col + 8 * c < a.dv ? load8(v + t * a.v_strides[0] + 8 * c, vec & 2)
                                                      : make_uint4(0, 0, 0, 0);
    };
    // the peaks that step ch starts from
    const auto note_peaks = [&](int ch) {
      float m = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) m = fmaxf(m, fabsf(S[c]));
      const uint32_t ms = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
      if (lane == 0) atomicMax(&peak[g][ch & 1][0], ms);
      if (lower) {
        uint32_t w = 0;  // 16-bit patterns of non-negative values order like the values
#pragma unroll
        for (int c = 0; c < CT / 8; ++c) {
          w = __vmaxu2(w, vr[c].x & 0x7FFF7FFFu);
          w = __vmaxu2(w, vr[c].y & 0x7FFF7FFFu);
          w = __vmaxu2(w, vr[c].z & 0x7FFF7FFFu);
          w = __vmaxu2(w, vr[c].w & 0x7FFF7FFFu);
        }
        const uint16_t top = (uint16_t)__reduce_max_sync(0xFFFFFFFFu, max(w & 0xFFFFu, w >> 16));
        if (lane == 0)
          atomicMax(&peak[g][ch & 1][1], __float_as_uint(to_f32(*reinterpret_cast<const T*>(&top))));
      }
    };
    // S times its scale, as 16-column pieces (CT is 16 or 32)
    const auto store_state = [&](float scale) {
#pragma unroll
      for (int c = 0; c < CT; c += 16) {
        float f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = S[c + i] * scale;
        store_op(s_op, 128 * 128, row, c, f);
      }
    };
#pragma unroll
    for (int c = 0; c < CT; c += 4) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (a.state_in && row < a.dk && col + c < a.dv)
        x = *reinterpret_cast<const float4*>(a.state_in + state_at + (int64_t)row * a.dv + col + c);
      S[c] = x.x;
      S[c + 1] = x.y;
      S[c + 2] = x.z;
      S[c + 3] = x.w;
    }
    load_v(0);
    note_peaks(0);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(128 * L::kWG) : "memory");
    float scale_s, inv_s;
    pow2_scale(__uint_as_float(peak[g][0][0]), scale_s, inv_s);
    store_state(scale_s);
    ready(0);
    bool ok = true;
    for (int ch = 0; ch < chunks && ok; ++ch) {
      const uint32_t ph = ch & 1;
      const float* vecs = reinterpret_cast<const float*>(img + ch * img_step + kImageBytes);
      float ab = vecs[row];                           // a of K S rows, b of Q S rows
      const float cc = lower ? vecs[128 + row] : 0.f;
      const float gamma = vecs[kGamma], bound_a = vecs[kBoundA], bound_u = vecs[kBoundU],
                  bound_s = vecs[kBoundS], image_scale = vecs[lower ? kScaleT : kScalePT];
      const int64_t t = t0 + (int64_t)ch * kChunk + (row & 63);
      // 1. K S -> R = V - a K S
      ok = bar_wait(gbar(g, 3), ph, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      fence_after();
      const float smax = __uint_as_float(peak[g][ph][0]), vmax = __uint_as_float(peak[g][ph][1]);
      // read by all before this step's first product was issued; filled again
      // after its last one
      if ((warp & (4 * L::kWG - 1)) == 0 && lane == 0) peak[g][ph ^ 1][0] = peak[g][ph ^ 1][1] = 0;
      const float bound_r = fmaf(bound_a, smax, vmax);
      float scale_r, inv_r, scale_u, inv_u;
      pow2_scale(bound_r, scale_r, inv_r);
      pow2_scale(bound_u * bound_r, scale_u, inv_u);
      ab *= inv_s;
      if (lower) {
        const float m = -ab * scale_r;
#pragma unroll
        for (int c = 0; c < CT; c += 16) {
          float f[16];
          product(d1, c, f);
          const T* ve = reinterpret_cast<const T*>(vr + c / 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = fmaf(m, f[i], to_f32(ve[i]) * scale_r);
          store_op(r_op, 64 * 128, row, c, f);
        }
        ready(1);
        if (ch + 1 < chunks) load_v(ch + 1);
      }
      // 2. U -> c U, and O = b Q S + P U
      ok = bar_wait(gbar(g, 4), ph, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      fence_after();
      const float from_image = inv_r * image_scale;
      if (lower) {
        const float m = from_image * cc * scale_u;
#pragma unroll
        for (int c = 0; c < CT; c += 16) {
          float f[16];
          product(d2, c, f);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] *= m;
          store_op(r_op, 64 * 128, row, c, f);
        }
        ready(2);
      } else {
#pragma unroll
        for (int c = 0; c < CT; c += 16) {
          float f[16], p[16];
          product(d1, c, f);
          product(d2, c, p);
          Vec<T, 8> o[2];
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i / 8].e[i % 8] = from_f32<T>(fmaf(ab, f[i], from_image * p[i]));
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (t < t1 && col + c + 8 * e < a.dv)
              *reinterpret_cast<uint4*>(out + t * a.heads * a.dv + c + 8 * e) =
                  *reinterpret_cast<const uint4*>(&o[e]);
        }
      }
      // 3. the state moves on
      ok = bar_wait(gbar(g, 5), ph, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
      fence_after();
#pragma unroll
      for (int c = 0; c < CT; c += 16) {
        float f[16];
        product(d3, c, f);
#pragma unroll
        for (int i = 0; i < 16; ++i) S[c + i] = fmaf(gamma, S[c + i], inv_u * f[i]);
      }
      if (ch + 1 < chunks) {
        pow2_scale(fmaf(bound_s, bound_r, gamma * smax), scale_s, inv_s);
        store_state(scale_s);
        note_peaks(ch + 1);
        ready(0);
      }
    }
#pragma unroll
    for (int c = 0; c < CT; c += 4)
      if (row < a.dk && col + c < a.dv)
        *reinterpret_cast<float4*>(a.state_out + state_at + (int64_t)row * a.dv + col + c) =
            make_float4(S[c], S[c + 1], S[c + 2], S[c + 3]);
  } else if (warp < L::kEpiWarps + GROUPS) {
    // ---------------- products: one thread per group ----------------
    const int g = warp - L::kEpiWarps;
    if (lane == 0) {
      const uint32_t d1 = tmem + (uint32_t)(g * L::kCols), d2 = d1 + 64, d3 = d1 + 128;
      const uint32_t s_op = smem_u32(s_base + g * L::kSBytes);
      const uint32_t r_op = smem_u32(r_base + g * L::kRBytes);
      const int ksteps = (a.dk + 15) / 16;
      bool ok = true;
      for (int ch = 0; ch < chunks && ok; ++ch) {
        const uint32_t ph = ch & 1;
        const int ks = ch % L::kKQStages, ts = ch % L::kTStages;
        const uint32_t kq = smem_u32(kq_base + ks * L::kKQ);
        const uint32_t ti = smem_u32(t_base + ts * kImageBytes);
        // [K; Q] S
        ok = bar_wait(kq_full(ks), (ch / L::kKQStages) & 1, abort_flag) &&
             bar_wait(gbar(g, 0), ph, abort_flag);
        if (!ok) break;
        fence_after();
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t ao = kq + (k >> 2) * L::kBox + (k & 3) * 32, bo = s_op + k * 2048;
          mma(d1, desc(ao, 16), desc(bo, 16), idesc(64, false), k > 0);
          if constexpr (!kPacked) mma(d1, desc(ao, 16), desc(bo + 128 * 128, 16), idesc(64, false), true);
        }
        commit(gbar(g, 3));
        // [T; P T] R
        ok = bar_wait(t_full(ts), (ch / L::kTStages) & 1, abort_flag) &&
             bar_wait(gbar(g, 1), ph, abort_flag);
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t ao = ti + k * 32, bo = r_op + k * 2048;
          mma(d2, desc(ao, 16), desc(bo, 16), idesc(64, false), k > 0);
          if constexpr (!kPacked) mma(d2, desc(ao, 16), desc(bo + 64 * 128, 16), idesc(64, false), true);
          mma(d2, desc(ao + kImageBytes / 2, 16), desc(bo, 16), idesc(NV, false), true);
        }
        commit(gbar(g, 4));
        commit(t_empty(ts));
        // K^T U
        ok = bar_wait(gbar(g, 2), ph, abort_flag);
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t ao = kq + k * 2048, bo = r_op + k * 2048;
          mma(d3, desc(ao, L::kBox), desc(bo, 16), idesc(64, true), k > 0);
          if constexpr (!kPacked)
            mma(d3, desc(ao, L::kBox), desc(bo + 64 * 128, 16), idesc(64, true), true);
        }
        commit(gbar(g, 5));
        commit(kq_empty(ks));
      }
      // whatever was issued has finished before tensor memory is freed
      commit(gbar(g, 6));
      bar_drain(gbar(g, 6), 0);
    }
  } else {
    // ---------------- producers ----------------
    const int pt = tid - 32 * (L::kEpiWarps + GROUPS);
    const int pieces = a.dk / 8;
    const T* qp = static_cast<const T*>(a.q) + kh * a.q_strides[1];
    const T* kp = static_cast<const T*>(a.k) + kh * a.k_strides[1];
    int issued = 0;
    bool ok = true;
    for (int ch = 0; ch < chunks && ok; ++ch) {
      const int ks = ch % L::kKQStages, ts = ch % L::kTStages;
      if (pt == 0) {
        if (ch >= L::kTStages)
          ok = bar_wait(t_empty(ts), (ch / L::kTStages - 1) & 1, abort_flag);
        if (ok) {
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(t_full(ts)),
                       "r"(kImageBytes)
                       : "memory");
          asm volatile(
              "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
                  "r"(smem_u32(t_base + ts * kImageBytes)),
              "l"(img + ch * img_step), "r"(kImageBytes), "r"(t_full(ts))
              : "memory");
          issued = ch + 1;
        }
      }
      if (ok && ch >= L::kKQStages)
        ok = bar_wait(kq_empty(ks), (ch / L::kKQStages - 1) & 1, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      uint8_t* kq = kq_base + ks * L::kKQ;
      const float* scales = reinterpret_cast<const float*>(img + ch * img_step + kImageBytes) + kRowScale;
      const int64_t tc = t0 + (int64_t)ch * kChunk;
      const int n = (int)(t1 - tc < kChunk ? t1 - tc : kChunk);
      for (int i0 = pt; i0 < 128 * pieces; i0 += 32 * L::kProducers * 4) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * 32 * L::kProducers;
          const int r = i / pieces, q = i - r * pieces, row = r & 63;
          x[u] = make_uint4(0, 0, 0, 0);
          if (r < 128 && row < n)
            x[u] = r < 64 ? load8(kp + (tc + row) * a.k_strides[0] + 8 * q, vec & 1)
                          : load8(qp + (tc + row) * a.q_strides[0] + 8 * q, vec & 1);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * 32 * L::kProducers;
          const int r = i / pieces, q = i - r * pieces;
          if (r >= 128) break;
          uint8_t* dst = kq + (q >> 3) * L::kBox + swz(r, q & 7);
          if constexpr (!std::is_same<T, __half>::value) {
            const float f = scales[r];
            const T* e = reinterpret_cast<const T*>(&x[u]);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __half2 p = __floats2half2_rn(to_f32(e[2 * j]) * f, to_f32(e[2 * j + 1]) * f);
              w[j] = *reinterpret_cast<const uint32_t*>(&p);
            }
            x[u] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(dst) = x[u];
        }
      }
      fence_async();
      bar_arrive(kq_full(ks));
    }
    // stopped early: copies in flight land before the CTA exits
    if (pt == 0 && *abort_flag)
      for (int ch = issued > L::kTStages ? issued - L::kTStages : 0; ch < issued; ++ch)
        bar_drain(t_full(ch % L::kTStages), (ch / L::kTStages) & 1);
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicAdd(&g_delta_faults, 1u);
  if (warp == L::kEpiWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kAlloc));
  }
}

template <typename T, int GROUPS, int NV, int CT>
int launch_chain(const exl3_delta_args& a, const uint8_t* ws, int vec, cudaStream_t stream) {
  using L = Geo<T, GROUPS, NV, CT>;
  static DeviceBits attr_done;
  int dev = 0;
  EXL3_CUDA(cudaGetDevice(&dev));
  if (!attr_done.has(dev)) {
    EXL3_CUDA(cudaFuncSetAttribute(delta_chain_kernel<T, GROUPS, NV, CT>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem));
    attr_done.set(dev);
  }
  const int64_t ctas = a.seqs * a.heads * ((a.dv + GROUPS * NV - 1) / (GROUPS * NV));
  EXL3_REQUIRE(ctas < (1ll << 31), "too many sequences and heads");
  delta_chain_kernel<T, GROUPS, NV, CT><<<(unsigned)ctas, L::kThreads, L::kSmem, stream>>>(a, ws, vec);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

template <typename T>
int launch_chunks(const exl3_delta_args& a, uint8_t* ws, cudaStream_t stream) {
  static DeviceBits attr_done;
  int dev = 0;
  EXL3_CUDA(cudaGetDevice(&dev));
  if (!attr_done.has(dev)) {
    EXL3_CUDA(cudaFuncSetAttribute(delta_prep_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)sizeof(PrepSmem)));
    attr_done.set(dev);
  }
  const auto fits = [](const void* p, const int64_t* st) {
    return aligned_to(p, 16) && st[0] % 8 == 0 && st[1] % 8 == 0;
  };
  const int vec = (fits(a.q, a.q_strides) && fits(a.k, a.k_strides) ? 1 : 0) |
                  (fits(a.v, a.v_strides) ? 2 : 0);
  const int64_t slots = a.tokens / kChunk + a.seqs;
  EXL3_REQUIRE(slots < (1ll << 31) && a.key_heads < 65536, "too many tokens or heads");
  delta_prep_kernel<T><<<dim3((unsigned)slots, (unsigned)a.key_heads), kPrepThreads, sizeof(PrepSmem),
                         stream>>>(a, ws, vec & 1);
  EXL3_LAUNCHED();
  const int64_t chains = a.seqs * a.heads;
  if (chains * ((a.dv + 31) / 32) <= sm_count())
    return launch_chain<T, 1, 32, 16>(a, ws, vec, stream);
  return launch_chain<T, 2, 64, 32>(a, ws, vec, stream);
}

}  // namespace

size_t delta_chunk_ws_bytes(const exl3_delta_args& a) {
  return (size_t)(a.tokens / kChunk + a.seqs) * a.heads * kSlotBytes;
}

int delta_chunks(const exl3_delta_args& a, void* ws, cudaStream_t stream) {
  return a.dtype == EXL3_F16 ? launch_chunks<__half>(a, static_cast<uint8_t*>(ws), stream)
                             : launch_chunks<__nv_bfloat16>(a, static_cast<uint8_t*>(ws), stream);
}

}  // namespace exl3

extern "C" int exl3_delta_fault_count(unsigned int* count) {
  using namespace exl3;
  EXL3_REQUIRE(count != nullptr, "count is NULL");
  EXL3_CUDA(cudaMemcpyFromSymbol(count, g_delta_faults, sizeof(unsigned int)));
  return EXL3_OK;
}
