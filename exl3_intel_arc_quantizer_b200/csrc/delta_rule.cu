// The gated delta rule, token by token, and the entry points of both forms.
//
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t)
//   o_t = scale S_t^T q_t
//
// Both dot products of a token go over the old state: with a = S^T k,
// b = S^T q and G = e^g,
//   u = beta (v - G a),  o = scale (G b + (q . k) u),
// so one pass over the state's registers and one set of shuffles give u and
// o, and the update follows. The norms of q and k are factors of a, b and
// q . k and are summed by the same shuffles.
//
// A warp owns 4 CL columns of one head's state in registers: CL lanes hold
// four columns each (CL = 4: a row of the slice is 64 bytes), 32 / CL lanes
// share the rows. No two warps exchange anything. Single tokens are
// bound by HBM: the state is read and written once (8 bytes per element).
//
// B200: 128 tokens of 32 heads of 128 x 128: 106.5 us, 5.1 TB/s (0.78 of the
// measured copy rate) with 16 columns per warp; with 32, twice the registers
// per thread and half the warps, 127 us.
#include "common.cuh"
#include "delta_rule.cuh"

namespace exl3 {
namespace {

constexpr int kWarps = 4;  // per CTA

// N consecutive elements from p, zero where the row of k or q ends
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, int at, int d, bool vec, float (&out)[N]) {
  if (vec) {
#pragma unroll
    for (int c = 0; c < N; c += 8) {
      if (at + c < d) {  // d is a multiple of 8
        float f[8];
        unpack(load_raw<T, 8>(p + at + c), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) out[c + i] = f[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[c + i] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = at + i < d ? to_f32(p[at + i]) : 0.f;
  }
}

// ROWS: state rows of a thread (dk <= ROWS * 32 / CL). STEP: one token per sequence,
// states picked by slot and written in place.
template <typename T, int ROWS, int CL, bool STEP>
__global__ void __launch_bounds__(32 * kWarps)
delta_tokens_kernel(const __grid_constant__ exl3_delta_args a, int vec) {
  const int lane = threadIdx.x & 31;
  constexpr int kCols = 4 * CL;
  const int slices = (a.dv + kCols - 1) / kCols;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t sh = w / slices;
  if (sh >= a.seqs * a.heads) return;
  const int64_t s = sh / a.heads;
  const int h = (int)(sh - s * a.heads), kh = h / (a.heads / a.key_heads);
  const int col = (int)(w - sh * slices) * kCols + (lane % CL) * 4;
  const int row0 = (lane / CL) * ROWS;
  const bool in = col < a.dv;  // dv is a multiple of 8: four columns are all in or all out

  int64_t t0, t1, from, to;
  if (STEP) {
    t0 = s;
    t1 = s + 1;
    from = to = a.slots ? a.slots[s] : s;
    if (from < 0 || from >= a.num_slots) {
      if (in && lane < CL) {
        T* o = static_cast<T*>(a.out) + (t0 * a.heads + h) * a.dv + col;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = from_f32<T>(0.f);
      }
      return;
    }
  } else {
    seq_bounds(a, s, t0, t1);
    from = to = s;
    if (in && lane < CL) zero_outside<T>(a, s, t0, t1, h, col, 4);
  }
  float S[ROWS][4];
  const int64_t state_at = ((int64_t)from * a.heads + h) * a.dk * a.dv;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.state_in && in && row0 + i < a.dk)
      v = *reinterpret_cast<const float4*>(a.state_in + state_at + (int64_t)(row0 + i) * a.dv + col);
    S[i][0] = v.x;
    S[i][1] = v.y;
    S[i][2] = v.z;
    S[i][3] = v.w;
  }
  const T* q = static_cast<const T*>(a.q) + kh * a.q_strides[1];
  const T* k = static_cast<const T*>(a.k) + kh * a.k_strides[1];
  const T* v = static_cast<const T*>(a.v) + h * a.v_strides[1];
  for (int64_t t = t0; t < t1; ++t) {
    float kr[ROWS], qr[ROWS], vr[4];
    load_row<T, ROWS>(k + t * a.k_strides[0], row0, a.dk, vec & 1, kr);
    load_row<T, ROWS>(q + t * a.q_strides[0], row0, a.dk, vec & 1, qr);
#pragma unroll
    for (int c = 0; c < 4; ++c) vr[c] = in ? to_f32(v[t * a.v_strides[0] + col + c]) : 0.f;
    const float G = expf(a.g[t * a.g_stride + h]), beta = a.beta[t * a.beta_stride + h];
    // kk, qq, qk, then the four columns of S^T k and S^T q
    float r[11];
#pragma unroll
    for (int j = 0; j < 11; ++j) r[j] = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      r[0] = fmaf(kr[i], kr[i], r[0]);
      r[1] = fmaf(qr[i], qr[i], r[1]);
      r[2] = fmaf(qr[i], kr[i], r[2]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        r[3 + c] = fmaf(S[i][c], kr[i], r[3 + c]);
        r[7 + c] = fmaf(S[i][c], qr[i], r[7 + c]);
      }
    }
#pragma unroll
    for (int o = CL; o < 32; o <<= 1)
#pragma unroll
      for (int j = 0; j < 11; ++j) r[j] += __shfl_xor_sync(0xFFFFFFFFu, r[j], o);
    const float rk = a.normalize_qk ? rsqrtf(r[0] + kNormEps) : 1.f;
    const float rq = (a.normalize_qk ? rsqrtf(r[1] + kNormEps) : 1.f) * a.scale;
    float u[4], o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = beta * (vr[c] - G * rk * r[3 + c]);
      o[c] = rq * (G * r[7 + c] + r[2] * rk * u[c]);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float ki = kr[i] * rk;
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = fmaf(ki, u[c], G * S[i][c]);
    }
    if (in && lane < CL)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (t * a.heads + h) * a.dv + col) =
          make_uint2(f32_to_word<T>(make_float2(o[0], o[1])), f32_to_word<T>(make_float2(o[2], o[3])));
  }
  if (in)
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (row0 + i < a.dk)
        *reinterpret_cast<float4*>(a.state_out + ((int64_t)to * a.heads + h) * a.dk * a.dv +
                                   (int64_t)(row0 + i) * a.dv + col) =
            make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
}

template <typename T, bool STEP>
int launch_tokens(const exl3_delta_args& a, cudaStream_t stream) {
  constexpr int kCols = 16;
  const int64_t warps = a.seqs * a.heads * ((a.dv + kCols - 1) / kCols);
  const int64_t ctas = (warps + kWarps - 1) / kWarps;
  EXL3_REQUIRE(ctas < (1ll << 31), "too many sequences and heads");
  const auto fits = [](const void* p, const int64_t* st) {
    return aligned_to(p, 16) && st[0] % 8 == 0 && st[1] % 8 == 0;
  };
  const int vec = fits(a.q, a.q_strides) && fits(a.k, a.k_strides);
  if (a.dk <= 64)
    delta_tokens_kernel<T, 8, 4, STEP><<<(unsigned)ctas, 32 * kWarps, 0, stream>>>(a, vec);
  else if (a.dk <= 128)
    delta_tokens_kernel<T, 16, 4, STEP><<<(unsigned)ctas, 32 * kWarps, 0, stream>>>(a, vec);
  else
    delta_tokens_kernel<T, 32, 4, STEP><<<(unsigned)ctas, 32 * kWarps, 0, stream>>>(a, vec);
  EXL3_LAUNCHED();
  return EXL3_OK;
}

// The chunked form for all but a handful of tokens and heads too wide for it.
bool chunked(const exl3_delta_args& a) { return a.dk <= 128 && a.tokens > 8; }

int check_args(const exl3_delta_args* args) {
  EXL3_REQUIRE(args != nullptr, "args is NULL");
  const exl3_delta_args& a = *args;
  EXL3_REQUIRE(a.dtype == EXL3_F16 || a.dtype == EXL3_BF16, "dtype must be 0 (fp16) or 1 (bf16), got %d",
               a.dtype);
  EXL3_REQUIRE(a.key_heads >= 1 && a.heads >= 1 && a.heads % a.key_heads == 0,
               "heads (%d) must be a positive multiple of key_heads (%d)", a.heads, a.key_heads);
  EXL3_REQUIRE(a.dk >= 8 && a.dk <= 256 && a.dk % 8 == 0, "dk must be a multiple of 8 up to 256, got %d",
               a.dk);
  EXL3_REQUIRE(a.dv >= 8 && a.dv <= 65536 && a.dv % 8 == 0, "dv must be a positive multiple of 8, got %d",
               a.dv);
  EXL3_REQUIRE(a.tokens >= 0 && a.seqs >= 0, "tokens and seqs must be non-negative");
  return EXL3_OK;
}

int check_pointers(const exl3_delta_args& a) {
  EXL3_REQUIRE(a.state_out && aligned_to(a.state_out, 16) && aligned_to(a.state_in, 16),
               "the states must be 16-byte aligned device pointers");
  EXL3_REQUIRE(a.tokens == 0 || (a.q && a.k && a.v && a.g && a.beta && a.out), "NULL pointer argument");
  EXL3_REQUIRE(aligned_to(a.out, 16), "out must be 16-byte aligned");
  return EXL3_OK;
}

}  // namespace
}  // namespace exl3

using namespace exl3;

extern "C" int exl3_delta_step(const exl3_delta_args* args, exl3_stream_t stream) {
  if (const int rc = check_args(args)) return rc;
  exl3_delta_args a = *args;
  EXL3_REQUIRE(a.tokens == a.seqs, "a step has one token per sequence");
  EXL3_REQUIRE(a.num_slots >= (a.slots ? 1 : a.seqs), "num_slots (%lld) is less than the sequences",
               (long long)a.num_slots);
  if (a.seqs == 0) return EXL3_OK;
  a.state_in = a.state_out;
  if (const int rc = check_pointers(a)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  return a.dtype == EXL3_F16 ? launch_tokens<__half, true>(a, s)
                             : launch_tokens<__nv_bfloat16, true>(a, s);
}

extern "C" size_t exl3_delta_rule_ws_bytes(const exl3_delta_args* args) {
  if (check_args(args)) return 0;
  return chunked(*args) ? delta_chunk_ws_bytes(*args) : 16;
}

extern "C" int exl3_delta_rule(const exl3_delta_args* args, void* ws, size_t ws_bytes,
                               exl3_stream_t stream) {
  if (const int rc = check_args(args)) return rc;
  const exl3_delta_args& a = *args;
  const size_t need = exl3_delta_rule_ws_bytes(args);
  EXL3_REQUIRE(ws && ws_bytes >= need, "workspace of %zu bytes is smaller than the %zu needed",
               ws_bytes, need);
  if (a.seqs == 0) return EXL3_OK;
  EXL3_REQUIRE(a.cu_seqlens, "cu_seqlens is NULL");
  if (const int rc = check_pointers(a)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (chunked(a)) {
    EXL3_REQUIRE(aligned_to(ws, 16), "the workspace must be 16-byte aligned");
    return delta_chunks(a, ws, s);
  }
  return a.dtype == EXL3_F16 ? launch_tokens<__half, false>(a, s)
                             : launch_tokens<__nv_bfloat16, false>(a, s);
}
