// Activations of the grouped linear layers, their derivatives, and the element-wise part
// of the layers' gradient.
#pragma once
#include "common.cuh"

namespace smoe {

// 2^v and 1/v as one instruction each: relative error 2^-22 and one unit in the last place,
// subnormal results flushed to 0.  The general forms handle subnormal operands in extra
// instructions, which the gradient's element-wise kernel has no time for.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 2^(2 v) to 2^-21, subnormal results rounded instead of flushed: times a few units they are
// normal numbers again.
__device__ __forceinline__ float exp2_twice(float v) {
  const float h = exp2_fast(v);
  return h * h;
}
constexpr float kLog2e = 1.4426950408889634f;

// v within [-lim, lim], NaN kept.
__device__ __forceinline__ float clamp_nan(float v, float lim) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(lim));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(-lim));
  return r;
}

// sigmoid(v) = 1 / (1 + e^-v) with numerator and denominator 2^-8 times as large, for the lower
// tail: 1 / e^-v would be flushed from v = -87.3 on, this from -93, where v sigmoid(v) (a
// normal number of bf16 down to v = -92) no longer matters.  e^-v may be infinite, the
// quotient is then 0.  One multiplication more; with e^v / (1 + e^v) for v < 0, three more,
// SiLU's gradient took 256 us instead of 234 for 16384 x 14336 bf16 values.
__device__ __forceinline__ float sigmoid_f(float v) {
  return 0.00390625f * rcp_fast(0.00390625f + exp2_fast(fmaf(-kLog2e, v, -8.0f)));
}

// gelu_tanh(z) = z/2 (1 + tanh u) = z sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3).
__device__ __forceinline__ float gelu_tanh_2u(float z) {
  constexpr float c = 1.5957691216057308f;  // 2 sqrt(2/pi)
  return c * fmaf(0.044715f * z * z, z, z);
}

// Phi(z), the normal distribution function, and e = exp(-z^2 / 2), which the derivative of
// z Phi(z) needs too.  The lower tail is Phi(-x) = e R(x) with Mills' ratio over sqrt(2 pi),
// R(x) = exp(x^2 / 2) erfc(x / sqrt 2) / 2, smooth and algebraic in x: with t = 1 / (1 + p x)
// it is t times a polynomial in t, here of degree 6, its coefficients and p fitted for the
// smallest RELATIVE error over 0 <= x <= 13.5 (a linear programme over Chebyshev points):
// 7e-7.  So small values far down the tail keep their digits -- with an absolutely accurate
// erfc (Abramowitz and Stegun 7.1.26, two terms less) z Phi(z) was off by 5e-4 at z = -4,
// half a step of fp16, and by 1e-2 at -8, five half steps of bf16.  One exponential and one
// reciprocal serve both, no cancellation for z < 0.  (erff and a separate exponential made
// the gradient of 16384 x 14336 bf16 values compute-bound, 448 us; with these it takes 273.)
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = rcp_fast(fmaf(0.3617f, fabsf(z), 1.0f));
  e = exp2_twice((-0.25f * kLog2e * z) * z);
  float q = fmaf(t, 0.04806739448f, -0.1808574259f);
  q = fmaf(t, q, 0.1784509820f);
  q = fmaf(t, q, 0.02768831198f);
  q = fmaf(t, q, 0.1397628274f);
  q = fmaf(t, q, 0.1424992758f);
  q = fmaf(t, q, 0.1443889928f);
  q *= t * e;
  return z < 0.0f ? q : 1.0f - q;
}

// ACT is a compile-time SMOE_ACT_*; NaN stays NaN in all of them.
template <int ACT> __device__ __forceinline__ float act_f(float z) {
  if constexpr (ACT == SMOE_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == SMOE_ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  if constexpr (ACT == SMOE_ACT_GELU_TANH) return z * sigmoid_f(gelu_tanh_2u(z));
  if constexpr (ACT == SMOE_ACT_SILU) return z * sigmoid_f(z);
  return z;
}

// z may be infinite where the forward was finite: it is kept rounded to the layer's type,
// and fp16 ends at 65504.  The slopes are 0 or 1 to fp32 long before the clamps' limits
// (GELU's beyond 15, SiLU's beyond 105), which keep 0 * infinity out of them.
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == SMOE_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;  // NaN: the gradient passes
  if constexpr (ACT == SMOE_ACT_GELU) {  // Phi(z) + z phi(z)
    z = clamp_nan(z, 30.0f);
    float e;
    const float phi = normal_cdf(z, e);
    return fmaf(z * 0.3989422804014327f, e, phi);
  }
  if constexpr (ACT == SMOE_ACT_GELU_TANH) {  // s + z s (1 - s) (2u)'
    z = clamp_nan(z, 30.0f);
    const float s = sigmoid_f(gelu_tanh_2u(z));
    return fmaf(z * s * (1.0f - s), 1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f), s);
  }
  if constexpr (ACT == SMOE_ACT_SILU) {
    z = clamp_nan(z, 128.0f);
    const float s = sigmoid_f(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return 1.0f;
}

// f(z[i]) for a run-time activation: one uniform branch around the whole array.
template <int N> __device__ __forceinline__ void apply_act(int act, float (&z)[N]) {
  switch (act) {
    case SMOE_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = act_f<SMOE_ACT_RELU>(z[i]);
      break;
    case SMOE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = act_f<SMOE_ACT_GELU>(z[i]);
      break;
    case SMOE_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = act_f<SMOE_ACT_GELU_TANH>(z[i]);
      break;
    case SMOE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = act_f<SMOE_ACT_SILU>(z[i]);
      break;
    default: break;
  }
}

// What the epilogue of a grouped linear layer adds to its products: out = act(acc +
// bias[g]) + residual[row], preact[row] = acc + bias[g] (kept for the gradient).  Null
// pointers leave a term out.  Column counts are multiples of 8, pointers 16-byte aligned.
struct LinearEpi {
  const void* bias = nullptr;      // [G, N], the layer's 16-bit type, or fp32
  const void* residual = nullptr;  // [rows_cap, N], the layer's type
  void* preact = nullptr;          // [rows_cap, N], the layer's type
  int bias_f32 = 0;
  int act = SMOE_ACT_NONE;
  int fill = 0;                    // rows of no group get residual (or 0) instead of staying as they were
};

// v[i] += bias[g, col + i] for W consecutive columns (W = 4 or a multiple of 8).
template <typename T, int W>
__device__ __forceinline__ void add_bias(const LinearEpi& lin, int64_t at, float (&v)[W]) {
  if (lin.bias == nullptr) return;
  if (lin.bias_f32) {
    const float* b = static_cast<const float*>(lin.bias) + at;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(b) + i);
      v[4 * i] += q.x;
      v[4 * i + 1] += q.y;
      v[4 * i + 2] += q.z;
      v[4 * i + 3] += q.w;
    }
  } else {
    const T* b = static_cast<const T*>(lin.bias) + at;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(b) + i);
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] += Num<T>::to_f(e[j]);
    }
  }
}

// ------------------------------------------------------------------ gradient, element-wise
// dz = dout * act'(z) for the rows of the groups, and the bias gradient db[g] = the sum
// of dz over the group's rows, from the unrounded fp32 products.  dz itself is rounded to the
// layer's type, as an operand of the 16-bit tensor-core products that make dA and dW of it.
// Memory-bound: dout and z read once, dz written once.  A block owns 256 columns (a lane 8 of
// them) of `slice` consecutive rows, its eight warps every eighth row; it walks the groups its
// rows belong to and writes one partial row of column sums per group to part[s + g], which is
// a different row for every (slice s, group g) pair that has rows, since both only grow along
// the rows.  bias_grad_reduce_kernel adds a group's partials in slice order, so no result
// depends on the order in which blocks run.
constexpr int kActCols = 256, kActGroups = 1024;

template <typename T, int ACT, bool BIAS>
__global__ void __launch_bounds__(256, 4) linear_act_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ z,
                                                             T* __restrict__ dz, const int32_t* __restrict__ offsets,
                                                             int G, int rows_cap, int N, int slice,
                                                             float* __restrict__ part) {
  __shared__ float s_sum[8][kActCols + 8];
  __shared__ int s_off[kActGroups + 1];  // the walk over (mostly empty) groups waits for no load
  for (int i = threadIdx.x; i <= G; i += 256) s_off[i] = offsets[i];
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * kActCols + lane * 8;
  const bool live = col < N;
  const int end_all = min(max(s_off[G], 0), rows_cap);
  int row = max(blockIdx.y * slice, max(s_off[0], 0));
  const int row_end = min((int)blockIdx.y * slice + slice, end_all);
  if (row >= row_end) return;
  int lo = 0, hi = G - 1;  // last group whose start <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_off[mid] <= row) lo = mid; else hi = mid - 1;
  }
  for (int g = lo; g < G && row < row_end; ++g) {
    const int stop = min(s_off[g + 1], row_end);
    if (stop <= row) continue;
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.f;
    if (live) {
#pragma unroll 2  // (4 rows take the registers of a fourth block per SM: 307 against 267 us with GELU)
      for (int r = row + warp; r < stop; r += 8) {
        float dy[8];
        load_vec_f<T, 8>(dout + (int64_t)r * N + col, dy);
        if constexpr (ACT != SMOE_ACT_NONE) {
          float zz[8];
          load_vec_f<T, 8>(z + (int64_t)r * N + col, zz);
          union {
            uint4 u;
            T e[8];
          } o;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dy[i] *= act_slope<ACT>(zz[i]);
            o.e[i] = Num<T>::from_f(dy[i]);
          }
          *reinterpret_cast<uint4*>(dz + (int64_t)r * N + col) = o.u;
        }
        if constexpr (BIAS)
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] += dy[i];
      }
    }
    if constexpr (BIAS) {
      __syncthreads();  // the previous group's sums have been read
#pragma unroll
      for (int i = 0; i < 8; ++i) s_sum[warp][lane * 8 + i] = sum[i];
      __syncthreads();
      const int c = blockIdx.x * kActCols + threadIdx.x;
      if (c < N) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += s_sum[q][threadIdx.x];
        part[((int64_t)blockIdx.y + g) * N + c] = s;
      }
    }
    row = stop;
  }
}

// dbias[g, n] = sum over the group's slices, in order; OutT is the bias's type.  One block:
// 32 columns of one group, each of its eight warps every eighth slice, then the eight sums
// in warp order.
template <typename OutT>
__global__ void __launch_bounds__(256) bias_grad_reduce_kernel(const float* __restrict__ part,
                                                               const int32_t* __restrict__ offsets, int G, int rows_cap,
                                                               int N, int slice, OutT* __restrict__ dbias) {
  __shared__ float s_sum[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, g = blockIdx.y;
  const int b = min(max(offsets[g], 0), rows_cap), e = min(max(offsets[g + 1], b), rows_cap);
  float s = 0.f;
  if (c < N && e > b)
#pragma unroll 4
    for (int q = b / slice + warp; q <= (e - 1) / slice; q += 8) s += part[((int64_t)q + g) * N + c];
  s_sum[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < N) {
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) t += s_sum[q][lane];
    dbias[(int64_t)g * N + c] = Num<OutT>::from_f(t);
  }
}

}  // namespace smoe
