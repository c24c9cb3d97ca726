// Tokens to expert-ordered rows and back, with the gate weights, and their gradients.
//
// With r(t, j) the row of slot j of token t (the dispatch plan's slot_row, -1: no row):
//   sort    rows[r(t,j)] = w_tj x_t                      (rows of no slot: zeros)
//   unsort  out_t = sum_j w_tj rows[r(t,j)] + residual_t
// Each is the other's adjoint, so two kernels serve both directions:
//   sort's gradient:    dx_t = sum_j w_tj drows[r(t,j)],   dw_tj = <x_t, drows[r(t,j)]>
//   unsort's gradient:  drows[r(t,j)] = w_tj dout_t,       dw_tj = <dout_t, rows[r(t,j)]>
// Both walk the tokens: a token's row is read once whatever k is, its k rows are read or
// written once, and the dot products of the weights' gradients use the pieces that are in
// registers anyway.  There is no scatter of sums: every output element has one writer,
// and sums run over j (and over a row's columns) in a fixed order.  All arithmetic is in
// fp32, rounded once to T; each product w * y is rounded before it is added, as in
// combine_kernel, so that the weighted sums agree with it bit for bit.
#pragma once
#include "common.cuh"

namespace smoe {
namespace rows {

// VEC consecutive elements of a row, loaded and stored as one word.
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <typename T, int VEC> struct Piece {
  using W = typename Word<sizeof(T) * VEC>::type;
  union {
    W w;
    T e[VEC];
  };
  __device__ Piece() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = Num<T>::from_f(0.f);
  }
  __device__ __forceinline__ float f(int i) const { return Num<T>::to_f(e[i]); }
};

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_K = 32;  // slots of a token: one lane each

// Sums of the WPT warps of a token, added in warp order; dw[t, j] is written by lane j of
// the token's first warp.  Every thread of the block calls this (block barriers inside).
template <int WPT>
__device__ __forceinline__ void store_dots(float my_dot, bool live, int64_t t, int k, float* __restrict__ dw) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (WPT == 1) {
    if (live && lane < k) dw[t * k + lane] = my_dot;
  } else {
    __shared__ float s_dot[WARPS][32];
    s_dot[warp][lane] = my_dot;
    __syncthreads();
    if (live && warp % WPT == 0 && lane < k) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < WPT; ++q) s += s_dot[warp + q][lane];
      dw[t * k + lane] = s;
    }
    __syncthreads();
  }
}

// sort (and the gradient of unsort).  WPT warps share a token's columns.  DOT: also
// dw[t, j] = <x_t, y[r(t,j)]>, 0 for slots without a row.
template <typename T, int VEC, int WPT, bool HAS_W, bool DOT>
__global__ void __launch_bounds__(THREADS) sort_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ slot_row,
                                                            const float* __restrict__ w, int T_, int k, int d,
                                                            const int32_t* __restrict__ row_token,
                                                            const int32_t* __restrict__ offsets, int E,
                                                            int64_t rows_cap, T* __restrict__ rows,
                                                            const T* __restrict__ y, float* __restrict__ dw) {
  pdl_wait_and_release();
  constexpr int U = 4, TPB = WARPS / WPT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % WPT;
  const int nv = d / VEC;
  for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < T_; t0 += (int64_t)gridDim.x * TPB) {
    const int64_t t = t0 + warp / WPT;
    const bool live = t < T_;
    int my_r = live && lane < k ? slot_row[t * k + lane] : -1;
    if (my_r >= rows_cap) my_r = -1;
    const float my_w = HAS_W && live && lane < k ? w[t * k + lane] : 1.f;
    const unsigned mask = __ballot_sync(0xffffffffu, my_r >= 0);
    float my_dot = 0.f;
    const T* xt = x + (live ? t : 0) * d;
    if (mask != 0) {
      for (int c0 = part * 32 + lane; c0 - lane < nv; c0 += 32 * WPT * U) {
        Piece<T, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * 32 * WPT;
          if (c < nv) v[u].load(xt + (int64_t)c * VEC);
          else v[u].zero();
        }
        for (unsigned m = mask; m != 0; m &= m - 1) {
          const int j = __ffs(m) - 1;
          const int64_t r = __shfl_sync(0xffffffffu, my_r, j);
          const float wj = HAS_W ? __shfl_sync(0xffffffffu, my_w, j) : 1.f;
          Piece<T, VEC> z[U];
          if constexpr (DOT) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = c0 + u * 32 * WPT;
              if (c < nv) z[u].load(y + r * d + (int64_t)c * VEC);
              else z[u].zero();
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 32 * WPT;
            if (c >= nv) continue;
            T* dst = rows + r * d + (int64_t)c * VEC;
            if constexpr (HAS_W) {
              Piece<T, VEC> o;
#pragma unroll
              for (int i = 0; i < VEC; ++i) o.e[i] = Num<T>::from_f(wj * v[u].f(i));
              o.store(dst);
            } else {
              v[u].store(dst);
            }
          }
          if constexpr (DOT) {
            float s = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (c0 + u * 32 * WPT < nv)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s = fmaf(v[u].f(i), z[u].f(i), s);
            s = warp_sum(s);
            if (lane == j) my_dot += s;
          }
        }
      }
    }
    if constexpr (DOT) store_dots<WPT>(my_dot, live, t, k, dw);
  }
  // rows of no slot: from the plan's total on, and (row_token given: a plan with group
  // starts rounded up) the padding rows, which carry token -1
  const int64_t total = min((int64_t)max(offsets[E], 0), rows_cap);
  const int64_t nw = (int64_t)gridDim.x * WARPS;
  const int64_t first = row_token != nullptr ? 0 : total / 32 * 32;
  for (int64_t r0 = first + ((int64_t)blockIdx.x * WARPS + warp) * 32; r0 < rows_cap; r0 += nw * 32) {
    const int64_t mine = r0 + lane;
    bool empty = mine >= total && mine < rows_cap;
    if (row_token != nullptr && mine < total) empty = row_token[mine] < 0;
    for (unsigned m = __ballot_sync(0xffffffffu, empty); m != 0; m &= m - 1) {
      T* dst = rows + (r0 + __ffs(m) - 1) * d;
      Piece<T, VEC> z;
      z.zero();
      for (int c = lane; c < nv; c += 32) z.store(dst + (int64_t)c * VEC);
    }
  }
}

// unsort (and the gradient of sort).  DOT: also dw[t, j] = <x_t, y[r(t,j)]>.
template <typename T, int VEC, int WPT, bool HAS_W, bool DOT>
__global__ void __launch_bounds__(THREADS) unsort_rows_kernel(const T* __restrict__ y, const int32_t* __restrict__ slot_row,
                                                              const float* __restrict__ w, int T_, int k, int d,
                                                              int64_t rows_cap, const T* __restrict__ residual,
                                                              T* __restrict__ out, const T* __restrict__ x,
                                                              float* __restrict__ dw) {
  pdl_wait_and_release();
  constexpr int U = 4, TPB = WARPS / WPT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % WPT;
  const int nv = d / VEC;
  for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < T_; t0 += (int64_t)gridDim.x * TPB) {
    const int64_t t = t0 + warp / WPT;
    const bool live = t < T_;
    int my_r = live && lane < k ? slot_row[t * k + lane] : -1;
    if (my_r >= rows_cap) my_r = -1;
    const float my_w = HAS_W && live && lane < k ? w[t * k + lane] : 1.f;
    const unsigned mask = __ballot_sync(0xffffffffu, my_r >= 0);
    float my_dot = 0.f;
    for (int c0 = part * 32 + lane; live && c0 - lane < nv; c0 += 32 * WPT * U) {
      float acc[U][VEC];
      Piece<T, VEC> xv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * 32 * WPT;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[u][i] = 0.f;
        if constexpr (DOT) {
          if (c < nv) xv[u].load(x + t * d + (int64_t)c * VEC);
          else xv[u].zero();
        }
      }
      for (unsigned m = mask; m != 0;) {  // two slots at a time: 2 U loads in flight
        const int j0 = __ffs(m) - 1;
        m &= m - 1;
        const int j1 = m != 0 ? __ffs(m) - 1 : -1;
        m &= m - 1;
        const int64_t r0 = __shfl_sync(0xffffffffu, my_r, j0);
        const int64_t r1 = j1 >= 0 ? __shfl_sync(0xffffffffu, my_r, j1) : -1;
        const float w0 = HAS_W ? __shfl_sync(0xffffffffu, my_w, j0) : 1.f;
        const float w1 = HAS_W && j1 >= 0 ? __shfl_sync(0xffffffffu, my_w, j1) : 1.f;
        Piece<T, VEC> v0[U], v1[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * 32 * WPT;
          if (c < nv) v0[u].load(y + r0 * d + (int64_t)c * VEC);
          else v0[u].zero();
          if (j1 >= 0 && c < nv) v1[u].load(y + r1 * d + (int64_t)c * VEC);
          else v1[u].zero();
        }
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float f = v0[u].f(i);
            acc[u][i] = __fadd_rn(acc[u][i], HAS_W ? __fmul_rn(w0, f) : f);
            if constexpr (DOT) s0 = fmaf(xv[u].f(i), f, s0);
          }
        if (j1 >= 0)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float f = v1[u].f(i);
              acc[u][i] = __fadd_rn(acc[u][i], HAS_W ? __fmul_rn(w1, f) : f);
              if constexpr (DOT) s1 = fmaf(xv[u].f(i), f, s1);
            }
        if constexpr (DOT) {
          s0 = warp_sum(s0);
          if (lane == j0) my_dot += s0;
          if (j1 >= 0) {
            s1 = warp_sum(s1);
            if (lane == j1) my_dot += s1;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * 32 * WPT;
        if (c >= nv) continue;
        if (residual != nullptr) {
          Piece<T, VEC> rv;
          rv.load(residual + t * d + (int64_t)c * VEC);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[u][i] = __fadd_rn(acc[u][i], rv.f(i));
        }
        Piece<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.e[i] = Num<T>::from_f(acc[u][i]);
        o.store(out + t * d + (int64_t)c * VEC);
      }
    }
    if constexpr (DOT) store_dots<WPT>(my_dot, live, t, k, dw);
  }
}

}  // namespace rows
}  // namespace smoe
