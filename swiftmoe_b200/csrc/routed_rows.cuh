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
#include <type_traits>

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
template <int N> using Int = std::integral_constant<int, N>;

// sort's dot products of a token with its slots' rows (DOT = 8 or MAX_K: the most slots).
// Up to 8 slots keep a partial sum each in registers over the whole row, and the eight sums
// meet in one transposing butterfly (9 shuffles); with more slots every step of the row
// ends in a warp sum per slot, kept by the slot's lane.  unsort, which also holds the sums
// over the slots, has no registers to spare for the first form (it measured 314 us with it
// against 225 for the gradient of 32768 x 8 fp16 rows of 2048).
template <int DOT> struct Dots {
  float s[DOT == 8 ? 8 : 1];
  __device__ __forceinline__ Dots() {
#pragma unroll
    for (int i = 0; i < (DOT == 8 ? 8 : 1); ++i) s[i] = 0.f;
  }
  // v: this lane's part of <x, y_j>; j is a constant after unrolling when DOT == 8
  __device__ __forceinline__ void add(int j, float v) {
    if constexpr (DOT == 8) {
      s[j] += v;
    } else {
      v = warp_sum(v);
      if ((threadIdx.x & 31) == j) s[0] += v;
    }
  }
  // lane j gets the warp's sum of slot j
  __device__ __forceinline__ float total() {
    if constexpr (DOT != 8) return s[0];
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 4; n >= 1; n >>= 1) {  // lanes with bit 4n keep the upper n of 2n sums
      const bool up = lane & (4 * n);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float give = up ? s[i] : s[i + n], keep = up ? s[i + n] : s[i];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * n);
      }
    }
    float v = s[0];
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return __shfl_sync(0xffffffffu, v, (lane & 7) * 4);  // the sum of slot j is in lanes 4j .. 4j+3
  }
};

// dw[t, j] by lane j of the token's first warp, the WPT warps' sums added in warp order.
// Every thread of the block calls this (block barriers inside for WPT > 1).
template <int WPT>
__device__ __forceinline__ void store_dots(float my, bool live, int64_t t, int k, float* __restrict__ dw) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (WPT == 1) {
    if (live && lane < k) dw[t * k + lane] = my;
  } else {
    __shared__ float s_dot[WARPS][32];
    s_dot[warp][lane] = my;
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

// sort (and the gradient of unsort).  WPT warps share a token's columns.  DOT > 0: also
// dw[t, j] = <x_t, y[r(t,j)]>, 0 for slots without a row; rows may then be null: dw alone, the
// same operation in both directions (32768 x 8 fp16 rows of 2048: 182 us, 222 and 348 together
// with unsort's and sort's other output; a form of unsort without its output took 210).
template <typename T, int VEC, int WPT, bool HAS_W, int DOT>
__global__ void __launch_bounds__(THREADS) sort_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ slot_row,
                                                            const float* __restrict__ w, int T_, int k, int d,
                                                            const int32_t* __restrict__ row_token,
                                                            const int32_t* __restrict__ offsets, int E,
                                                            int64_t rows_cap, T* __restrict__ rows,
                                                            const T* __restrict__ y, float* __restrict__ dw) {
  pdl_wait_and_release();
  constexpr int TPB = WARPS / WPT, STEP = 32 * WPT;
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
    const T* xt = x + (live ? t : 0) * d;
    Dots<DOT> dots;
    // U pieces per lane from column piece c0 on; FULL: all of them exist
    auto step = [&](auto u_, auto full_, int c0) {
      constexpr int U = decltype(u_)::value;
      constexpr bool FULL = decltype(full_)::value != 0;
      Piece<T, VEC> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (FULL || c0 + u * STEP < nv) v[u].load(xt + (int64_t)(c0 + u * STEP) * VEC);
      auto slot = [&](int j) {
        const int64_t r = __shfl_sync(0xffffffffu, my_r, j);
        [[maybe_unused]] const float wj = HAS_W ? __shfl_sync(0xffffffffu, my_w, j) : 1.f;
        [[maybe_unused]] Piece<T, VEC> z[U];
        if constexpr (DOT > 0) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (FULL || c0 + u * STEP < nv) z[u].load(y + r * d + (int64_t)(c0 + u * STEP) * VEC);
        }
        [[maybe_unused]] float s = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!FULL && c0 + u * STEP >= nv) continue;
          if (DOT == 0 || rows != nullptr) {
            T* dst = rows + r * d + (int64_t)(c0 + u * STEP) * VEC;
            if constexpr (HAS_W) {
              Piece<T, VEC> o;
#pragma unroll
              for (int i = 0; i < VEC; ++i) o.e[i] = Num<T>::from_f(wj * v[u].f(i));
              o.store(dst);
            } else {
              v[u].store(dst);
            }
          }
          if constexpr (DOT > 0)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s = fmaf(v[u].f(i), z[u].f(i), s);
        }
        if constexpr (DOT > 0) dots.add(j, s);
      };
      if constexpr (DOT == 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (mask >> j & 1u) slot(j);
      } else {
        for (unsigned m = mask; m != 0; m &= m - 1) slot(__ffs(m) - 1);
      }
    };
    if (mask != 0) {
      // a row of 4096 bf16 is 2 x 8 x 32 pieces, or 2 x 8 warps; single elements, more of them
      constexpr int U = (WPT == 1 ? 8 : 2) * (sizeof(T) * VEC < 16 ? 2 : 1);
      int c = part * 32;
      for (; c + (U - 1) * STEP + 32 <= nv; c += U * STEP) step(Int<U>(), Int<1>(), c + lane);
      for (; c < nv; c += STEP) step(Int<1>(), Int<0>(), c + lane);
    }
    if constexpr (DOT > 0) store_dots<WPT>(dots.total(), live, t, k, dw);
  }
  if (DOT > 0 && rows == nullptr) return;
  // rows of no slot become zeros: the rows from the plan's total on, all threads together,
  const int64_t total = min((int64_t)max(offsets[E], 0), rows_cap);
  Piece<T, VEC> z;
  z.zero();
  const int64_t pieces = (rows_cap - total) * nv;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * THREADS)
    z.store(rows + (total * nv + i) * VEC);
  // and (row_token given: a plan with group starts rounded up) the padding rows, which
  // carry token -1: a block looks at 32 rows and clears those it finds, all eight warps
  if (row_token != nullptr)
    for (int64_t r0 = (int64_t)blockIdx.x * 32; r0 < total; r0 += (int64_t)gridDim.x * 32) {
      const bool empty = r0 + lane < total && row_token[r0 + lane] < 0;
      for (unsigned m = __ballot_sync(0xffffffffu, empty); m != 0; m &= m - 1) {
        T* dst = rows + (r0 + __ffs(m) - 1) * d;
        for (int c = threadIdx.x; c < nv; c += THREADS) z.store(dst + (int64_t)c * VEC);
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
  constexpr int BYTES = sizeof(T) * VEC;
  constexpr int U = (DOT && WPT == 1 ? 4 : 2) * (BYTES == 16 ? 1 : BYTES == 8 ? 2 : 4), TPB = WARPS / WPT;
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
      Piece<T, VEC> xv[U], rv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * 32 * WPT;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[u][i] = 0.f;
        if constexpr (DOT) {
          if (c < nv) xv[u].load(x + t * d + (int64_t)c * VEC);
          else xv[u].zero();
        }
        // on its way with the first rows (DOT has no registers to spare for it)
        if (!DOT && residual != nullptr && c < nv) rv[u].load(residual + t * d + (int64_t)c * VEC);
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
          if (DOT) rv[u].load(residual + t * d + (int64_t)c * VEC);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[u][i] = __fadd_rn(acc[u][i], rv[u].f(i));
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
