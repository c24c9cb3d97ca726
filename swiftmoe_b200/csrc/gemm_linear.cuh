// Grouped linear layers on the sm_100a tensor cores: the products of the forward and of the
// input gradient (linear_gemm_kernel) and the weight gradient (linear_wgrad_kernel).
//
// The pipeline is grouped_gemm_kernel's -- TMA into a 4-stage ring of 48 KB, one thread
// issuing tcgen05.mma (128 x 256 x 16) into one of two TMEM accumulators, epilogue warps
// draining the other, every wait bounded -- with what these layers need besides:
//   * bias, activation, residual and pre-activations in the epilogue, by eight warps (two per
//     TMEM lane quarter, each 128 of the 256 columns).  A tile's epilogue takes them 4.3 us
//     without an activation, 6.3 with SiLU, 7.3 with the exact GELU (16384 x 14336 outputs, K = 64),
//     and 7.3 us are the products of a tile for K = 1700: four warps would take twice as long;
//   * weights in either layout: [N, K] K-major, or [K, N] as an MN-major operand (the input
//     gradient reads the weights as they are, no transposed copy);
//   * two producer warps, which share the four to six boxes of an MN-major stage (a stage's
//     MMAs take 512 cycles).  Input gradient of 16384 x 14336 x 4096: 1.38 to 1.42 ms; with one
//     warp 1.39 to 1.50, so what it gains is the slow end; 1.70 with one that also leaves out
//     boxes past N;
//   * launches of few tiles cut along K, the partial tiles summed by a second launch over the
//     whole GPU (split_units below);
//   * weight-gradient groups that start at any row, 16-bit gradients.
#pragma once
#include "activation.cuh"
#include "common.cuh"
#include "gemm_tc.cuh"
#include "gemv.cuh"

namespace smoe {
namespace lin {

using tc::A_BYTES;
using tc::B_BYTES;
using tc::BK;
using tc::BM;
using tc::BN;
using tc::kMnBox;
using tc::MAX_GROUPS;
using tc::STAGES;

constexpr int EPI_WARPS = 8;
constexpr int EPI_WARP0 = 2;                       // warps 2 .. 9: epilogue
constexpr int WARP_B = EPI_WARP0 + EPI_WARPS;      // warp 0: first producer, 1: MMA, 10: second
constexpr int THREADS = 32 * (WARP_B + 1);
constexpr int EPI_THREADS = 32 * EPI_WARPS;
constexpr int STAGE_OUT = 16 * 128;                // output stage of an epilogue warp: 16 rows x 128 bytes
constexpr int NUM_BARS = 2 * STAGES + 5;
constexpr int SMEM_BYTES = 1024 + STAGES * (A_BYTES + B_BYTES) + NUM_BARS * 8 + 16 + 3 * (MAX_GROUPS + 1) * 4 + 16 +
                           EPI_WARPS * STAGE_OUT;
constexpr int MAX_SPLIT = 16;

// The shared memory of both kernels: the ring, barriers, a few words, three int tables of
// the groups and the epilogue warps' output stages.
struct Smem {
  unsigned char *a, *b, *out;
  uint64_t* bars;
  uint32_t* tmem;
  volatile int *abort, *word;
  int *t0, *t1, *t2;
  __device__ __forceinline__ explicit Smem(unsigned char* raw) {
    a = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    b = a + STAGES * A_BYTES;
    bars = reinterpret_cast<uint64_t*>(b + STAGES * B_BYTES);
    tmem = reinterpret_cast<uint32_t*>(bars + NUM_BARS);
    abort = reinterpret_cast<volatile int*>(tmem + 1);  // set when a wait gives up
    word = reinterpret_cast<volatile int*>(tmem + 2);
    t0 = reinterpret_cast<int*>(tmem + 4);
    t1 = t0 + (MAX_GROUPS + 1);
    t2 = t1 + (MAX_GROUPS + 1);
    out = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(t2 + MAX_GROUPS + 1) + 15) & ~uintptr_t(15));
  }
  __device__ __forceinline__ uint32_t full(int s) const { return smem_u32(bars + s); }
  __device__ __forceinline__ uint32_t empty(int s) const { return smem_u32(bars + STAGES + s); }
  __device__ __forceinline__ uint32_t tfull(int i) const { return smem_u32(bars + 2 * STAGES + i); }
  __device__ __forceinline__ uint32_t tempty(int i) const { return smem_u32(bars + 2 * STAGES + 2 + i); }
  __device__ __forceinline__ uint32_t mma_done() const { return smem_u32(bars + 2 * STAGES + 4); }
  __device__ __forceinline__ void init(const CUtensorMap& ma, const CUtensorMap& mb) const {  // one thread
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 2);  // one arrive per producer
      mbar_init(empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull(i), 1);
      mbar_init(tempty(i), EPI_WARPS);
    }
    mbar_init(mma_done(), 1);
    fence_mbar_init();
    tma_prefetch_desc(&ma);
    tma_prefetch_desc(&mb);
  }
};

// Position in the ring (producers, MMA) or in the pair of accumulators.
template <int N> struct Cursor {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1;
    }
  }
};

// The producers' way out: the last armed phase of every stage has landed.
__device__ __forceinline__ void drain_loads(const Smem& sm, int64_t issued) {
  for (int s = 0; s < STAGES; ++s) {
    const int64_t n = issued / STAGES + (s < issued % STAGES ? 1 : 0);
    if (n > 0) tc::mbar_wait_drain(sm.full(s), (uint32_t)((n - 1) & 1));
  }
}

// The instruction descriptor with N cut to the columns that exist, in steps of 16.
__device__ __forceinline__ uint32_t idesc_cols(uint32_t idesc, int cols) {
  return cols >= BN ? idesc : (idesc & ~(63u << 17)) | ((uint32_t)((cols + 15) / 16 * 2) << 17);
}

// Eight 16-byte pieces per lane -- 128 bytes of the lane's row of a warp's 32 accumulator
// rows -- to global memory by way of the warp's 2 KB stage, 16 rows at a time, so that a
// warp store writes whole 128-byte lines of four rows instead of 16 bytes of 32 (the
// load/store unit takes one step per row; a weight gradient of 0.94 GB from one row per
// group: 214 us with 64-byte pieces of eight rows, 171 with these).  The pieces are XOR-swizzled by row: conflict-free both
// ways.  Row rr goes to p + rr * pitch bytes; rows from nrows on and bytes from `width` on
// are left out.
__device__ __forceinline__ void store_rows128(const uint4 (&u)[8], unsigned char* p, int64_t pitch, int nrows,
                                              int width, unsigned char* stage, int lane) {
  const int j = lane & 7;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (lane >> 4 == h)
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(stage + (lane & 15) * 128 + ((i ^ j) << 4)) = u[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = i * 4 + (lane >> 3);
      const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((j ^ (rr & 7)) << 4));
      if (h * 16 + rr < nrows && j * 16 < width)
        *reinterpret_cast<uint4*>(p + (h * 16 + rr) * pitch + j * 16) = v;
    }
    __syncwarp();
  }
}
// Half of it at once: four pieces, 64 bytes of all 32 rows (the products' epilogue, which has
// no registers for 64 columns and a residual).
__device__ __forceinline__ void store_rows64(const uint4 (&u)[4], unsigned char* p, int64_t pitch, int nrows, int width,
                                             unsigned char* stage, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) = u[j];
  __syncwarp();
  const int j = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 8 + (lane >> 2);
    const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 64 + ((j ^ (rr >> 1 & 3)) << 4));
    if (rr < nrows && j * 16 < width) *reinterpret_cast<uint4*>(p + rr * pitch + j * 16) = v;
  }
  __syncwarp();
}
// The same way in: v[i] holds 16 bytes of row i * 8 + lane / 4, u gets the lane's own row.
__device__ __forceinline__ void take_rows64(const uint4 (&v)[4], uint4 (&u)[4], unsigned char* stage, int lane) {
  const int j = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 8 + (lane >> 2);
    *reinterpret_cast<uint4*>(stage + rr * 64 + ((j ^ (rr >> 1 & 3)) << 4)) = v[i];
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) u[q] = *reinterpret_cast<const uint4*>(stage + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4));
  __syncwarp();
}

template <typename T, int W> __device__ __forceinline__ void pack_cols(const float (&f)[W], uint4 (&u)[W / 8]) {
#pragma unroll
  for (int j = 0; j < W / 8; ++j)
    u[j] = make_uint4(pack2<T>(f[8 * j], f[8 * j + 1]), pack2<T>(f[8 * j + 2], f[8 * j + 3]),
                      pack2<T>(f[8 * j + 4], f[8 * j + 5]), pack2<T>(f[8 * j + 6], f[8 * j + 7]));
}

// 64 accumulator columns of the lane's row.
__device__ __forceinline__ void load_acc64(uint32_t taddr, uint32_t (&v)[64]) {
  tmem_ld32(taddr, reinterpret_cast<uint32_t(&)[32]>(v[0]));
  tmem_ld32(taddr + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
}

// This warp's 32 accumulator rows (first row `row`, nrows valid), columns col0 .. col0 + 127
// below N: plus bias, pre-activation out, activation, plus residual, out.  Bias (the same
// pieces for every lane) and residual are requested before the accumulator is read.  The
// output is rounded once, from fp32; the pre-activation is kept for the gradient in 16 bits
// (fp32 would double its 0.47 GB out and back in for 16384 x 14336), which puts an error of
// half a step of z into the argument of act'.
template <typename T>
__device__ __forceinline__ void epilogue_tile(uint32_t tbase, int g, int row, int nrows, int col0, int N,
                                              T* __restrict__ C, const LinearEpi& lin, unsigned char* stage, int lane) {
  if (nrows <= 0) return;
  const int64_t pitch = (int64_t)N * sizeof(T);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const int col = col0 + c * 32;
    if (col >= N) break;  // warp-uniform
    const int width = (N - col) * (int)sizeof(T);
    const int64_t at = (int64_t)row * N + col;
    uint32_t v[32];
    tmem_ld32(tbase + c * 32, v);
    uint4 res[4];
    if (lin.residual != nullptr) {
      const unsigned char* src = reinterpret_cast<const unsigned char*>(static_cast<const T*>(lin.residual) + at);
      const int j = lane & 3;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = i * 8 + (lane >> 2);
        res[i] = rr < nrows && j * 16 < width ? *reinterpret_cast<const uint4*>(src + rr * pitch + j * 16)
                                             : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    uint4 bias[4];
    const bool bias16 = lin.bias != nullptr && !lin.bias_f32;
    if (bias16)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        bias[j] = col + 8 * j < N
                      ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(lin.bias) + (int64_t)g * N + col) + j)
                      : make_uint4(0u, 0u, 0u, 0u);
    tmem_ld_wait();
    float f[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
    if (bias16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T* e = reinterpret_cast<const T*>(&bias[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[8 * j + i] += Num<T>::to_f(e[i]);
      }
    } else if (lin.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + 8 * j < N) add_bias<T>(lin, (int64_t)g * N + col + 8 * j, reinterpret_cast<float(&)[8]>(f[8 * j]));
    }
    uint4 u[4];
    if (lin.preact != nullptr) {
      pack_cols<T, 32>(f, u);
      store_rows64(u, reinterpret_cast<unsigned char*>(static_cast<T*>(lin.preact) + at), pitch, nrows, width, stage, lane);
    }
    apply_act(lin.act, f);
    if (lin.residual != nullptr) {
      take_rows64(res, u, stage, lane);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const T* e = reinterpret_cast<const T*>(&u[q]);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[8 * q + i] += Num<T>::to_f(e[i]);
      }
    }
    pack_cols<T, 32>(f, u);
    store_rows64(u, reinterpret_cast<unsigned char*>(C + at), pitch, nrows, width, stage, lane);
  }
}

// lin.fill: the rows of no group, [0, first) and [last, rows_cap), become the residual
// (zeros without one).  Thread et of nt of block b of nb.
template <typename T>
__device__ __forceinline__ void fill_other_rows(const LinearEpi& lin, T* __restrict__ C, int first, int last,
                                                int rows_cap, int N, int b, int nb, int et, int nt) {
  const int64_t pieces = (int64_t)N / 8, head = (int64_t)first * pieces;
  const int64_t total = head + (int64_t)(rows_cap - last) * pieces;
  for (int64_t i = (int64_t)b * nt + et; i < total; i += (int64_t)nb * nt) {
    const int64_t p = i < head ? i : (int64_t)last * pieces + (i - head);
    reinterpret_cast<uint4*>(C)[p] =
        lin.residual != nullptr ? static_cast<const uint4*>(lin.residual)[p] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// ------------------------------------------------------------------------ split along K
// A launch of few tiles leaves SMs idle, or its last wave nearly empty.  Every tile's K range
// is then cut into ks slices, one work unit each, that store fp32 partial tiles; a second
// launch adds a tile's slices in order (so no result depends on which unit ends first) and
// applies the epilogue, spread over the whole GPU.  (With the last unit of a tile adding
// them up itself, its one CTA took longer than the products: 35 us for 64 rows against
// 4096 x 4096 weights, now 18; the bytes take 5.)  ks is the cheapest by a count of k-blocks per
// CTA: whole waves of units, each with its share of the K blocks, about 3 blocks' time to
// fill the ring and drain the tile, and for its partial tile's way out and back 8 blocks'
// time per 128 rows; the second launch counts 16.  Both launches compute it from the same
// numbers.  rows: rows of a slot.
// (32-bit divisions: one thread of every block works this out before the block can start.)
__host__ __device__ inline int split_units(uint32_t tiles, uint32_t kb, uint32_t rows, uint32_t ctas, uint32_t slots) {
  int best = 1;
  uint64_t best_cost = ~0ull;
  for (uint32_t ks = 1; ks <= MAX_SPLIT; ++ks) {
    if (ks > 1 && (tiles > slots / ks || kb < 4 * ks)) break;
    const uint32_t waves = (tiles * ks + ctas - 1) / ctas, blocks = (kb + ks - 1) / ks + 3;
    const uint64_t cost = (uint64_t)waves * (blocks * 16 + (ks > 1 ? rows : 0)) + (ks > 1 ? 16 * 16 : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = (int)ks;
    }
  }
  return best;
}

// 32 fp32 columns of a lane's row into a slot, piece-major: the 4-column piece p of row r is
// at float (p * rows + r) * 4, so the lanes of a warp store 512 contiguous bytes.
__device__ __forceinline__ void store_partial(uint32_t taddr, float* slot, int rows, int p0, int r, bool row_ok) {
  uint32_t v[32];
  tmem_ld32(taddr, v);
  tmem_ld_wait();
  if (row_ok)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4*>(slot + ((int64_t)(p0 + j) * rows + r) * 4) =
          make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}

// Columns 8 * p8 .. + 7 of row r: the sum of slots first .. first + n - 1, in order.
__device__ __forceinline__ void sum_partials(const float* ws, int64_t first, int n, int rows, int p8, int r,
                                             float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  const float* p = ws + first * rows * BN + ((int64_t)2 * p8 * rows + r) * 4;
#pragma unroll 8
  for (int q = 0; q < n; ++q, p += (int64_t)rows * BN) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldcg(reinterpret_cast<const float4*>(p + rows * 4));
    f[0] += a.x;
    f[1] += a.y;
    f[2] += a.z;
    f[3] += a.w;
    f[4] += b.x;
    f[5] += b.y;
    f[6] += b.z;
    f[7] += b.w;
  }
}

// ------------------------------------------------------------------------ products
// C = act(A W_g^T + bias[g]) + residual for the rows of group g; BMN: W [G, K, N], C = A W_g.
// ws: `slots` partial tiles of slot_rows x BN fp32, or null for no split.
template <typename T, bool BMN>
__global__ void __launch_bounds__(THREADS, 1)
    linear_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       T* __restrict__ C, const int32_t* __restrict__ offsets, int G, int N, int K, int rows_cap, int gm,
                       uint32_t idesc, const LinearEpi lin, float* __restrict__ ws, int slots, int slot_rows) {
  pdl_wait();
  extern __shared__ unsigned char smem_raw[];
  const Smem sm(smem_raw);
  int *s_beg = sm.t0, *s_fin = sm.t1, *s_ts = sm.t2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int NB = (N + BN - 1) / BN, KB = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    *sm.abort = 0;
    sm.init(tmA, tmB);
  }
  tc::load_group_table<BM>(offsets, nullptr, G, rows_cap, NB, s_beg, s_fin, s_ts);
  if (warp == 1) tmem_alloc(smem_u32(sm.tmem), 2 * BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) {
    tc::scan_group_table(G, s_ts);
    if (lane == 0) *sm.word = ws != nullptr ? split_units(s_ts[G], KB, slot_rows, gridDim.x, slots) : 1;
  }
  __syncthreads();
  const uint32_t tmem_base = *sm.tmem;
  const int ks_n = *sm.word, total = s_ts[G] * ks_n;
  auto tile_of = [&](int L) { return tc::decode_tile_t<BM>(L / ks_n, s_ts, s_beg, s_fin, G, NB, gm); };

  if (warp == 0 || warp == WARP_B) {
    if (lane == 0) {
      // ------------------------------------------------------------- TMA producers
      // warp 0 the A tile (and the first of four B boxes), the other the rest of B; boxes
      // of B whose columns all lie past N are not loaded
      constexpr int boxes = BMN ? 4 : 2, box_cols = BN / boxes, box_bytes = B_BYTES / boxes, own = BMN ? 1 : 0;
      Cursor<STAGES> st;
      int64_t issued = 0;
      bool ok = true;
      for (int L = blockIdx.x; L < total && ok; L += gridDim.x) {
        const tc::TileCoord t = tile_of(L);
        const int ks = L % ks_n, n0 = t.nb * BN;
        const int live = min(boxes, (N - n0 + box_cols - 1) / box_cols);
        for (int kb = ks * KB / ks_n; kb < (ks + 1) * KB / ks_n; ++kb) {
          if (!mbar_wait(sm.empty(st.i), st.phase ^ 1, sm.abort)) { ok = false; break; }
          const uint32_t fb = sm.full(st.i);
          const uint32_t b_dst = smem_u32(sm.b + st.i * B_BYTES);
          auto b_box = [&](int i) {
            if constexpr (BMN) tma_load_3d(b_dst + i * box_bytes, &tmB, fb, n0 + box_cols * i, kb * BK, t.g);
            else tma_load_3d(b_dst + i * box_bytes, &tmB, fb, kb * BK, n0 + box_cols * i, t.g);
          };
          if (warp == 0) {
            mbar_arrive_expect_tx(fb, A_BYTES + own * box_bytes);
            tma_load_2d(smem_u32(sm.a + st.i * A_BYTES), &tmA, fb, kb * BK, t.row0);
            if constexpr (own > 0) b_box(0);
          } else {
            mbar_arrive_expect_tx(fb, (live - own) * box_bytes);
            if (live == boxes) {
#pragma unroll
              for (int i = own; i < boxes; ++i) b_box(i);
            } else {
              for (int i = own; i < live; ++i) b_box(i);
            }
          }
          ++issued;
          st.next();
        }
      }
      drain_loads(sm, issued);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------------------- MMA issuer
      const uint64_t a0 = umma_desc_sw128(smem_u32(sm.a));
      const uint64_t b0 = BMN ? umma_desc_mn_sw128(smem_u32(sm.b), kMnBox, 1024) : umma_desc_sw128(smem_u32(sm.b));
      constexpr int b_step = BMN ? 2048 >> 4 : 2;  // a K step of 16: two 1 KB atoms, or 32 bytes of a row
      Cursor<STAGES> st;
      Cursor<2> acc;
      bool ok = true;
      for (int L = blockIdx.x; L < total && ok; L += gridDim.x) {
        const int ks = L % ks_n;
        const uint32_t id = idesc_cols(idesc, N - tile_of(L).nb * BN);
        if (!mbar_wait(sm.tempty(acc.i), acc.phase ^ 1, sm.abort)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc.i * BN);
        const int kb0 = ks * KB / ks_n, kb1 = (ks + 1) * KB / ks_n;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(sm.full(st.i), st.phase, sm.abort)) { ok = false; break; }
          tc_fence_after();
          const uint64_t a = a0 + (uint64_t)(st.i * (A_BYTES >> 4)), b = b0 + (uint64_t)(st.i * (B_BYTES >> 4));
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_f16(d, a + 2 * kk, b + b_step * kk, id, (kb != kb0 || kk != 0) ? 1u : 0u);
          umma_commit(sm.empty(st.i));
          st.next();
        }
        if (!ok) break;
        umma_commit(sm.tfull(acc.i));
        acc.next();
      }
      umma_commit(sm.mma_done());
      tc::mbar_wait_drain(sm.mma_done(), 0);
    }
  } else {
    // --------------------------------------------------------------- epilogue
    const int q = warp & 3;                      // TMEM lane quarter this warp may access
    const int half = (warp - EPI_WARP0) >> 2;    // columns 128 * half .. + 127 of the tile
    unsigned char* stage = sm.out + (warp - EPI_WARP0) * STAGE_OUT;
    if (lin.fill)  // while the first tile is computed
      fill_other_rows<T>(lin, C, s_beg[0], s_fin[G - 1], rows_cap, N, blockIdx.x, gridDim.x,
                         (int)threadIdx.x - 32 * EPI_WARP0, EPI_THREADS);
    Cursor<2> acc;
    for (int L = blockIdx.x; L < total; L += gridDim.x) {
      const tc::TileCoord t = tile_of(L);
      const int nrows = t.rows_valid - q * 32, col0 = t.nb * BN + half * 128;
      if (!mbar_wait(sm.tfull(acc.i), acc.phase, sm.abort)) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc.i * BN + half * 128);
      if (ks_n == 1) {
        epilogue_tile<T>(tbase, t.g, t.row0 + q * 32, nrows, col0, N, C, lin, stage, lane);
      } else if (nrows > 0) {
        float* slot = ws + (int64_t)L * slot_rows * BN;
#pragma unroll 1
        for (int c = 0; c < 4 && col0 + c * 32 < N; ++c)
          store_partial(tbase + c * 32, slot, slot_rows, half * 32 + c * 8, q * 32 + lane, lane < nrows);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.tempty(acc.i));
      acc.next();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// The second launch of a split product: every (tile, row, 8 columns) once.  ctas: the first
// launch's grid.  Nothing to do where the groups' tiles made no split worth it.
template <typename T>
__global__ void __launch_bounds__(256) linear_sum_kernel(T* __restrict__ C, const int32_t* __restrict__ offsets, int G,
                                                         int N, int K, int rows_cap, int gm, const LinearEpi lin,
                                                         const float* __restrict__ ws, int slots, int slot_rows,
                                                         int ctas) {
  pdl_wait_and_release();
  __shared__ int s_beg[MAX_GROUPS + 1], s_fin[MAX_GROUPS + 1], s_ts[MAX_GROUPS + 1], s_ks;
  const int NB = (N + BN - 1) / BN, KB = (K + BK - 1) / BK;
  tc::load_group_table<BM>(offsets, nullptr, G, rows_cap, NB, s_beg, s_fin, s_ts);
  __syncthreads();
  if (threadIdx.x < 32) {
    tc::scan_group_table(G, s_ts);
    if (threadIdx.x == 0) s_ks = split_units(s_ts[G], KB, slot_rows, ctas, slots);
  }
  __syncthreads();
  const int tiles = s_ts[G], ks_n = s_ks;
  if (ks_n == 1) return;
  const int per = slot_rows * (BN / 8);  // (8 columns, row) pairs of a tile, rows fastest
  const int64_t total = (int64_t)tiles * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int tile = (int)(i / per), rem = (int)(i - (int64_t)tile * per);
    const int p8 = rem / slot_rows, r = rem - p8 * slot_rows;
    const tc::TileCoord t = tc::decode_tile_t<BM>(tile, s_ts, s_beg, s_fin, G, NB, gm);
    const int col = t.nb * BN + p8 * 8;
    if (r >= t.rows_valid || col >= N) continue;
    float f[8];
    sum_partials(ws, (int64_t)tile * ks_n, ks_n, slot_rows, p8, r, f);
    add_bias<T>(lin, (int64_t)t.g * N + col, f);
    const int64_t at = (int64_t)(t.row0 + r) * N + col;
    auto out = [&](T* p) {
      *reinterpret_cast<uint4*>(p + at) =
          make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    };
    if (lin.preact != nullptr) out(static_cast<T*>(lin.preact));
    apply_act(lin.act, f);
    if (lin.residual != nullptr) {
      float v[8];
      load_vec_f<T, 8>(static_cast<const T*>(lin.residual) + at, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += v[j];
    }
    out(C);
  }
}

// ------------------------------------------------------------------------ one or two rows
// A decode step of one token: at most two rows in at most two groups, bound by reading those
// groups' weights once.  A warp owns an output column: its lanes read the weight row in
// 16-byte pieces, eight in flight each, multiply them with the rows (from shared memory) and
// add up across the warp.  The pieces of the next step -- of the same column or the warp's
// next one -- are requested before the current ones are used, so a column's reduction does
// not leave the memory idle (one token's two of eight experts, 14336 x 4096: 50.4 us without,
// 38 to 41 with it; the 235 MB take 36.  Both rows in one expert: 35, where its 117 MB take
// 18 -- two multiplications per weight from shared memory set the time).  The choice is by
// rows_cap, which the host knows; how many of a larger buffer's rows are in groups, it does not.
constexpr int GEMV_ROWS = 2, GEMV_U = 8, GEMV_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(GEMV_THREADS, 2)
    linear_gemv_kernel(const T* __restrict__ A, const T* __restrict__ W, T* __restrict__ C,
                       const int32_t* __restrict__ offsets, int G, int N, int K, int rows_cap, const LinearEpi lin) {
  pdl_wait_and_release();
  extern __shared__ unsigned char smem_raw[];
  uint4* s_a = reinterpret_cast<uint4*>(smem_raw);  // [rows_cap][K / 8]
  __shared__ int s_group[GEMV_ROWS], s_first, s_last;
  const int lane = threadIdx.x & 31;
  const int chunks = K / 8;
  if (threadIdx.x < GEMV_ROWS) s_group[threadIdx.x] = -1;
  if (threadIdx.x == 0) {
    s_first = min(max(offsets[0], 0), rows_cap);
    s_last = min(max(offsets[G], s_first), rows_cap);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < G; g += GEMV_THREADS) {
    const int b = max(offsets[g], 0), e = min(offsets[g + 1], rows_cap);
    for (int r = b; r < e; ++r) s_group[r] = g;  // at most two rows
  }
  for (int i = threadIdx.x; i < rows_cap * chunks; i += GEMV_THREADS)
    s_a[i] = __ldg(reinterpret_cast<const uint4*>(A) + i);
  __syncthreads();
  if (lin.fill)  // rows of no group: the residual, or zeros
    for (int r = 0; r < rows_cap; ++r)
      if (r < s_first || r >= s_last)
        for (int n = blockIdx.x * GEMV_THREADS + threadIdx.x; n < N; n += gridDim.x * GEMV_THREADS)
          C[(int64_t)r * N + n] = lin.residual != nullptr ? static_cast<const T*>(lin.residual)[(int64_t)r * N + n]
                                                          : Num<T>::from_f(0.f);
  // the groups with rows: both rows in one, one each, or fewer
  const int g0 = s_group[0], g1 = rows_cap > 1 ? s_group[1] : -1;
  int group[GEMV_ROWS], row[GEMV_ROWS], nr[GEMV_ROWS], nact = 0;
  if (g0 >= 0) {
    group[0] = g0;
    row[0] = 0;
    nr[0] = g1 == g0 ? 2 : 1;
    nact = 1;
  }
  if (g1 >= 0 && g1 != g0) {
    group[nact] = g1;
    row[nact] = 1;
    nr[nact++] = 1;
  }
  const int64_t tasks = (int64_t)nact * N;
  const int64_t warps = (int64_t)gridDim.x * (GEMV_THREADS / 32);
  int64_t task = (int64_t)blockIdx.x * (GEMV_THREADS / 32) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  auto weight_row = [&](int64_t t) {
    const int second = t >= N;
    return reinterpret_cast<const uint4*>(W + ((int64_t)(second ? group[nact - 1] : group[0]) * N + (t - second * (int64_t)N)) * K);
  };
  uint4 next[GEMV_U];
  auto request = [&](const uint4* p, int c0) {
#pragma unroll
    for (int u = 0; u < GEMV_U; ++u) {
      const int c = c0 + u * 32 + lane;
      next[u] = c < chunks ? __ldcs(p + c) : make_uint4(0u, 0u, 0u, 0u);  // streamed once
    }
  };
  const uint4* wrow = weight_row(task);
  request(wrow, 0);
  float acc[GEMV_ROWS] = {0.f, 0.f};
  for (int c0 = 0;;) {
    uint4 w[GEMV_U];
#pragma unroll
    for (int u = 0; u < GEMV_U; ++u) w[u] = next[u];
    const int second = task >= N;
    const int rows = second ? nr[nact - 1] : nr[0], r0 = second ? row[nact - 1] : row[0];
    const int this_c0 = c0;
    const int64_t this_task = task;
    c0 += 32 * GEMV_U;
    if (c0 >= chunks) {  // the next step belongs to the warp's next column
      c0 = 0;
      task += warps;
      if (task < tasks) wrow = weight_row(task);
    }
    const bool more = task < tasks;
    if (more) request(wrow, c0);
    // (row by row: with the rows inside the pieces' loop the compiler keeps fewer loads ahead,
    // 49.0 us)
#pragma unroll
    for (int r = 0; r < GEMV_ROWS; ++r)
      if (r < rows) {
        const uint4* a = s_a + (r0 + r) * chunks;
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u) {
          const int c = this_c0 + u * 32 + lane;
          if (c < chunks) gemv::fma8<T>(a[c], w[u], acc[r]);
        }
      }
    if (c0 == 0) {  // the column is complete
      const int n = (int)(this_task - second * (int64_t)N);
      const int g = second ? group[nact - 1] : group[0];
#pragma unroll
      for (int r = 0; r < GEMV_ROWS; ++r) {
        float v[1] = {warp_sum(acc[r])};
        acc[r] = 0.f;
        if (r < rows && lane == 0) {
          const int64_t at = (int64_t)(r0 + r) * N + n;
          if (lin.bias != nullptr)
            v[0] += lin.bias_f32 ? static_cast<const float*>(lin.bias)[(int64_t)g * N + n]
                                 : Num<T>::to_f(static_cast<const T*>(lin.bias)[(int64_t)g * N + n]);
          if (lin.preact != nullptr) static_cast<T*>(lin.preact)[at] = Num<T>::from_f(v[0]);
          apply_act(lin.act, v);
          if (lin.residual != nullptr) v[0] += Num<T>::to_f(static_cast<const T*>(lin.residual)[at]);
          C[at] = Num<T>::from_f(v[0]);
        }
      }
    }
    if (!more) break;
  }
}

// ------------------------------------------------------------------------ weight gradients
// C[g] [M, N] = sum over the rows k of group g of A[k, m] * B[k, n] (A: the output gradients
// [rows, M], B: the layer's input [rows, N]), both read as MN-major tiles: TMA boxes of 64
// columns x 64 rows.  A group's K tiles run from its own first row -- rows are the outer
// coordinate of a box, which needs no alignment -- and the last one reaches up to 63 rows
// past its end, into the next group.  Those rows must not count, and they may hold anything
// (Inf and NaN times zero is not zero), so they are overwritten with zeros in both operands'
// boxes (a K row is 128 contiguous bytes of every box, whatever the swizzle) before the
// tile's MMAs, of which only the 16-row steps that hold rows of the group are issued: at
// most 15 rows x 6 boxes x 128 bytes are written.
//
// cmd: stage | valid rows << 8.  Lanes 1 to 31 of the MMA warp do the writing; they wait on
// the warp barrier (with all lanes following the pipeline's mbarriers instead, the gradient
// of 8 x 14336 x 4096 weights took 2.06 ms against 1.82 at the power cap).
__device__ __forceinline__ void zero_tile_rows(const Smem& sm, int cmd, int lane) {
  const int stage = cmd & 255, valid = cmd >> 8;
  const int n = ((valid + 15) / 16 * 16 - valid) * 8;  // 16-byte pieces per box
  for (int i = lane - 1; i < 6 * n; i += 31) {         // row by row, eight pieces in each of six boxes
    const int r = i / 48, p = i - r * 48, box = p >> 3;
    unsigned char* base = box < 2 ? sm.a + stage * A_BYTES + box * kMnBox : sm.b + stage * B_BYTES + (box - 2) * kMnBox;
    *reinterpret_cast<uint4*>(base + (valid + r) * 128 + (p & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Unit L of a launch with ks slices per tile: its tile and its rows [k0, k1), 64-row blocks
// from the group's first row (k0 == k1: no rows).
struct WgUnit {
  int g, m0, n0, k0, k1;
};
__device__ __forceinline__ WgUnit wgrad_unit(int L, int ks_n, int MT, int NB, int band, const int* s_k0, const int* s_k1) {
  WgUnit u;
  const int tile = ks_n == 1 ? L : L / ks_n;
  tc::wgrad_tile(tile, MT, NB, band, u.g, u.m0, u.n0);
  u.k0 = s_k0[u.g];
  u.k1 = s_k1[u.g];
  if (ks_n > 1) {
    const int ks = L - tile * ks_n, lo = u.k0, kb = (u.k1 - lo + BK - 1) / BK;  // ks kb < 2^31
    u.k0 = lo + ks * kb / ks_n * BK;
    u.k1 = min(u.k1, lo + (ks + 1) * kb / ks_n * BK);
  }
  return u;
}

__device__ __forceinline__ void load_k_ranges(const int32_t* koff, int G, int rows, int* s_k0, int* s_k1) {
  for (int g = threadIdx.x; g < G; g += blockDim.x) {
    s_k0[g] = min(max(koff[g], 0), rows);
    s_k1[g] = min(max(koff[g + 1], s_k0[g]), rows);
  }
}

template <typename OutT>
__global__ void __launch_bounds__(THREADS, 1)
    linear_wgrad_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        OutT* __restrict__ C, const int32_t* __restrict__ koff, int G, int M, int N, int rows, int band,
                        uint32_t idesc, float* __restrict__ ws, int ks_n) {
  pdl_wait();
  extern __shared__ unsigned char smem_raw[];
  const Smem sm(smem_raw);
  int *s_k0 = sm.t0, *s_k1 = sm.t1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int MT = (M + BM - 1) / BM, NB = (N + BN - 1) / BN;
  const int total = G * MT * NB * ks_n;

  if (threadIdx.x == 0) {
    *sm.abort = 0;
    sm.init(tmA, tmB);
  }
  load_k_ranges(koff, G, rows, s_k0, s_k1);
  if (warp == 1) tmem_alloc(smem_u32(sm.tmem), 2 * BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *sm.tmem;
  auto unit = [&](int L) { return wgrad_unit(L, ks_n, MT, NB, band, s_k0, s_k1); };

  if (warp == 0 || warp == WARP_B) {
    if (lane == 0) {
      // ------------------------------------------------------------- TMA producers
      Cursor<STAGES> st;
      int64_t issued = 0;
      bool ok = true;
      for (int L = blockIdx.x; L < total && ok; L += gridDim.x) {
        const WgUnit u = unit(L);
        const int live = min(4, (N - u.n0 + 63) / 64);  // boxes of B that hold columns below N
        for (int k = u.k0; k < u.k1; k += BK) {
          if (!mbar_wait(sm.empty(st.i), st.phase ^ 1, sm.abort)) { ok = false; break; }
          const uint32_t fb = sm.full(st.i);
          const uint32_t a_dst = smem_u32(sm.a + st.i * A_BYTES), b_dst = smem_u32(sm.b + st.i * B_BYTES);
          if (warp == 0) {
            mbar_arrive_expect_tx(fb, 3 * kMnBox);
            tma_load_2d(a_dst, &tmA, fb, u.m0, k);
            tma_load_2d(a_dst + kMnBox, &tmA, fb, u.m0 + 64, k);
            tma_load_2d(b_dst, &tmB, fb, u.n0, k);
          } else {
            mbar_arrive_expect_tx(fb, (live - 1) * kMnBox);
            if (live == 4) {
#pragma unroll
              for (int i = 1; i < 4; ++i) tma_load_2d(b_dst + i * kMnBox, &tmB, fb, u.n0 + 64 * i, k);
            } else {
              for (int i = 1; i < live; ++i) tma_load_2d(b_dst + i * kMnBox, &tmB, fb, u.n0 + 64 * i, k);
            }
          }
          ++issued;
          st.next();
        }
      }
      drain_loads(sm, issued);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------------------- MMA issuer
      const uint64_t a0 = umma_desc_mn_sw128(smem_u32(sm.a), kMnBox, 1024);
      const uint64_t b0 = umma_desc_mn_sw128(smem_u32(sm.b), kMnBox, 1024);
      Cursor<STAGES> st;
      Cursor<2> acc;
      bool ok = true;
      for (int L = blockIdx.x; L < total && ok; L += gridDim.x) {
        const WgUnit u = unit(L);
        if (u.k1 <= u.k0) continue;  // no rows: the epilogue knows
        const uint32_t id = idesc_cols(idesc, N - u.n0);
        if (!mbar_wait(sm.tempty(acc.i), acc.phase ^ 1, sm.abort)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc.i * BN);
        for (int k = u.k0; k < u.k1; k += BK) {
          if (!mbar_wait(sm.full(st.i), st.phase, sm.abort)) { ok = false; break; }
          const int valid = min(BK, u.k1 - k), steps = (valid + 15) / 16;
          if (valid < 16 * steps) {  // the group's last rows: wake the other lanes, wait for them
            *sm.word = st.i | valid << 8;
            __syncwarp();
            __syncwarp();
          }
          tc_fence_after();
          const uint64_t a = a0 + (uint64_t)(st.i * (A_BYTES >> 4)), b = b0 + (uint64_t)(st.i * (B_BYTES >> 4));
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {  // 16 rows of K: two 1 KB atoms
            if (kk >= steps) break;
            umma_f16(d, a + 128 * kk, b + 128 * kk, id, (k != u.k0 || kk != 0) ? 1u : 0u);
          }
          umma_commit(sm.empty(st.i));
          st.next();
        }
        if (!ok) break;
        umma_commit(sm.tfull(acc.i));
        acc.next();
      }
      *sm.word = -1;  // the other lanes may leave
      __syncwarp();
      umma_commit(sm.mma_done());
      tc::mbar_wait_drain(sm.mma_done(), 0);
    } else {
      while (true) {
        __syncwarp();
        const int cmd = *sm.word;
        if (cmd < 0) break;
        zero_tile_rows(sm, cmd, lane);
        __syncwarp();
      }
    }
  } else {
    // --------------------------------------------------------------- epilogue
    const int q = warp & 3, half = (warp - EPI_WARP0) >> 2;
    unsigned char* stage = sm.out + (warp - EPI_WARP0) * STAGE_OUT;
    const int64_t pitch = (int64_t)N * sizeof(OutT);
    Cursor<2> acc;
    for (int L = blockIdx.x; L < total; L += gridDim.x) {
      const WgUnit u = unit(L);
      const int row = u.m0 + q * 32, nrows = M - row, col0 = u.n0 + half * 128;
      const bool none = u.k1 <= u.k0;
      if (none && ks_n > 1) continue;          // the sum leaves empty slices out
      if (!none) {
        if (!mbar_wait(sm.tfull(acc.i), acc.phase, sm.abort)) break;
        tc_fence_after();
      }
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc.i * BN + half * 128);
      if (ks_n > 1) {
        if (nrows > 0)
#pragma unroll 1
          for (int c = 0; c < 4 && col0 + c * 32 < N; ++c)
            store_partial(tbase + c * 32, ws + (int64_t)L * BM * BN, BM, half * 32 + c * 8, q * 32 + lane, lane < nrows);
      } else if (none) {                       // a group without rows: zeros
        constexpr int W = 16 / sizeof(OutT), L_ROW = 128 / W;  // columns per lane, lanes per row
        const int col = col0 + lane % L_ROW * W;
        for (int rr = lane / L_ROW; rr < min(nrows, 32); rr += 32 / L_ROW)
          if (col < N)
            *reinterpret_cast<uint4*>(C + ((int64_t)u.g * M + row + rr) * N + col) = make_uint4(0u, 0u, 0u, 0u);
      } else if (nrows > 0) {
#pragma unroll 1
        for (int c = 0; c < 2 && col0 + c * 64 < N; ++c) {
          uint32_t v[64];
          load_acc64(tbase + c * 64, v);
          tmem_ld_wait();
          unsigned char* p = reinterpret_cast<unsigned char*>(C + ((int64_t)u.g * M + row) * N + col0 + c * 64);
          const int width = (N - col0 - c * 64) * (int)sizeof(OutT);
          uint4 w[8];
          if constexpr (sizeof(OutT) == 2) {
            float f[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) f[j] = __uint_as_float(v[j]);
            pack_cols<OutT, 64>(f, w);
            store_rows128(w, p, pitch, nrows, width, stage, lane);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {      // 32 fp32 columns at a time
#pragma unroll
              for (int j = 0; j < 8; ++j)
                w[j] = make_uint4(v[32 * h + 4 * j], v[32 * h + 4 * j + 1], v[32 * h + 4 * j + 2], v[32 * h + 4 * j + 3]);
              store_rows128(w, p + 128 * h, pitch, nrows, width - 128 * h, stage, lane);
            }
          }
        }
      }
      if (none) continue;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.tempty(acc.i));
      acc.next();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// The second launch of a split weight gradient: the slices of a tile that have rows, in order.
template <typename OutT>
__global__ void __launch_bounds__(256) linear_wgrad_sum_kernel(OutT* __restrict__ C, const int32_t* __restrict__ koff,
                                                               int G, int M, int N, int rows, int band,
                                                               const float* __restrict__ ws, int ks_n) {
  pdl_wait_and_release();
  __shared__ int s_k0[MAX_GROUPS], s_k1[MAX_GROUPS];
  load_k_ranges(koff, G, rows, s_k0, s_k1);
  __syncthreads();
  const int MT = (M + BM - 1) / BM, NB = (N + BN - 1) / BN;
  constexpr int per = BM * (BN / 8);
  const int64_t total = (int64_t)G * MT * NB * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int tile = (int)(i / per), rem = (int)(i - (int64_t)tile * per);
    const int p8 = rem / BM, r = rem - p8 * BM;
    const WgUnit u = wgrad_unit(tile * ks_n, ks_n, MT, NB, band, s_k0, s_k1);
    const int row = u.m0 + r, col = u.n0 + p8 * 8;
    if (row >= M || col >= N) continue;
    // Of ks slices over kb row blocks, slice q has floor((q+1) kb / ks) - floor(q kb / ks): none
    // for some q where kb < ks.  Those hold nothing.
    const int kb = (s_k1[u.g] - s_k0[u.g] + BK - 1) / BK;
    float f[8];
    if (kb >= ks_n) {
      sum_partials(ws, (int64_t)tile * ks_n, ks_n, BM, p8, r, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
      for (int q = 0; q < ks_n; ++q)
        if ((q + 1) * kb / ks_n > q * kb / ks_n) {
          float one[8];
          sum_partials(ws, (int64_t)tile * ks_n + q, 1, BM, p8, r, one);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] += one[j];
        }
    }
    OutT* p = C + ((int64_t)u.g * M + row) * N + col;
    if constexpr (sizeof(OutT) == 2) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<OutT>(f[0], f[1]), pack2<OutT>(f[2], f[3]),
                                                pack2<OutT>(f[4], f[5]), pack2<OutT>(f[6], f[7]));
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
}

}  // namespace lin
}  // namespace smoe
