// Products of few rows: C [M, N] = A [M, K] B with M up to 32, which are bound by reading
// B once.
//
// The 32-wide tile of gemm_direct.hip spends a 32x32x2 MFMA, 64 cycles, on each two k of
// 32 columns whatever the rows: 256 cycles per KB of B, so that the card's MFMAs keep up
// with 8.8 TB/s only if they never wait. Here a tile has 16 rows (or 2 x 16): a 16x16x4
// MFMA takes 32 cycles per four k of 16 columns, half as much. A wave covers 64 columns
// (float64, B contiguous in n: 32) of its share of k, the block's waves share k, and the
// partial tiles are added through LDS.
//   B contiguous in k: a lane's 16 bytes are consecutive k of one column.
//   B contiguous in n: a lane's 16 bytes are consecutive columns of one k; column VEC c + t
//   is lane c's in MFMA tile t, so each 16-byte load feeds VEC tiles.
// k within a chunk of 4 VEC is permuted alike for A and B: lane group g takes k = VEC g + s
// at step s. Loads need element alignment only.
#pragma once

#include "gemm_common.h"
#include "gemm_direct_tile.h"

namespace dtmi {

template <typename T>
struct RowsMma;
template <>
struct RowsMma<float> {
  typedef float acc_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int r, int g) { return 4 * g + r; }
};
template <>
struct RowsMma<double> {
  typedef double acc_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t mma(double a, double b, acc_t c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int r, int g) { return g + 4 * r; }
};

template <typename T>
using RowsAcc = typename RowsMma<T>::acc_t;

constexpr int kRowsMaxWaves = 8;

template <typename T, bool BKC>
struct RowsTile {
  static constexpr int VEC = MF<T>::VEC;
  static constexpr int NT = BKC ? 4 : VEC;     // MFMA tiles along n
  static constexpr int COLS = 16 * NT;
  static constexpr int CHUNK = 4 * VEC;        // k of one 16-byte load of a lane
  static constexpr int BATCH = 2 * CHUNK;      // k in flight
  // column of lane position c in tile t
  static __device__ __forceinline__ int col(int c, int t) { return BKC ? 16 * t + c : VEC * c + t; }
};

// acc += the rows m0 .. m0 + 16 MR of A times the columns n0 .. n0 + COLS of B over kbeg <=
// k < kend: one wave. Rows and columns past the last are the last one's again.
template <typename T, int MR, bool BKC, int NT>
__device__ __forceinline__ void rows_product(RowsAcc<T> (&acc)[MR][NT], const T* __restrict__ A,
                                             int64_t lda, int64_t M, int64_t m0, const T* __restrict__ B, int64_t ldb,
                                             int64_t N, int64_t n0, int kbeg, int kend, int g, int c) {
  using RT = RowsTile<T, BKC>;
  constexpr int VEC = RT::VEC, CHUNK = RT::CHUNK, BATCH = RT::BATCH, NB = BATCH / CHUNK;
  constexpr int BV = BKC ? NT : VEC;  // B vectors of a chunk
  typedef typename MF<T>::vec_t VT;
  typedef typename UVec<T>::type UV;
  const T* pa[MR];
#pragma unroll
  for (int i = 0; i < MR; ++i) {
    const int64_t m = m0 + 16 * i + c;
    pa[i] = A + (m < M ? m : M - 1) * lda;
  }
  const T* pb[NT];  // k-contiguous: a column each; n-contiguous: the lane's columns (of k row 0)
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + RT::col(c, t), nc = n < N ? n : N - 1;
    pb[t] = BKC ? B + nc * ldb : B + nc;
  }
  const bool whole = BKC || n0 + RT::COLS <= N;  // wave-uniform
  struct Regs {
    VT a[MR][NB], b[BV][NB];
  };
  auto load = [&](Regs& r, int k0) {
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const int k = k0 + q * CHUNK + VEC * g;
#pragma unroll
      for (int i = 0; i < MR; ++i) r.a[i][q] = *reinterpret_cast<const UV*>(pa[i] + k);
      if constexpr (BKC) {
#pragma unroll
        for (int t = 0; t < NT; ++t) r.b[t][q] = *reinterpret_cast<const UV*>(pb[t] + k);
      } else if (whole) {
#pragma unroll
        for (int s = 0; s < VEC; ++s) r.b[s][q] = *reinterpret_cast<const UV*>(pb[0] + (int64_t)(k + s) * ldb);
      } else {
#pragma unroll
        for (int s = 0; s < VEC; ++s)
#pragma unroll
          for (int t = 0; t < NT; ++t) r.b[s][q][t] = pb[t][(int64_t)(k + s) * ldb];
      }
    }
  };
  // the last k of a range: element by element, zeros from kend on
  auto load_tail = [&](Regs& r, int k0) {
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int s = 0; s < VEC; ++s) {
        const int k = k0 + q * CHUNK + VEC * g + s;
        const int kc = k < kend ? k : kend - 1;
#pragma unroll
        for (int i = 0; i < MR; ++i) {
          const T x = pa[i][kc];
          r.a[i][q][s] = k < kend ? x : T(0);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const T x = BKC ? pb[t][kc] : pb[t][(int64_t)kc * ldb];
          if (BKC)
            r.b[t][q][s] = k < kend ? x : T(0);
          else
            r.b[s][q][t] = k < kend ? x : T(0);
        }
      }
  };
  auto mul = [&](const Regs& r) {
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int s = 0; s < VEC; ++s)
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[i][t] = RowsMma<T>::mma(r.a[i][q][s], BKC ? r.b[BKC ? t : 0][q][s] : r.b[BKC ? 0 : s][q][t], acc[i][t]);
  };
  const int nb = (kend - kbeg) / BATCH;
  Regs r0, r1;
  if (nb > 0) {
    load(r0, kbeg);
    int b = 0;
    for (; b + 2 <= nb; b += 2) {
      load(r1, kbeg + (b + 1) * BATCH);
      mul(r0);
      if (b + 2 < nb) load(r0, kbeg + (b + 2) * BATCH);
      mul(r1);
    }
    if (b < nb) mul(r0);
  }
  if (kbeg + nb * BATCH < kend) {
    load_tail(r0, kbeg + nb * BATCH);
    mul(r0);
  }
}

// The block's sum of its waves' tiles: every wave writes its own, then value(q) is register
// q = (i NT + t) 4 + r of this lane, added in wave order.
template <typename T, int MR, bool BKC>
struct RowsSum {
  static constexpr int NT = RowsTile<T, BKC>::NT, REGS = MR * NT * 4;
  T* part;
  int lane, nw;
  __device__ __forceinline__ void put(const RowsAcc<T> (&acc)[MR][NT], int wave) const {
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[(wave * REGS + (i * NT + t) * 4 + r) * 64 + lane] = acc[i][t][r];
  }
  __device__ __forceinline__ T value(int q) const {
    T v[kRowsMaxWaves];  // all read before the first is added
#pragma unroll
    for (int w = 0; w < kRowsMaxWaves; ++w) v[w] = w < nw ? part[(w * REGS + q) * 64 + lane] : T(0);
    T s = v[0];
#pragma unroll
    for (int w = 1; w < kRowsMaxWaves; ++w) s = s + v[w];
    return s;
  }
};

}  // namespace dtmi
