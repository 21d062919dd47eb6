// The 32 x 32 tile of small products: the k loop of one wave, its operands read
// straight into MFMA fragments (gemm_direct.hip says why and when).
#pragma once

#include "gemm_common.h"
#include "gemm_direct.h"

namespace dtmi {

// 16-byte vector at an element-aligned address
template <typename T>
struct UVec;
template <>
struct UVec<float> {
  typedef MF<float>::vec_t __attribute__((aligned(4))) type;
};
template <>
struct UVec<double> {
  typedef MF<double>::vec_t __attribute__((aligned(8))) type;
};

// One operand's share of a wave: R MFMA tiles of MT rows (columns) along m/n by
// KB of k per batch.
template <typename T, bool KCONTIG, int R, int KB>
struct DirectSrc {
  static constexpr int MT = MF<T>::MT, VEC = MF<T>::VEC, NCH = KB / 8;
  typedef typename MF<T>::vec_t VT;
  const char* base;  // wave-uniform: the current batch's first k
  unsigned off[R];   // this lane's byte offset from it
  int64_t ldb;       // bytes between k-rows (m/n-contiguous)

  __device__ __forceinline__ void init(const T* __restrict__ P, int64_t ld, int64_t mn0, int64_t MN, int64_t k0, int g,
                                       int c) {
    base = reinterpret_cast<const char*>(KCONTIG ? P + mn0 * ld + k0 : P + k0 * ld + mn0);
    ldb = ld * (int64_t)sizeof(T);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      int64_t r = mn0 + i * MT + c;
      r = (r < MN ? r : MN - 1) - mn0;
      off[i] = (unsigned)((KCONTIG ? r * ld + VEC * g : (int64_t)VEC * g * ld + r) * (int64_t)sizeof(T));
    }
  }
  __device__ __forceinline__ void load(VT (&v)[R][NCH]) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        if constexpr (KCONTIG) {
          v[i][ch] = *reinterpret_cast<const typename UVec<T>::type*>(base + off[i] + 8 * ch * sizeof(T));
        } else {
#pragma unroll
          for (int s = 0; s < VEC; ++s) v[i][ch][s] = *reinterpret_cast<const T*>(base + (8 * ch + s) * ldb + off[i]);
        }
      }
    base += KCONTIG ? (int64_t)KB * (int64_t)sizeof(T) : (int64_t)KB * ldb;
  }
  // the last `left` (< KB) values of k: element loads clamped to k = left - 1,
  // zeros from `left` on
  __device__ __forceinline__ void load_tail(VT (&v)[R][NCH], int left, int g) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int s = 0; s < VEC; ++s) {
          const int k = 8 * ch + VEC * g + s;
          const int64_t kc = (k < left ? k : left - 1) - VEC * g;  // relative to this lane's offset
          const T x = *reinterpret_cast<const T*>(base + (int64_t)off[i] + kc * (KCONTIG ? (int64_t)sizeof(T) : ldb));
          v[i][ch][s] = k < left ? x : T(0);
        }
  }
};

template <typename T>
struct DirectTile {
  static constexpr int EDGE = 32;                      // block tile
  static constexpr int R = EDGE / MF<T>::MT;           // MFMA tiles per edge
  static constexpr int REGS = R * R * MF<T>::NACC;     // accumulators per lane
  static constexpr int KB = kDirectBatch<T>;
};

// acc += A(m0.., k) B(k, n0..) over the kn values of k from kbeg: one wave, lane group g,
// position c. on_b(y) is called with every batch of B's fragments (k past the range as
// zeros). (gemm_direct_kernel has this loop written out: called from here, its float32
// form of two k-contiguous operands took 128 registers and spilled.)
template <typename T, bool AKC, bool BKC, typename F>
__device__ __forceinline__ void direct_product(
    typename MF<T>::acc_t (&acc)[DirectTile<T>::R][DirectTile<T>::R], const T* A, int64_t lda, int64_t M,
    int64_t m0, const T* B, int64_t ldb, int64_t N, int64_t n0, int64_t kbeg, int kn, int g, int c, F on_b) {
  using MFT = MF<T>;
  using D = DirectTile<T>;
  constexpr int VEC = MFT::VEC, R = D::R, KB = D::KB, NCH = KB / 8;
  typedef typename MFT::vec_t VT;
  DirectSrc<T, AKC, R, KB> sa;
  DirectSrc<T, BKC, R, KB> sb;
  sa.init(A, lda, m0, M, kbeg, g, c);
  sb.init(B, ldb, n0, N, kbeg, g, c);
  auto mul = [&](const VT (&x)[R][NCH], const VT (&y)[R][NCH], int chunks) {
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      if (ch >= chunks) break;
#pragma unroll
      for (int s = 0; s < VEC; ++s)
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int j = 0; j < R; ++j) acc[i][j] = MFT::mma(x[i][ch][s], y[j][ch][s], acc[i][j]);
    }
    on_b(y);
  };
  const int nb = kn / KB, left = kn - nb * KB;
  VT x0[R][NCH], y0[R][NCH], x1[R][NCH], y1[R][NCH];
  if (nb > 0) {
    sa.load(x0);
    sb.load(y0);
    int b = 0;
    for (; b + 2 <= nb; b += 2) {
      sa.load(x1);
      sb.load(y1);
      mul(x0, y0, NCH);
      if (b + 2 < nb) {
        sa.load(x0);
        sb.load(y0);
      }
      mul(x1, y1, NCH);
    }
    if (b < nb) mul(x0, y0, NCH);
  }
  if (left > 0) {
    sa.load_tail(x0, left, g);
    sb.load_tail(y0, left, g);
    mul(x0, y0, (left + 7) / 8);
  }
}

}  // namespace dtmi
