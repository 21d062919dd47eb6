// The kernels behind gemm_group.h.
#pragma once

#include "gemm_group.h"
#include "gemm_tiles.h"
#include "seqmath.h"

namespace dtmi {

// Blocks are dealt to the 8 XCDs in turn: this order gives each a contiguous range of
// tiles, whose operands its L2 then holds. The last tiles % 8 keep their place.
__device__ __forceinline__ int xcd_tile(int b, int tiles) {
  const int per = tiles >> 3;
  return b < 8 * per ? (b & 7) * per + (b >> 3) : b;
}

// Tile t of a task's own grid: groups of 8 rows of tiles, as tile_coords_of; or, of a
// symmetric product, row by row the tiles on and below the diagonal.
__device__ __forceinline__ void group_coords(int t, int tiles_m, int tiles_n, int sym, int& tm, int& tn) {
  if (sym) {
    tm = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > t) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
    tn = t - tm * (tm + 1) / 2;
    return;
  }
  constexpr int GROUP = 8;
  const int per_group = GROUP * tiles_n;
  const int group = t / per_group;
  const int first_m = group * GROUP;
  const int gsz = tiles_m - first_m < GROUP ? tiles_m - first_m : GROUP;
  const int r = t - group * per_group;
  tm = first_m + r % gsz;
  tn = r / gsz;
}

// The task of tile t: every lane holds the first tile of one task (64 at most).
__device__ __forceinline__ int group_task(const GroupArgs& a, int t) {
  const int lane = threadIdx.x & 63;
  const int first = lane < a.count ? a.t[lane].tile0 : 0x7fffffff;
  const uint64_t mask = __ballot(first <= t);
  return __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(mask));
}

// One output element: s (alpha v + beta D) + gamma C.
template <typename T>
struct GroupEpi {
  T alpha, beta, gamma, s;
  int dmode;
  bool mirror;
  const T* D;
  T* C;
  int64_t N;
  __device__ __forceinline__ T value(T v, T d, T old) const {
    v = alpha * v;
    if (dmode == kDMatrix) v = fma(beta, d, v);
    if (dmode == kDRow) v = v + d;
    v = s * v;
    if (gamma != T(0)) v = fma(gamma, old, v);
    return v;
  }
  __device__ __forceinline__ void store(int64_t m, int64_t n, T v) const {
    const int64_t o = m * N + n;
    const T d = dmode == kDMatrix ? D[o] : dmode == kDRow ? D[n] : T(0);
    v = value(v, d, gamma != T(0) ? C[o] : T(0));
    C[o] = v;
    if (mirror) C[n * N + m] = v;
  }
};

template <typename T>
__device__ __forceinline__ GroupEpi<T> group_epi(const GroupArgs& a, const GroupTask& k, bool mirror) {
  return {(T)a.alpha, (T)a.beta, (T)a.gamma, (T)k.s, a.dmode, mirror, (const T*)k.D, (T*)k.C, (int64_t)k.N};
}

template <typename T, int BM, bool AKC, bool BKC, bool VEC>
__global__ void __launch_bounds__(256, 2) gemm_group_kernel(GroupArgs a) {
  using MFT = MF<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC;
  constexpr int W = BM / 2, TW = W / MT;
  __shared__ __attribute__((aligned(1024))) T lds[kDmaLds<T, BM, BM>];

  const int t = xcd_tile((int)blockIdx.x, a.tiles);
  const int ti = group_task(a, t);
  const GroupTask k = a.t[ti];
  int tm, tn;
  group_coords(t - k.tile0, (k.M + BM - 1) / BM, (k.N + BM - 1) / BM, a.sym, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BM;
  const int split = blockIdx.y;
  constexpr int BK = 64 / (int)sizeof(T);
  const int64_t kps = a.splits > 1 ? ((k.K + a.splits - 1) / a.splits + BK - 1) / BK * BK : k.K;
  const int64_t kbeg = split * kps < k.K ? split * kps : k.K;
  const int64_t kend = kbeg + kps < k.K ? kbeg + kps : k.K;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane / MT, c = lane % MT;
  typename MFT::acc_t acc[TW][TW];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) acc[i][j] = typename MFT::acc_t(0);
  const bool take_colsum = a.dmode == kDColsum && tm == 0 && (int)threadIdx.x < BM;
  double csum = 0.0;
  dma_product<T, BM, BM, AKC, BKC, VEC, VEC>(acc, lds, (const T*)k.A, AKC ? k.K : k.M, k.M, m0, (const T*)k.B,
                                             BKC ? k.K : k.N, k.N, n0, kbeg, kend, sizeof(T) == 4 ? 2 : 4,
                                             take_colsum, csum);
  if (take_colsum && n0 + threadIdx.x < k.N) {
    const int64_t n = n0 + threadIdx.x;
    if (a.csws)
      ((T*)a.csws)[((int64_t)split * a.count + ti) * k.N + n] = (T)csum;
    else if (k.D)
      ((T*)k.D)[n] = (T)csum;
  }
  const int64_t wm = m0 + (wave >> 1) * W, wn = n0 + (wave & 1) * W;
  if (a.ws) {  // the raw partial, tile by tile
    T* P = (T*)a.ws + ((int64_t)split * a.tiles + t) * (BM * BM);
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j)
#pragma unroll
        for (int r = 0; r < NACC; ++r)
          P[((wave >> 1) * W + i * MT + MFT::row(r, g)) * BM + (wave & 1) * W + j * MT + c] = acc[i][j][r];
    return;
  }
  const GroupEpi<T> e = group_epi<T>(a, k, a.sym && tm != tn);
  if constexpr (sizeof(T) == 4) {
    if (wm + W <= k.M && wn + W <= k.N) {
      // a wave tile in range: buffer accesses off its corner, one lane offset and a
      // wave-uniform offset per element (as write_acc); D and C of a row of MFMA tiles
      // are read before its first store
      const int64_t corner = wm * e.N + wn;
      const Rsrc rc = make_rsrc(e.C + corner, ~0ull);
      const Rsrc rd = make_rsrc(e.dmode == kDMatrix ? e.D + corner : e.C + corner, ~0ull);
      const uint32_t voff = (uint32_t)((4 * g * e.N + c) * 4);
      float row[TW];
#pragma unroll
      for (int j = 0; j < TW; ++j) row[j] = e.dmode == kDRow ? e.D[wn + j * MT + c] : 0.f;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        float d[TW][NACC];
#pragma unroll
        for (int j = 0; j < TW; ++j)
#pragma unroll
          for (int r = 0; r < NACC; ++r) d[j][r] = row[j];
        if (e.dmode == kDMatrix)
#pragma unroll
          for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int r = 0; r < NACC; ++r)
              d[j][r] = buf_load1(rd, voff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.N + j * MT) * 4));
        float old[TW][NACC];
#pragma unroll
        for (int j = 0; j < TW; ++j)
#pragma unroll
          for (int r = 0; r < NACC; ++r) old[j][r] = 0.f;
        if (e.gamma != 0.f)
#pragma unroll
          for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int r = 0; r < NACC; ++r)
              old[j][r] = buf_load1(rc, voff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.N + j * MT) * 4));
#pragma unroll
        for (int j = 0; j < TW; ++j) {
          float v[NACC];
#pragma unroll
          for (int r = 0; r < NACC; ++r) {
            v[r] = e.value(acc[i][j][r], d[j][r], old[j][r]);
            buf_store1(v[r], rc, voff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.N + j * MT) * 4));
          }
          if (e.mirror) {
            // a lane's registers 4q .. 4q + 3 are four rows of one column, so four
            // elements in a row of the mirror image
            float* R = e.C + (wn + j * MT + c) * e.N + wm + i * MT + 4 * g;
            if constexpr (VEC) {
#pragma unroll
              for (int q = 0; q < NACC / 4; ++q)
                *reinterpret_cast<f32x4*>(R + 8 * q) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            } else {
#pragma unroll
              for (int r = 0; r < NACC; ++r) R[8 * (r / 4) + r % 4] = v[r];
            }
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) {
      const int64_t n = wn + j * MT + c;
      if (n >= k.N) continue;
#pragma unroll
      for (int r = 0; r < NACC; ++r) {
        const int64_t m = wm + i * MT + MFT::row(r, g);
        if (m < k.M) e.store(m, n, acc[i][j][r]);
      }
    }
}

// The splits' partials of a tile, added in split order, and the epilogue.
template <typename T, int BM>
__global__ void __launch_bounds__(256) group_sum_kernel(GroupArgs a) {
  const int t = blockIdx.x;
  const int ti = group_task(a, t);
  const GroupTask k = a.t[ti];
  int tm, tn;
  group_coords(t - k.tile0, (k.M + BM - 1) / BM, (k.N + BM - 1) / BM, a.sym, tm, tn);
  const GroupEpi<T> e = group_epi<T>(a, k, a.sym && tm != tn);
  const T* P = (const T*)a.ws + (int64_t)t * (BM * BM);
  const int64_t step = (int64_t)a.tiles * (BM * BM);
  constexpr int PER = 8;
  for (int i0 = threadIdx.x; i0 < BM * BM; i0 += 256 * PER) {
    T v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = P[i0 + 256 * u];
    for (int s = 1; s < a.splits; ++s)
#pragma unroll
      for (int u = 0; u < PER; ++u) v[u] = v[u] + P[s * step + i0 + 256 * u];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = i0 + 256 * u;
      const int64_t m = (int64_t)tm * BM + i / BM, n = (int64_t)tn * BM + i % BM;
      if (m < k.M && n < k.N) e.store(m, n, v[u]);
    }
  }
  const int64_t n = (int64_t)tn * BM + threadIdx.x;
  if (a.csws && tm == 0 && threadIdx.x < BM && n < k.N && k.D) {
    const T* S = (const T*)a.csws;
    T v = S[(int64_t)ti * k.N + n];
    for (int s = 1; s < a.splits; ++s) v = v + S[((int64_t)s * a.count + ti) * k.N + n];
    ((T*)k.D)[n] = v;
  }
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// Z = A B + bias and, per row, the maximum and sum of exponentials of each wave's
// columns. A wave turns its tile through LDS (the k loop's stages, free by then), one
// row of MFMA tiles at a time, so that a lane owns part of a row: 64 reads and 64
// exponentials a lane at BM = 128, where a butterfly over the columns' lanes would
// take ten exchanges for each of 32 rows.
template <typename T, int BM, bool BKC, bool VEC>
__global__ void __launch_bounds__(256, 2) gemm_stats_kernel(StatsArgs a) {
  using MFT = MF<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC, V = MFT::VEC;
  constexpr int W = BM / 2, TW = W / MT;
  constexpr int LD = W + V;            // of a wave's turned rows: conflict-free column writes
  constexpr int PARTS = 64 / MT;       // lanes per row
  constexpr int COLS = W / PARTS;      // columns per lane
  static_assert(4 * MT * LD <= kDmaLds<T, BM, BM>, "turned rows fit the stages");
  __shared__ __attribute__((aligned(1024))) T lds[kDmaLds<T, BM, BM>];

  const int t = xcd_tile((int)blockIdx.x, a.tiles_m * a.tiles_n);
  int tm, tn;
  group_coords(t, a.tiles_m, a.tiles_n, 0, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BM;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane / MT, c = lane % MT;
  typename MFT::acc_t acc[TW][TW];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) acc[i][j] = typename MFT::acc_t(0);
  double csum = 0.0;
  dma_product<T, BM, BM, true, BKC, VEC, VEC>(acc, lds, (const T*)a.A, a.lda, a.M, m0, (const T*)a.B, a.ldb, a.N, n0,
                                              0, a.K, sizeof(T) == 4 ? 2 : 4, false, csum);
  const int64_t wm = m0 + (wave >> 1) * W, wn = n0 + (wave & 1) * W;
  T* C = (T*)a.C;
  T* R = lds + wave * (MT * LD);
  __syncthreads();  // every wave is done with the stages
  const int64_t part = 2 * (int64_t)tn + (wave & 1);
#pragma unroll
  for (int i = 0; i < TW; ++i) {
#pragma unroll
    for (int j = 0; j < TW; ++j) {
      const int64_t n = wn + j * MT + c;
      const bool in = n < a.N;
      const T b = in && a.bias ? ((const T*)a.bias)[n] : T(0);
#pragma unroll
      for (int r = 0; r < NACC; ++r) {
        const int row = MFT::row(r, g);
        const T z = a.bias ? acc[i][j][r] + b : acc[i][j][r];
        R[row * LD + j * MT + c] = in ? z : -INFINITY;
        if (C && in && wm + i * MT + row < a.M) C[(wm + i * MT + row) * a.ldc + n] = z;
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int row = lane % MT, q = lane / MT;
    const int64_t m = wm + i * MT + row;
    typedef T vt __attribute__((ext_vector_type(V)));
    vt x[COLS / V];
#pragma unroll
    for (int u = 0; u < COLS / V; ++u) x[u] = *reinterpret_cast<const vt*>(R + row * LD + q * COLS + u * V);
    T mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < COLS / V; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) mx = fmax(mx, x[u][e]);
#pragma unroll
    for (int o = MT; o < 64; o <<= 1) mx = fmax(mx, __shfl_xor(mx, o, 64));
    // a NaN is dropped by the maximum and comes back through the sum; a part of -inf
    // alone has sum 0
    const T ref = mx == -INFINITY ? T(0) : mx;
    T s = T(0);
#pragma unroll
    for (int u = 0; u < COLS / V; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) s += exp_of(x[u][e] - ref);
#pragma unroll
    for (int o = MT; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if (m < a.M) {
      const int64_t tc = a.targets ? a.targets[m] - (wn + q * COLS) : -1;
      if (tc >= 0 && tc < COLS) ((T*)a.zt)[m] = R[row * LD + q * COLS + (int)tc];
      if (q == 0) {
        ((T*)a.pmax)[part * a.M + m] = mx;
        ((T*)a.psum)[part * a.M + m] = s;
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T, int BM>
void launch_group(const GroupArgs& a, int akc, int bkc, bool vec) {
  const dim3 grid((unsigned)a.tiles, (unsigned)a.splits);
#define DTMI_GROUP(AK, BKK)                                                  \
  if (vec)                                                                   \
    gemm_group_kernel<T, BM, AK, BKK, true><<<grid, 256, 0, stream()>>>(a);  \
  else                                                                       \
    gemm_group_kernel<T, BM, AK, BKK, false><<<grid, 256, 0, stream()>>>(a)
  if (akc && bkc) {
    DTMI_GROUP(true, true);
  } else if (akc) {
    DTMI_GROUP(true, false);
  } else {
    DTMI_GROUP(false, false);
  }
#undef DTMI_GROUP
  if (a.ws) group_sum_kernel<T, BM><<<(unsigned)a.tiles, 256, 0, stream()>>>(a);
}

template <typename T, int BM>
void launch_stats(const StatsArgs& a, int bkc, bool vec) {
  const unsigned grid = (unsigned)(a.tiles_m * a.tiles_n);
  if (bkc) {
    if (vec)
      gemm_stats_kernel<T, BM, true, true><<<grid, 256, 0, stream()>>>(a);
    else
      gemm_stats_kernel<T, BM, true, false><<<grid, 256, 0, stream()>>>(a);
  } else {
    if (vec)
      gemm_stats_kernel<T, BM, false, true><<<grid, 256, 0, stream()>>>(a);
    else
      gemm_stats_kernel<T, BM, false, false><<<grid, 256, 0, stream()>>>(a);
  }
}

}  // namespace dtmi
